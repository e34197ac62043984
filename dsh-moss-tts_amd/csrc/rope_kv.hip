// rope_kv.hip -- rotary positions of rows, and rows into and out of a paged K/V cache (gfx950).
//
// Rotation of pair i of a row at position p: with w_i the pair's angle per position,
//   a' = m (a cos(p w_i) - b sin(p w_i)),  b' = m (b cos(p w_i) + a sin(p w_i)).
// The pair is (2i, 2i + 1) or (i, i + rot / 2); elements from rot on are copied.  p w_i is formed in
// 64 bits and reduced to a fraction of a turn before anything is rounded to 32, so that far
// positions lose nothing; a sine then costs one sincospif per (row, pair), shared by every head
// of the row through LDS.  The reference rotates in its QKV step from a table of the same values
// (csrc/src/llm.cpp:90-102,173-187); scaled frequencies, halves and part of a head have no
// counterpart there.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256;

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};

// Memory is read and written 16 bytes at a time at any address that an element may have (the hardware takes
// them unaligned).

// 8 values to p.
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    uint32_t w[2 * sizeof(T)];  // (words: from an array of halves the compiler makes 2-byte stores)
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(T); ++i) {
        if constexpr (sizeof(T) == 2)
            w[i] = (uint32_t)f2h(x[2 * i]) | (uint32_t)f2h(x[2 * i + 1]) << 16;
        else
            w[i] = __float_as_uint(x[i]);
    }
    __builtin_memcpy(p, w, sizeof(w));
}

// V elements as they lie in memory.
template <class T, int V>
struct Raw {
    T e[V];
};
template <class T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T *p) {
    Raw<T, V> x;
    if constexpr (V * sizeof(T) >= 16) {
        uint4 w[V * sizeof(T) / 16];
        __builtin_memcpy(w, p, sizeof(w));
        __builtin_memcpy(&x, w, sizeof(w));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x.e[i] = p[i];
    }
    return x;
}
template <class T, int V>
__device__ __forceinline__ void store_raw(T *p, const Raw<T, V> &x) {
    if constexpr (V * sizeof(T) >= 16) {
        uint4 w[V * sizeof(T) / 16];
        __builtin_memcpy(w, &x, sizeof(w));
        __builtin_memcpy(p, w, sizeof(w));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = x.e[i];
    }
}

// cos and sin (times mscale) of position p at `w` radians a position.
__device__ __forceinline__ float2 turn(int p, double w, float mscale) {
    const double t = (double)p * w * 0.15915494309189533577;  // turns
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    return make_float2(c * mscale, s * mscale);
}

__device__ __forceinline__ void rotate(float a, float b, float2 cs, float &x, float &y) {
    x = a * cs.x - b * cs.y;
    y = b * cs.x + a * cs.y;
}

// One workgroup per `rpb` rows (and a share of their units where there are few rows).  A unit is
// what one thread turns at a time: V neighbouring elements of interleaved pairs, or V elements
// and their V partners half a rotation further; then the V-element pieces behind rot.
// Memory bound: every element is read and written once, in 16-byte pieces where head_dim and
// (halves) rot / 2 are made of such, and a thread has N units' loads in flight, the first N before the
// angles are formed.  8191 rows of 40 heads x 128 fp16, three quarters of each turned: 33.5 us, 5.0 TB/s,
// what a 1 GiB copy reaches (5.08); one unit at a time, a row a workgroup: 51.
template <class T, bool HALVES, int V, int N>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeRowsArgs a, int rpb, int per_head) {
    extern __shared__ float2 cs[];  // [rpb][rot / 2]
    const int half = a.rope.rot / 2, t = threadIdx.x;
    const int row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    const int per_row = a.heads * per_head, units = nrow * per_row, turned = HALVES ? half / V : per_head;
    const int step = kThreads * gridDim.y;
    constexpr int SIDES = HALVES ? 2 : 1;
    Raw<T, V> x[N][SIDES];
    T *to[N];
    int at[N], angle[N];  // first element (of the lower half), and where its angles are; -1: copied
    auto load = [&](int u0) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = min(u0 + n * step, units - 1);
            const int r = u / per_row, hu = u - r * per_row, h = hu / per_head, p = hu - h * per_head;
            const T *from = (const T *)a.x + (row0 + r) * a.x_row + h * a.x_head;
            to[n] = (T *)a.y + (row0 + r) * a.y_row + h * a.y_head;
            const bool turn_it = HALVES ? p < turned : p * V < 2 * half;
            at[n] = HALVES && !turn_it ? 2 * half + (p - turned) * V : p * V;
            angle[n] = turn_it ? r * half + (HALVES ? p * V : p * V / 2) : -1;
            x[n][0] = load_raw<T, V>(from + at[n]);
            if (HALVES) x[n][SIDES - 1] = load_raw<T, V>(from + (turn_it ? half + at[n] : at[n]));
        }
    };
    const int first = blockIdx.y * kThreads + t;
    load(first);
    for (int i = t; i < nrow * half; i += kThreads) {
        const int r = i / half;
        cs[i] = turn(a.pos[row0 + r], a.rope.freqs[i - r * half], a.rope.mscale);
    }
    __syncthreads();
    for (int u0 = first; u0 < units; u0 += N * step) {
        if (u0 != first) load(u0);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (u0 + n * step >= units) break;
            if (angle[n] >= 0) {
                const float2 *c = cs + angle[n];
                if constexpr (HALVES) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float lo, hi;
                        rotate(Elem<T>::get(x[n][0].e[i]), Elem<T>::get(x[n][SIDES - 1].e[i]), c[i], lo, hi);
                        x[n][0].e[i] = Elem<T>::put(lo);
                        x[n][SIDES - 1].e[i] = Elem<T>::put(hi);
                    }
                    store_raw<T, V>(to[n] + half + at[n], x[n][SIDES - 1]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 2)
                        if (at[n] + i < 2 * half) {
                            float lo, hi;
                            rotate(Elem<T>::get(x[n][0].e[i]), Elem<T>::get(x[n][0].e[i + 1]), c[i / 2], lo, hi);
                            x[n][0].e[i] = Elem<T>::put(lo);
                            x[n][0].e[i + 1] = Elem<T>::put(hi);
                        }
                }
            }
            store_raw<T, V>(to[n] + at[n], x[n][0]);
        }
    }
}

template <class T, bool HALVES, int V>
hipError_t rope_rows(const RopeRowsArgs &a, hipStream_t s) {
    const int half = a.rope.rot / 2;
    const int per_head = HALVES ? half / V + (a.dim - a.rope.rot) / V : a.dim / V;
    const int units = a.heads * per_head;
    (void)hipGetLastError();
    // 4 units a thread once that leaves 1024 workgroups
    const int rpb4 = std::min(std::max(1, 4 * kThreads / units), 16);
    if ((a.rows + rpb4 - 1) / rpb4 >= 1024) {
        hipLaunchKernelGGL((rope_rows_kernel<T, HALVES, V, 4>), dim3((a.rows + rpb4 - 1) / rpb4), dim3(kThreads),
                           rpb4 * half * sizeof(float2), s, a, rpb4, per_head);
        return hipGetLastError();
    }
    const int rpb = std::min(std::max(1, kThreads / units), 16);
    const int split = a.rows < 512 ? std::min((units + kThreads - 1) / kThreads, 64) : 1;
    hipLaunchKernelGGL((rope_rows_kernel<T, HALVES, V, 1>), dim3((a.rows + rpb - 1) / rpb, split), dim3(kThreads),
                       rpb * half * sizeof(float2), s, a, rpb, per_head);
    return hipGetLastError();
}

template <class T>
hipError_t rope_rows_t(const RopeRowsArgs &a, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    auto whole = [](int n) { return n % V == 0; };
    if (a.rope.halves)
        return whole(a.dim) && whole(a.rope.rot) && whole(a.rope.rot / 2) ? rope_rows<T, true, V>(a, s) : rope_rows<T, true, 1>(a, s);
    return whole(a.dim) ? rope_rows<T, false, V>(a, s) : rope_rows<T, false, 2>(a, s);
}

// ---------------------------------------------------------------- the paged cache

// Where row r of a call lives in the pools: the index of its first vector ([page][head 0][slot]) and
// whether there is such a place.  A wave has one row at a time, so all of this is scalar work.
struct Place {
    size_t at;
    bool ok;
};
__device__ __forceinline__ Place place_of(const KvCacheArgs &c, int stream, int pos) {
    Place p{0, false};
    if (stream < 0 || stream >= c.streams || pos < 0) return p;
    const int j = pos / c.page_size;
    if (j >= c.table_stride) return p;
    const int page = __builtin_amdgcn_readfirstlane(c.table[(size_t)stream * c.table_stride + j]);
    if (page < 0 || page >= c.n_pages) return p;
    p.at = (size_t)page * c.heads * c.page_size + (pos - j * c.page_size);
    p.ok = true;
    return p;
}

// max over the L lanes of a group (L = 8 or 16 consecutive lanes)
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    v = max(v, (uint32_t)xshfl<1>((int)v));
    v = max(v, (uint32_t)xshfl<2>((int)v));
    v = max(v, (uint32_t)xshfl<4>((int)v));
    if constexpr (L == 16) v = max(v, (uint32_t)xshfl<8>((int)v));
    return v;
}

constexpr int kUnits = 4;  // of a lane at a time

// Rows into the pools: a wave a row.  A unit is 8 elements of K or V; the row's units, K's heads then V's, go to the
// lanes in turn, kUnits a lane at a time and their loads before the angles are formed, which lane p keeps
// in LDS for the row.  A group of D / 8 lanes holds one head.
// 8-bit caches: with t = max|x| over the head and d = t / 127 (int8) or t / 448 (e4m3), the stored
// value is x (1 / d) rounded to nearest even, so |x - q d| <= d / 2 (int8) or |q d| 2^-4 (e4m3).  A d
// under 2^-126 is stored as 0 (its reciprocal would not be finite).  A head with an Inf or NaN gets
// the scale NaN and reads back as NaN, as quantising it would otherwise hide it.  The maximum is
// taken over the magnitudes' bit patterns, in which Inf and NaN are largest.
// Memory and vector work are near each other (about 180 instructions a unit: the quotients, the rotation, the
// packing); the rotation of the keys is done here so that they do not go through memory twice.  16001 rows of
// 8 x 128 fp16 into e4m3, keys turned: 30.4 us, 3.3 TB/s (a thread a unit of any row, its place in vector
// registers: 42.8).  2603 rows of 12 x 64 into int8: 7.9 us.
template <class T, int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvRowsArgs a, int table_words) {
    extern __shared__ float2 cs[];  // [waves][rot / 2], rounded up to what lanes read at once
    constexpr int L = D / 8;
    const int lane = threadIdx.x & 63, l = lane % L;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = blockIdx.x * (blockDim.x >> 6) + w;
    if (r >= a.rows) return;
    const int half = a.rope.rot / 2, of_k = a.c.heads * L, units = 2 * of_k;
    const bool rope = a.rope.freqs != nullptr, apart = a.rope.halves && half % 8 == 0;
    const T *k = (const T *)a.k + r * a.k_row, *v = (const T *)a.v + r * a.v_row - (size_t)of_k * 8;
    // with halves of whole pieces, the partners of this lane's 8 elements are 8 others
    const bool upper = 8 * l >= half, turned = 8 * l < 2 * half;
    const int mate = !turned ? 0 : (upper ? -half : half);
    // a lane reads the angles of its 8 elements (4 pairs): angle p is kept at (p % per lane) * pitch + p / per lane, so that
    // lanes read neighbouring words
    const int lanes_at = apart ? 3 : (a.rope.halves ? 0 : 2), pitch = (half + (1 << lanes_at) - 1) >> lanes_at;
    float2 *angles = cs + w * table_words;
    Raw<T, 8> raw[kUnits], other[kUnits];
    auto load = [&](int u0) {
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            const int u = u0 + 64 * n;
            if (u < units) {
                raw[n] = load_raw<T, 8>((u < of_k ? k : v) + 8 * u);
                if (rope && apart && u < of_k) other[n] = load_raw<T, 8>(k + 8 * u + mate);
            }
        }
    };
    load(lane);
    const Place place = place_of(a.c, __builtin_amdgcn_readfirstlane(a.stream[r]), __builtin_amdgcn_readfirstlane(a.pos[r]));
    if (!place.ok) return;
    if (rope) {
        const int pos = __builtin_amdgcn_readfirstlane(a.rope_pos != nullptr ? a.rope_pos[r] : a.pos[r]);
        for (int p = lane; p < half; p += 64)
            angles[(p & ((1 << lanes_at) - 1)) * pitch + (p >> lanes_at)] = turn(pos, a.rope.freqs[p], a.rope.mscale);
        // written and read by lanes of this one wave
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    for (int u0 = lane; u0 < units; u0 += 64 * kUnits) {
        if (u0 != lane) load(u0);
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            const int u = u0 + 64 * n;
            if (u >= units) break;  // (whole groups of lanes)
            const bool is_v = u >= of_k;
            const int h = (is_v ? u - of_k : u) / L;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Elem<T>::get(raw[n].e[i]);
            if (rope && !is_v) {
                if (apart) {
                    if (turned) {
                        const float2 *c = angles + l - (upper ? half / 8 : 0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float b = Elem<T>::get(other[n].e[i]);
                            const float2 t = c[i * pitch];
                            x[i] = fmaf(upper ? b : -b, t.y, x[i] * t.x);
                        }
                    }
                } else if (a.rope.halves) {
                    const T *src = k + h * D;
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        const int e = 8 * l + i;
                        if (e < 2 * half) {
                            const bool up = e >= half;
                            const float b = Elem<T>::get(src[up ? e - half : e + half]);
                            const float2 t = angles[up ? e - half : e];
                            const float y = fmaf(up ? b : -b, t.y, Elem<T>::get(src[e]) * t.x);
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[j] = j == i ? y : x[j];
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        if (8 * l + i < 2 * half) rotate(x[i], x[i + 1], angles[i / 2 * pitch + l], x[i], x[i + 1]);
                }
            }
            const size_t vec = place.at + (size_t)(unsigned)(h * a.c.page_size), o = vec * D + 8 * l;
            void *pool = is_v ? a.c.v : a.c.k;
            if constexpr (KV == ELEM_F32) {
                store8((float *)pool + o, x);
            } else if constexpr (KV == ELEM_F16) {
                store8((__half *)pool + o, x);
            } else {
                constexpr float top = KV == ELEM_I8 ? 127.0f : 448.0f;
                uint32_t mb = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) mb = max(mb, __float_as_uint(x[i]) & 0x7fffffffu);
                mb = group_max<L>(mb);
                const bool bad = mb >= 0x7f800000u;
                float d = __uint_as_float(mb) / top;
                if (bad || d < 1.17549435e-38f) d = 0.0f;
                const float id = d > 0.0f ? 1.0f / d : 0.0f;
                // |x id| passes the top by 2^-22 of it at most (three roundings), which rounds back to it: no clamp
                uint32_t q[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma clang fp contract(off)  // the product is rounded before it is rounded to a whole number
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = x[4 * i + j] * id;
                    if constexpr (KV == ELEM_I8) {
                        // 1.5 * 2^23 + y: the sum's low byte is y rounded to nearest even
                        uint32_t b[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(y[j] + 12582912.0f);
                        q[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                                     0x05040100u);
                    } else {
                        const int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                        q[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
                    }
                    if (bad) q[i] = 0;
                }
                *(uint2 *)((uint8_t *)pool + o) = make_uint2(q[0], q[1]);
                if (l == 0) (is_v ? a.c.v_scale : a.c.k_scale)[vec] = bad ? __uint_as_float(0x7fc00000u) : d;
            }
        }
    }
}

// Rows out of the pools, a wave a row: q d in 32 bits, rounded once to the output's type.  Rows with no place in
// the cache (a position past the table, a page outside the pools) are NaN; a negative position is
// padding and its row stays as it was.  Memory bound: 16001 rows of 8 x 128 out of e4m3 as fp16 17.9 us, 5.5 TB/s.
template <class T, int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvRowsArgs a) {
    constexpr int L = D / 8;
    constexpr int E = KV == ELEM_F32 ? 4 : (KV == ELEM_F16 ? 2 : 1);
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = blockIdx.x * (blockDim.x >> 6) + w;
    if (r >= a.rows) return;
    const int of_k = a.c.heads * L, units = 2 * of_k;
    const int pos = __builtin_amdgcn_readfirstlane(a.pos[r]);
    if (pos < 0) return;
    const Place place = place_of(a.c, __builtin_amdgcn_readfirstlane(a.stream[r]), pos);
    T *k = (T *)a.k_out + r * a.k_row, *v = (T *)a.v_out + r * a.v_row - (size_t)of_k * 8;
    for (int u0 = lane; u0 < units; u0 += 64 * kUnits) {
        uint32_t raw[kUnits][2 * E];
        float d[kUnits];
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            const int u = u0 + 64 * n;
            if (u < units && place.ok) {
                const bool is_v = u >= of_k;
                const int h = (is_v ? u - of_k : u) / L;
                const size_t vec = place.at + (size_t)(unsigned)(h * a.c.page_size);
                __builtin_memcpy(raw[n], __builtin_assume_aligned((const char *)(is_v ? a.c.v : a.c.k) + (vec * D + 8 * (u % L)) * E, 8 * E > 16 ? 16 : 8 * E),
                                 8 * E);
                if constexpr (E == 1) d[n] = (is_v ? a.c.v_scale : a.c.k_scale)[vec];
            }
        }
#pragma unroll
        for (int n = 0; n < kUnits; ++n) {
            const int u = u0 + 64 * n;
            if (u >= units) break;
            float x[8];
            if constexpr (KV == ELEM_F32) {
                __builtin_memcpy(x, raw[n], 32);
            } else if constexpr (KV == ELEM_F16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = h2f((uint16_t)(raw[n][i / 2] >> (16 * (i & 1))));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (KV == ELEM_I8) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int8_t)(raw[n][i] >> (8 * j)) * d[n];
                    } else {
                        x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)raw[n][i], 0) * d[n];
                        x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)raw[n][i], 1) * d[n];
                        x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)raw[n][i], 2) * d[n];
                        x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)raw[n][i], 3) * d[n];
                    }
                }
            }
            if (!place.ok)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(0x7fc00000u);
            store8((u < of_k ? k : v) + 8 * u, x);
        }
    }
}

// A workgroup of 4 rows, or of one where rows are few (a step's 64 rows of
// 12 x 64, written and read: 5.8 us, by fours 6.1).
template <class T, bool READ, int KV, int D>
hipError_t kv_launch(const KvRowsArgs &a, hipStream_t s) {
    const int waves = a.rows >= 2048 ? kThreads / 64 : 1, blocks = (a.rows + waves - 1) / waves;
    const int words = a.rope.freqs ? (a.rope.rot / 2 + 7) / 8 * 8 : 0;
    (void)hipGetLastError();
    if constexpr (READ)
        hipLaunchKernelGGL((kv_read_kernel<T, KV, D>), dim3(blocks), dim3(64 * waves), 0, s, a);
    else
        hipLaunchKernelGGL((kv_write_kernel<T, KV, D>), dim3(blocks), dim3(64 * waves), waves * words * sizeof(float2), s, a, words);
    return hipGetLastError();
}

template <class T, bool READ, int D>
hipError_t kv_rows_d(const KvRowsArgs &a, hipStream_t s) {
    switch (a.c.dtype) {
        case ELEM_F32: return kv_launch<T, READ, ELEM_F32, D>(a, s);
        case ELEM_F16: return kv_launch<T, READ, ELEM_F16, D>(a, s);
        case ELEM_I8: return kv_launch<T, READ, ELEM_I8, D>(a, s);
        default: return kv_launch<T, READ, ELEM_E4M3, D>(a, s);
    }
}

template <class T, bool READ>
hipError_t kv_rows(const KvRowsArgs &a, hipStream_t s) {
    return a.c.dim == 64 ? kv_rows_d<T, READ, 64>(a, s) : kv_rows_d<T, READ, 128>(a, s);
}

}  // namespace

hipError_t launch_rope_rows(const RopeRowsArgs &a, hipStream_t s) {
    return a.dtype == ELEM_F16 ? rope_rows_t<__half>(a, s) : rope_rows_t<float>(a, s);
}
hipError_t launch_kv_write(const KvRowsArgs &a, hipStream_t s) {
    return a.dtype == ELEM_F16 ? kv_rows<__half, false>(a, s) : kv_rows<float, false>(a, s);
}
hipError_t launch_kv_read(const KvRowsArgs &a, hipStream_t s) {
    return a.dtype == ELEM_F16 ? kv_rows<__half, true>(a, s) : kv_rows<float, true>(a, s);
}

}  // namespace mh
