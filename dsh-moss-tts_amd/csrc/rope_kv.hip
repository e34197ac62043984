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
// angles are formed.
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

// Divisions of a launch by numbers that it does not change, as products.
struct KvShape {
    uint32_t row_magic;  // u / (units of a row): u times 2^32 / that, rounded up (exact while their product is under 2^32)
    int page_shift;      // page_size = 1 << page_shift, or -1
};
__device__ __forceinline__ int row_of(const KvShape &k, int u) { return (int)__umulhi((uint32_t)u, k.row_magic); }

// Where row r of a call lives in the pools: the index of its first vector ([page][head 0][slot]) and
// whether there is such a place.
struct Place {
    size_t at;
    bool ok;
};
__device__ __forceinline__ Place place_of(const KvCacheArgs &c, const KvShape &k, int stream, int pos) {
    Place p{0, false};
    if (stream < 0 || stream >= c.streams || pos < 0) return p;
    const int j = k.page_shift >= 0 ? pos >> k.page_shift : pos / c.page_size;
    if (j >= c.table_stride) return p;
    const int page = c.table[(size_t)stream * c.table_stride + j];
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

// Rows into the pools.  A group of D / 8 lanes holds one (row, head) of K or V, 8 elements a lane.
// 8-bit caches: with t = max|x| over the head and d = t / 127 (int8) or t / 448 (e4m3), the stored
// value is x (1 / d) rounded to nearest even, so |x - q d| <= d / 2 (int8) or |q d| 2^-4 (e4m3).  A d
// under 2^-126 is stored as 0 (its reciprocal would not be finite).  A head with an Inf or NaN gets
// the scale NaN and reads back as NaN, as quantising it would otherwise hide it.  The maximum is
// taken over the magnitudes' bit patterns, in which Inf and NaN are largest.
// Memory bound; the rotation of the keys is done here so that they do not go through memory twice.
// A thread has N units (8 elements of K or V of one head) in flight at a time, the first before the angles.
template <class T, int KV, int D, int N>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvRowsArgs a, KvShape shape, int rpb) {
    extern __shared__ float2 cs[];  // [rpb][rot / 2]
    constexpr int L = D / 8;
    const int t = threadIdx.x, l = t % L;
    const int row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    const int half = a.rope.rot / 2, heads = a.c.heads;
    const bool rope = a.rope.freqs != nullptr, apart = a.rope.halves && half % 8 == 0;
    const int per_row = 2 * heads * L, units = nrow * per_row;  // K then V
    // with halves of whole pieces, the partners of this lane's 8 elements are 8 others
    const bool upper = 8 * l >= half, turned = 8 * l < 2 * half;
    const int mate = !turned ? 0 : (upper ? -half : half);
    Raw<T, 8> raw[N], other[N];
    const T *src[N];
    size_t vecs[N];
    int row[N];
    bool is_v[N], ok[N];
    auto load = [&](int u0) {
#pragma unroll
        for (int n = 0; n < N; ++n) {  // (a unit past the last is the last, and not written: groups are whole)
            const int u = u0 + n * kThreads < units ? u0 + n * kThreads : units - L + l;
            row[n] = row_of(shape, u);
            const int g = (u - row[n] * per_row) / L, r = row0 + row[n];
            is_v[n] = g >= heads;
            const int h = is_v[n] ? g - heads : g;
            src[n] = (is_v[n] ? (const T *)a.v + r * a.v_row : (const T *)a.k + r * a.k_row) + h * D;
            raw[n] = load_raw<T, 8>(src[n] + 8 * l);
            if (rope && apart && !is_v[n]) other[n] = load_raw<T, 8>(src[n] + 8 * l + mate);
            vecs[n] = (size_t)h * a.c.page_size;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const Place at = place_of(a.c, shape, a.stream[row0 + row[n]], a.pos[row0 + row[n]]);
            vecs[n] += at.at;
            ok[n] = at.ok && u0 + n * kThreads < units;
        }
    };
    load(t);
    if (rope) {
        const int *pos = a.rope_pos != nullptr ? a.rope_pos : a.pos;
        for (int i = t; i < nrow * half; i += kThreads) {
            const int r = i / half;
            cs[i] = turn(pos[row0 + r], a.rope.freqs[i - r * half], a.rope.mscale);
        }
        __syncthreads();
    }
    for (int u0 = t; u0 < units; u0 += N * kThreads) {
        if (u0 != t) load(u0);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Elem<T>::get(raw[n].e[i]);
            if (rope && !is_v[n]) {
                const float2 *c = cs + row[n] * half;
                if (apart) {
                    if (turned) {
                        c += 8 * l - (upper ? half : 0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float b = Elem<T>::get(other[n].e[i]);
                            x[i] = fmaf(upper ? b : -b, c[i].y, x[i] * c[i].x);
                        }
                    }
                } else if (a.rope.halves) {
#pragma unroll 1
                    for (int i = 0; i < 8; ++i) {
                        const int e = 8 * l + i;
                        if (e < 2 * half) {
                            const bool up = e >= half;
                            const float b = Elem<T>::get(src[n][up ? e - half : e + half]);
                            const float2 w = c[up ? e - half : e];
                            const float y = fmaf(up ? b : -b, w.y, Elem<T>::get(src[n][e]) * w.x);
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[j] = j == i ? y : x[j];
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        if (8 * l + i < 2 * half) rotate(x[i], x[i + 1], c[4 * l + i / 2], x[i], x[i + 1]);
                }
            }
            const size_t o = vecs[n] * D + 8 * l;
            void *pool = is_v[n] ? a.c.v : a.c.k;
            if constexpr (KV == ELEM_F32) {
                if (ok[n]) store8((float *)pool + o, x);
            } else if constexpr (KV == ELEM_F16) {
                if (ok[n]) store8((__half *)pool + o, x);
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
                uint32_t w[2] = {0, 0};
                if (!bad) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i] * id, -top), top);
                    if constexpr (KV == ELEM_I8) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i / 4] |= ((uint32_t)(int)rintf(x[i]) & 0xffu) << (8 * (i & 3));
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
                            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], p, true);
                        }
                    }
                }
                if (ok[n]) {
                    *(uint2 *)((uint8_t *)pool + o) = make_uint2(w[0], w[1]);
                    if (l == 0) (is_v[n] ? a.c.v_scale : a.c.k_scale)[vecs[n]] = bad ? __uint_as_float(0x7fc00000u) : d;
                }
            }
        }
    }
}

// Rows out of the pools: q d in 32 bits, rounded once to the output's type.  Rows with no place in
// the cache (a position past the table, a page outside the pools) are NaN; a negative position is
// padding and its row stays as it was.  N units of a thread in flight, as in the write.
template <class T, int KV, int D, int N>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvRowsArgs a, KvShape shape, int rpb) {
    constexpr int L = D / 8;
    constexpr int RAW = KV == ELEM_F32 ? 32 : (KV == ELEM_F16 ? 16 : 8);  // bytes of a unit
    const int row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    const int per_row = 2 * a.c.heads * L, units = nrow * per_row;
    for (int u0 = threadIdx.x; u0 < units; u0 += N * kThreads) {
        T *dst[N];
        size_t vecs[N];
        bool is_v[N], ok[N], put[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int u = min(u0 + n * kThreads, units - 1);
            const int rl = row_of(shape, u), rest = u - rl * per_row, g = rest / L, l = rest - g * L, r = row0 + rl;
            is_v[n] = g >= a.c.heads;
            const int h = is_v[n] ? g - a.c.heads : g, pos = a.pos[r];
            const Place at = place_of(a.c, shape, a.stream[r], pos);
            ok[n] = at.ok;
            put[n] = pos >= 0 && u0 + n * kThreads < units;
            vecs[n] = at.ok ? at.at + (size_t)h * a.c.page_size : 0;  // (0: any vector that exists)
            dst[n] = (is_v[n] ? (T *)a.v_out + r * a.v_row : (T *)a.k_out + r * a.k_row) + h * D + 8 * l;
        }
        const int l = threadIdx.x % L;
        uint4 raw[N][RAW > 16 ? 2 : 1];
        float d[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const char *p = (const char *)(is_v[n] ? a.c.v : a.c.k) + (vecs[n] * D + 8 * l) * elem_size(KV);
            if constexpr (RAW == 8) {
                const uint2 w = *(const uint2 *)p;
                raw[n][0] = make_uint4(w.x, w.y, 0, 0);
                d[n] = (is_v[n] ? a.c.v_scale : a.c.k_scale)[vecs[n]];
            } else {
#pragma unroll
                for (int i = 0; i < RAW / 16; ++i) raw[n][i] = ((const uint4 *)p)[i];
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float x[8];
            if constexpr (KV == ELEM_F32) {
                __builtin_memcpy(x, raw[n], 32);
            } else if constexpr (KV == ELEM_F16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __half2float(((const __half *)raw[n])[i]);
            } else {
                const uint32_t w[2] = {raw[n][0].x, raw[n][0].y};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (KV == ELEM_I8) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int8_t)(w[i] >> (8 * j)) * d[n];
                    } else {
                        x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * d[n];
                        x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * d[n];
                        x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * d[n];
                        x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * d[n];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!ok[n]) x[i] = __uint_as_float(0x7fc00000u);
            if (put[n]) store8(dst[n], x);
        }
    }
}

// Several units a thread once that leaves 512 workgroups, else one (a step's few rows).
constexpr int kWriteUnits = 2;
template <class T, bool READ, int KV, int D>
hipError_t kv_launch(const KvRowsArgs &a, hipStream_t s) {
    constexpr int N = READ ? 4 : kWriteUnits;
    const int units = 2 * a.c.heads * (D / 8), rpb_n = std::max(1, N * kThreads / units);
    const bool many = (a.rows + rpb_n - 1) / rpb_n >= 512;
    const int rpb = many ? rpb_n : std::max(1, kThreads / units), blocks = (a.rows + rpb - 1) / rpb;
    const size_t lds = a.rope.freqs ? (size_t)rpb * (a.rope.rot / 2) * sizeof(float2) : 0;
    const KvShape shape{(uint32_t)(((1ull << 32) + units - 1) / units),
                        (a.c.page_size & (a.c.page_size - 1)) == 0 ? __builtin_ctz(a.c.page_size) : -1};
    (void)hipGetLastError();
    if constexpr (READ) {
        if (many)
            hipLaunchKernelGGL((kv_read_kernel<T, KV, D, 4>), dim3(blocks), dim3(kThreads), 0, s, a, shape, rpb);
        else
            hipLaunchKernelGGL((kv_read_kernel<T, KV, D, 1>), dim3(blocks), dim3(kThreads), 0, s, a, shape, rpb);
    } else {
        if (many)
            hipLaunchKernelGGL((kv_write_kernel<T, KV, D, kWriteUnits>), dim3(blocks), dim3(kThreads), lds, s, a, shape, rpb);
        else
            hipLaunchKernelGGL((kv_write_kernel<T, KV, D, 1>), dim3(blocks), dim3(kThreads), lds, s, a, shape, rpb);
    }
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
