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

// N elements at p as 32-bit floats: 16-byte accesses where `vec` (p is then 16-byte aligned),
// one element at a time elsewhere.
template <class T, int N>
__device__ __forceinline__ void load_n(const T *p, bool vec, float (&x)[N]) {
    constexpr int B = N * (int)sizeof(T);
    if (B % 16 == 0 && vec) {
        uint4 raw[B / 16 ? B / 16 : 1];
#pragma unroll
        for (int i = 0; i < B / 16; ++i) raw[i] = ((const uint4 *)p)[i];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Elem<T>::get(((const T *)raw)[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Elem<T>::get(p[i]);
    }
}
template <class T, int N>
__device__ __forceinline__ void store_n(T *p, bool vec, const float (&x)[N]) {
    constexpr int B = N * (int)sizeof(T);
    if (B % 16 == 0 && vec) {
        uint4 raw[B / 16 ? B / 16 : 1];
#pragma unroll
        for (int i = 0; i < N; ++i) ((T *)raw)[i] = Elem<T>::put(x[i]);
#pragma unroll
        for (int i = 0; i < B / 16; ++i) ((uint4 *)p)[i] = raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = Elem<T>::put(x[i]);
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
// Memory bound: every element is read and written once, in 16-byte pieces where base, strides
// and (halves) rot / 2 allow it.
template <class T, bool HALVES, int V>
__global__ __launch_bounds__(kThreads) void rope_rows_kernel(RopeRowsArgs a, int rpb, int per_head) {
    extern __shared__ float2 cs[];  // [rpb][rot / 2]
    const int half = a.rope.rot / 2, t = threadIdx.x;
    const int row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    for (int i = t; i < nrow * half; i += kThreads) {
        const int r = i / half;
        cs[i] = turn(a.pos[row0 + r], a.rope.freqs[i - r * half], a.rope.mscale);
    }
    __syncthreads();
    const int units = a.heads * per_head, turned = HALVES ? half / V : per_head;
    for (int u = blockIdx.y * kThreads + t; u < nrow * units; u += kThreads * gridDim.y) {
        const int r = u / units, hu = u - r * units, h = hu / per_head, p = hu - h * per_head;
        const T *x = (const T *)a.x + (row0 + r) * a.x_row + h * a.x_head;
        T *y = (T *)a.y + (row0 + r) * a.y_row + h * a.y_head;
        const float2 *c = cs + r * half;
        if (HALVES && p < turned) {
            float lo[V], hi[V];
            load_n<T, V>(x + p * V, true, lo);
            load_n<T, V>(x + half + p * V, true, hi);
#pragma unroll
            for (int i = 0; i < V; ++i) rotate(lo[i], hi[i], c[p * V + i], lo[i], hi[i]);
            store_n<T, V>(y + p * V, true, lo);
            store_n<T, V>(y + half + p * V, true, hi);
        } else {
            const int e = HALVES ? 2 * half + (p - turned) * V : p * V;
            float v[V];
            load_n<T, V>(x + e, true, v);
            if constexpr (!HALVES) {
#pragma unroll
                for (int i = 0; i < V; i += 2)
                    if (e + i < 2 * half) rotate(v[i], v[i + 1], c[(e + i) / 2], v[i], v[i + 1]);
            }
            store_n<T, V>(y + e, true, v);
        }
    }
}

template <class T, bool HALVES, int V>
hipError_t rope_rows(const RopeRowsArgs &a, hipStream_t s) {
    const int half = a.rope.rot / 2;
    const int per_head = HALVES ? half / V + (a.dim - a.rope.rot) / V : a.dim / V;
    const long long units = (long long)a.heads * per_head;
    const int rpb = units >= kThreads ? 1 : (int)std::min<long long>(kThreads / units, 16);
    const int blocks = (a.rows + rpb - 1) / rpb;
    const int split = rpb == 1 && a.rows < 512 ? (int)std::min<long long>((units + kThreads - 1) / kThreads, 64) : 1;
    (void)hipGetLastError();
    hipLaunchKernelGGL((rope_rows_kernel<T, HALVES, V>), dim3(blocks, split), dim3(kThreads), rpb * half * sizeof(float2), s, a,
                       rpb, per_head);
    return hipGetLastError();
}

template <class T>
hipError_t rope_rows_t(const RopeRowsArgs &a, hipStream_t s) {
    constexpr int V = 16 / (int)sizeof(T);
    auto whole = [](int64_t n) { return n % V == 0; };
    const bool vec = ((uintptr_t)a.x | (uintptr_t)a.y) % 16 == 0 && whole(a.x_row) && whole(a.x_head) && whole(a.y_row) &&
                     whole(a.y_head) && whole(a.dim);
    if (a.rope.halves)
        return vec && whole(a.rope.rot / 2) ? rope_rows<T, true, V>(a, s) : rope_rows<T, true, 1>(a, s);
    return vec ? rope_rows<T, false, V>(a, s) : rope_rows<T, false, 2>(a, s);
}

// ---------------------------------------------------------------- the paged cache

// Where row r of a call lives in the pools: the index of its first vector ([page][head 0][slot]) and
// whether there is such a place.
struct Place {
    size_t at;
    bool ok;
};
__device__ __forceinline__ Place place_of(const KvCacheArgs &c, int stream, int pos) {
    Place p{0, false};
    if (stream < 0 || stream >= c.streams || pos < 0) return p;
    const int j = pos / c.page_size;
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
template <class T, int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvRowsArgs a, int rpb, bool vec) {
    extern __shared__ float2 cs[];  // [rpb][rot / 2]
    constexpr int L = D / 8;
    const int t = threadIdx.x, l = t % L;
    const int row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    const int half = a.rope.rot / 2, heads = a.c.heads;
    if (a.rope.freqs != nullptr) {
        const int *pos = a.rope_pos != nullptr ? a.rope_pos : a.pos;
        for (int i = t; i < nrow * half; i += kThreads) {
            const int r = i / half;
            cs[i] = turn(pos[row0 + r], a.rope.freqs[i - r * half], a.rope.mscale);
        }
        __syncthreads();
    }
    const int units = 2 * heads * L;  // K then V
    for (int u = t; u < nrow * units; u += kThreads) {
        const int rl = u / units, g = (u - rl * units) / L, r = row0 + rl;
        const bool is_v = g >= heads;
        const int h = is_v ? g - heads : g;
        const T *src = (is_v ? (const T *)a.v + r * a.v_row : (const T *)a.k + r * a.k_row) + h * D;
        float x[8];
        load_n<T, 8>(src + 8 * l, vec, x);
        const Place at = place_of(a.c, a.stream[r], a.pos[r]);
        if (!is_v && a.rope.freqs != nullptr) {
            const float2 *c = cs + rl * half;
            if (a.rope.halves) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = 8 * l + i;
                    if (e < 2 * half) {
                        const bool up = e >= half;
                        const float b = Elem<T>::get(src[up ? e - half : e + half]);
                        const float2 w = c[up ? e - half : e];
                        x[i] = up ? x[i] * w.x + b * w.y : x[i] * w.x - b * w.y;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    if (8 * l + i < 2 * half) rotate(x[i], x[i + 1], c[4 * l + i / 2], x[i], x[i + 1]);
            }
        }
        const size_t vecs = at.at + (size_t)h * a.c.page_size;
        const size_t o = vecs * D + 8 * l;
        void *pool = is_v ? a.c.v : a.c.k;
        if constexpr (KV == ELEM_F32) {
            if (at.ok) store_n<float, 8>((float *)pool + o, true, x);
        } else if constexpr (KV == ELEM_F16) {
            if (at.ok) store_n<__half, 8>((__half *)pool + o, true, x);
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
                        int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
                        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], p, true);
                    }
                }
            }
            if (at.ok) {
                *(uint2 *)((uint8_t *)pool + o) = make_uint2(w[0], w[1]);
                if (l == 0) (is_v ? a.c.v_scale : a.c.k_scale)[vecs] = bad ? __uint_as_float(0x7fc00000u) : d;
            }
        }
    }
}

// Rows out of the pools: q d in 32 bits, rounded once to the output's type.  Rows with no place in
// the cache (a position past the table, a page outside the pools) are NaN; a negative position is
// padding and its row stays as it was.
template <class T, int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvRowsArgs a, int rpb, bool vec) {
    constexpr int L = D / 8;
    const int units = 2 * a.c.heads * L, row0 = blockIdx.x * rpb, nrow = min(rpb, a.rows - row0);
    for (int u = threadIdx.x; u < nrow * units; u += kThreads) {
        const int rl = u / units, rest = u - rl * units, g = rest / L, l = rest - g * L, r = row0 + rl;
        const bool is_v = g >= a.c.heads;
        const int h = is_v ? g - a.c.heads : g;
        const int pos = a.pos[r];
        if (pos < 0) continue;
        const Place at = place_of(a.c, a.stream[r], pos);
        float x[8];
        if (at.ok) {
            const size_t vecs = at.at + (size_t)h * a.c.page_size;
            const size_t o = vecs * D + 8 * l;
            const void *pool = is_v ? a.c.v : a.c.k;
            if constexpr (KV == ELEM_F32) {
                load_n<float, 8>((const float *)pool + o, true, x);
            } else if constexpr (KV == ELEM_F16) {
                load_n<__half, 8>((const __half *)pool + o, true, x);
            } else {
                const uint2 w = *(const uint2 *)((const uint8_t *)pool + o);
                const float d = (is_v ? a.c.v_scale : a.c.k_scale)[vecs];
                const uint32_t ww[2] = {w.x, w.y};
    #pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (KV == ELEM_I8) {
    #pragma unroll
                        for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int8_t)(ww[i] >> (8 * j)) * d;
                    } else {
                        x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)ww[i], 0) * d;
                        x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)ww[i], 1) * d;
                        x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)ww[i], 2) * d;
                        x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)ww[i], 3) * d;
                    }
                }
            }
        } else {
    #pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(0x7fc00000u);
        }
        T *dst = (is_v ? (T *)a.v_out + r * a.v_row : (T *)a.k_out + r * a.k_row) + h * D;
        store_n<T, 8>(dst + 8 * l, vec, x);
    }
}

template <class T>
bool rows_vec(const void *k, const void *v, int64_t k_row, int64_t v_row) {
    constexpr int V = 16 / (int)sizeof(T);
    return ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_row % V == 0 && v_row % V == 0;
}

template <class T, int KV, int D>
hipError_t kv_write(const KvRowsArgs &a, hipStream_t s) {
    const int units = 2 * a.c.heads * (D / 8);
    const int rpb = units >= kThreads ? 1 : kThreads / units;
    const size_t lds = a.rope.freqs ? (size_t)rpb * (a.rope.rot / 2) * sizeof(float2) : 0;
    (void)hipGetLastError();
    hipLaunchKernelGGL((kv_write_kernel<T, KV, D>), dim3((a.rows + rpb - 1) / rpb), dim3(kThreads), lds, s, a, rpb,
                       rows_vec<T>(a.k, a.v, a.k_row, a.v_row));
    return hipGetLastError();
}

template <class T, int KV, int D>
hipError_t kv_read(const KvRowsArgs &a, hipStream_t s) {
    const int units = 2 * a.c.heads * (D / 8);
    const int rpb = units >= kThreads ? 1 : kThreads / units;
    (void)hipGetLastError();
    hipLaunchKernelGGL((kv_read_kernel<T, KV, D>), dim3((a.rows + rpb - 1) / rpb), dim3(kThreads), 0, s, a, rpb,
                       rows_vec<T>(a.k_out, a.v_out, a.k_row, a.v_row));
    return hipGetLastError();
}

template <class T, bool READ, int D>
hipError_t kv_rows_d(const KvRowsArgs &a, hipStream_t s) {
    switch (a.c.dtype) {
        case ELEM_F32: return READ ? kv_read<T, ELEM_F32, D>(a, s) : kv_write<T, ELEM_F32, D>(a, s);
        case ELEM_F16: return READ ? kv_read<T, ELEM_F16, D>(a, s) : kv_write<T, ELEM_F16, D>(a, s);
        case ELEM_I8: return READ ? kv_read<T, ELEM_I8, D>(a, s) : kv_write<T, ELEM_I8, D>(a, s);
        default: return READ ? kv_read<T, ELEM_E4M3, D>(a, s) : kv_write<T, ELEM_E4M3, D>(a, s);
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
