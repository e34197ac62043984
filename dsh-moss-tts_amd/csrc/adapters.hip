// adapters.hip -- low-rank adapters of many requests beside a shared projection (gfx950).
//
// y_r = base_r + s_a B_a (A_a x_r), with a = which[r] the row's own adapter, A_a of rank x cols and B_a of
// out x rank.  Rows without an adapter are base_r.
//
// One launch: a workgroup takes a tile of 16 or 32 neighbouring rows and one of the adapters among them, forms
// t = A x for the tile's rows of that adapter, and goes from there to its share of the outputs; t stays on the
// chip.  Both products are matrix instructions with the weights as the one operand and the rows as the other, so
// a lane keeps one row throughout: what scales a row is one number of the lane.  With one row of an adapter, 15
// of 16 columns of a product idle; the instructions are still fewer than the vector unit would need.
//
// Weights are fp16.  fp16 rows are multiplied as they are.  32-bit rows, and t, go in as two fp16 numbers, hi + lo,
// 22 bits: of 128 columns of a row (of all ranks of t) the largest is put at 2^14 by a power of two, which leaves
// 2^-39 of the largest as the finest step, and the power is taken out again in 32 bits.  The matrix
// instructions cut their sums towards zero, so no more than 8 of them go into one sum before it is added up in 32
// bits with rounding.  A row's sums do not depend on where in a tile it stands, nor on the other rows.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kSlices = 8;    // of the columns: a wave each
constexpr int kThreads = 64 * kSlices;
constexpr int kChunk = 128;   // columns under one power of two
constexpr int kTPitch = 17;   // of t in LDS, 16 rows wide

template <class T>
__device__ __forceinline__ float get(T x) {
    if constexpr (sizeof(T) == 2)
        return __half2float(x);
    else
        return x;
}

union Frag {
    uint4 u;
    half8 h;
    __half e[8];
};

// The power of two that puts `top` at 2^14 .. 2^15, and its reciprocal; 1 where there is none.
struct Power {
    float up, down;
};
__device__ __forceinline__ Power power_of(float top) {
    const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent of a number >= 0
    if (e == 0 && top == 0.0f) return Power{1.0f, 1.0f};
    if (e == 255) return Power{1.0f, 1.0f};
    const int up = min(127 + 14 + 127 - e, 253);
    return Power{__uint_as_float((unsigned)up << 23), __uint_as_float((unsigned)(254 - up) << 23)};
}
// 8 values times a power of two as hi + lo.
__device__ __forceinline__ void split8(const float (&x)[8], float up, Frag &hi, Frag &lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = x[i] * up;
        hi.e[i] = __float2half_rn(v);
        lo.e[i] = __float2half_rn(v - __half2float(hi.e[i]));
    }
}
__device__ __forceinline__ float row_max(float v) {  // over the lanes of one row
    v = fmaxf(v, xshfl<16>(v));
    return fmaxf(v, xshfl<32>(v));
}

// 8 elements of a row at any address that an element may have.
template <class X>
__device__ __forceinline__ void load8(const X *p, uint4 (&raw)[sizeof(X) / 2]) {
    __builtin_memcpy(raw, p, sizeof(raw));
}

// STEPS * 32 columns of RT tiles of rows from x and the weights' rows on (STEPS <= 4), added to sum.  No load depends on a rank or
// on which rows are the adapter's: ranks past the last give rows of t that are dropped later, and lanes of other rows
// read one that is.
template <class X, int RK, int RT, int STEPS>
__device__ __forceinline__ void shrink_chunk(const X *const (&x)[RT], const __half *const (&w)[RK], int c, f32x4_t (&sum)[RT][RK]) {
    constexpr int W = sizeof(X) / 2;  // 16-byte loads, and operands, of 8 elements
    uint4 raw[RT][STEPS][W];
    Frag f[STEPS][RK];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) load8(x[rt] + c + 32 * s, raw[rt][s]);
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int k = 0; k < RK; ++k) f[s][k].u = *(const uint4 *)(w[k] + c + 32 * s);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        f32x4_t acc[RK] = {};
        float down = 1.0f;
        Power p{1.0f, 1.0f};
        if constexpr (W == 2) {
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                float v[8];
                __builtin_memcpy(v, raw[rt][s], sizeof(v));
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
            }
            p = power_of(row_max(top));
            down = p.down;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            Frag h[W];
            if constexpr (W == 1) {
                h[0].u = raw[rt][s][0];
            } else {
                float v[8];
                __builtin_memcpy(v, raw[rt][s], sizeof(v));
                split8(v, p.up, h[0], h[W - 1]);
            }
#pragma unroll
            for (int k = 0; k < RK; ++k)
#pragma unroll
                for (int i = 0; i < W; ++i) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[s][k].h, h[i].h, acc[k], 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < RK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[rt][k][i] = fmaf(acc[k][i], down, sum[rt][k][i]);
    }
}

// RK: ranks of 16 that max_rank has; RT: tiles of 16 rows.
template <class X, class Y, int RK, int RT>
__global__ __launch_bounds__(kThreads) void adapter_kernel(AdapterArgs a, int outs_each) {
    constexpr int KS = RK == 1 ? 1 : RK / 2;  // steps of 32 ranks (RK 1: one half of a step)
    __shared__ float part[RT][kSlices][16 * RK][kTPitch];
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int m = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16 * RT;
    const int out0 = blockIdx.z * outs_each, out1 = min(out0 + outs_each, a.out);
    // the tile's adapters: this workgroup takes the blockIdx.y-th and so on
    int id = -2;
    if (lane < 16 * RT && row0 + lane < a.rows) {
        id = a.which[row0 + lane];
        if (id < 0 || id >= a.n) id = -1;
    }
    uint64_t todo = __ballot(id != -2);
    for (int j = 0; todo; ++j) {
        const int mine = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const uint64_t who = __ballot(id == mine);
        todo &= ~who;
        if (j % gridDim.y != blockIdx.y) continue;
        const int rank = mine < 0 ? 0 : (a.rank == nullptr ? a.max_rank : min(max(a.rank[mine], 0), a.max_rank));
        if (rank == 0) {  // y is base
            if (a.y == a.base) continue;
            const int units = (out1 - out0) * (int)sizeof(Y) / 16;
            for (int r = w; r < 16 * RT; r += kSlices) {
                if (!(who >> r & 1)) continue;
                const char *from = (const char *)((const Y *)a.base + (row0 + r) * a.base_row + out0);
                char *to = (char *)((Y *)a.y + (row0 + r) * a.y_row + out0);
                for (int u = lane; u < units; u += 64) {
                    uint4 v;
                    __builtin_memcpy(&v, from + 16 * u, 16);
                    __builtin_memcpy(to + 16 * u, &v, 16);
                }
            }
            continue;
        }
        const float scale = a.scale == nullptr ? 1.0f : a.scale[mine];
        // t = A x: a wave an eighth of the chunks of columns
        {
            f32x4_t sum[RT][RK] = {};
            const X *x[RT];
            const int some = __builtin_ctzll(who);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                x[rt] = (const X *)a.x + (row0 + (who >> (16 * rt + m) & 1 ? 16 * rt + m : some)) * a.x_row + 8 * g;
            const __half *wa[RK];
#pragma unroll
            for (int k = 0; k < RK; ++k)
                wa[k] = (const __half *)a.a + ((size_t)mine * a.max_rank + min(16 * k + m, a.max_rank - 1)) * a.cols + 8 * g;
            int c = kChunk * w;
            for (; c + kChunk <= a.cols; c += kChunk * kSlices) shrink_chunk<X, RK, RT, 4>(x, wa, c, sum);
            const int left = (a.cols - c) / 32;  // of this wave's last chunk
            if (left == 1)
                shrink_chunk<X, RK, RT, 1>(x, wa, c, sum);
            else if (left == 2)
                shrink_chunk<X, RK, RT, 2>(x, wa, c, sum);
            else if (left == 3)
                shrink_chunk<X, RK, RT, 3>(x, wa, c, sum);
            __syncthreads();  // (the last adapter's t is no longer read)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < RK; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[rt][w][16 * k + 4 * g + i][m] = sum[rt][k][i];
        }
        __syncthreads();
        // this lane's row of t in each tile: the operands of B t
        Frag hi[RT][KS], lo[RT][KS];
        float factor[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float v[KS][8], top = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = 32 * s + 8 * g + i, at = min(k, 16 * RK - 1);
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < kSlices; ++j) sum += part[rt][j][at][m];
                    v[s][i] = k < rank ? sum : 0.0f;
                    top = fmaxf(top, fabsf(v[s][i]));
                }
            const Power p = power_of(row_max(top));
            factor[rt] = p.down * scale;
#pragma unroll
            for (int s = 0; s < KS; ++s) split8(v[s], p.up, hi[rt][s], lo[rt][s]);
        }
        // B's elements past the rank may be anything: the bits of a lane's 8 that count
        uint4 keep[KS];
        int at_k[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int k = 32 * s + 8 * g;
            at_k[s] = min(k, a.max_rank - 8);
            auto two = [&](int i) { return (k + i < rank ? 0xffffu : 0u) | (k + i + 1 < rank ? 0xffff0000u : 0u); };
            keep[s] = make_uint4(two(0), two(2), two(4), two(6));
        }
        // B t: a wave 64 outputs of all rows
        constexpr int P = 16 / (int)sizeof(Y);  // outputs of a lane that lie together: output i of tile q is the lane's q * 4 + i-th
        for (int o = out0 + 64 * w; o < out1; o += 64 * kSlices) {
            Frag f[4][KS];
            uint4 raw[RT][16 / P];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                // row m of the product's tile q is this output
                const int at = P == 4 ? o + 16 * q + m : o + 32 * (q >> 1) + 8 * (m >> 2) + 4 * (q & 1) + (m & 3);
                const __half *wb = (const __half *)a.b + ((size_t)mine * a.out + min(at, a.out - 1)) * a.max_rank;
#pragma unroll
                for (int s = 0; s < KS; ++s) f[q][s].u = *(const uint4 *)(wb + at_k[s]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int q = 0; q < 16 / P; ++q) {
                    const int at = P == 4 ? o + 16 * q + 4 * g : o + 32 * q + 8 * g;
                    if ((who >> (16 * rt + m) & 1) && at < out1)
                        __builtin_memcpy(&raw[rt][q], (const Y *)a.base + (row0 + 16 * rt + m) * a.base_row + at, 16);
                }
            f32x4_t acc[RT][4] = {};
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    f[q][s].u.x &= keep[s].x;
                    f[q][s].u.y &= keep[s].y;
                    f[q][s].u.z &= keep[s].z;
                    f[q][s].u.w &= keep[s].w;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        acc[rt][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q][s].h, hi[rt][s].h, acc[rt][q], 0, 0, 0);
                        acc[rt][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[q][s].h, lo[rt][s].h, acc[rt][q], 0, 0, 0);
                    }
                }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int q = 0; q < 16 / P; ++q) {
                    const int at = P == 4 ? o + 16 * q + 4 * g : o + 32 * q + 8 * g;
                    if (!(who >> (16 * rt + m) & 1) || at >= out1) continue;
                    Y v[P];
                    __builtin_memcpy(v, &raw[rt][q], 16);
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        const float y = fmaf(acc[rt][q * (P / 4) + i / 4][i & 3], factor[rt], get(v[i]));
                        if constexpr (sizeof(Y) == 2)
                            v[i] = __float2half_rn(y);
                        else
                            v[i] = y;
                    }
                    __builtin_memcpy((Y *)a.y + (row0 + 16 * rt + m) * a.y_row + at, v, 16);
                }
        }
    }
}

template <class X, class Y, int RK>
hipError_t launch(const AdapterArgs &a, hipStream_t s) {
    (void)hipGetLastError();
    const int tiles = (a.rows + 15) / 16, groups = (a.out + 63) / 64;
    constexpr int kMost = RK == 8 ? 1 : 2;  // (t of two tiles of 128 ranks takes a whole unit's LDS)
    const int rt = tiles >= 512 ? kMost : 1;
    const int blocks = (tiles + rt - 1) / rt;
    const int of_tile = std::min({16 * rt, a.rows, a.n + 1});
    const int each = std::min(of_tile, std::max(2, 2048 / blocks));  // workgroups for the adapters of a tile
    const int want = std::max(1, 512 / (blocks * each));
    const int slices = std::min(want, std::max(1, groups / kSlices));
    const int outs = (groups + slices - 1) / slices * 64;
    const dim3 grid(blocks, each, (a.out + outs - 1) / outs);
    if (rt == kMost)
        hipLaunchKernelGGL((adapter_kernel<X, Y, RK, kMost>), grid, dim3(kThreads), 0, s, a, outs);
    else
        hipLaunchKernelGGL((adapter_kernel<X, Y, RK, 1>), grid, dim3(kThreads), 0, s, a, outs);
    return hipGetLastError();
}

template <class X, class Y>
hipError_t launch_xy(const AdapterArgs &a, hipStream_t s) {
    return a.max_rank <= 16 ? launch<X, Y, 1>(a, s) : a.max_rank <= 32 ? launch<X, Y, 2>(a, s) : a.max_rank <= 64 ? launch<X, Y, 4>(a, s) : launch<X, Y, 8>(a, s);
}

}  // namespace

hipError_t launch_adapter_rows(const AdapterArgs &a, hipStream_t s) {
    if (a.x_dtype == ELEM_F16) return a.y_dtype == ELEM_F16 ? launch_xy<__half, __half>(a, s) : launch_xy<__half, float>(a, s);
    return a.y_dtype == ELEM_F16 ? launch_xy<float, __half>(a, s) : launch_xy<float, float>(a, s);
}

}  // namespace mh
