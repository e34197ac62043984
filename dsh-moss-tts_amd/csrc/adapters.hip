// adapters.hip -- low-rank adapters of many requests beside a shared projection (gfx950).
//
// y_r = base_r + s_a B_a (A_a x_r), with a = which[r] the row's own adapter, A_a of rank x cols and B_a of
// out x rank.  Rows without an adapter are base_r.
//
// Both products are matrix instructions with the weights as the one operand and a tile of 16 neighbouring rows as the
// other, one of the adapters among them at a time, so a lane keeps one row throughout: what scales a row is one
// number of the lane.  With one row of an adapter, 15 of 16 columns of a product idle; the instructions are still
// fewer than the vector unit would need.  One launch: a workgroup takes a tile, one of the adapters among its rows and a
// share of the outputs, and keeps t = A x on the chip.  (Two launches with t in memory were as fast at 8191 rows of 4096, 84 and
// 86 us, 19 and 16 at 2896 of 768 -> 2304, and slower below: 84 and 39 at 1086 rows of 64 adapters.)
//
// Weights are fp16, laid out once in the order in which a wave's lanes hold them, so that a load is 1 KiB in one piece.
// Rows go through LDS for the same reason: as an operand, lanes next to each other hold different rows, and 64 separate
// accesses a load made the L1 the limit: 8191 fp16 rows of 4096 -> 4096, rank 64, took 129 us, now 86 (2.4 TB/s; a copy of
// those sizes reaches 3.2).  What is left is that a workgroup's registers fill a compute unit, so that its two products
// do not overlap with another's.  2896 fp32 rows of 768 -> 2304, rank 16: 16.3 us, 3.9 TB/s.  One row: 5.7 us, a chain of loads.
//
// fp16 rows are multiplied as they are.  32-bit rows, and t, go in as two fp16 numbers, hi + lo, 22 bits: of 128 columns of a
// row (of all ranks of t) the largest is put at 2^14 by a power of two, which leaves 2^-39 of the largest as the
// finest step, and the power is taken out again in 32 bits.  The matrix instructions cut their sums towards zero, so no more
// than 8 of them go into one sum before it is added up in 32 bits with rounding.  A row's sums do not depend on where in a
// tile it stands, nor on the other rows.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

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
    half4_t q[2];
    __half e[8];
};

// The power of two that puts `top` at 2^14 .. 2^15, and its reciprocal; 1 where there is none.
struct Power {
    float up, down;
};
__device__ __forceinline__ Power power_of(float top) {
    const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent of a number >= 0
    if (top == 0.0f || e == 255) return Power{1.0f, 1.0f};
    const int up = min(127 + 14 + 127 - e, 253);
    return Power{__uint_as_float((unsigned)up << 23), __uint_as_float((unsigned)(254 - up) << 23)};
}
// Values times a power of two as hi + lo.
template <int N>
__device__ __forceinline__ void split(const float (&x)[N], float up, Frag &hi, Frag &lo) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = x[i] * up;
        hi.e[i] = __float2half_rn(v);
        lo.e[i] = __float2half_rn(v - __half2float(hi.e[i]));
    }
}
__device__ __forceinline__ float row_max(float v) {  // over the lanes of one row
    v = fmaxf(v, xshfl<16>(v));
    return fmaxf(v, xshfl<32>(v));
}
// What lanes of this wave wrote to LDS can be read by others of it.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------- the weights' order

// Of one adapter: A [cols / 32][ranks / 16][64 lanes][8], lane l with rank l % 16 of the 16, columns 8 (l / 16) .. of the 32;
// B, of up to 16 ranks, [outs / 32][64 lanes][2][4], lane l with output l % 16 of each of two 16, ranks 4 (l / 16) ..; of
// more, [outs / 64][ranks / 32][4][64 lanes][8], with output l % 16 of each of four 16, ranks 8 (l / 16) .. of the
// 32.  ranks is max_rank as 16, 32, 64 or 128, outs is out in whole 64s; what is past the adapter's own is 0.
__host__ __device__ constexpr int ranks_of(int max_rank) { return max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : max_rank <= 64 ? 64 : 128; }
__host__ __device__ constexpr int outs_of(int out) { return (out + 63) / 64 * 64; }
__host__ __device__ constexpr size_t a_size(int max_rank, int cols) { return (size_t)ranks_of(max_rank) * cols; }
__host__ __device__ constexpr size_t b_size(int max_rank, int out) { return (size_t)ranks_of(max_rank) * outs_of(out); }

// A lane's 8 elements a thread.
__global__ __launch_bounds__(256) void pack_kernel(AdapterPackArgs p, int per_a, int per_b) {
    const int i = blockIdx.x * 256 + threadIdx.x, n = blockIdx.y;
    const int rank = p.rank == nullptr ? p.max_rank : min(max(p.rank[n], 0), p.max_rank), R = ranks_of(p.max_rank);
    const int l = i & 63, m = l & 15, g = l >> 4;
    Frag f{uint4{}};
    if (i < per_a) {
        const int k = (i >> 6) % (R / 16), step = (i >> 6) / (R / 16), r = 16 * k + m;
        if (r < rank) f.u = *(const uint4 *)((const __half *)p.a + ((size_t)n * p.max_rank + r) * p.cols + 32 * step + 8 * g);
        *(uint4 *)((__half *)p.to_a + (p.first + n) * a_size(p.max_rank, p.cols) + 8 * (size_t)i) = f.u;
    }
    if (i < per_b) {
        const int u = i >> 6;
        const __half *b = (const __half *)p.b + (size_t)n * p.out * p.max_rank;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int o = R == 16 ? 32 * u + 16 * (e >> 2) + m : 64 * (u / (R / 8)) + 16 * (u & 3) + m;
            const int r = R == 16 ? 4 * g + (e & 3) : 32 * ((u >> 2) % (R / 32)) + 8 * g + e;
            if (o < p.out && r < rank) f.e[e] = b[(size_t)o * p.max_rank + r];
            else f.e[e] = __half(0.0f);
        }
        *(uint4 *)((__half *)p.to_b + (p.first + n) * b_size(p.max_rank, p.out) + 8 * (size_t)i) = f.u;
    }
}

// ---------------------------------------------------------------- t = A x

// 16 rows of 128 columns in LDS, one wave's: 16-byte pieces, piece c of row r at c ^ r of its 256 bytes, so that neither the
// rows' pieces as they are written nor the same piece of all rows as they are read fall on the same banks.
template <class X>
struct Tile {
    static constexpr int W = sizeof(X) / 2;        // pieces of 8 elements
    static constexpr int N = 4 * W;                // loads of a lane
    static constexpr int kBytes = 16 * kChunk * (int)sizeof(X);
    static __device__ __forceinline__ int at(int row, int piece) { return row * 16 * W + (piece & ~15) + ((piece ^ row) & 15); }
    // Lane l of load i: row and piece.
    static __device__ __forceinline__ int row_of(int i) { return W == 1 ? 4 * i + ((threadIdx.x & 63) >> 4) : 2 * i + ((threadIdx.x & 63) >> 5); }
    static __device__ __forceinline__ int piece_of() { return threadIdx.x & (16 * W - 1); }
};

template <class X, int RK>
struct Shrink {
    using T = Tile<X>;
    static constexpr int W = T::W;
    const X *x[T::N];  // the rows of this lane's pieces
    const __half *w;
    int cols;

    __device__ __forceinline__ Shrink(const AdapterArgs &a, int id, int row0, uint64_t who) : cols(a.cols) {
        const int some = __builtin_ctzll(who);  // rows of others are not read: their lanes read this one
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            const int r = T::row_of(i);
            x[i] = (const X *)a.x + (row0 + (who >> r & 1 ? r : some)) * a.x_row;
        }
        w = (const __half *)a.a + id * a_size(a.max_rank, a.cols) + 8 * (threadIdx.x & 63);
    }
    __device__ __forceinline__ void load(int c, uint4 (&raw)[T::N]) const {
        const int col = c + T::piece_of() * (8 / W);
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            __builtin_memcpy(&raw[i], x[i] + min(col, cols - 8 / W), 16);
            if (col >= cols) raw[i] = uint4{};  // (of the last chunk)
        }
    }
    // Chunks c, c + step, ... of the columns, into sum.  The rows' loads run a chunk ahead.
    __device__ __forceinline__ void run(int c, int step, uint4 *lds, f32x4_t (&sum)[RK]) const {
        if (c >= cols) return;
        const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
        uint4 raw[T::N];
        load(c, raw);
        while (true) {
            Frag f[4][RK];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int k = 0; k < RK; ++k) f[s][k].u = *(const uint4 *)(w + ((size_t)min(c / 32 + s, cols / 32 - 1) * RK + k) * 512);
            wave_fence();  // (the last chunk has been read)
#pragma unroll
            for (int i = 0; i < T::N; ++i) lds[T::at(T::row_of(i), T::piece_of())] = raw[i];
            wave_fence();
            const int next = c + step;
            if (next < cols) load(next, raw);
            f32x4_t acc[RK] = {};
            float down = 1.0f;
            if constexpr (W == 1) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const Frag v{lds[T::at(m, 4 * s + g)]};
#pragma unroll
                    for (int k = 0; k < RK; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[s][k].h, v.h, acc[k], 0, 0, 0);
                }
            } else {
                float v[4][8], top = 0.0f;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const uint4 two[2] = {lds[T::at(m, 8 * s + 2 * g)], lds[T::at(m, 8 * s + 2 * g + 1)]};
                    __builtin_memcpy(v[s], two, 32);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[s][i]));
                }
                const Power p = power_of(row_max(top));
                down = p.down;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    Frag hi, lo;
                    split(v[s], p.up, hi, lo);
#pragma unroll
                    for (int k = 0; k < RK; ++k) {
                        acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[s][k].h, hi.h, acc[k], 0, 0, 0);
                        acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[s][k].h, lo.h, acc[k], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < RK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[k][i] = fmaf(acc[k][i], down, sum[k][i]);
            if (next >= cols) break;
            c = next;
        }
    }
};

// ---------------------------------------------------------------- y = base + B t

// This lane's row of t as operands: steps of 32 ranks, or one of 16.
template <int RK>
struct Rows {
    static constexpr int KS = (RK + 1) / 2, N = RK == 1 ? 4 : 8;  // elements of a lane in a step
    Frag hi[KS], lo[KS];
    float factor;
    template <class Get>
    __device__ __forceinline__ void set(float scale, Get &&get_t) {
        const int g = (threadIdx.x & 63) >> 4;
        float v[KS][N], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            get_t(32 * s + N * g, v[s]);
#pragma unroll
            for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(v[s][i]));
        }
        const Power p = power_of(row_max(top));
        factor = p.down * scale;
#pragma unroll
        for (int s = 0; s < KS; ++s) split(v[s], p.up, hi[s], lo[s]);
    }
};

// Groups of 64 outputs of a tile's rows, a wave each.  The products' lanes hold one row and four outputs of 16; through LDS they come to
// lanes that hold 16 bytes of y next to each other.
template <class Y, int RK>
struct Expand {
    static constexpr int KS = Rows<RK>::KS, F = RK == 1 ? 2 : 4 * KS;  // 16-byte loads of weights
    static constexpr int P = 16 / (int)sizeof(Y), N = 16 / P;          // outputs of a piece of y, pieces of a lane
    struct In {
        Frag f[F];
        uint4 raw[N];
    };
    const Y *base[N];
    Y *y[N];
    bool mine[N];
    int out1;
    const __half *w;

    static __device__ __forceinline__ int row_of(int i) { return (i * 64 + ((int)threadIdx.x & 63)) / (64 / P); }
    static __device__ __forceinline__ int first() { return ((int)threadIdx.x & (64 / P - 1)) * P; }
    __device__ __forceinline__ Expand(const AdapterArgs &a, int id, int64_t row0, uint64_t who, int end) : out1(end) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row_of(i);
            mine[i] = who >> r & 1;
            base[i] = (const Y *)a.base + (row0 + r) * a.base_row + first();
            y[i] = (Y *)a.y + (row0 + r) * a.y_row + first();
        }
        w = (const __half *)a.b + id * b_size(a.max_rank, a.out) + 8 * (threadIdx.x & 63);
    }
    __device__ __forceinline__ void load(int o, In &in) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (mine[i] && o + first() < out1) __builtin_memcpy(&in.raw[i], base[i] + o, 16);
#pragma unroll
        for (int i = 0; i < F; ++i) in.f[i].u = *(const uint4 *)(w + ((size_t)(o / 64) * F + i) * 512);
    }
    __device__ __forceinline__ void finish(int o, const Rows<RK> &t, const In &in, uint4 *lds) const {
        const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
        f32x4_t acc[4] = {};
        if constexpr (RK == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x16f16(in.f[q >> 1].q[q & 1], t.hi[0].q[0], acc[q], 0, 0, 0);
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x16f16(in.f[q >> 1].q[q & 1], t.lo[0].q[0], acc[q], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(in.f[4 * s + q].h, t.hi[s].h, acc[q], 0, 0, 0);
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(in.f[4 * s + q].h, t.lo[s].h, acc[q], 0, 0, 0);
                }
        }
        wave_fence();  // (the last group has been read)
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // outputs 16 q + 4 g .. of row m: piece 4 q + g of its 256 bytes, at that ^ m
            f32x4_t v = acc[q] * t.factor;
            lds[16 * m + ((4 * q + g) ^ m)] = __builtin_bit_cast(uint4, v);
        }
        wave_fence();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row_of(i);
            if (!mine[i] || o + first() >= out1) continue;
            Y v[P];
            float d[P];
            __builtin_memcpy(v, &in.raw[i], 16);
#pragma unroll
            for (int j = 0; j < P / 4; ++j) {
                const uint4 u = lds[16 * r + ((first() / 4 + j) ^ r)];
                __builtin_memcpy(d + 4 * j, &u, 16);
            }
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float z = get(v[j]) + d[j];
                if constexpr (sizeof(Y) == 2)
                    v[j] = __float2half_rn(z);
                else
                    v[j] = z;
            }
            __builtin_memcpy(y[i] + o, v, 16);
        }
    }
    // Groups o, o + step, ...; the next one's loads run ahead.
    __device__ __forceinline__ void run(int o, int step, const Rows<RK> &t, uint4 *lds) const {
        if (o >= out1) return;
        In in, next;
        load(o, in);
        while (true) {
            const bool more = o + step < out1;
            if (more) load(o + step, next);
            finish(o, t, in, lds);
            if (!more) break;
            in = next;
            o += step;
        }
    }
};

// ---------------------------------------------------------------- tiles

// Rows `who` without an adapter, or one of rank 0: y is base.
template <class Y>
__device__ __forceinline__ void copy_rows(const AdapterArgs &a, int64_t row0, int rows, uint64_t who, int out0, int out1) {
    if (a.y == a.base) return;
    const int units = (out1 - out0) * (int)sizeof(Y) / 16;
    for (int r = threadIdx.x >> 6; r < rows; r += blockDim.x >> 6) {
        if (!(who >> r & 1)) continue;
        const char *from = (const char *)((const Y *)a.base + (row0 + r) * a.base_row + out0);
        char *to = (char *)((Y *)a.y + (row0 + r) * a.y_row + out0);
        for (int u = threadIdx.x & 63; u < units; u += 64) {
            uint4 v;
            __builtin_memcpy(&v, from + 16 * u, 16);
            __builtin_memcpy(to + 16 * u, &v, 16);
        }
    }
}

// The adapters among a tile's rows, one after the other: take(adapter or -1, its rows) for every gridDim.y-th.
template <class Take>
__device__ __forceinline__ void each_adapter(const AdapterArgs &a, int row0, int rows, Take &&take) {
    const int lane = threadIdx.x & 63;
    int id = -2;
    if (lane < rows && row0 + lane < a.rows) {
        id = a.which[row0 + lane];
        if (id < 0 || id >= a.n) id = -1;
    }
    uint64_t todo = __ballot(id != -2);
    for (int j = 0; todo; ++j) {
        const int mine = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        const uint64_t who = __ballot(id == mine);
        todo &= ~who;
        if (j % gridDim.y == blockIdx.y) take(mine, who);
    }
}
__device__ __forceinline__ float sum8(const float *p, int step) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kSlices; ++j) s += p[j * step];
    return s;
}

// Both products of a tile of 16 rows (RK: ranks of 16), for outs_each outputs.
template <class X, class Y, int RK>
__global__ __launch_bounds__(kThreads) void adapter_kernel(AdapterArgs a, int outs_each) {
    constexpr int kPart = kSlices * 16 * RK * kTPitch * 4, kTiles = kSlices * Tile<X>::kBytes;
    __shared__ uint4 lds[std::max({kPart, kTiles, kSlices * 4096}) / 16];
    float *part = (float *)lds;  // [slice][rank][row]
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16, out0 = blockIdx.z * outs_each, out1 = min(out0 + outs_each, a.out);
    each_adapter(a, row0, 16, [&](int id, uint64_t who) {
        if (id < 0) return copy_rows<Y>(a, row0, 16, who, out0, out1);
        f32x4_t sum[RK] = {};
        const Shrink<X, RK> shrink(a, id, row0, who);
        __syncthreads();  // (the last adapter's outputs have left LDS)
        shrink.run(kChunk * w, kChunk * kSlices, lds + w * Tile<X>::kBytes / 16, sum);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[(w * 16 * RK + 16 * k + 4 * g + i) * kTPitch + m] = sum[k][i];
        __syncthreads();
        Rows<RK> t;
        t.set(a.scale == nullptr ? 1.0f : a.scale[id], [&](int k, auto &v) {
#pragma unroll
            for (int i = 0; i < Rows<RK>::N; ++i) v[i] = sum8(part + (k + i) * kTPitch + m, 16 * RK * kTPitch);
        });
        __syncthreads();
        const Expand<Y, RK> expand(a, id, row0, who, out1);
        expand.run(out0 + 64 * w, 64 * kSlices, t, lds + w * 256);
    });
}

template <class X, class Y, int RK>
hipError_t launch(const AdapterArgs &a, hipStream_t s) {
    (void)hipGetLastError();
    const int tiles = (a.rows + 15) / 16, groups = (a.out + 63) / 64;
    // Workgroups for the adapters of a tile, and for shares of the outputs (each share forms t again), until there are 512. Most
    // of them find no adapter left and end; 2048 of them took 23 us in place of 16 at 2896 rows, 256 56 in place of 39 at
    // 1086 rows of 64 adapters.
    const int of_tile = std::min({16, a.rows, a.n + 1});
    const int each = std::min(of_tile, std::max(2, 512 / tiles));
    const int slices = std::min(std::max(1, 512 / (tiles * each)), std::max(1, groups / kSlices));
    const int outs = (groups + slices - 1) / slices * 64;
    hipLaunchKernelGGL((adapter_kernel<X, Y, RK>), dim3(tiles, each, (a.out + outs - 1) / outs), dim3(kThreads), 0, s, a, outs);
    return hipGetLastError();
}

template <class X, class Y>
hipError_t launch_xy(const AdapterArgs &a, hipStream_t s) {
    switch (ranks_of(a.max_rank)) {
        case 16: return launch<X, Y, 1>(a, s);
        case 32: return launch<X, Y, 2>(a, s);
        case 64: return launch<X, Y, 4>(a, s);
        default: return launch<X, Y, 8>(a, s);
    }
}

}  // namespace

void adapter_sizes(const AdapterArgs &a, size_t *a_bytes, size_t *b_bytes) {
    *a_bytes = a.n * a_size(a.max_rank, a.cols) * 2;
    *b_bytes = a.n * b_size(a.max_rank, a.out) * 2;
}

hipError_t launch_adapter_pack(const AdapterPackArgs &all, hipStream_t s) {
    (void)hipGetLastError();
    constexpr int kMost = 65535;  // of a grid's y
    const int per_a = (int)(a_size(all.max_rank, all.cols) / 8), per_b = (int)(b_size(all.max_rank, all.out) / 8);
    for (int from = 0; from < all.count; from += kMost) {
        AdapterPackArgs p = all;
        p.a = (const __half *)all.a + (size_t)from * all.max_rank * all.cols;
        p.b = (const __half *)all.b + (size_t)from * all.out * all.max_rank;
        if (all.rank != nullptr) p.rank = all.rank + from;
        p.first = all.first + from;
        p.count = std::min(all.count - from, kMost);
        hipLaunchKernelGGL(pack_kernel, dim3((std::max(per_a, per_b) + 255) / 256, p.count), dim3(256), 0, s, p, per_a, per_b);
    }
    return hipGetLastError();
}

hipError_t launch_adapter_rows(const AdapterArgs &a, hipStream_t s) {
    if (a.x_dtype == ELEM_F16) return a.y_dtype == ELEM_F16 ? launch_xy<__half, __half>(a, s) : launch_xy<__half, float>(a, s);
    return a.y_dtype == ELEM_F16 ? launch_xy<float, __half>(a, s) : launch_xy<float, float>(a, s);
}

}  // namespace mh
