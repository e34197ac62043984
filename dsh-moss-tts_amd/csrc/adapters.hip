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
// accesses a load made the L1 the limit: 8191 fp16 rows of 4096 -> 4096, rank 64, took 129 us, 86 through LDS, now 77 (2.6 TB/s of the
// 201 MB that it reads and writes; a copy of 134 MB in tiles of 16 rows reaches 3.2).  What is left is that a workgroup's registers
// fill a compute unit, so that its two products do not overlap with another's.  2896 fp32 rows of 768 -> 2304, rank 16: 13.8 us, 4.6
// TB/s.  One row: 5.3 us, a chain of loads.
//
// No kernel keeps anything in scratch memory: weights are held as far as they have to run ahead, in places that the next ones take as
// soon as they have been used; places in LDS are worked out anew for each tile; and the eight partial sums of t are added up once
// where ranks are many.  Before that, 4260 fp32 rows that change between 5 adapters of rank 128, 768 -> 768, took 170 us, now 66; 7434 of 14,
// 32 -> 544, 346, now 134.  Such rows read every adapter among 16 of them again for each 16.
//
// fp16 rows are multiplied as they are.  32-bit rows, and t, go in as two fp16 numbers, hi + lo, 22 bits: of 128 columns of a
// row (of all ranks of t) the largest is put at 2^14 by a power of two, which leaves 2^-39 of the largest as the
// finest step, and the power is taken out again in 32 bits.  The matrix instructions cut their sums towards zero, so no more
// than 8 of them go into one sum before it is added up in 32 bits with rounding.  A row's sums do not depend on where in a
// tile it stands, nor on the other rows.
#include <algorithm>
#include <type_traits>

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

template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F &&f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, I + 1>(f);
    }
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
// This thread's number, as one that the compiler does not know: places in LDS that follow from it are not held in registers from one
// tile to the next, which took 60 of them.
__device__ __forceinline__ int own_thread() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
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

// A tile's rows of one adapter: row0 + r for the bits r of who.
struct TileRows {
    int64_t row0;
    uint64_t who;
};

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
    static __device__ __forceinline__ int row_of(int lane, int i) { return W == 1 ? 4 * i + (lane >> 4) : 2 * i + (lane >> 5); }
    static __device__ __forceinline__ int piece_of(int lane) { return lane & (16 * W - 1); }
};

template <class X, int RK>
struct Shrink {
    using T = Tile<X>;
    static constexpr int W = T::W;
    static constexpr bool kPeel = RK < 8;  // whether the last chunk has code of its own
    static constexpr int KB = std::min(RK, 2), R = std::min(RK, 4);  // 16s of ranks at a time, and whose weights are held
    const X *x[T::N];  // the rows of this lane's pieces
    const __half *w;
    int cols, lane;

    __device__ __forceinline__ Shrink(const AdapterArgs &a, int id, const TileRows &rows, int own) : cols(a.cols), lane(own) {
        const int some = __builtin_ctzll(rows.who);  // rows of others are not read: their lanes read this one
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            const int r = T::row_of(lane, i);
            x[i] = (const X *)a.x + (rows.row0 + (rows.who >> r & 1 ? r : some)) * a.x_row;
        }
        w = (const __half *)a.a + id * a_size(a.max_rank, a.cols) + 8 * lane;
    }
    __device__ __forceinline__ void load(int c, uint4 (&raw)[T::N]) const {
        const int col = c + T::piece_of(lane) * (8 / W);
#pragma unroll
        for (int i = 0; i < T::N; ++i) {
            __builtin_memcpy(&raw[i], x[i] + min(col, cols - 8 / W), 16);
            if (!kPeel && col >= cols) raw[i] = uint4{};  // (of the last chunk; else in LDS, so that nothing waits here)
        }
    }
    __device__ __forceinline__ void load_weights(int c, int k, Frag (&f)[4]) const {
#pragma unroll
        for (int s = 0; s < 4; ++s) f[s].u = *(const uint4 *)(w + ((size_t)min(c / 32 + s, cols / 32 - 1) * RK + k) * 512);
    }
    // Chunks c, c + step, ... of the columns, into sum.  The rows' loads run a chunk ahead, the weights' R 16s of ranks: all of a
    // chunk's at rank 128 would be half of the registers.  No load stands behind a branch, so that each is waited for by itself, but at rank
    // 128, where a last chunk of its own takes too many registers (271 -> 286 us, 7784 fp32 rows of 3 adapters in turn, 4096 -> 4096).
    __device__ __forceinline__ void run(int c, int step, uint4 *lds, f32x4_t (&sum)[RK]) const {
        if (c >= cols) return;
        uint4 raw[T::N];
        Frag f[R][4];
        load(c, raw);
#pragma unroll
        for (int k = 0; k < R; ++k) load_weights(c, k, f[k]);
        if constexpr (kPeel) {
            for (; c + step < cols; c += step) chunk(c, c + step, true, lds, raw, f, sum);
            chunk(c, c, false, lds, raw, f, sum);
        } else {
            for (; c < cols; c += step) chunk(c, c + step, c + step < cols, lds, raw, f, sum);
        }
    }
    // Chunk c, and with `more` the loads of chunk next.
    __device__ __forceinline__ void chunk(int c, int next, bool more, uint4 *lds, uint4 (&raw)[T::N], Frag (&f)[R][4], f32x4_t (&sum)[RK]) const {
        const int m = lane & 15, g = lane >> 4;
        if (kPeel && c + kChunk > cols && c + T::piece_of(lane) * (8 / W) >= cols)
#pragma unroll
            for (int i = 0; i < T::N; ++i) raw[i] = uint4{};
        wave_fence();  // (the last chunk has been read)
#pragma unroll
        for (int i = 0; i < T::N; ++i) lds[T::at(T::row_of(lane, i), T::piece_of(lane))] = raw[i];
        wave_fence();
        Frag hi[4], lo[4];
        float down = 1.0f;
        if constexpr (W == 1) {
#pragma unroll
            for (int s = 0; s < 4; ++s) hi[s].u = lds[T::at(m, 4 * s + g)];
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
            for (int s = 0; s < 4; ++s) split(v[s], p.up, hi[s], lo[s]);
        }
#pragma unroll
        for (int k0 = 0; k0 < RK; k0 += KB) {
            if (more && k0 == RK - R) load(next, raw);  // (behind the last weights of this chunk, which are waited for first)
            f32x4_t acc[KB] = {};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int k = 0; k < KB; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[(k0 + k) % R][s].h, hi[s].h, acc[k], 0, 0, 0);
                if constexpr (W == 2)
#pragma unroll
                    for (int k = 0; k < KB; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[(k0 + k) % R][s].h, lo[s].h, acc[k], 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                if (k0 + k + R < RK)
                    load_weights(c, k0 + k + R, f[(k0 + k) % R]);
                else if (more)
                    load_weights(next, k0 + k + R - RK, f[(k0 + k) % R]);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[k0 + k][i] = fmaf(acc[k][i], down, sum[k0 + k][i]);
            }
        }
    }
};

// ---------------------------------------------------------------- y = base + B t

// This lane's row of t as operands: steps of 32 ranks, or one of 16.
template <int RK>
struct Rows {
    static constexpr int KS = (RK + 1) / 2, N = RK == 1 ? 4 : 8;  // elements of a lane in a step
    Frag hi[KS], lo[KS];
    float scale, down;
    template <class Get>
    __device__ __forceinline__ void set(float by, int lane, Get &&get_t) {
        const int g = lane >> 4;
        float v[KS][N], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            get_t(32 * s + N * g, v[s]);
#pragma unroll
            for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(v[s][i]));
        }
        const Power p = power_of(row_max(top));
        scale = by;
        down = p.down;
#pragma unroll
        for (int s = 0; s < KS; ++s) split(v[s], p.up, hi[s], lo[s]);
    }
};

// Groups of 64 outputs of a tile's rows, a wave each.  The products' lanes hold one row and four outputs of 16; through LDS they come to
// lanes that hold 16 bytes of y next to each other.
template <class Y, int RK>
struct Expand {
    static constexpr int KS = Rows<RK>::KS, F = RK == 1 ? 2 : 4 * KS;  // 16-byte loads of weights
    static constexpr bool kPeel = RK < 8;
    static constexpr int P = 16 / (int)sizeof(Y), N = 16 / P;          // outputs of a piece of y, pieces of a lane
    const Y *base[N];
    Y *y[N];
    bool mine[N];
    int out1, lane;
    const __half *w;

    __device__ __forceinline__ int row_of(int i) const { return (i * 64 + lane) / (64 / P); }
    __device__ __forceinline__ int first() const { return (lane & (64 / P - 1)) * P; }
    __device__ __forceinline__ Expand(const AdapterArgs &a, int id, const TileRows &rows, int end, int own) : out1(end), lane(own) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row_of(i);
            mine[i] = rows.who >> r & 1;
            base[i] = (const Y *)a.base + (rows.row0 + (mine[i] ? r : __builtin_ctzll(rows.who))) * a.base_row;  // (others read that one)
            y[i] = (Y *)a.y + (rows.row0 + r) * a.y_row + first();
        }
        w = (const __half *)a.b + id * b_size(a.max_rank, a.out) + 8 * lane;
    }
    __device__ __forceinline__ void load_base(int o, uint4 (&raw)[N]) const {
        const int at = min(o + first(), out1 - P);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (kPeel || mine[i]) __builtin_memcpy(&raw[i], base[i] + at, 16);  // (rows of others only where it saves a branch)
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void load_weights(int o, Frag (&f)[F]) const {
#pragma unroll
        for (int i = FROM; i < TO; ++i) f[i].u = *(const uint4 *)(w + ((size_t)(o / 64) * F + i) * 512);
    }
    // Group o; with `more`, the weights of group next take the places of those that have been used.
    __device__ __forceinline__ void finish(int o, int next, bool more, const Rows<RK> &t, Frag (&f)[F], const uint4 (&raw)[N], uint4 *lds) const {
        const int m = lane & 15, g = lane >> 4;
        f32x4_t acc[4] = {};
        if constexpr (RK == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x16f16(f[q >> 1].q[q & 1], t.hi[0].q[0], acc[q], 0, 0, 0);
                acc[q] = __builtin_amdgcn_mfma_f32_16x16x16f16(f[q >> 1].q[q & 1], t.lo[0].q[0], acc[q], 0, 0, 0);
            }
            if (more) load_weights<0, F>(next, f);
        } else {
            static_for<KS>([&](auto step) {
                constexpr int s = decltype(step)::value;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[4 * s + q].h, t.hi[s].h, acc[q], 0, 0, 0);
                    acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[4 * s + q].h, t.lo[s].h, acc[q], 0, 0, 0);
                }
                if (more) load_weights<4 * s, 4 * s + 4>(next, f);
            });
        }
        wave_fence();  // (the last group has been read)
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // outputs 16 q + 4 g .. of row m: piece 4 q + g of its 256 bytes, at that ^ m
            f32x4_t v = acc[q] * t.scale * t.down;  // (the power of two last: it rounds only what leaves the range)
            lds[16 * m + ((4 * q + g) ^ m)] = __builtin_bit_cast(uint4, v);
        }
        wave_fence();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row_of(i);
            if (!mine[i] || o + first() >= out1) continue;
            Y v[P];
            float d[P];
            __builtin_memcpy(v, &raw[i], 16);
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
        Frag f[F];
        uint4 raw[N], ahead[N];
        load_base(o, raw);
        load_weights<0, F>(o, f);
        if constexpr (kPeel) {
            for (; o + step < out1; o += step) {
                load_base(o + step, ahead);
                finish(o, o + step, true, t, f, raw, lds);
                __builtin_memcpy(raw, ahead, sizeof(raw));
            }
            finish(o, o, false, t, f, raw, lds);
        } else {
            for (; o < out1; o += step) {
                const bool more = o + step < out1;
                if (more) load_base(o + step, ahead);
                finish(o, o + step, more, t, f, raw, lds);
                __builtin_memcpy(raw, ahead, sizeof(raw));
            }
        }
    }
};

// ---------------------------------------------------------------- tiles

// Rows without an adapter: y is base.
template <class Y>
__device__ __forceinline__ void copy_rows(const AdapterArgs &a, const TileRows &rows, int out0, int out1) {
    if (a.y == a.base) return;
    const int units = (out1 - out0) * (int)sizeof(Y) / 16;
    for (int r = threadIdx.x >> 6; r < 16; r += blockDim.x >> 6) {
        if (!(rows.who >> r & 1)) continue;
        const char *from = (const char *)((const Y *)a.base + (rows.row0 + r) * a.base_row + out0);
        char *to = (char *)((Y *)a.y + (rows.row0 + r) * a.y_row + out0);
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

// Both products of a tile of up to 16 rows of one adapter (RK: ranks of 16), for outputs out0 .. out1.
template <class X, class Y, int RK>
struct Products {
    static constexpr int kPart = kSlices * 16 * RK * kTPitch * 4, kTiles = kSlices * Tile<X>::kBytes;
    static constexpr int kBytes = std::max({kPart, kTiles, kSlices * 4096});
    static __device__ __forceinline__ void of(const AdapterArgs &a, int id, const TileRows &rows, int out0, int out1, uint4 *lds) {
        if (id < 0) return copy_rows<Y>(a, rows, out0, out1);
        float *part = (float *)lds;  // [slice][rank][row]
        const int t = own_thread(), lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), m = lane & 15, g = lane >> 4;
        f32x4_t sum[RK] = {};
        const Shrink<X, RK> shrink(a, id, rows, lane);
        __syncthreads();  // (the last adapter's outputs have left LDS)
        shrink.run(kChunk * w, kChunk * kSlices, lds + w * Tile<X>::kBytes / 16, sum);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[(w * 16 * RK + 16 * k + 4 * g + i) * kTPitch + m] = sum[k][i];
        __syncthreads();
        // The slices' sums: of many ranks each by one thread, of few by every wave for itself, which saves a barrier.
        constexpr int kSlice = 16 * RK * kTPitch;
        constexpr bool kShared = RK >= 4;
        if constexpr (kShared) {
#pragma unroll
            for (int i = 0; i < 256 * RK / kThreads; ++i) {
                float *p = part + (i * kThreads + t) / 16 * kTPitch + (t & 15);
                *p = sum8(p, kSlice);
            }
            __syncthreads();
        }
        Rows<RK> tr;
        tr.set(a.scale == nullptr ? 1.0f : a.scale[id], lane, [&](int k, auto &v) {
#pragma unroll
            for (int i = 0; i < Rows<RK>::N; ++i) {
                const float *p = part + (k + i) * kTPitch + m;
                v[i] = kShared ? *p : sum8(p, kSlice);
            }
        });
        __syncthreads();
        const Expand<Y, RK> expand(a, id, rows, out1, lane);
        expand.run(out0 + 64 * w, 64 * kSlices, tr, lds + w * 256);
    }
};

template <class X, class Y, int RK>
__global__ __launch_bounds__(kThreads) void adapter_kernel(AdapterArgs a, int outs_each) {
    __shared__ uint4 lds[Products<X, Y, RK>::kBytes / 16];
    const int row0 = blockIdx.x * 16, out0 = blockIdx.z * outs_each, out1 = min(out0 + outs_each, a.out);
    each_adapter(a, row0, 16, [&](int id, uint64_t who) { Products<X, Y, RK>::of(a, id, TileRows{row0, who}, out0, out1, lds); });
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
    // Two workgroups of fp16 kernels of up to 32 ranks fit a compute unit, and where there is about one for each, some share one while others
    // have none.  More than half of the LDS keeps them apart: 3560 rows in runs, 4096 -> 4096, rank 32, 25.4 -> 20.6 us, in turn 43 -> 53; with
    // more tiles it costs (8192 rows in runs 47 -> 53), with fewer, where more of a tile's workgroups have work, too (285 rows of
    // 58 adapters 11 -> 16), and of up to 16 ranks rows in turn lose more (1221: 11.4 -> 16.5) than runs gain (21.6 -> 18.4).
    constexpr bool kTwo = RK == 2 && sizeof(X) == 2 && sizeof(Y) == 2;
    const unsigned spare = kTwo && each <= 2 && tiles <= 256 ? 82 * 1024 - Products<X, Y, RK>::kBytes : 0;
    hipLaunchKernelGGL((adapter_kernel<X, Y, RK>), dim3(tiles, each, (a.out + outs - 1) / outs), dim3(kThreads), spare, s, a, outs);
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
