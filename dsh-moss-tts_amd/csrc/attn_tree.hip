// attn_tree.hip -- attention of a few rows per stream (one token, or a tree of drafted ones) over a
// paged K/V cache in fp32, fp16, int8 or e4m3, with grouped heads (gfx950).
//
// Row i of a stream attends the stream's whole context, keys 0 .. ctx - 1, and those of the drafted
// positions ctx + j (j < n, the stream's row count) whose bit j its mask has:
//   s_p = scale (q . k_p),  o = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m),  lse = m + log(sum).
// A row that sees nothing is 0 with lse = -inf.
//
// The n rows x (heads / kv_heads) queries that share a key head are packed into tiles of 16, the
// columns of the matrix instructions, so a key is loaded once for all of them.  A workgroup's 4 or 8
// waves take every 4th or 8th span of keys with a running maximum and sum each, and are joined through LDS; with
// few workgroups the keys are also cut over workgroups, whose partial results a second launch
// joins in their order (no atomics: the same call gives the same bits).
//
// Per 16 keys, S^T = K Q^T (A = K: lane l holds key l % 16; B = Q: row l % 16), so a lane has the
// scores of one row and 4 neighbouring keys; O^T = V^T P^T takes them as its B operand as they are,
// with the 8 values of a lane being keys 4g .. 4g + 3 (g = l / 16) of two 16-key blocks.  V's A
// operand wants 8 keys of one dim in a lane: lane (c, g) loads the D / 16 neighbouring dims from
// c D / 16 of those 8 keys and turns that little block over in its own registers with byte
// permutes, so V needs no LDS and both loads cover whole rows.  Output dim c D / 16 + j is then
// row c of the j-th product.
//
// Arithmetic: fp16, int8 and e4m3 values are exact in the fp16 products; a 32-bit query (scaled by a
// power of two to below 2) and the softmax weights go in as fp16 hi + lo: 22 bits, but no finer than 2^-35 of the
// largest (fp16's smallest step, with the largest near its range's end), which shows where nearly all the weight is
// on keys whose values are 0.  int8 / e4m3 scales multiply the scores and the weights; weights are kept in
// fp16's range by a power of two of each row's own, which falls as the row's largest weight times value scale
// rises.  An fp32 cache runs on the fp32 matrix instructions.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr float kSlack = 5.0f;  // log 2 of how far below its place a row's largest weight may lie
constexpr float kPlace = 16.0f;  // log 2 of that place: what passes fp16's 65504 is left to lo
// Scores past this are rounded before ref is taken off: past 2^31 a product's last bits alone can leave exp2's range.
constexpr float kFar = 16384.0f;
// log 2 of the least product of weight and value scale that is put in its place: 2^(kPlace - kLeast) has to be a float.
constexpr float kLeast = -109.0f;

struct TreePlan {
    int tiles, group, row_groups;  // row tiles of 16, of which a workgroup takes `group`
    int waves;                     // of a workgroup of the kernel for few rows
    int slots;                     // pieces that all streams' keys are cut into; streams: no cuts, and no workspace
    int chunk;                     // keys of a piece where every stream has as many slots
    uint64_t page_magic;           // block of 16 keys / blocks of a page, as a product
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }

__device__ __forceinline__ uint32_t bias_off(uint32_t w) {  // two halves 1024 + (q + 128) -> q
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w) - bias);
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}

struct Frag {  // 8 halves
    uint32_t w[4];
    __device__ __forceinline__ half8 h() const { return __builtin_bit_cast(half8, *this); }
};
__device__ __forceinline__ floatx4 mfma(const Frag &a, const Frag &b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h(), b.h(), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// x as hi + lo halves, hi towards zero and lo to nearest: off by half of 2^-21 of it, or of 2^-24 where that is more
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    float x = fmaf((float)h[0], -1.0f, a), y = fmaf((float)h[1], -1.0f, b);
    asm("" : "+v"(x), "+v"(y));  // (as fma_mixlo and fma_mixhi these are 5 % of the kernel for many rows)
    const h2 l = {(_Float16)x, (_Float16)y};
    lo = __builtin_bit_cast(uint32_t, l);
}

// A lane's share of 32 keys x D of one head, as they lie in memory: of K the A operand of S^T (key
// l % 16 of each block of 16), of V the lane's dims of keys 4g .. 4g + 3 of each block.
template <int KV, int D>
struct Keys {
    static constexpr int NW = D * elem_size(KV) / 64;
    uint4 k[2][NW];
    uint32_t v[2][4][NW];
    float4 ks[2], vs[2];
};

// The block of keys kb .. kb + 15 of a stream, or of the last one that has any up to key `last`: the index of its
// first vector.  A block lies in one page, so all of it can be read; what lies behind the last key is masked like a key
// that no row sees.  A page outside the pools sets `bad` (and page 0 is read in its place).
__device__ __forceinline__ size_t block_of(const TreeArgs &a, const TreePlan &plan, const int *table, int h, int kb, int last,
                                           bool &bad) {
    kb = min(kb, last & ~15);
    const uint32_t blk = (uint32_t)kb >> 4, pg = (uint32_t)((blk * plan.page_magic) >> 40);
    int page = __builtin_amdgcn_readfirstlane(table[pg]);
    if (page < 0 || page >= a.c.n_pages) {
        page = 0;
        bad = true;
    }
    return ((size_t)page * a.c.heads + h) * a.c.page_size + (blk - pg * (a.c.page_size >> 4)) * 16;
}

// Loads of the block at vector `at`: K as NW 16-byte pieces of a key, V as NW words of each of 4 keys; a lane's
// offsets are the same for every block.
template <int KV, int D>
__device__ __forceinline__ void load_k(const TreeArgs &a, size_t at, int c, int g, uint4 (&k)[Keys<KV, D>::NW]) {
    const char *p = (const char *)a.c.k + at * (D * elem_size(KV));
#pragma unroll
    for (int u = 0; u < Keys<KV, D>::NW; ++u) k[u] = *(const uint4 *)(p + (unsigned)(c * (D * elem_size(KV)) + 16 * g + 64 * u));
}
template <int KV, int D>
__device__ __forceinline__ void load_v(const TreeArgs &a, size_t at, int c, int g, uint32_t (&v)[4][Keys<KV, D>::NW]) {
    constexpr int NW = Keys<KV, D>::NW;
    const char *p = (const char *)a.c.v + at * (D * elem_size(KV));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        __builtin_memcpy(v[i], __builtin_assume_aligned(p + (unsigned)((4 * g + i) * (D * elem_size(KV)) + c * (NW * 4)), NW < 4 ? NW * 4 : 16),
                         NW * 4);
}

// The 8 dims of K fragment s (f16 products) start at this one, for lane group g.
template <int KV>
__device__ __forceinline__ constexpr int frag_dim(int s, int g) {
    return KV == ELEM_F16 ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
}

template <int KV, int D>
__device__ __forceinline__ Frag k_frag(const uint4 (&k)[Keys<KV, D>::NW], int s) {
    Frag f;
    if constexpr (KV == ELEM_F16) {
        f.w[0] = k[s].x, f.w[1] = k[s].y, f.w[2] = k[s].z, f.w[3] = k[s].w;
    } else {
        const uint2 q = s % 2 ? make_uint2(k[s / 2].z, k[s / 2].w) : make_uint2(k[s / 2].x, k[s / 2].y);
        if constexpr (KV == ELEM_I8) {
            f = __builtin_bit_cast(Frag, i8x8_to_h8(q));
        } else {
            f.w[0] = e4m3_pair(q.x, false), f.w[1] = e4m3_pair(q.x, true);
            f.w[2] = e4m3_pair(q.y, false), f.w[3] = e4m3_pair(q.y, true);
        }
    }
    return f;
}

// The half of V's fragments that one block of 16 keys gives: words w[0], w[1] of the fragments of dims
// 4n .. 4n + 3 (8 bit) or 2n, 2n + 1 (fp16) of the lane's D / 16.
template <int KV>
constexpr int dims_per_word() {
    return KV == ELEM_F16 ? 2 : 4;
}
template <int KV, int NW>
__device__ __forceinline__ void v_halves(const uint32_t (&v)[4][NW], int n, uint32_t (&f)[dims_per_word<KV>()][2]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const uint32_t a = v[2 * q][n], b = v[2 * q + 1][n];
        if constexpr (KV == ELEM_F16) {
            f[0][q] = perm(b, a, 0x05040100u);
            f[1][q] = perm(b, a, 0x07060302u);
        } else {
            const uint32_t x = KV == ELEM_I8 ? 0x80808080u : 0u;
            const uint32_t t01 = perm(b ^ x, a ^ x, 0x05010400u), t23 = perm(b ^ x, a ^ x, 0x07030602u);
            if constexpr (KV == ELEM_I8) {
                f[0][q] = bias_off(perm(0x64646464u, t01, 0x04010400u));
                f[1][q] = bias_off(perm(0x64646464u, t01, 0x04030402u));
                f[2][q] = bias_off(perm(0x64646464u, t23, 0x04010400u));
                f[3][q] = bias_off(perm(0x64646464u, t23, 0x04030402u));
            } else {
                f[0][q] = e4m3_pair(t01, false), f[1][q] = e4m3_pair(t01, true);
                f[2][q] = e4m3_pair(t23, false), f[3][q] = e4m3_pair(t23, true);
            }
        }
    }
}

// One element of V in 32 bits.
template <int KV>
__device__ __forceinline__ float v_value(const void *p, size_t i) {
    if constexpr (KV == ELEM_F32) return ((const float *)p)[i];
    if constexpr (KV == ELEM_F16) return __half2float(((const __half *)p)[i]);
    if constexpr (KV == ELEM_I8) return (float)((const int8_t *)p)[i];
    return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t *)p)[i], 0);
}

// The raw V values of a word with each Inf or NaN among them as 0.
template <int KV>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    if constexpr (KV == ELEM_F32) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    if constexpr (KV == ELEM_F16)
        return ((w & 0x7c00u) == 0x7c00u ? 0u : w & 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : w & 0xffff0000u);
    if constexpr (KV == ELEM_E4M3) {  // NaN is 0x7f: plus one carries into the byte's top bit
        const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
        return w & ~(nan * 0xffu);
    }
    return w;
}

// A stream's rows and keys; n = 0 where there is nothing to do.
struct Stream {
    int row0, n, ctx, total;
    bool bad;  // more keys than the launch or the table has room for
};
__device__ __forceinline__ Stream stream_at(const TreeArgs &a, int row0, int end, int ctx) {
    Stream t;
    t.row0 = row0;
    t.n = row0 < 0 || end > a.rows || end <= row0 ? 0 : min(end - row0, a.max_rows);
    t.ctx = ctx;
    const long long room = min((long long)a.c.table_stride * a.c.page_size, (long long)a.max_keys);
    t.bad = ctx < 0 || (long long)ctx + t.n > room;
    t.total = t.bad ? 0 : ctx + t.n;
    return t;
}
__device__ __forceinline__ Stream stream_of(const TreeArgs &a, int s) {
    return stream_at(a, __builtin_amdgcn_readfirstlane(a.row_start[s]), __builtin_amdgcn_readfirstlane(a.row_start[s + 1]),
                     __builtin_amdgcn_readfirstlane(a.ctx_len[s]));
}

// One piece of the keys: those from beg to end of a stream (-1: none), whose pieces are the slots from `first` on.
struct Cut {
    int stream, beg, end, first, pieces;
};
// Up to 64 streams share the slots out by their lengths: pieces of the fewest keys (a multiple of 128, at least 256)
// of which there are no more than slots, so that no workgroup has much more to do than another, however
// ragged the streams (7 of 8192 to 16384 keys and one just begun: 203 us with as many pieces each, 172 so, both
// before later steps).  Every wave finds that size for itself, lane s holding stream s.  More streams: as many slots each.
__device__ __forceinline__ int sum64(int v) {
    v += xshfl<32>(v);
    v += xshfl<16>(v);
    v += xshfl<8>(v);
    v += xshfl<4>(v);
    v += xshfl<2>(v);
    v += xshfl<1>(v);
    return v;
}
__device__ __forceinline__ int max64(int v) {
    v = max(v, xshfl<32>(v));
    v = max(v, xshfl<16>(v));
    v = max(v, xshfl<8>(v));
    v = max(v, xshfl<4>(v));
    v = max(v, xshfl<2>(v));
    return max(v, xshfl<1>(v));
}
// The sum over the lanes below: shifts within rows of 16, then row ends handed on.
__device__ __forceinline__ int sum_below(int v) {
    int sum = v;
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xF, 0xF, false);  // row_shr:1
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xF, 0xF, false);
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    sum += __builtin_amdgcn_update_dpp(0, sum, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return sum - v;
}
// The size of a piece and how many of it the lane's stream has, in blocks of 128 keys.
__device__ __forceinline__ int even_chunk(const TreeArgs &a, const TreePlan &plan, int &pieces) {
    const int lane = threadIdx.x & 63;
    int mine = 0;
    if (lane < a.c.streams) {
        const Stream st = stream_at(a, a.row_start[lane], a.row_start[lane + 1], a.ctx_len[lane]);
        mine = st.n == 0 ? 0 : (max(st.total, 1) + 127) / 128;  // (rows that are to be NaN need a piece too)
    }
    const int most = max64(mine), even = (sum64(mine) + plan.slots - 1) / plan.slots;
    int chunk = __builtin_amdgcn_readfirstlane(max(max(even, (most + kMaxSplits - 1) / kMaxSplits), 2));
    const int step = (chunk + 15) / 16;
    while (true) {  // (ends at the longest stream's keys at the latest: then there are no more pieces than streams)
        pieces = (mine + chunk - 1) / chunk;
        if (__builtin_amdgcn_readfirstlane(sum64(pieces)) <= plan.slots) return chunk * 128;
        chunk += step;
    }
}
__device__ __forceinline__ bool even_cuts(const TreeArgs &a, const TreePlan &plan) { return a.c.streams > 1 && a.c.streams <= 64; }
__device__ __forceinline__ Cut cut_of_slot(const TreeArgs &a, const TreePlan &plan, int slot) {
    if (plan.slots == a.c.streams) return Cut{slot, 0, 0x7fffffff, slot, 1};
    if (!even_cuts(a, plan)) {
        const int per = plan.slots / a.c.streams, s = slot / per, z = slot - s * per;
        return Cut{s, z * plan.chunk, (z + 1) * plan.chunk, s * per, per};
    }
    int pieces;
    const int chunk = even_chunk(a, plan, pieces), before = sum_below(pieces);
    const uint64_t who = __ballot(slot >= before && slot < before + pieces);
    if (who == 0) return Cut{-1, 0, 0, 0, 0};
    const int s = __builtin_ctzll(who), first = __builtin_amdgcn_readlane(before, s), z = slot - first;
    return Cut{s, z * chunk, (z + 1) * chunk, first, __builtin_amdgcn_readlane(pieces, s)};
}
// N values of a query in 32 bits, at element i.
template <int N>
__device__ __forceinline__ void load_q(const TreeArgs &a, bool f32, size_t i, float (&x)[N]) {
    if (f32) {
        const float *p = (const float *)a.q + i;
        if (a.q_vec) {
#pragma unroll
            for (int e = 0; e < N; e += 4) *(float4 *)&x[e] = *(const float4 *)(p + e);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = p[e];
        }
    } else {
        const __half *p = (const __half *)a.q + i;
        if (a.q_vec) {
            __half h[N];
            __builtin_memcpy(h, __builtin_assume_aligned(p, N >= 8 ? 16 : 2 * N), 2 * N);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = __half2float(h[e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = __half2float(p[e]);
        }
    }
}

// One packed query of a lane's row: fp16 fragments (hi, and lo of a 32-bit query) or 32-bit values.  Its
// scores in units of log 2 are qs times the products; qs > 0 (the sign of the scale goes into the query, and
// a scale of 0 is one so small that it makes no score differ from 0).
template <int KV, int D, bool LO>
struct Query {
    static constexpr bool F32 = KV == ELEM_F32;
    Frag hi[F32 ? 1 : D / 32], lo[F32 || !LO ? 1 : D / 32];
    float f[F32 ? D / 4 : 1];
    float qs;
    uint64_t mask;

    __device__ __forceinline__ void load(const TreeArgs &a, const Stream &st, int grp, int h, int i, int packed, int g) {
        const bool ok = i < packed;
        const int node = ok ? i / grp : 0, row = st.row0 + node, head = h * grp + (ok ? i - node * grp : 0);
        const size_t base = (size_t)((int64_t)row * a.q_row + head * D);
        mask = !ok ? 0 : (a.row_mask != nullptr ? a.row_mask[row] : (2ull << node) - 1);
        if (st.n < 64) mask &= (1ull << st.n) - 1;
        const bool minus = a.scale < 0.0f;
        qs = fmaxf(fabsf(a.scale) * kLog2e, 1.17549435e-38f);
        if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < D / 16; ++u) {
                float x[4];
                load_q<4>(a, a.q_dtype == ELEM_F32, base + 16 * u + 4 * g, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) f[4 * u + e] = !ok ? 0.0f : (minus ? -x[e] : x[e]);
            }
        } else {
            float x[D / 32][8];
#pragma unroll
            for (int k = 0; k < D / 32; ++k) {
                load_q<8>(a, LO, base + frag_dim<KV>(k, g), x[k]);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e] = !ok ? 0.0f : (minus ? -x[k][e] : x[k][e]);
            }
            if constexpr (LO) {
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
                top = max(top, (uint32_t)xshfl<16>((int)top));
                top = max(top, (uint32_t)xshfl<32>((int)top));
                const int e2 = (int)(top >> 23) - 127;  // a power of two: exact (an Inf or NaN stays one)
                qs = fmaxf(__builtin_amdgcn_ldexpf(qs, e2), 1.17549435e-38f);
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        split2(__builtin_amdgcn_ldexpf(x[k][e], -e2), __builtin_amdgcn_ldexpf(x[k][e + 1], -e2), hi[k].w[e / 2],
                               lo[k].w[e / 2]);
            } else {
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        hi[k].w[e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[k][e], x[k][e + 1]));
            }
        }
    }
};

// Whether a row whose mask is `bits` sees key `pos` (of a stream's ctx + n).
__device__ __forceinline__ bool visible(const Stream &st, uint64_t bits, int pos) {
    const int j = pos - st.ctx;
    return j < 0 || (j < st.n && ((bits >> (j & 63)) & 1));
}

// Softmax state of a lane's rows, one per tile: l = sum w, o = sum w v with weights w = 2^(x - ref) of the scores x so far,
// l of this lane's keys only, summed span by span with what each addition rounds off kept in `lost` (equal weights round
// the same way each time: 2e-4 of 131072 that were added one by one).  ref is a whole number, so scaling by its changes is
// exact.  No score passes it, and the largest is at most kSlack + 1/2 below: it moves (and o and l are scaled) only when a
// score passes it, which after the first spans is rare, where the largest itself still moves in every other span for some
// row of a tile.  kSlack is what a weight's place costs in bits: with 3 the kernel for many rows takes 10 % longer, with 8
// no less than with 5.
// For the fp16 products the weights are multiplied by 2^kPlace; with value scales (SCALED) a weight times its scale
// is, by 2^(kPlace - top), where no such product of the row so far has passed 2^top: top moves like ref.  Both are a
// row's own business: what other rows of a tile see changes nothing.  `settle` takes these factors out.
template <int MT, int ND, bool SCALED, bool F32>
struct Rows {
    static constexpr float kUp = F32 || SCALED ? 0.0f : kPlace;  // log 2 of what w itself is multiplied by
    float ref[MT], l[MT], lost[MT];
    float top[SCALED ? MT : 1], g[SCALED ? MT : 1];  // g = 2^(kPlace - top)
    floatx4 o[MT][ND];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            ref[mt] = -INFINITY;
            l[mt] = lost[mt] = 0.0f;
            if constexpr (SCALED) {
                top[mt] = kLeast;
                g[mt] = exp2_(kPlace - kLeast);
            }
#pragma unroll
            for (int j = 0; j < ND; ++j) o[mt][j] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void settle(int mt) {
        l[mt] = (l[mt] - lost[mt]) * exp2_(-kUp);
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)  // (2^(top - kPlace) itself can be below what fp32 holds)
                o[mt][j][r] = SCALED ? __builtin_amdgcn_ldexpf(o[mt][j][r], (int)(top[mt] - kPlace)) : o[mt][j][r] * exp2_(-kUp);
    }
    // Products x (times key scales) of 32 keys, -inf where the row does not see the key, become weights (times 2^kUp).
    // Returns how far the largest of these scores is from ref.
    __device__ __forceinline__ float weigh(int mt, float qs, float (&x)[2][4]) {
        float mx = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
        mx = fmaxf(mx, xshfl<16>(mx));
        mx = fmaxf(mx, xshfl<32>(mx)) * qs;
        if (__any(mx > ref[mt])) {
            const bool up = mx > ref[mt];
            const float r = up ? rintf(mx) + kSlack : ref[mt], by = up ? ref[mt] - r : 0.0f;
            ref[mt] = r;
            float fade = exp2_(by);
            l[mt] *= fade;
            lost[mt] *= fade;
            if constexpr (SCALED) {  // top stays where it was, unless it would fall under kLeast
                const float t = fmaxf(top[mt] + by, kLeast);
                fade = exp2_(top[mt] + by - t);
                top[mt] = t;
                g[mt] = exp2_(kPlace - t);
            }
#pragma unroll
            for (int j = 0; j < ND; ++j) o[mt][j] *= fade;
        }
        const float r0 = ref[mt] == -INFINITY ? 0.0f : ref[mt];
        const bool far = fabsf(mx) > kFar && fabsf(mx) < INFINITY;
        if (__any(far)) {
#pragma clang fp contract(off)  // rounded as mx was
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float z = x[b][i] * qs;
                    x[b][i] = exp2_(far ? (z - r0) + kUp : fmaf(x[b][i], qs, kUp - r0));
                }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[b][i] = exp2_(fmaf(x[b][i], qs, kUp - r0));
        }
        const float add = (((x[0][0] + x[0][1]) + (x[0][2] + x[0][3])) + ((x[1][0] + x[1][1]) + (x[1][2] + x[1][3]))) - lost[mt];
        const float sum = l[mt] + add;
        lost[mt] = (sum - l[mt]) - add;
        l[mt] = sum;
        return mx - r0;
    }
    // Weights times value scales, 0 where the row does not see the key, are put in place: `most` is what weigh returned and
    // `vmax` log 2 of what no scale of the 32 keys reaches, seen or not.
    __device__ __forceinline__ void place(int mt, float most, float vmax, float (&y)[2][4]) {
        // (less a margin for the roundings of `most`: where this is false, no product passes top)
        if (__any(most + vmax > top[mt] - 0.015625f)) {
            float m = fmaxf(fmaxf(fmaxf(fabsf(y[0][0]), fabsf(y[0][1])), fmaxf(fabsf(y[0][2]), fabsf(y[0][3]))),
                            fmaxf(fmaxf(fabsf(y[1][0]), fabsf(y[1][1])), fmaxf(fabsf(y[1][2]), fabsf(y[1][3]))));
            m = fmaxf(m, xshfl<16>(m));
            m = fmaxf(m, xshfl<32>(m));
            const float e = (float)((int)(__float_as_uint(m) >> 23) - 126);  // m < 2^e
            const float t = e > top[mt] ? e + kSlack : top[mt], fade = exp2_(top[mt] - t);
            top[mt] = t;
            g[mt] = exp2_(kPlace - t);
#pragma unroll
            for (int j = 0; j < ND; ++j) o[mt][j] *= fade;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[b][i] *= g[mt];
    }
};

// log 2 of what no value with a magnitude up to this one's reaches.
__device__ __forceinline__ float above(uint32_t bits) { return (float)((int)(bits >> 23) - 126); }

// x of the keys that a row does not see becomes `v` (32 keys at p0).
template <class Q, int MT>
__device__ __forceinline__ void hide(const Stream &st, const Q (&q)[MT], int p0, int g, float v, float (&x)[MT][2][4]) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!visible(st, q[mt].mask, p0 + 16 * b + 4 * g + i)) x[mt][b][i] = v;
}
// Weights times value scales; 0 for what a row does not see, whatever its scale holds.
template <class Q, int MT>
__device__ __forceinline__ void scale_weights(const Stream &st, const Q (&q)[MT], bool tail, int p0, int g, const float4 (&vs)[2],
                                              float (&x)[MT][2][4]) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const float v[4] = {vs[b].x, vs[b].y, vs[b].z, vs[b].w};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[mt][b][i] *= v[i];
    }
    if (tail) hide(st, q, p0, g, 0.0f, x);
}

// The Inf and NaN elements of V among 32 keys, added key by key to the rows that see them (x: weights,
// `room` the wave's [16][ >= 32] floats of LDS).
template <int KV, int D, class Room, class R>
__device__ __forceinline__ void add_odd_values(const TreeArgs &a, const Stream &st, const size_t (&blk)[2], int p0, int mt,
                                               uint64_t mask, const float (&x)[2][4], Room &room, R &rows) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) room[c][16 * b + 4 * g + i] = x[b][i];
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int kk = 0; kk < 32; ++kk) {
        const int b = kk >> 4;
        const size_t at = ((b ? blk[1] : blk[0]) + (kk & 15)) * D + (D / 4) * g;
        const float wt = room[c][kk];
        const bool see = visible(st, mask, p0 + kk);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                const float v = v_value<KV>(a.c.v, at + (D / 16) * r + j);
                rows.o[mt][j][r] += see && !(fabsf(v) < INFINITY) ? wt * v : 0.0f;
            }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The workspace: each stream's first slot and how many it has (4 words a stream), (maximum, sum) of each slot's
// rows, [slots][max_rows][heads], then their unnormalised outputs.
__device__ __forceinline__ float2 *row_sums(const TreeArgs &a) { return (float2 *)((int4 *)a.ws + a.c.streams); }
__device__ __forceinline__ float *partials(const TreeArgs &a, const TreePlan &plan) {
    return (float *)(row_sums(a) + ((size_t)plan.slots * a.max_rows * a.heads + 1) / 2 * 2);
}
// Says so to the join: by the first piece's workgroup of the first head and rows.
__device__ __forceinline__ void put_cut(const TreeArgs &a, const TreePlan &plan, const Cut &cut, int slot, int h, int rg) {
    if (plan.slots > a.c.streams && slot == cut.first && h == 0 && rg == 0 && threadIdx.x == 0)
        *((int4 *)a.ws + cut.stream) = make_int4(cut.first, cut.pieces, 0, 0);
}
// Whether a row attends anything.
__device__ __forceinline__ bool sees_any(const TreeArgs &a, const Stream &st, int node) {
    const uint64_t m = a.row_mask != nullptr ? a.row_mask[st.row0 + node] : 1;
    return st.ctx > 0 || (m << (64 - st.n)) != 0;
}
// N elements from d0 on of packed row i, normalised, or, where the keys are cut, as they are with the
// row's maximum and sum (a lane of d0 = 0 writes those) for the slot.
template <int D, int N>
__device__ __forceinline__ void put_row(const TreeArgs &a, const TreePlan &plan, const Stream &st, int slot, int grp, int h, int i,
                                        int d0, float M, float L, const float (&x)[N]) {
    const int node = i / grp, head = h * grp + i - node * grp;
    if (slot >= 0 && plan.slots > a.c.streams) {
        const size_t at = (size_t)slot * a.max_rows * a.heads + node * a.heads + head;
        if (d0 == 0) row_sums(a)[at] = make_float2(M, L);
        if (L == 0.0f) return;
        float *po = partials(a, plan) + at * D + d0;
#pragma unroll
        for (int j = 0; j < N; j += 4) *(float4 *)(po + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        return;
    }
    const size_t at = (size_t)(st.row0 + node) * a.heads + head;
    if (L == 0.0f && sees_any(a, st, node)) L = __uint_as_float(0x7fc00000u);  // (no score above -inf: 0 / 0)
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const size_t o = (size_t)((int64_t)(st.row0 + node) * a.out_row + head * D + d0);
    if (a.out_dtype == ELEM_F16) {
        __half *p = (__half *)a.out + o;
        __half y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = __float2half_rn(x[j] * inv);
        if (a.out_vec) {
            __builtin_memcpy(__builtin_assume_aligned(p, N < 8 ? 2 * N : 16), y, 2 * N);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = y[j];
        }
    } else {
        float *p = (float *)a.out + o;
        if (a.out_vec) {
#pragma unroll
            for (int j = 0; j < N; j += 4) *(float4 *)(p + j) = make_float4(x[j] * inv, x[j + 1] * inv, x[j + 2] * inv, x[j + 3] * inv);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) p[j] = x[j] * inv;
        }
    }
    if (a.lse != nullptr && d0 == 0) a.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Few rows (up to 4 tiles, 2 of a workgroup): memory bound.  Each of the W = 4 or 8 waves takes every W-th span of 32 keys,
// the next span's loads in flight while one is worked on, and the waves are joined through LDS.
// LO: 32-bit queries, as hi + lo.
// One row over 130001 e4m3 keys of 8 x 128, 32 heads: 51.7 us and 4.8 of the join, 5.3 TB/s.  64 streams of 270 to 541
// int8 keys of 12 x 64: 16.1 us; 16 trees of 14 to 27 over 507 to 1015 fp16 keys of 12 x 64, by 8 waves: 15.8.  The last two
// are short of it by their chain of dependent loads (row range, page, keys, then 4 or 5 spans a wave), by the longest of
// the streams, which are not cut there, and by vector work, about 310 instructions a span.
template <int KV, int D, int MT, bool LO, int W>
__global__ __launch_bounds__(64 * W, W > kWaves ? 2 : KV == ELEM_F32 ? (D == 64 ? 2 : 1) : (D == 64 && MT == 1 ? 3 : 2)) void attn_tree_kernel(TreeArgs a, TreePlan plan) {
    constexpr bool F32 = KV == ELEM_F32, SCALED = quantised(KV);
    constexpr int NW = Keys<KV, D>::NW, ND = D / 16;
    __shared__ float so[W][16][D + 4];
    __shared__ float sm[W][16], sl[W][16];

    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // workgroups that read the same keys follow each other on one XCD, whose L2 then serves them
    const int b8 = blockIdx.x >> 3, rg = b8 % plan.row_groups, unit = (b8 / plan.row_groups) * 8 + (blockIdx.x & 7);
    if (unit >= plan.slots * a.c.heads) return;
    const int slot = unit / a.c.heads, h = unit - slot * a.c.heads;
    const Cut cut = cut_of_slot(a, plan, slot);
    const int s = cut.stream;
    if (s < 0) return;
    const Stream st = stream_of(a, s);
    const int grp = a.heads / a.c.heads, packed = st.n * grp, first = rg * MT * 16;
    if (first >= packed) return;
    const int live = min(MT, (packed - first + 15) / 16);
    bool bad = st.bad;
    const int beg = cut.beg, end = min(cut.end, st.total), last = end - 1;
    const int *table = a.c.table + (size_t)s * a.c.table_stride;

    Keys<KV, D> cur;
    size_t blk[2];
    auto fetch = [&](int p, Keys<KV, D> &to, size_t (&at)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) at[b] = block_of(a, plan, table, h, p + 16 * b, last, bad);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            load_k<KV, D>(a, at[b], c, g, to.k[b]);
            if constexpr (SCALED) {
                to.ks[b] = *(const float4 *)(a.c.k_scale + at[b] + 4 * g);
                to.vs[b] = *(const float4 *)(a.c.v_scale + at[b] + 4 * g);
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) load_v<KV, D>(a, at[b], c, g, to.v[b]);
    };
    int p0 = beg + 32 * w;
    if (p0 < end) fetch(p0, cur, blk);

    Query<KV, D, LO> q[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) q[mt].load(a, st, grp, h, first + mt * 16 + c, packed, g);
    Rows<MT, ND, SCALED, F32> rows;
    rows.clear();

#pragma unroll 1
    for (; p0 < end; p0 += 32 * W) {
        const bool tail = p0 + 32 > st.ctx;
        Keys<KV, D> next;
        size_t nblk[2];
        fetch(p0 + 32 * W, next, nblk);  // (past the end: the last block again)

        float x[MT][2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            floatx4 acc[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt] = floatx4{0.f, 0.f, 0.f, 0.f};
            if constexpr (F32) {
#pragma unroll
                for (int u = 0; u < NW; ++u) {
                    const float kf[4] = {__uint_as_float(cur.k[b][u].x), __uint_as_float(cur.k[b][u].y),
                                         __uint_as_float(cur.k[b][u].z), __uint_as_float(cur.k[b][u].w)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) acc[mt] = mfma(kf[e], q[mt].f[4 * u + e], acc[mt]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < D / 32; ++k) {
                    const Frag f = k_frag<KV, D>(cur.k[b], k);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        acc[mt] = mfma(f, q[mt].hi[k], acc[mt]);
                        if constexpr (LO) acc[mt] = mfma(f, q[mt].lo[k], acc[mt]);
                    }
                }
            }
            const float ks[4] = {cur.ks[b].x, cur.ks[b].y, cur.ks[b].z, cur.ks[b].w};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[mt][b][i] = SCALED ? acc[mt][i] * ks[i] : acc[mt][i];
        }
        if (tail) hide(st, q, p0, g, -INFINITY, x);
        float most[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) most[mt] = rows.weigh(mt, q[mt].qs, x[mt]);
        if constexpr (SCALED) {
            scale_weights(st, q, tail, p0, g, cur.vs, x);
            float v = fmaxf(fmaxf(fmaxf(fabsf(cur.vs[0].x), fabsf(cur.vs[0].y)), fmaxf(fabsf(cur.vs[0].z), fabsf(cur.vs[0].w))),
                            fmaxf(fmaxf(fabsf(cur.vs[1].x), fabsf(cur.vs[1].y)), fmaxf(fabsf(cur.vs[1].z), fabsf(cur.vs[1].w))));
            v = fmaxf(v, xshfl<16>(v));
            v = fmaxf(v, xshfl<32>(v));
            const float vmax = above((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) rows.place(mt, most[mt], vmax, x[mt]);
        }
        Frag ph[MT], pl[MT];
        if constexpr (!F32)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) split2(x[mt][b][i], x[mt][b][i + 1], ph[mt].w[2 * b + i / 2], pl[mt].w[2 * b + i / 2]);
        // drafted values that some row does not see may hold anything, and 0 times an Inf or NaN is not 0: such
        // elements go into the products as 0, and are added to the rows that see them
        if constexpr (KV != ELEM_I8) {
            if (tail) {
                bool odd = false;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < NW; ++n) {
                            const uint32_t y = cur.v[b][i][n];
                            cur.v[b][i][n] = finite_part<KV>(y);
                            odd |= cur.v[b][i][n] != y;
                        }
                if (__any(odd))
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) add_odd_values<KV, D>(a, st, blk, p0, mt, q[mt].mask, x[mt], so[w], rows);
            }
        }
        if constexpr (F32) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < ND; ++j)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            rows.o[mt][j] = mfma(__uint_as_float(cur.v[b][i][j]), x[mt][b][i], rows.o[mt][j]);
        } else {
            constexpr int DW = dims_per_word<KV>();
#pragma unroll
            for (int n = 0; n < NW; ++n) {
                uint32_t f0[DW][2], f1[DW][2];
                v_halves<KV, NW>(cur.v[0], n, f0);
                v_halves<KV, NW>(cur.v[1], n, f1);
#pragma unroll
                for (int d = 0; d < DW; ++d) {
                    const Frag f{{f0[d][0], f0[d][1], f1[d][0], f1[d][1]}};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        rows.o[mt][DW * n + d] = mfma(f, ph[mt], rows.o[mt][DW * n + d]);
                        rows.o[mt][DW * n + d] = mfma(f, pl[mt], rows.o[mt][DW * n + d]);
                    }
                }
            }
        }
        cur = next;
        blk[0] = nblk[0], blk[1] = nblk[1];
    }

    // ---- the waves joined, one row tile at a time
    put_cut(a, plan, cut, slot, h, rg);
    bad = __any(bad);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (mt >= live) break;
        rows.settle(mt);
        float sum = rows.l[mt];
        sum += xshfl<16>(sum);
        sum += xshfl<32>(sum);
        if (mt > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < ND; j += 4)
                *(float4 *)&so[w][c][ND * (4 * g + r) + j] =
                    make_float4(rows.o[mt][j][r], rows.o[mt][j + 1][r], rows.o[mt][j + 2][r], rows.o[mt][j + 3][r]);
        if (g == 0) {
            sm[w][c] = rows.ref[mt];
            sl[w][c] = bad ? __uint_as_float(0x7fc00000u) : sum;
        }
        __syncthreads();
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * ND;
        const int i = first + mt * 16 + row;
        if (row >= 16 || i >= packed) continue;
        float M = sm[0][row];
#pragma unroll
        for (int v = 1; v < W; ++v) M = fmaxf(M, sm[v][row]);
        const float M0 = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, acc[ND];
#pragma unroll
        for (int j = 0; j < ND; ++j) acc[j] = 0.0f;
#pragma unroll
        for (int v = 0; v < W; ++v) {
            const float f = exp2_(sm[v][row] - M0);
            L = fmaf(sl[v][row], f, L);
#pragma unroll
            for (int j = 0; j < ND; ++j) acc[j] = fmaf(so[v][row][d0 + j], f, acc[j]);
        }
        put_row<D, ND>(a, plan, st, slot, grp, h, i, d0, M, L, acc);
    }
}

// Many rows (more than 64): bound by the matrix and vector units.  Every wave has MT row tiles of its own and all
// of them the same keys, which they prepare together: of a stage of 16 keys a wave each turns its block into
// fragments, K and V, and puts them into LDS in the order in which the products read them (16 bytes a lane, without
// bank conflicts; the few that are counted are likely V's stores, 8 bytes at a stride of 16), so a key is converted once
// for up to 256 rows.  Two stages: while one is worked on the next one's loads are in flight, and it is written before
// the only barrier of a stage.
// LO: 32-bit queries, as hi + lo; the weights are hi + lo whatever the output's type is.
// 8 streams with trees of 33 to 64, 32 heads of 128 on 8 key heads, 8192 to 16384 int8 keys: 185 to 214 us from run to
// run, and 9.5 of the join.
// The vector unit is what is busy most: 218 thousand cycles of the softmax (a score: scale, maximum, exponential of 4 slots,
// sum, value scale, packing) and the conversions, 117 of the matrix unit, of 394 that a wave lives: little of the one falls
// under the other with two waves to a SIMD.  Tried when it took 172, with weights of 11 bits: products of the next span
// issued ahead of the weights of one, 182; the row tiles dealt to the waves in turn, so that none is idle where rows are
// fewer than 256, 184, as each then reads all fragments for half the rows.
template <int KV, int D, int NWV>
struct WideLds {
    uint4 k[2][NWV][D / 32][64];
    uint4 v[2][NWV / 2][D / 16][64];
    float ks[2][NWV][16], vs[2][NWV][16];
    uint32_t top[2][NWV];
    int odd[2][NWV];
    int bad[NWV];
    float room[KV == ELEM_I8 ? 1 : NWV][16][36];
};

template <int KV, int D, int NWV, int MT, bool LO>
__global__ __launch_bounds__(64 * NWV, 2) void attn_tree_wide_kernel(TreeArgs a, TreePlan plan) {
    constexpr bool SCALED = quantised(KV);
    constexpr int NW = Keys<KV, D>::NW, NS = D / 32, ND = D / 16, DW = dims_per_word<KV>();
    constexpr int STAGE = 16 * NWV;
    __shared__ WideLds<KV, D, NWV> lds;

    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b8 = blockIdx.x >> 3, rg = b8 % plan.row_groups, unit = (b8 / plan.row_groups) * 8 + (blockIdx.x & 7);
    if (unit >= plan.slots * a.c.heads) return;
    const int slot = unit / a.c.heads, h = unit - slot * a.c.heads;
    const Cut cut = cut_of_slot(a, plan, slot);
    const int s = cut.stream;
    if (s < 0) return;
    const Stream st = stream_of(a, s);
    const int grp = a.heads / a.c.heads, packed = st.n * grp;
    if (rg * NWV * MT * 16 >= packed) return;
    const int first = (rg * NWV + w) * MT * 16;
    bool bad = st.bad;
    const int beg = cut.beg, end = min(cut.end, st.total), last = end - 1;
    const int *table = a.c.table + (size_t)s * a.c.table_stride;

    uint4 kraw[NW];
    uint32_t vraw[4][NW];
    float ksr = 0.0f, vsr = 0.0f;
    auto fetch = [&](int p) {
        const size_t b = block_of(a, plan, table, h, p + 16 * w, last, bad);
        load_k<KV, D>(a, b, c, g, kraw);
        load_v<KV, D>(a, b, c, g, vraw);
        if constexpr (SCALED) {
            ksr = a.c.k_scale[b + c];
            vsr = a.c.v_scale[b + c];
        }
    };
    if (beg < end) fetch(beg);

    Query<KV, D, LO> q[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) q[mt].load(a, st, grp, h, first + mt * 16 + c, packed, g);

    auto put = [&](int buf, int p) {  // this wave's block of the stage at p
        const int pos = p + 16 * w;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            const Frag f = k_frag<KV, D>(kraw, k);
            lds.k[buf][w][k][lane] = make_uint4(f.w[0], f.w[1], f.w[2], f.w[3]);
        }
        if constexpr (KV != ELEM_I8) {
            bool odd = false;
            if (pos + 16 > st.ctx) {  // (as in the kernel for few rows)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int n = 0; n < NW; ++n) {
                        const uint32_t y = vraw[i][n];
                        vraw[i][n] = finite_part<KV>(y);
                        odd |= vraw[i][n] != y;
                    }
            }
            odd = __any(odd);
            if (lane == 0) lds.odd[buf][w] = odd;
        }
#pragma unroll
        for (int n = 0; n < NW; ++n) {
            uint32_t f[DW][2];
            v_halves<KV, NW>(vraw, n, f);
#pragma unroll
            for (int d = 0; d < DW; ++d) ((uint2 *)&lds.v[buf][w / 2][DW * n + d][lane])[w & 1] = make_uint2(f[d][0], f[d][1]);
        }
        if constexpr (SCALED) {
            uint32_t top = __float_as_uint(vsr) & 0x7fffffffu;
            top = max(top, (uint32_t)xshfl<1>((int)top));
            top = max(top, (uint32_t)xshfl<2>((int)top));
            top = max(top, (uint32_t)xshfl<4>((int)top));
            top = max(top, (uint32_t)xshfl<8>((int)top));
            if (lane == 0) lds.top[buf][w] = top;
            if (g == 0) {
                lds.ks[buf][w][c] = ksr;
                lds.vs[buf][w][c] = vsr;
            }
        }
    };

    Rows<MT, ND, SCALED, false> rows;
    rows.clear();
    if (beg < end) put(0, beg);
    lds_barrier();
    int buf = 0;
#pragma unroll 1
    for (int p = beg; p < end; p += STAGE) {
        const bool more = p + STAGE < end;
        if (more) fetch(p + STAGE);
        if (first < packed) {
#pragma unroll 1
            for (int u = 0; u < NWV / 2; ++u) {
                const int p0 = p + 32 * u;
                if (p0 >= end) break;
                const bool tail = p0 + 32 > st.ctx;
                float x[MT][2][4];
                float4 ks[2], vs[2];
                float vmax = 0.0f;
                if constexpr (SCALED) {
                    vmax = above((uint32_t)__builtin_amdgcn_readfirstlane((int)max(lds.top[buf][2 * u], lds.top[buf][2 * u + 1])));
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        ks[b] = *(const float4 *)&lds.ks[buf][2 * u + b][4 * g];
                        vs[b] = *(const float4 *)&lds.vs[buf][2 * u + b][4 * g];
                    }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    floatx4 acc[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) acc[mt] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < NS; ++k) {
                        const uint4 y = lds.k[buf][2 * u + b][k][lane];
                        const Frag f{{y.x, y.y, y.z, y.w}};
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            acc[mt] = mfma(f, q[mt].hi[k], acc[mt]);
                            if constexpr (LO) acc[mt] = mfma(f, q[mt].lo[k], acc[mt]);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[mt][b][i] = SCALED ? acc[mt][i] * ((const float *)&ks[b])[i] : acc[mt][i];
                }
                if (tail) hide(st, q, p0, g, -INFINITY, x);
                float most[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) most[mt] = rows.weigh(mt, q[mt].qs, x[mt]);
                if constexpr (SCALED) {
                    scale_weights(st, q, tail, p0, g, vs, x);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) rows.place(mt, most[mt], vmax, x[mt]);
                }
                Frag ph[MT], pl[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) split2(x[mt][b][i], x[mt][b][i + 1], ph[mt].w[2 * b + i / 2], pl[mt].w[2 * b + i / 2]);
                if constexpr (KV != ELEM_I8) {
                    if (tail && (lds.odd[buf][2 * u] | lds.odd[buf][2 * u + 1])) {
                        size_t blk[2];
#pragma unroll
                        for (int b = 0; b < 2; ++b) blk[b] = block_of(a, plan, table, h, p0 + 16 * b, last, bad);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) add_odd_values<KV, D>(a, st, blk, p0, mt, q[mt].mask, x[mt], lds.room[w], rows);
                    }
                }
#pragma unroll
                for (int j = 0; j < ND; ++j) {
                    const uint4 y = lds.v[buf][u][j][lane];
                    const Frag f{{y.x, y.y, y.z, y.w}};
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        rows.o[mt][j] = mfma(f, ph[mt], rows.o[mt][j]);
                        rows.o[mt][j] = mfma(f, pl[mt], rows.o[mt][j]);
                    }
                }
            }
        }
        buf ^= 1;
        if (more) put(buf, p + STAGE);
        lds_barrier();
    }
    put_cut(a, plan, cut, slot, h, rg);
    bad = __any(bad);
    if (lane == 0) lds.bad[w] = bad;
    lds_barrier();
#pragma unroll
    for (int v = 0; v < NWV; ++v) bad |= lds.bad[v] != 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int i = first + mt * 16 + c;
        rows.settle(mt);
        float L = rows.l[mt];
        L += xshfl<16>(L);
        L += xshfl<32>(L);
        if (bad) L = __uint_as_float(0x7fc00000u);
        float y[4 * ND];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < ND; ++j) y[ND * r + j] = rows.o[mt][j][r];
        if (i < packed) put_row<D, 4 * ND>(a, plan, st, slot, grp, h, i, (D / 4) * g, rows.ref[mt], L, y);
    }
}

// The pieces of each (row, head) joined in their order: lane c holds piece c's maximum and sum, and D / 4
// lanes add up a vector with SIDE = 256 / D pieces side by side, several loads of a wave at once.  One wave does a
// row where pieces are few (about 4 of 12400 rows of 128: 9.3 us; a workgroup a row: 16.8), else they are shared out to the
// 4 waves of a workgroup and joined through LDS (64 of 32 rows: 4.8 us; one wave a row: 14).
template <int D, bool ONE_WAVE>
__global__ __launch_bounds__(kThreads) void attn_tree_join_kernel(TreeArgs a, TreePlan plan) {
    constexpr int G = D / 4, SIDE = 64 / G, ROUNDS = kMaxSplits / (kWaves * SIDE);
    __shared__ float4 part[kWaves][G];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int of_stream = a.max_rows * a.heads, per = ONE_WAVE ? (of_stream + kWaves - 1) / kWaves : of_stream;
    const int s = blockIdx.x / per, i = ONE_WAVE ? (blockIdx.x - s * per) * kWaves + w : blockIdx.x - s * per;
    const Stream st = stream_of(a, s);
    if (i >= st.n * a.heads) return;
    const int4 cut = ((const int4 *)a.ws)[s];
    const int splits = __builtin_amdgcn_readfirstlane(cut.y);
    const size_t slot_rows = (size_t)of_stream, at = cut.x * slot_rows + i;
    float2 mine = make_float2(-INFINITY, 0.0f);
    if (lane < splits) mine = row_sums(a)[lane * slot_rows + at];
    const int d = (lane % G) * 4, side = lane / G;
    const int first = ONE_WAVE ? side : w * SIDE + side, step = ONE_WAVE ? SIDE : kWaves * SIDE;
    const float *po = partials(a, plan) + at * D + d;
    const float M = wave_max(mine.x), M0 = M == -INFINITY ? 0.0f : M;
    const float f = exp2_(mine.x - M0), L = wave_sum(mine.y * f);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < splits; k0 += ROUNDS * step) {  // (one wave: more rounds where a stream has most of the slots)
        float4 x[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)  // (a piece without keys has written none: what is read there is not used)
            if (k0 + r * step < splits) x[r] = *(const float4 *)(po + (size_t)min(k0 + first + r * step, splits - 1) * slot_rows * D);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (k0 + r * step < splits) {
                const int k = k0 + first + r * step;
                const float fk = __shfl(f, k & 63), lk = __shfl(mine.y, k & 63);
                const bool use = k < splits && lk != 0.0f;
                o.x = use ? fmaf(x[r].x, fk, o.x) : o.x;
                o.y = use ? fmaf(x[r].y, fk, o.y) : o.y;
                o.z = use ? fmaf(x[r].z, fk, o.z) : o.z;
                o.w = use ? fmaf(x[r].w, fk, o.w) : o.w;
            }
    }
    if constexpr (G == 16) o.x += xshfl<16>(o.x), o.y += xshfl<16>(o.y), o.z += xshfl<16>(o.z), o.w += xshfl<16>(o.w);
    o.x += xshfl<32>(o.x), o.y += xshfl<32>(o.y), o.z += xshfl<32>(o.z), o.w += xshfl<32>(o.w);
    float y[4] = {o.x, o.y, o.z, o.w};
    if constexpr (!ONE_WAVE) {
        if (side == 0) part[w][lane % G] = o;
        __syncthreads();
        if (w != 0) return;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = (((const float *)&part[0][lane % G])[j] + ((const float *)&part[1][lane % G])[j]) +
                   (((const float *)&part[2][lane % G])[j] + ((const float *)&part[3][lane % G])[j]);
    }
    if (side != 0) return;
    put_row<D, 4>(a, plan, st, -1, a.heads, 0, i, d, M, L, y);
}

// Rows of 16 of a workgroup: 1 or 2 in the kernel for few rows, 8 or 16 in the wide one.  With 3 and 4 tiles the keys are
// read twice by the one and still sooner done (16 trees of 64 over 1015 fp16 keys of 12 x 64: 21.9 us, a wide workgroup of 4
// waves 27.4; 4 over 4000 int8 keys 22.6 and 25.1); with 5 to 8 they are not (8 trees of 32 x 4 heads a key head over 16384
// int8 keys of 128: 172 and 142; 80 rows over 8000 fp16 keys: 162 and 67 of 128 dims, 56 and 46 of 64).  An fp32 cache, which the wide one's fp16 fragments
// cannot hold, takes the first always.
int group_tiles(const KvCacheArgs &c, int tiles) {
    if (tiles <= 4 || c.dtype == ELEM_F32) return std::min(tiles, 2);
    return tiles <= 8 ? 8 : 16;
}

TreePlan plan_of(const KvCacheArgs &c, int heads, int max_rows, int max_keys) {
    TreePlan p;
    p.tiles = (max_rows * (heads / c.heads) + 15) / 16;
    p.group = group_tiles(c, p.tiles);
    p.row_groups = (p.tiles + p.group - 1) / p.group;
    const long long base = (long long)c.streams * c.heads * p.row_groups;
    // as many workgroups as are resident at once (3 or 2 of the kernel for few rows on a CU, one wide one), and keys
    // enough in a piece for its start and end to pay
    const int least = 256, want = 256 * (p.group > 2 ? 1 : (c.dim == 64 && p.group == 1 ? 3 : 2));
    int splits = (int)std::min<long long>(want / base, kMaxSplits);
    splits = std::max(1, std::min(splits, (max_keys + least - 1) / least));
    // Short keys that would be cut are given to 8 waves of a workgroup instead, without the join: 16 trees of 27 over 1000
    // fp16 keys of 12 x 64 19.9 -> 15.2 us, 64 rows over 300 int8 keys of 4 x 128 14.4 -> 9.1.  That pays while the cuts
    // that the workgroups leave room for are few and the spans of a wave are few: where one stream is much longer than
    // the others, cuts serve it better (1500 keys among 100s: 13.5 us cut, 16.4 so).  Two tiles of 128 dims cost most a
    // span (16 x 27 over 500 keys of 8 x 128: 22.0 cut in 4, 24.4 so).
    const int room = (int)std::min<long long>(want / base, kMaxSplits);
    const int eight_to = c.dim == 128 && p.group == 2 ? (room <= 2 ? 512 : 0) : (room <= 2 ? 1536 : (room <= 4 ? 1024 : 512));
    p.waves = kWaves;
    if (p.group <= 2 && c.dtype != ELEM_F32 && splits > 1 && max_keys <= eight_to) {
        p.waves = 2 * kWaves;
        splits = 1;
    }
    // The matrix instructions cut what they add towards zero, so a sum of one sign falls short by about 2^-25 for each (1.6e-4
    // and, of equal weights, 4.8e-4 over 131072 keys of a wide workgroup).  No wave gets more than 1024 in a row: two for 32
    // keys, or eight in fp32; the wide workgroup's waves see every key, the others a fourth.
    const int most = p.group > 2 || c.dtype == ELEM_F32 ? 16384 : 65536;
    // That is as far as it goes with partial results of 2^20 rows (0.5 GB of 128 dims), and so with a grid that can be launched.
    const int room_for = (int)std::max<long long>(1, (1 << 20) / ((long long)c.streams * max_rows * heads));
    splits = std::max(splits, std::min({(max_keys + most - 1) / most, kMaxSplits, room_for}));
    p.chunk = ((max_keys + splits - 1) / splits + 127) / 128 * 128;
    p.slots = splits * c.streams;
    // blk / (page_size / 16) for blk < 2^24 and a divisor up to 2^11: 2^40 / d rounded up is off by
    // less than d, and blk * d < 2^40
    const uint64_t d = (uint64_t)c.page_size / 16;
    p.page_magic = ((1ull << 40) + d - 1) / d;
    return p;
}

template <int KV, int D, int MT, bool LO>
void launch_few(dim3 grid, const TreeArgs &a, const TreePlan &p, hipStream_t s) {
    if constexpr (KV != ELEM_F32) {
        if (p.waves > kWaves) {
            hipLaunchKernelGGL((attn_tree_kernel<KV, D, MT, LO, 2 * kWaves>), grid, dim3(2 * kThreads), 0, s, a, p);
            return;
        }
    }
    hipLaunchKernelGGL((attn_tree_kernel<KV, D, MT, LO, kWaves>), grid, dim3(kThreads), 0, s, a, p);
}

template <int KV, int D, bool LO>
void launch_group(const TreeArgs &a, const TreePlan &p, hipStream_t s) {
    const long long units = (long long)p.slots * a.c.heads;
    const dim3 grid((unsigned)((units + 7) / 8 * 8 * p.row_groups));
    if (p.group == 1) {
        launch_few<KV, D, 1, LO>(grid, a, p, s);
    } else if (p.group == 2) {
        launch_few<KV, D, 2, LO>(grid, a, p, s);
    } else if constexpr (KV != ELEM_F32) {
        if (p.group == 8)
            hipLaunchKernelGGL((attn_tree_wide_kernel<KV, D, 8, 1, LO>), grid, dim3(512), 0, s, a, p);
        else
            hipLaunchKernelGGL((attn_tree_wide_kernel<KV, D, 8, 2, LO>), grid, dim3(512), 0, s, a, p);
    }
}

template <int KV, int D>
hipError_t launch_kv(const TreeArgs &a, hipStream_t s) {
    const TreePlan p = plan_of(a.c, a.heads, a.max_rows, a.max_keys);
    (void)hipGetLastError();
    if constexpr (KV == ELEM_F32)
        launch_group<KV, D, false>(a, p, s);
    else if (a.q_dtype == ELEM_F32)
        launch_group<KV, D, true>(a, p, s);
    else
        launch_group<KV, D, false>(a, p, s);
    const unsigned rows = (unsigned)(a.max_rows * a.heads), streams = (unsigned)a.c.streams;
    if (p.slots > 1024 / D * a.c.streams)
        hipLaunchKernelGGL((attn_tree_join_kernel<D, false>), dim3(streams * rows), dim3(kThreads), 0, s, a, p);
    else if (p.slots > a.c.streams)
        hipLaunchKernelGGL((attn_tree_join_kernel<D, true>), dim3(streams * ((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0, s, a, p);
    return hipGetLastError();
}

template <int D>
hipError_t launch_d(const TreeArgs &a, hipStream_t s) {
    switch (a.c.dtype) {
        case ELEM_F32: return launch_kv<ELEM_F32, D>(a, s);
        case ELEM_F16: return launch_kv<ELEM_F16, D>(a, s);
        case ELEM_I8: return launch_kv<ELEM_I8, D>(a, s);
        default: return launch_kv<ELEM_E4M3, D>(a, s);
    }
}

}  // namespace

size_t tree_workspace(const KvCacheArgs &c, int heads, int rows, int max_rows, int max_keys) {
    max_rows = std::min(max_rows, rows);
    const TreePlan p = plan_of(c, heads, max_rows, max_keys);
    return p.slots == c.streams ? 0 : c.streams * sizeof(int4) + ((size_t)p.slots * max_rows * heads * (2 + c.dim) + 2) * sizeof(float);
}

hipError_t launch_attn_tree(const TreeArgs &args, hipStream_t s) {
    TreeArgs a = args;
    a.max_rows = std::min(a.max_rows, a.rows);
    a.q_vec = (uintptr_t)a.q % 16 == 0 && a.q_row * elem_size(a.q_dtype) % 16 == 0;
    a.out_vec = (uintptr_t)a.out % 16 == 0 && a.out_row * elem_size(a.out_dtype) % 16 == 0;
    return a.c.dim == 64 ? launch_d<64>(a, s) : launch_d<128>(a, s);
}

}  // namespace mh
