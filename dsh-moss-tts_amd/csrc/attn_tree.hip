// attn_tree.hip -- attention of a few rows per stream (one token, or a tree of drafted ones) over a
// paged K/V cache in fp32, fp16, int8 or e4m3, with grouped heads (gfx950).
//
// Row i of a stream attends the stream's whole context, keys 0 .. ctx - 1, and those of the drafted
// positions ctx + j (j < n, the stream's row count) whose bit j its mask has:
//   s_p = scale (q . k_p),  o = sum_p e^(s_p - m) v_p / sum_p e^(s_p - m),  lse = m + log(sum).
// A row that sees nothing is 0 with lse = -inf.
//
// The n rows x (heads / kv_heads) queries that share a key head are packed into tiles of 16, the
// columns of the matrix instructions, so a key is loaded once for all of them.  A workgroup's 4 waves
// take every 4th span of keys with a running maximum and sum each, and are joined through LDS; with
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
// power of two to below 2) and the softmax weights go in as fp16 hi + lo, 22 bits, so results are as
// good as 32-bit ones.  int8 / e4m3 scales multiply the scores and the weights; weights are kept in
// fp16's range by the largest value scale seen, a power of two E that is wave-uniform and rises like the
// running maximum.  An fp32 cache runs on the fp32 matrix instructions.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kMaxSplits = 64;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr int kWeightExp = 13;  // weights are scaled to at most 2^14

struct TreePlan {
    int tiles, row_groups, splits, chunk;  // row tiles of 16, groups of MT of them, key splits of `chunk` keys
    uint64_t page_magic;                   // block of 16 keys / blocks of a page, as a product
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

// x as hi + lo halves, both towards zero: 22 bits
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]));
}

// 16 keys x D of one head as a lane's share of 32 keys: K as the A operand of S^T, V as that of O^T.
template <int KV, int D>
struct Keys {
    static constexpr int NW = D * elem_size(KV) / 64;
    uint4 k[2][NW];
    uint32_t v[8][NW];
    float4 ks[2], vs[2];
};

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

// V fragments of dims 4n .. 4n + 3 (8 bit) or 2n, 2n + 1 (fp16) of the lane's D / 16.
template <int KV>
constexpr int dims_per_word() {
    return KV == ELEM_F16 ? 2 : 4;
}
template <int KV, int NW>
__device__ __forceinline__ void v_frags(const uint32_t (&v)[8][NW], int n, Frag (&f)[dims_per_word<KV>()]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t a = v[2 * q][n], b = v[2 * q + 1][n];
        if constexpr (KV == ELEM_F16) {
            f[0].w[q] = perm(b, a, 0x05040100u);
            f[1].w[q] = perm(b, a, 0x07060302u);
        } else {
            const uint32_t x = KV == ELEM_I8 ? 0x80808080u : 0u;
            const uint32_t t01 = perm(b ^ x, a ^ x, 0x05010400u), t23 = perm(b ^ x, a ^ x, 0x07030602u);
            if constexpr (KV == ELEM_I8) {
                f[0].w[q] = bias_off(perm(0x64646464u, t01, 0x04010400u));
                f[1].w[q] = bias_off(perm(0x64646464u, t01, 0x04030402u));
                f[2].w[q] = bias_off(perm(0x64646464u, t23, 0x04010400u));
                f[3].w[q] = bias_off(perm(0x64646464u, t23, 0x04030402u));
            } else {
                f[0].w[q] = e4m3_pair(t01, false), f[1].w[q] = e4m3_pair(t01, true);
                f[2].w[q] = e4m3_pair(t23, false), f[3].w[q] = e4m3_pair(t23, true);
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

__device__ __forceinline__ float load_q(const TreeArgs &a, size_t i) {
    return a.q_dtype == ELEM_F16 ? __half2float(((const __half *)a.q)[i]) : ((const float *)a.q)[i];
}

// A stream's rows and keys; n = 0 where there is nothing to do.
struct Stream {
    int row0, n, ctx, total;
    bool bad;  // more keys than the launch or the table has room for
};
__device__ __forceinline__ Stream stream_of(const TreeArgs &a, int s) {
    Stream t;
    t.row0 = __builtin_amdgcn_readfirstlane(a.row_start[s]);
    const int end = __builtin_amdgcn_readfirstlane(a.row_start[s + 1]);
    t.n = t.row0 < 0 || end > a.rows || end <= t.row0 ? 0 : min(end - t.row0, a.max_rows);
    t.ctx = __builtin_amdgcn_readfirstlane(a.ctx_len[s]);
    const long long room = min((long long)a.c.table_stride * a.c.page_size, (long long)a.max_keys);
    t.bad = t.ctx < 0 || (long long)t.ctx + t.n > room;
    t.total = t.bad ? 0 : t.ctx + t.n;
    return t;
}

// HB: spans of HB * 32 keys; MT row tiles; LO: 32-bit queries, as hi + lo.
template <int KV, int D, int MT, int HB, bool LO>
__global__ __launch_bounds__(kThreads) void attn_tree_kernel(TreeArgs a, TreePlan plan) {
    constexpr bool F32 = KV == ELEM_F32, SCALED = quantised(KV);
    constexpr int NW = Keys<KV, D>::NW, NS = D / 32, ND = D / 16;
    constexpr int KT = 32 * HB;
    constexpr int ESZ = elem_size(KV);
    __shared__ float so[kWaves][16][D + 4];
    __shared__ float sm[kWaves][16], sl[kWaves][16];

    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // workgroups that read the same keys follow each other on one XCD, whose L2 then serves them
    const int units = a.c.streams * a.c.heads * plan.splits;
    const int b8 = blockIdx.x >> 3, rg = b8 % plan.row_groups, unit = (b8 / plan.row_groups) * 8 + (blockIdx.x & 7);
    if (unit >= units) return;
    const int z = unit % plan.splits, sh = unit / plan.splits, h = sh % a.c.heads, s = sh / a.c.heads;
    const Stream st = stream_of(a, s);
    const int grp = a.heads / a.c.heads, packed = st.n * grp, first = rg * MT * 16;
    if (first >= packed) return;
    const int live = min(MT, (packed - first + 15) / 16);

    // ---- queries
    Frag qh[MT][F32 ? 1 : NS], ql[MT][F32 || !LO ? 1 : NS];
    float qf[MT][F32 ? D / 4 : 1];
    float qs[MT];
    uint64_t mask[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int i = first + mt * 16 + c;
        const bool ok = i < packed;
        const int node = ok ? i / grp : 0, row = st.row0 + node, head = h * grp + (ok ? i - node * grp : 0);
        const size_t base = (size_t)((int64_t)row * a.q_row + head * D);
        mask[mt] = !ok ? 0 : (a.row_mask != nullptr ? a.row_mask[row] : (2ull << node) - 1);
        if (st.n < 64) mask[mt] &= (1ull << st.n) - 1;
        qs[mt] = a.scale * kLog2e;
        if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < D / 16; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) qf[mt][4 * u + e] = ok ? load_q(a, base + 16 * u + 4 * g + e) : 0.0f;
        } else {
            float x[NS][8];
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < NS; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[k][e] = ok ? load_q(a, base + frag_dim<KV>(k, g) + e) : 0.0f;
                    top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
                }
            if constexpr (LO) {
                top = max(top, (uint32_t)xshfl<16>((int)top));
                top = max(top, (uint32_t)xshfl<32>((int)top));
                const int e2 = (int)(top >> 23) - 127;  // a power of two: exact (an Inf or NaN stays one)
                qs[mt] = ldexpf(qs[mt], e2);
#pragma unroll
                for (int k = 0; k < NS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        split2(ldexpf(x[k][e], -e2), ldexpf(x[k][e + 1], -e2), qh[mt][k].w[e / 2], ql[mt][k].w[e / 2]);
            } else {
#pragma unroll
                for (int k = 0; k < NS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        qh[mt][k].w[e / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[k][e], x[k][e + 1]));
            }
        }
    }
    uint64_t seen = 0;  // drafted positions that any of these rows sees
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) seen |= mask[mt];
    {
        uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
        lo |= xshfl<1>((int)lo), hi |= xshfl<1>((int)hi);
        lo |= xshfl<2>((int)lo), hi |= xshfl<2>((int)hi);
        lo |= xshfl<4>((int)lo), hi |= xshfl<4>((int)hi);
        lo |= xshfl<8>((int)lo), hi |= xshfl<8>((int)hi);
        seen = ((uint64_t)hi << 32) | lo;
    }

    // ---- keys
    float m[MT], l[MT];
    floatx4 o[MT][ND];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = -INFINITY;
        l[mt] = 0.0f;
#pragma unroll
        for (int j = 0; j < ND; ++j) o[mt][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    int top_exp = 0;       // biased exponent of the largest value scale so far
    bool bad = st.bad;
    const int beg = z * plan.chunk, end = min(beg + plan.chunk, st.total), last = st.total - 1;
    const int *table = a.c.table + (size_t)s * a.c.table_stride;
    const uint32_t page16 = a.c.page_size >> 4;

#pragma unroll 1
    for (int p0 = beg + KT * w; p0 < end; p0 += KT * kWaves) {
        const bool tail = p0 + KT > st.ctx;
        Keys<KV, D> keys[HB];
        size_t vec[HB][2];  // first vector of each block of 16 keys
        int lim[HB][2];     // its last key that exists
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int kb = min(p0 + 32 * hb + 16 * b, last & ~15);
                const uint32_t blk = (uint32_t)kb >> 4, pg = (uint32_t)((blk * plan.page_magic) >> 40);
                int page = __builtin_amdgcn_readfirstlane(table[pg]);
                if (page < 0 || page >= a.c.n_pages) {
                    page = 0;
                    bad = true;
                }
                vec[hb][b] = ((size_t)page * a.c.heads + h) * a.c.page_size + (blk - pg * page16) * 16;
                lim[hb][b] = min(15, last - kb);
            }
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const char *kp = (const char *)a.c.k + vec[hb][b] * (D * ESZ);
                const int off = min(c, lim[hb][b]) * (D * ESZ) + 16 * g;
#pragma unroll
                for (int u = 0; u < NW; ++u) keys[hb].k[b][u] = *(const uint4 *)(kp + off + 64 * u);
                if constexpr (SCALED) {
                    keys[hb].ks[b] = *(const float4 *)(a.c.k_scale + vec[hb][b] + 4 * g);
                    keys[hb].vs[b] = *(const float4 *)(a.c.v_scale + vec[hb][b] + 4 * g);
                }
            }
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const char *vp = (const char *)a.c.v + vec[hb][b] * (D * ESZ);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int off = min(4 * g + i, lim[hb][b]) * (D * ESZ) + c * (NW * 4);
                    __builtin_memcpy(keys[hb].v[4 * b + i], __builtin_assume_aligned(vp + off, NW < 4 ? NW * 4 : 16), NW * 4);
                }
            }

        // scores, in units of log 2
        float sc[MT][HB][2][4];
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                floatx4 acc[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) acc[mt] = floatx4{0.f, 0.f, 0.f, 0.f};
                if constexpr (F32) {
#pragma unroll
                    for (int u = 0; u < NW; ++u) {
                        const float *kf = (const float *)&keys[hb].k[b][u];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt)
                                if (mt < live) acc[mt] = mfma(kf[e], qf[mt][4 * u + e], acc[mt]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < NS; ++k) {
                        const Frag f = k_frag<KV, D>(keys[hb].k[b], k);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            if (mt < live) {
                                acc[mt] = mfma(f, qh[mt][k], acc[mt]);
                                if constexpr (LO) acc[mt] = mfma(f, ql[mt][k], acc[mt]);
                            }
                    }
                }
                const float *ks = (const float *)&keys[hb].ks[b];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[mt][hb][b][i] = acc[mt][i] * (SCALED ? ks[i] * qs[mt] : qs[mt]);
            }
        auto visible = [&](uint64_t rows_mask, int key) {  // key p0 + key
            const int j = p0 + key - st.ctx;
            return j < 0 || (j < st.n && ((rows_mask >> (j & 63)) & 1));
        };
        if (tail) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!visible(mask[mt], 32 * hb + 16 * b + 4 * g + i)) sc[mt][hb][b][i] = -INFINITY;
        }

        // value scales against the largest so far
        float vs[HB][2][4];
        float shrink = 1.0f;
        if constexpr (SCALED) {
            uint32_t top = 0;
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = __float_as_uint(((const float *)&keys[hb].vs[b])[i]) & 0x7fffffffu;
                        const bool use = x < 0x7f800000u && (!tail || visible(seen, 32 * hb + 16 * b + 4 * g + i));
                        top = max(top, use ? x : 0u);
                    }
            top = max(top, (uint32_t)xshfl<16>((int)top));
            top = max(top, (uint32_t)xshfl<32>((int)top));
            const int e = __builtin_amdgcn_readfirstlane(top >> 23);
            if (e > top_exp) {
                shrink = ldexpf(1.0f, top_exp - e);
                top_exp = e;
            }
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        vs[hb][b][i] = ldexpf(((const float *)&keys[hb].vs[b])[i], kWeightExp + 127 - top_exp);
        }

        // weights
        Frag ph[MT][HB], pl[MT][HB];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float mx = -INFINITY;
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[mt][hb][b][i]);
            mx = fmaxf(mx, xshfl<16>(mx));
            mx = fmaxf(mx, xshfl<32>(mx));
            const float m_new = fmaxf(m[mt], mx), m0 = m_new == -INFINITY ? 0.0f : m_new;
            const float fade = exp2_(m[mt] - m0);
            if (__any(fade != 1.0f) || (SCALED && shrink != 1.0f)) {
                l[mt] *= fade;
                const float f = SCALED ? fade * shrink : fade;
#pragma unroll
                for (int j = 0; j < ND; ++j) o[mt][j] *= f;
            }
            m[mt] = m_new;
#pragma unroll
            for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &x = sc[mt][hb][b][i];
                        const float e = exp2_(x - m0);
                        l[mt] += e;
                        x = SCALED ? e * vs[hb][b][i] : (F32 ? e : e * (float)(1 << kWeightExp));
                        if (SCALED && tail && !visible(mask[mt], 32 * hb + 16 * b + 4 * g + i)) x = 0.0f;  // whatever its scale holds
                    }
            if constexpr (!F32) {
#pragma unroll
                for (int hb = 0; hb < HB; ++hb)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 4; i += 2)
                            split2(sc[mt][hb][b][i], sc[mt][hb][b][i + 1], ph[mt][hb].w[2 * b + i / 2], pl[mt][hb].w[2 * b + i / 2]);
            }
        }

        // values
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) {
            if constexpr (KV != ELEM_I8) {
                // drafted values that some row does not see may hold anything, and 0 times an Inf or NaN
                // is not 0: such elements go into the products as 0, and are added, key by key, to the rows
                // that see them
                if (tail) {
                    bool odd = false;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int n = 0; n < NW; ++n) {
                            const uint32_t x = keys[hb].v[e][n];
                            keys[hb].v[e][n] = finite_part<KV>(x);
                            odd |= keys[hb].v[e][n] != x;
                        }
                    if (__any(odd)) {
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                            for (int b = 0; b < 2; ++b)
#pragma unroll
                                for (int i = 0; i < 4; ++i) so[w][c][16 * b + 4 * g + i] = sc[mt][hb][b][i];
                            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
                            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                            for (int kk = 0; kk < 32; ++kk) {
                                const int b = kk >> 4;
                                const size_t at = ((b ? vec[hb][1] : vec[hb][0]) + min(kk & 15, b ? lim[hb][1] : lim[hb][0])) * D +
                                                  (D / 4) * g;
                                const float x = so[w][c][kk];
                                const bool see = visible(mask[mt], 32 * hb + kk);
#pragma unroll
                                for (int r = 0; r < 4; ++r)
#pragma unroll
                                    for (int j = 0; j < ND; ++j) {
                                        const float v = v_value<KV>(a.c.v, at + ND * r + j);
                                        const bool add = see && !(fabsf(v) < INFINITY);
                                        o[mt][j][r] += add ? x * v : 0.0f;
                                    }
                            }
                            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
                            __builtin_amdgcn_wave_barrier();
                        }
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int j = 0; j < ND; ++j)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            if (mt < live) o[mt][j] = mfma(__uint_as_float(keys[hb].v[e][j]), sc[mt][hb][e / 4][e % 4], o[mt][j]);
            } else {
                constexpr int DW = dims_per_word<KV>();
#pragma unroll
                for (int n = 0; n < NW; ++n) {
                    Frag f[DW];
                    v_frags<KV, NW>(keys[hb].v, n, f);
#pragma unroll
                    for (int d = 0; d < DW; ++d)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
                            if (mt < live) {
                                o[mt][DW * n + d] = mfma(f[d], ph[mt][hb], o[mt][DW * n + d]);
                                o[mt][DW * n + d] = mfma(f[d], pl[mt][hb], o[mt][DW * n + d]);
                            }
                }
            }
        }
    }

    // ---- the waves joined, one row tile at a time
    bad = __any(bad);
    const size_t all_rows = (size_t)a.rows * a.heads;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (mt >= live) break;
        const int unscale = F32 ? 0 : (SCALED ? top_exp - 127 - kWeightExp : -kWeightExp);
        float sum = l[mt];
        sum += xshfl<16>(sum);
        sum += xshfl<32>(sum);
        if (mt > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < ND; j += 4) {
                float4 x;
                x.x = ldexpf(o[mt][j][r], unscale);
                x.y = ldexpf(o[mt][j + 1][r], unscale);
                x.z = ldexpf(o[mt][j + 2][r], unscale);
                x.w = ldexpf(o[mt][j + 3][r], unscale);
                *(float4 *)&so[w][c][ND * (4 * g + r) + j] = x;
            }
        if (g == 0) {
            sm[w][c] = m[mt];
            sl[w][c] = bad ? __uint_as_float(0x7fc00000u) : sum;
        }
        __syncthreads();
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * ND;
        const int i = first + mt * 16 + row;
        if (i >= packed) continue;
        float M = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row]));
        const float M0 = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, acc[ND];
#pragma unroll
        for (int j = 0; j < ND; ++j) acc[j] = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const float f = exp2_(sm[v][row] - M0);
            L = fmaf(sl[v][row], f, L);
#pragma unroll
            for (int j = 0; j < ND; ++j) acc[j] = fmaf(so[v][row][d0 + j], f, acc[j]);
        }
        const int node = i / grp, head = h * grp + i - node * grp;
        const size_t at = (size_t)(st.row0 + node) * a.heads + head;
        if (plan.splits > 1) {
            float *ws = (float *)a.ws + ((size_t)z * all_rows + at) * 2;
            if (d0 == 0) *(float2 *)ws = make_float2(M, L);
            float *po = (float *)a.ws + (size_t)plan.splits * all_rows * 2 + ((size_t)z * all_rows + at) * D + d0;
            if (L != 0.0f)
#pragma unroll
                for (int j = 0; j < ND; j += 4) *(float4 *)(po + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            continue;
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        const size_t oi = (size_t)((int64_t)(st.row0 + node) * a.out_row + head * D + d0);
#pragma unroll
        for (int j = 0; j < ND; ++j) {
            if (a.out_dtype == ELEM_F16)
                ((__half *)a.out)[oi + j] = __float2half_rn(acc[j] * inv);
            else
                ((float *)a.out)[oi + j] = acc[j] * inv;
        }
        if (a.lse != nullptr && d0 == 0) a.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
}

// The key splits of each (row, head) joined in their order: one wave each, lane c holding split c's
// maximum and sum, then D / 4 lanes a vector with 256 / D splits side by side.
template <int D>
__global__ __launch_bounds__(kThreads) void attn_tree_join_kernel(TreeArgs a, int splits) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int per = (a.max_rows * a.heads + kWaves - 1) / kWaves;
    const int s = blockIdx.x / per, i = (blockIdx.x - s * per) * kWaves + w;
    const Stream st = stream_of(a, s);
    if (i >= st.n * a.heads) return;
    const size_t all_rows = (size_t)a.rows * a.heads, at = (size_t)st.row0 * a.heads + i;
    const float2 *ml = (const float2 *)a.ws;
    float2 mine = make_float2(-INFINITY, 0.0f);
    if (lane < splits) mine = ml[(size_t)lane * all_rows + at];
    const float M = wave_max(mine.x), M0 = M == -INFINITY ? 0.0f : M;
    const float f = exp2_(mine.x - M0);
    const float L = wave_sum(mine.y * f);
    constexpr int G = D / 4, SIDE = 64 / G;
    const int d = (lane % G) * 4, side = lane / G;
    const float *po = (const float *)a.ws + (size_t)splits * all_rows * 2;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < splits; c0 += SIDE) {
        const int k = c0 + side;
        const float fk = __shfl(f, k & 63), lk = __shfl(mine.y, k & 63);
        if (k < splits && lk != 0.0f) {
            const float4 x = *(const float4 *)(po + ((size_t)k * all_rows + at) * D + d);
            o.x = fmaf(x.x, fk, o.x);
            o.y = fmaf(x.y, fk, o.y);
            o.z = fmaf(x.z, fk, o.z);
            o.w = fmaf(x.w, fk, o.w);
        }
    }
#define MH_FOLD(M_) o.x += xshfl<M_>(o.x), o.y += xshfl<M_>(o.y), o.z += xshfl<M_>(o.z), o.w += xshfl<M_>(o.w)
    if constexpr (G == 16) MH_FOLD(16);
    MH_FOLD(32);
#undef MH_FOLD
    if (side != 0) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int node = i / a.heads, head = i - node * a.heads;
    const size_t oi = (size_t)((int64_t)(st.row0 + node) * a.out_row + head * D + d);
    const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (a.out_dtype == ELEM_F16)
            ((__half *)a.out)[oi + j] = __float2half_rn(x[j]);
        else
            ((float *)a.out)[oi + j] = x[j];
    }
    if (a.lse != nullptr && lane == 0) a.lse[at] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Row tiles of a workgroup.  An fp32 cache's queries and keys take four times the registers.
int row_tiles_of(const KvCacheArgs &c, int tiles) { return std::min(tiles >= 3 ? 4 : tiles, c.dtype == ELEM_F32 ? 2 : 4); }

TreePlan plan_of(const KvCacheArgs &c, int heads, int max_rows, int max_keys) {
    TreePlan p;
    p.tiles = (max_rows * (heads / c.heads) + 15) / 16;
    const int mt = row_tiles_of(c, p.tiles);
    p.row_groups = (p.tiles + mt - 1) / mt;
    const long long base = (long long)c.streams * c.heads * p.row_groups;
    const int spans = (max_keys + 255) / 256;  // every wave of a split should have a span
    int splits = base >= 512 ? 1 : (int)std::min<long long>((1024 + base - 1) / base, kMaxSplits);
    splits = std::max(1, std::min(splits, spans));
    p.chunk = (spans + splits - 1) / splits * 256;
    p.splits = (max_keys + p.chunk - 1) / p.chunk;
    // blk / (page_size / 16) for blk < 2^24 and a divisor up to 2^11: 2^40 / d rounded up is off by
    // less than d, and blk * d < 2^40
    const uint64_t d = (uint64_t)c.page_size / 16;
    p.page_magic = ((1ull << 40) + d - 1) / d;
    return p;
}

template <int KV, int D, int MT, int HB>
void launch_tiles(const TreeArgs &a, const TreePlan &p, hipStream_t s) {
    const long long units = (long long)a.c.streams * a.c.heads * p.splits;
    const dim3 grid((unsigned)((units + 7) / 8 * 8 * p.row_groups));
    constexpr bool LO = KV != ELEM_F32;  // there is a kernel of its own for 32-bit queries
    if (LO && a.q_dtype == ELEM_F32)
        hipLaunchKernelGGL((attn_tree_kernel<KV, D, MT, HB, LO>), grid, dim3(kThreads), 0, s, a, p);
    else
        hipLaunchKernelGGL((attn_tree_kernel<KV, D, MT, HB, false>), grid, dim3(kThreads), 0, s, a, p);
}

template <int KV, int D>
hipError_t launch_kv(const TreeArgs &a, hipStream_t s) {
    const TreePlan p = plan_of(a.c, a.heads, a.max_rows, a.max_keys);
    (void)hipGetLastError();
    constexpr int HB = KV == ELEM_F32 ? 1 : 2;
    switch (row_tiles_of(a.c, p.tiles)) {
        case 1: launch_tiles<KV, D, 1, HB>(a, p, s); break;
        case 2: launch_tiles<KV, D, 2, HB>(a, p, s); break;
        default:
            if constexpr (KV != ELEM_F32) launch_tiles<KV, D, 4, 1>(a, p, s);
    }
    if (p.splits > 1) {
        const int per = (a.max_rows * a.heads + kWaves - 1) / kWaves;
        hipLaunchKernelGGL((attn_tree_join_kernel<D>), dim3((unsigned)a.c.streams * per), dim3(kThreads), 0, s, a, p.splits);
    }
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
    const TreePlan p = plan_of(c, heads, max_rows, max_keys);
    return p.splits == 1 ? 0 : (size_t)p.splits * rows * heads * (2 + c.dim) * sizeof(float);
}

hipError_t launch_attn_tree(const TreeArgs &a, hipStream_t s) {
    return a.c.dim == 64 ? launch_d<64>(a, s) : launch_d<128>(a, s);
}

}  // namespace mh
