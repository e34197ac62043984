// verify.hip -- drafted tokens against the target's probabilities, from given random numbers (gfx950).
//
// p = softmax(x / T) after each node, q the draft's.  A chain whose tokens were drawn from q accepts node i
// where u_i q(t_i) < p(t_i), and draws the token behind the first one that it rejects from (p - q)+.  Tokens
// that were picked outright are point masses: of a node's children, in order, c is accepted where
// u_c (1 - the rejected ones' p) < p(t_c), and the token behind them is drawn from p without them.  Both leave the
// target's own distribution.  A draw with u is the first token whose cumulative sum passes u times the whole.
//
// A draw compares u with as many borders as the vocabulary has tokens, and sums of 32-bit exponentials move each by up
// to 2^-24: one draw in a hundred over 2^17 tokens.  So the row that is drawn from is weighed in 64 bits, at
// 20 instructions of 8 cycles a logit; all others, of which only the sum is wanted, with the hardware's exponential (the sum's
// error is some 2^-26 of it, and within 2^-18), which hides behind the reading.  Where a number then comes so near to the border of a
// child that the walk asks about that such errors could decide, the walk stops for the sums of that row in 64 bits: one
// question in 2^16, but many more behind likely children that were rejected, as what they leave of 1 is a small difference.
//
// A row is cut into pieces of a wave's values, four pieces a part.  First launch: every row, a workgroup a part, leaves each
// part's maximum and sum.  Second: a workgroup for each part of a stream; each one walks by itself, weighs its part of the row that
// the walk ended at, and the last one to finish draws: it finds the piece that u falls into by the pieces' masses and reads
// that one again.  What is drawn from (p - q)+ needs the exact sums of p and q first, and gets its masses and its
// draw in a third launch.  Which workgroup finishes last changes nothing but who draws.  Streams of few short rows take one launch.
//
// 24 chains of 9 over 130001 fp16 logits and the draft's: 27.5 us for all rows (4 TB/s), 17 for the walk and the two sums, 19 for
// (p - q)+ and the draw, both of which are 64-bit exponentials on 3.1 million logits (6 us each at best) and a chain of
// loads, one after the other: the bound of a row's end is each lane's own, so a lane waits for every 16 bytes before it asks for
// more.  64 chains of 6 over 16384: 10 + 13 + 12.  16 trees of 27 over 16384: 7 + 17.  All rows in 64 bits took 50 us in place
// of 28.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxPieces = 512;  // of a row
constexpr double kLog2e = 1.4426950408889634074;

// Of a part of a row, or of a row: the largest logit, where it is first, and sum of e^{(x - m) / T}.  Nothing
// above -inf: s is 0; a NaN or +inf among them: s is NaN.
struct Stat {
    float m;
    int best;  // -1: none
    double s;
};

// 2^a for a <= 0, as 2^n 2^f with a polynomial through Chebyshev's nodes of |f| <= 1/2, within 2^-44.5; under
// 2^-1010, and for NaN, it is 2^-1010.  n comes out of the low bits of a + 1.5 * 2^52 and goes into the exponent as an
// integer.
template <int N>
__device__ __forceinline__ void exp2_64(double (&a)[N]) {
    constexpr double magic = 6755399441055744.0;
    constexpr double c[] = {1.3259645243929057e-06, 1.5252672925346873e-05, 0.00015403433751254997, 0.0013333558200793719, 0.009618129193934304,
                            0.05550410866465168, 0.2402265069564034, 0.6931471805599462, 1.0};
    double t[N], y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a[i] = fmax(a[i], -1010.0);
        t[i] = a[i] + magic;
        a[i] -= t[i] - magic;
        y[i] = 1.0205905320493103e-07;
    }
#pragma unroll
    for (int j = 0; j < 9; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = fma(y[i], a[i], c[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = __hiloint2double(__double2hiint(y[i]) + (__double2loint(t[i]) << 20), __double2loint(y[i]));
}
// e^{(x - m) / T}, k = log2(e) / T.  The difference first: logits may be far from 0.  -inf is 2^-1010, and what is under kNone of
// the largest, a million of those together too, counts as nothing.
constexpr double kNone = 0x1p-980;
template <int N>
__device__ __forceinline__ void weights(const float (&x)[N], float m, double k, double (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ((double)x[i] - (double)m) * k;
    exp2_64(v);
}
__device__ __forceinline__ double weight(float x, float m, double k) {  // (0 for what counts as nothing)
    const float in[1] = {x};
    double v[1];
    weights<1>(in, m, k, v);
    return v[0] > kNone ? v[0] : 0.0;
}

template <int M>
__device__ __forceinline__ double xshfl64(double v) {
    return __hiloint2double(xshfl<M>(__double2hiint(v)), xshfl<M>(__double2loint(v)));
}
__device__ __forceinline__ double wave_sum64(double v) {
    v += xshfl64<32>(v);
    v += xshfl64<16>(v);
    v += xshfl64<8>(v);
    v += xshfl64<4>(v);
    v += xshfl64<2>(v);
    v += xshfl64<1>(v);
    return v;
}

template <class T>
__device__ __forceinline__ float logit(const T *p) {
    if constexpr (sizeof(T) == 2)
        return __half2float(*(const __half *)p);
    else
        return *p;
}
// N neighbouring logits from place e of a row on, at any address that a logit may have; -inf behind the row.
template <class T, int N>
__device__ __forceinline__ void load_logits(const T *p, int e, int vocab, float (&x)[N]) {
    if (e + N <= vocab) {
        T raw[N];
        __builtin_memcpy(raw, p + e, sizeof(raw));
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = logit(raw + j);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = e + j < vocab ? logit(p + e + j) : -INFINITY;
    }
}

// The workspace: statistics [streams][max_rows][parts] of the target, then of the draft; the masses [streams][pieces] of the row
// that is drawn from, and with a draft those of q and of (p - q)+; how many workgroups of a stream are done, in the second and the
// third launch; and what the draft's streams draw from.
struct Draw {
    float pm, qm;  // the row's largest logits
    int row, mode;
};
enum { DRAW_NONE = 0, DRAW_P = 1, DRAW_REST = 2 };
struct VerifyWs {
    Stat *p, *q;
    double *mass, *mass_q, *rest;
    int2 *done;
    Draw *draw;
};
__host__ __device__ __forceinline__ VerifyWs verify_ws(int streams, int max_rows, int parts, bool draft, void *ws) {
    VerifyWs w;
    const size_t n = (size_t)streams * max_rows * parts, m = (size_t)streams * parts * kWaves;
    w.p = (Stat *)ws;
    w.q = w.p + n;
    w.mass = (double *)(w.q + (draft ? n : 0));
    w.mass_q = w.mass + m;
    w.rest = w.mass_q + (draft ? m : 0);
    w.done = (int2 *)(w.rest + (draft ? m : 0));
    w.draw = (Draw *)(w.done + streams);
    return w;
}

// Rows of stream s: first and how many take part.
__device__ __forceinline__ int2 nodes_of(const VerifyArgs &a, int s) {
    const int r0 = a.row_start[s], r1 = a.row_start[s + 1];
    return r0 >= 0 && r1 >= r0 && r1 <= a.rows ? make_int2(r0, min(r1 - r0, a.max_rows)) : make_int2(0, 0);
}

// ---------------------------------------------------------------- all rows

// One piece of a row, by one wave: EPT values a lane, read V at a time.  Lane 0's is right.
template <class T, int EPT, bool GREEDY>
__device__ __forceinline__ Stat piece_stat(const T *p, int c, int vocab, float inv_t) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    const int base = c * EPT * 64 + ((int)threadIdx.x & 63) * V;
    float x[EPT / V][V];
#pragma unroll
    for (int i = 0; i < EPT / V; ++i) load_logits<T, V>(p, base + i * 64 * V, vocab, x[i]);
    float m = -INFINITY;
    int best = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPT / V; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (GREEDY && x[i][j] > m) best = base + i * 64 * V + j;
            m = fmaxf(m, x[i][j]);
        }
    if constexpr (GREEDY) {
        wave_argmax(m, best);
        return Stat{m, m > -INFINITY ? best : -1, 0.0};
    } else {
        m = wave_max(m);
        // half of the difference: that of a type's two ends stays within it
        const float h = m == -INFINITY ? 0.0f : -0.5f * m;
        float more[4] = {};
#pragma unroll
        for (int i = 0; i < EPT / V; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) more[j & 3] += __builtin_amdgcn_exp2f(fmaf(x[i][j], 0.5f, h) * inv_t * (float)(2.0 * kLog2e));
        return Stat{m, -1, wave_sum64(((double)more[0] + more[1]) + ((double)more[2] + more[3]))};
    }
}

// One part of one row of the target (blockIdx.y 0) or the draft (1).
template <class T, int EPT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void stat_kernel(VerifyArgs a, int parts) {
    __shared__ Stat ls[kWaves];
    const int at = blockIdx.x / parts, part = blockIdx.x - at * parts;
    const int s = at / a.max_rows, node = at - s * a.max_rows;
    const bool of_draft = blockIdx.y == 1;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, parts, a.y != nullptr, a.ws);
    if (node == 0 && part == 0 && !of_draft && threadIdx.x == 0) ws.done[s] = make_int2(0, 0);
    const int2 rows = nodes_of(a, s);
    if (node >= rows.y - of_draft) return;  // (nothing was drawn behind the last row)
    const T *p = of_draft ? (const T *)a.y + (rows.x + node) * a.y_row : (const T *)a.x + (rows.x + node) * a.x_row;
    const float inv_t = of_draft ? a.draft_inv_t : a.inv_t;
    const int w = threadIdx.x >> 6;
    const Stat mine = piece_stat<T, EPT, GREEDY>(p, part * kWaves + w, a.vocab, inv_t);
    if ((threadIdx.x & 63) == 0) ls[w] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double k = (double)inv_t * kLog2e;
        Stat r{-INFINITY, -1, 0.0};
#pragma unroll
        for (int i = 0; i < kWaves; ++i)
            if (ls[i].m > r.m) {
                r.m = ls[i].m;
                r.best = ls[i].best;
            }
        if constexpr (!GREEDY)
#pragma unroll
            for (int i = 0; i < kWaves; ++i)
                if (!(ls[i].s == 0.0)) r.s += ls[i].m == r.m ? ls[i].s : ls[i].s * weight(ls[i].m, r.m, k);
        (of_draft ? ws.q : ws.p)[(size_t)at * parts + part] = r;
    }
}

// ---------------------------------------------------------------- the walk

struct WalkLds {
    Stat p[kTreeMax], q[kTreeMax];
    Draw draw;
    int gone[kTreeMax], n_gone;  // the children of the last node, all rejected
    int unsure;                  // the node whose children the walk cannot tell apart by these sums, -1: none
    double part[kWaves];
};

// The parts of a row together, by 8 lanes; `mine` is the lane's first.
template <bool LARGEST>
__device__ __forceinline__ Stat row_stat(const Stat &mine, const Stat *c, int parts, double k) {
    const int l = threadIdx.x & 7;
    float m = mine.m;
    int best = LARGEST && m > -INFINITY ? mine.best : 0x7fffffff;
    for (int i = l + 8; i < parts; i += 8) {
        if (LARGEST && c[i].m > m) best = c[i].best;
        m = fmaxf(m, c[i].m);
    }
    if constexpr (LARGEST) {
        argmax_step<4>(m, best);
        argmax_step<2>(m, best);
        argmax_step<1>(m, best);
        return Stat{m, m > -INFINITY ? best : -1, 0.0};
    } else {
        m = fmaxf(m, xshfl<4>(m));
        m = fmaxf(m, xshfl<2>(m));
        m = fmaxf(m, xshfl<1>(m));
        double s = 0.0;
        if (!(mine.s == 0.0)) s = mine.m == m ? mine.s : mine.s * weight(mine.m, m, k);
        for (int i = l + 8; i < parts; i += 8)
            if (!(c[i].s == 0.0)) s += c[i].m == m ? c[i].s : c[i].s * weight(c[i].m, m, k);
        s += xshfl64<4>(s);
        s += xshfl64<2>(s);
        s += xshfl64<1>(s);
        return Stat{m, -1, s};
    }
}

// Sum of a row's weights in 64 bits, by the workgroup; every thread has it.
template <class T>
__device__ __forceinline__ double row_sum64(const T *p, int vocab, float m, double k, double (&part)[kWaves]) {
    constexpr int V = 4;
    double sum = 0.0;
#pragma unroll 1
    for (int e = threadIdx.x * V; e < vocab; e += kThreads * V) {
        float x[V];
        double v[V];
        load_logits<T, V>(p, e, vocab, x);
        weights<V>(x, m, k, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[j];
    }
    sum = wave_sum64(sum);
    __syncthreads();  // (the last row's have been read)
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += part[i];
    return sum;
}

__device__ __forceinline__ double uniform(double u) { return u < 1.0 ? (u > 0.0 ? u : 0.0) : 1.0; }  // (NaN: 1)

// What a thread of the walk needs of its node, asked for before everything that does not wait for it.
struct Node {
    bool in, known;  // known: a child with a token of the vocabulary
    int tok, parent;
    double u;
    float lx, ly;  // its token's logits behind the parent
};
template <class T, bool LARGEST>
__device__ __forceinline__ Node node_of(const VerifyArgs &a, int2 rows) {
    const int t = threadIdx.x, n = rows.y;
    Node d{t < n, false, -1, t - 1, 0.0, -INFINITY, -INFINITY};
    if (d.in) d.tok = a.tokens[rows.x + t];
    if (d.in && a.row_mask != nullptr) {
        const uint64_t mask = a.row_mask[rows.x + t], up = mask & ((1ull << t) - 1);
        d.parent = (mask >> t & 1) && up ? 63 - __builtin_clzll(up) : -1;
    }
    if (!d.in || t == 0) d.parent = -1;
    d.known = d.tok >= 0 && d.tok < a.vocab && d.parent >= 0;
    if (!LARGEST && d.known) {
        d.u = uniform(a.uniforms[rows.x + t]);
        d.lx = logit((const T *)a.x + (rows.x + d.parent) * a.x_row + d.tok);
        if (a.y != nullptr) d.ly = logit((const T *)a.y + (rows.x + d.parent) * a.y_row + d.tok);
    }
    return d;
}

// What decides a child: `number` < p(t), where number is u q(t), or u times what its elder siblings leave of 1.
struct Choice {
    bool accept;
    bool unsure;  // the sums' errors could decide it
};
template <bool LARGEST>
__device__ __forceinline__ Choice choice_of(const VerifyArgs &a, int n, const Node &d, const Stat &p, const Stat &q, double kp, double kq) {
    // Errors of 2^-18 of each probability, twice over; of what is left they are as large as of what is gone.
    constexpr double kNear = 0x1p-17;
    if constexpr (LARGEST) return Choice{d.known && d.tok == p.best, false};
    const int t = threadIdx.x, tok = d.tok, parent = d.parent;
    double prob = 0.0, number = 0.0, gone = 0.0;
    bool fine = d.known && p.s > 0.0;  // (not NaN)
    if (fine) prob = weight(d.lx, p.m, kp) / p.s;
    if (a.y != nullptr) {
        fine &= q.s > 0.0;
        if (fine) number = gone = d.u * (weight(d.ly, q.m, kq) / q.s);
    } else {
        double left = 1.0;
        bool again = false;  // an elder sibling is the same token
        if (a.row_mask != nullptr)
            for (int j = 1; j < n; ++j) {
                const int pj = __builtin_amdgcn_readlane(parent, j), tj = __builtin_amdgcn_readlane(tok, j);
                const bool aj = __builtin_amdgcn_readlane((int)again, j);
                const double bj = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(prob), j),
                                                   __builtin_amdgcn_readlane(__double2loint(prob), j));
                if (t > j && parent == pj && pj >= 0) {
                    again |= tok == tj;
                    if (!aj) left -= bj;
                }
            }
        fine &= !again;
        number = d.u * (left > 0.0 ? left : 0.0);
        gone = d.u * (1.0 - left);
    }
    return Choice{fine && number < prob, fine && prob > 0.0 && fabs(number - prob) <= kNear * (prob + gone)};
}

// The walk of one stream, by one workgroup: the rows' sums by all threads, then a lane a node.  pp, qq: the stream's parts; `writes`:
// whether this workgroup leaves the outputs.
template <class T, bool LARGEST>
__device__ __forceinline__ void walk(const VerifyArgs &a, int s, int2 rows, const Node &d, const Stat *pp, const Stat *qq, int parts, bool writes, WalkLds &lds) {
    const int t = threadIdx.x, n = rows.y;
    const bool drafted = a.y != nullptr, in = d.in, known = d.known;
    const int all = LARGEST || !drafted ? a.max_rows : 2 * a.max_rows;  // the target's rows, then the draft's; what is past n is not used
    auto row_at = [&](int i) { return (i < a.max_rows ? pp + (size_t)i * parts : qq + (size_t)(i - a.max_rows) * parts); };
    Stat first{-INFINITY, -1, 0.0};
    if ((t >> 3) < all && (t & 7) < parts) first = row_at(t >> 3)[t & 7];
    const double kp = (double)a.inv_t * kLog2e, kq = (double)a.draft_inv_t * kLog2e;
    const int tok = d.tok, parent = d.parent, of = max(parent, 0);
    for (int i = t >> 3; i < all; i += kThreads / 8) {
        const bool q = i >= a.max_rows;
        if (i >= kThreads / 8) first = (t & 7) < parts ? row_at(i)[t & 7] : Stat{-INFINITY, -1, 0.0};
        const Stat r = row_stat<LARGEST>(first, row_at(i), parts, q ? kq : kp);
        if ((t & 7) == 0) (q ? lds.q[i - a.max_rows] : lds.p[i]) = r;
    }
    __syncthreads();
    // From node to node by the first child that is accepted.
    int cur = 0;
    uint64_t on = 1, exact = 0;  // nodes on the path, and those whose rows' sums are of 64 bits
    while (true) {
        if (t < 64) {
            const Choice c = choice_of<LARGEST>(a, n, d, lds.p[of], drafted ? lds.q[of] : Stat{}, kp, kq);
            const uint64_t doubt = __ballot(c.unsure && !(exact >> of & 1)), stops = __ballot(c.accept) | doubt;
            bool unsure = false;
            while (const uint64_t next = __ballot(parent == cur) & stops) {
                unsure = doubt >> __builtin_ctzll(next) & 1;
                if (unsure) break;
                cur = __builtin_ctzll(next);
                on |= 1ull << cur;
            }
            if (!unsure) {
                if (in && writes) {  // entry j of the path is the j-th node on it
                    const int taken = __popcll(on);
                    if (on >> t & 1) a.path[rows.x + __popcll(on & ((1ull << t) - 1))] = t;
                    if (t >= taken) a.path[rows.x + t] = -1;
                }
                const bool child = !LARGEST && !drafted && parent == cur && known;
                const uint64_t children = __ballot(child);
                if (child) lds.gone[__popcll(children & ((1ull << t) - 1))] = tok;
                if (t == 0) {
                    const Stat pl = lds.p[cur];
                    Stat ql{};
                    if (drafted && cur < n - 1) ql = lds.q[cur];
                    lds.n_gone = __popcll(children);
                    lds.draw = Draw{pl.m, ql.m, rows.x + cur, !(pl.s > 0.0) ? DRAW_NONE : (ql.s > 0.0 ? DRAW_REST : DRAW_P)};
                    if (writes) {
                        a.accepted[s] = __popcll(on) - 1;
                        if (LARGEST) a.next[s] = pl.best;
                    }
                }
            }
            if (!LARGEST && t == 0) lds.unsure = unsure ? cur : -1;
        }
        __syncthreads();
        if (LARGEST || __builtin_expect(lds.unsure < 0, 1)) return;
        const int row = lds.unsure;
        const double sum = row_sum64((const T *)a.x + (rows.x + row) * a.x_row, a.vocab, lds.p[row].m, kp, lds.part);
        double sum_q = 0.0;
        if (drafted) sum_q = row_sum64((const T *)a.y + (rows.x + row) * a.y_row, a.vocab, lds.q[row].m, kq, lds.part);
        if (t == 0) {
            lds.p[row].s = sum;
            if (drafted) lds.q[row].s = sum_q;
        }
        exact |= 1ull << row;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- the draw

// Inclusive sums over a wave, and over the workgroup: what earlier threads hold, this thread's among them.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    return v + __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false),
                                __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ double scan64(double v, double *lds, double &all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    v = dpp_add<0x111, 0xf>(v);  // one lane up, two, four, eight, within rows of 16
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);  // the last lane of rows 0 and 2 to rows 1 and 3, of row 1 to the upper half
    v = dpp_add<0x143, 0xc>(v);
    __syncthreads();
    if (lane == 63) lds[w] = v;
    __syncthreads();
    double before = 0.0;
    all = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i < w) before += lds[i];
        all += lds[i];
    }
    return before + v;
}

struct PickLds {
    double scan[kWaves];
    double before;
    int found, last;
};

// Of values in order, N a thread: the first whose cumulative sum, on top of `before`, passes u of `whole` (or, whole < 0, of
// their own sum), else the last that counts; -1 where there is none.  `before` becomes the sum in front of it, whole theirs.
template <int N>
__device__ __forceinline__ int pick_of(const double (&v)[N], double u, double &before, double &whole, PickLds &lds) {
    const int t = threadIdx.x;
    double sum = 0.0, all;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += v[i];
    if (t == 0) {
        lds.found = 0x7fffffff;
        lds.last = -1;
    }
    double run = before + (scan64(sum, lds.scan, all) - sum);
    if (whole < 0.0) whole = all;
    const double aim = u * whole;
    int found = -1, last = -1;
    double front = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (v[i] > kNone) {
            last = t * N + i;
            if (found < 0) front = run;
            if (run + v[i] > aim && found < 0) found = t * N + i;
        }
        run += v[i];
    }
    if (found >= 0) atomicMin(&lds.found, found);
    if (last >= 0) atomicMax(&lds.last, last);
    __syncthreads();
    const int got = lds.found != 0x7fffffff ? lds.found : lds.last;
    if (got >= 0 && got / N == t) lds.before = front;  // (the last positive value's, where none was found)
    __syncthreads();
    before = lds.before;
    return got;
}

// Masses go from workgroup to workgroup of one launch by stores and loads that are coherent across the XCDs' L2 caches; a
// fence instead (which writes a whole L2 back, and empties it) took 20 us with 256 workgroups.
__device__ __forceinline__ void put_mass(double *p, double v) {
    __hip_atomic_store((uint64_t *)p, (uint64_t)__double_as_longlong(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get_mass(const double *p) {
    return __longlong_as_double((long long)__hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// What the tokens of a row weigh, up to a factor of the row.
template <class T>
struct Weights {
    const T *x, *y;
    float pm, qm;
    double kp, kq, ps = 1.0, qs = 1.0;  // ps, qs: 1 / sum
    bool rest = false;                  // (p - q)+
    __device__ __forceinline__ Weights(const VerifyArgs &a, const Draw &d)
        : x((const T *)a.x + d.row * a.x_row), y((const T *)a.y + d.row * a.y_row), pm(d.pm), qm(d.qm), kp((double)a.inv_t * kLog2e),
          kq((double)a.draft_inv_t * kLog2e) {}
    // of N tokens from e on
    template <int N>
    __device__ __forceinline__ void of(int e, int vocab, double (&v)[N]) const {
        float lx[N], ly[N];
        load_logits<T, N>(x, e, vocab, lx);
        if (rest) load_logits<T, N>(y, e, vocab, ly);
        weights<N>(lx, pm, kp, v);
        if (rest) {
            double q[N];
            weights<N>(ly, qm, kq, q);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const double d = v[i] * ps - q[i] * qs;
                v[i] = d > 0.0 ? d : 0.0;
            }
        }
    }
};

struct KeepAll {
    template <int N>
    __device__ __forceinline__ void operator()(int, double (&)[N]) const {}
};
// Leaves the rejected tokens out.
struct Drop {
    const int *gone;
    int n;
    template <int N>
    __device__ __forceinline__ void operator()(int first, double (&v)[N]) const {
        for (int i = 0; i < n; ++i) {
            const unsigned d = (unsigned)(gone[i] - first);
            if (d < (unsigned)N)
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = (int)d == j ? 0.0 : v[j];
        }
    }
};

// The mass of piece c, by one wave; every lane has it.
template <class T, int EPT, class D>
__device__ __forceinline__ double piece_mass(const Weights<T> &w, int vocab, int c, const D &drop) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPT / V; ++i) {
        const int e = c * EPT * 64 + (i * 64 + ((int)threadIdx.x & 63)) * V;
        double v[V];
        w.template of<V>(e, vocab, v);
        drop(e, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[j];
    }
    return wave_sum64(sum);
}

// The token drawn with u; mass(c): the pieces'.  -1 where none counts.
template <class T, int EPT, class M, class D>
__device__ __forceinline__ int pick(const Weights<T> &w, const M &mass, int vocab, int pieces, double u, PickLds &lds, const D &drop) {
    constexpr int N = EPT * 64 / kThreads, NP = kMaxPieces / kThreads;
    const int t = threadIdx.x;
    double m[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) m[i] = t * NP + i < pieces ? mass(t * NP + i) : 0.0;
    double before = 0.0, whole = -1.0;
    const int c = pick_of<NP>(m, u, before, whole, lds);
    if (c < 0) return -1;
    const int first = c * EPT * 64 + t * N;
    double v[N];
    w.template of<N>(first, vocab, v);
    drop(first, v);
    const int got = pick_of<N>(v, u, before, whole, lds);
    return got < 0 ? -1 : c * EPT * 64 + got;
}

// Sum of a stream's pieces, the same in every workgroup: by one wave.
__device__ __forceinline__ double sum_of(const double *mass, int pieces) {
    double s = 0.0;
    for (int i = threadIdx.x & 63; i < pieces; i += 64) s += mass[i];
    return wave_sum64(s);
}

// Whether this workgroup is the last of `all` to come here: then get_mass has what the others put before.
__device__ __forceinline__ bool last_of(int *done, int all, int *lds) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's masses have arrived
    __syncthreads();
    if (threadIdx.x == 0) *lds = __hip_atomic_fetch_add(done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    __syncthreads();
    return *lds != 0;
}

// A stream without rows.
__device__ __forceinline__ bool no_rows(const VerifyArgs &a, int s, int2 rows, bool writes) {
    if (rows.y > 0) return false;
    if (threadIdx.x == 0 && writes) {
        a.accepted[s] = 0;
        a.next[s] = -1;
    }
    return true;
}

// The other distribution of a row, as one to be weighed by itself.
template <class T>
__device__ __forceinline__ Weights<T> draft_of(const Weights<T> &w) {
    Weights<T> q = w;
    q.x = w.y;
    q.pm = w.qm;
    q.kp = w.kq;
    return q;
}

// A workgroup for each part of a stream.  With a draft, what has to come from (p - q)+ is left to the next launch.
template <class T, int EPT, bool DRAFT>
__global__ __launch_bounds__(kThreads) void walk_kernel(VerifyArgs a, int pieces, int parts) {
    __shared__ WalkLds wl;
    __shared__ PickLds lds;
    __shared__ int last;
    const int s = blockIdx.x / parts, part = blockIdx.x - s * parts, t = threadIdx.x;
    const int2 rows = nodes_of(a, s);
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, parts, DRAFT, a.ws);
    if (no_rows(a, s, rows, part == 0)) {
        if (DRAFT && t == 0 && part == 0) ws.draw[s].mode = DRAW_NONE;
        return;
    }
    const double u = uniform(a.uniforms[rows.x]);
    const Node node = node_of<T, false>(a, rows);
    walk<T, false>(a, s, rows, node, ws.p + (size_t)s * a.max_rows * parts, ws.q + (size_t)s * a.max_rows * parts, parts, part == 0, wl);
    const Draw d = wl.draw;
    if (DRAFT && t == 0 && part == 0) ws.draw[s] = d;
    if (d.mode == DRAW_NONE) {
        if (t == 0 && part == 0) a.next[s] = -1;
        return;
    }
    const int c = part * kWaves + (t >> 6);
    const Weights<T> w(a, d);
    double *mass = ws.mass + (size_t)s * parts * kWaves;
    const Drop drop{wl.gone, DRAFT ? 0 : wl.n_gone};
    if (c < pieces) {
        const double v = piece_mass<T, EPT>(w, a.vocab, c, drop);
        if ((t & 63) == 0) put_mass(mass + c, v);
        if (DRAFT && d.mode == DRAW_REST) {
            const double vq = piece_mass<T, EPT>(draft_of(w), a.vocab, c, KeepAll());
            if ((t & 63) == 0) put_mass(ws.mass_q + (size_t)s * parts * kWaves + c, vq);
        }
    }
    if (DRAFT && d.mode == DRAW_REST) return;
    if (!last_of(&ws.done[s].x, parts, &last)) return;
    auto masses = [&](int i) { return get_mass(mass + i); };
    int got = pick<T, EPT>(w, masses, a.vocab, pieces, u, lds, drop);
    if (!DRAFT && got < 0) {  // nothing is left: p itself
        __syncthreads();
        for (int i = t >> 6; i < pieces; i += kWaves) {
            const double v = piece_mass<T, EPT>(w, a.vocab, i, KeepAll());
            if ((t & 63) == 0) put_mass(mass + i, v);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        got = pick<T, EPT>(w, masses, a.vocab, pieces, u, lds, KeepAll());
    }
    if (t == 0) a.next[s] = got;
}

__global__ __launch_bounds__(kThreads) void greedy_kernel(VerifyArgs a, int parts) {
    __shared__ WalkLds wl;
    const int s = blockIdx.x;
    const int2 rows = nodes_of(a, s);
    if (no_rows(a, s, rows, true)) return;
    const Stat *p = verify_ws(a.streams, a.max_rows, parts, false, a.ws).p + (size_t)s * a.max_rows * parts;
    walk<float, true>(a, s, rows, node_of<float, true>(a, rows), p, p, parts, true, wl);  // (no logit is read)
}

// The draw behind a rejected token: a workgroup for each part of a stream has its masses of (p - q)+, the last one draws.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void rest_kernel(VerifyArgs a, int pieces, int parts) {
    __shared__ PickLds lds;
    __shared__ int last;
    const int s = blockIdx.x / parts, part = blockIdx.x - s * parts, t = threadIdx.x;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, parts, true, a.ws);
    const double *mass = ws.mass + (size_t)s * parts * kWaves, *mass_q = ws.mass_q + (size_t)s * parts * kWaves;
    const Draw d = ws.draw[s];
    const int root = a.row_start[s];
    if (d.mode != DRAW_REST) return;
    const double u = uniform(a.uniforms[root]);
    Weights<T> w(a, d);
    w.ps = 1.0 / sum_of(mass, pieces);
    w.qs = 1.0 / sum_of(mass_q, pieces);
    w.rest = true;
    double *rest = ws.rest + (size_t)s * parts * kWaves;
    const int c = part * kWaves + (t >> 6);
    if (c < pieces) {
        const double v = piece_mass<T, EPT>(w, a.vocab, c, KeepAll());
        if ((t & 63) == 0) put_mass(rest + c, v);
    }
    if (!last_of(&ws.done[s].y, parts, &last)) return;
    int got = pick<T, EPT>(w, [&](int i) { return get_mass(rest + i); }, a.vocab, pieces, u, lds, KeepAll());
    if (got < 0) {  // nothing is left over: p itself
        __syncthreads();
        w.rest = false;
        got = pick<T, EPT>(w, [&](int i) { return mass[i]; }, a.vocab, pieces, u, lds, KeepAll());
    }
    if (t == 0) a.next[s] = got;
}

// All of it in one launch, a workgroup a stream, where its rows have no more than kSmallPieces pieces: the smallest calls are
// launches and chains of loads.
constexpr int kSmallPieces = 32, kSmallEpt = 16;
template <class T, bool GREEDY>
__global__ __launch_bounds__(kThreads) void small_kernel(VerifyArgs a, int pieces) {
    constexpr int EPT = kSmallEpt;
    __shared__ Stat p[kSmallPieces], q[kSmallPieces];
    __shared__ double mass[kSmallPieces], mass_q[kSmallPieces];
    __shared__ WalkLds wl;
    __shared__ PickLds lds;
    const int s = blockIdx.x, t = threadIdx.x, w = t >> 6;
    const int2 rows = nodes_of(a, s);
    if (no_rows(a, s, rows, true)) return;
    const bool drafted = a.y != nullptr;
    const Node mine = node_of<T, GREEDY>(a, rows);
    const int units = rows.y * pieces;
    for (int i = w; i < units; i += kWaves) {
        const int node = i / pieces, c = i - node * pieces;
        const Stat m = piece_stat<T, EPT, GREEDY>((const T *)a.x + (rows.x + node) * a.x_row, c, a.vocab, a.inv_t);
        if ((t & 63) == 0) p[i] = m;
        if (drafted && node < rows.y - 1) {
            const Stat n = piece_stat<T, EPT, GREEDY>((const T *)a.y + (rows.x + node) * a.y_row, c, a.vocab, a.draft_inv_t);
            if ((t & 63) == 0) q[i] = n;
        }
    }
    __syncthreads();
    walk<T, GREEDY>(a, s, rows, mine, p, q, pieces, true, wl);
    if constexpr (!GREEDY) {
        const Draw d = wl.draw;
        int got = -1;
        if (d.mode != DRAW_NONE) {
            const double u = uniform(a.uniforms[rows.x]);
            Weights<T> wt(a, d);
            auto weigh = [&](const Weights<T> &x, double *to, const auto &drop) {
                for (int c = w; c < pieces; c += kWaves) {
                    const double v = piece_mass<T, EPT>(x, a.vocab, c, drop);
                    if ((t & 63) == 0) to[c] = v;
                }
            };
            const Drop drop{wl.gone, drafted ? 0 : wl.n_gone};
            weigh(wt, mass, drop);
            if (d.mode == DRAW_REST) {
                weigh(draft_of(wt), mass_q, KeepAll());
                __syncthreads();
                wt.ps = 1.0 / sum_of(mass, pieces);
                wt.qs = 1.0 / sum_of(mass_q, pieces);
                wt.rest = true;
                __syncthreads();
                weigh(wt, mass, KeepAll());
            }
            __syncthreads();
            got = pick<T, EPT>(wt, [&](int i) { return mass[i]; }, a.vocab, pieces, u, lds, drop);
            if (got < 0) {  // nothing is left: p itself
                wt.rest = false;
                __syncthreads();
                weigh(wt, mass, KeepAll());
                __syncthreads();
                got = pick<T, EPT>(wt, [&](int i) { return mass[i]; }, a.vocab, pieces, u, lds, KeepAll());
            }
        }
        if (t == 0) a.next[s] = got;
    }
}

// Whether a stream's rows are few and short enough for one workgroup.
bool small(int max_rows, int vocab) { return max_rows * ((vocab + kSmallEpt * 64 - 1) / (kSmallEpt * 64)) <= kSmallPieces; }

// Values of a lane of a piece: few while that fills the chip, many where the parts' sums would be much work themselves.
constexpr int kFinePieces = 16, kFineRows = 1024;  // parts of 4 values a lane: most of a row, and of all rows
int ept_of(int rows, int vocab) {
    const int few = (vocab + 1023) / 1024;
    if (few <= kFinePieces && (long long)rows * few <= kFineRows) return 4;
    return vocab <= 64 * 1024 ? 16 : 32;
}
int parts_of(int rows, int vocab) {
    const int n = ept_of(rows, vocab) * kThreads;
    return (vocab + n - 1) / n;
}
static_assert(kMaxPieces * 32 * 64 >= kVocabMax, "a row's pieces");

template <class T, int EPT>
hipError_t verify_e(const VerifyArgs &a, hipStream_t s) {
    const int parts = parts_of(a.streams * a.max_rows, a.vocab), pieces = (a.vocab + EPT * 64 - 1) / (EPT * 64);
    const dim3 rows((unsigned)a.streams * a.max_rows * parts, a.y != nullptr ? 2 : 1), of_streams((unsigned)a.streams * parts);
    if (a.greedy) {
        hipLaunchKernelGGL((stat_kernel<T, EPT, true>), rows, dim3(kThreads), 0, s, a, parts);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;  // (what follows trusts what it leaves)
        hipLaunchKernelGGL(greedy_kernel, dim3(a.streams), dim3(kThreads), 0, s, a, parts);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((stat_kernel<T, EPT, false>), rows, dim3(kThreads), 0, s, a, parts);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.y != nullptr) {
        hipLaunchKernelGGL((walk_kernel<T, EPT, true>), of_streams, dim3(kThreads), 0, s, a, pieces, parts);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        hipLaunchKernelGGL((rest_kernel<T, EPT>), of_streams, dim3(kThreads), 0, s, a, pieces, parts);
    } else {
        hipLaunchKernelGGL((walk_kernel<T, EPT, false>), of_streams, dim3(kThreads), 0, s, a, pieces, parts);
    }
    return hipGetLastError();
}

template <class T>
hipError_t verify_t(const VerifyArgs &a, hipStream_t s) {
    (void)hipGetLastError();
    if (small(a.max_rows, a.vocab)) {
        const int pieces = (a.vocab + kSmallEpt * 64 - 1) / (kSmallEpt * 64);
        if (a.greedy)
            hipLaunchKernelGGL((small_kernel<T, true>), dim3(a.streams), dim3(kThreads), 0, s, a, pieces);
        else
            hipLaunchKernelGGL((small_kernel<T, false>), dim3(a.streams), dim3(kThreads), 0, s, a, pieces);
        return hipGetLastError();
    }
    switch (ept_of(a.streams * a.max_rows, a.vocab)) {
        case 4: return verify_e<T, 4>(a, s);
        case 16: return verify_e<T, 16>(a, s);
        default: return verify_e<T, 32>(a, s);
    }
}

}  // namespace

size_t verify_need(int streams, int max_rows, int vocab, bool draft) {
    if (small(max_rows, vocab)) return 0;
    const VerifyWs w = verify_ws(streams, max_rows, parts_of(streams * max_rows, vocab), draft, nullptr);
    return (size_t)(uintptr_t)(w.draw + (draft ? streams : 0));
}
// What calls of up to so many streams and rows need.  Few rows are cut finer (ept_of), so the most can be that of the largest call that
// still is.
size_t verify_workspace(int streams, int max_rows, int vocab, bool draft) {
    size_t most = verify_need(streams, max_rows, vocab, draft);
    const int few = (vocab + 1023) / 1024;
    for (int r = 1; r <= max_rows && few <= kFinePieces; ++r)
        if (const int s = std::min(streams, kFineRows / (few * r)); s > 0) most = std::max(most, verify_need(s, r, vocab, draft));
    return most;
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) { return a.dtype == ELEM_F16 ? verify_t<__half>(a, s) : verify_t<float>(a, s); }

}  // namespace mh
