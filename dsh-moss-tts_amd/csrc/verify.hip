// verify.hip -- drafted tokens against the target's probabilities, from given random numbers (gfx950).
//
// p = softmax(x / T) after each node, q the draft's.  A chain whose tokens were drawn from q accepts node i
// where u_i q(t_i) < p(t_i), and draws the token behind the first one that it rejects from (p - q)+.  Tokens
// that were picked outright are point masses: of a node's children, in order, c is accepted where
// u_c (1 - the rejected ones' p) < p(t_c), and the token behind them is drawn from p without them.  Both leave the
// target's own distribution.  A draw with u is the first token whose cumulative sum passes u times the whole.
//
// A draw compares u with as many borders as the vocabulary has tokens, and sums of 32 bits move each by up to
// 2^-24: one draw in a hundred over 2^17 tokens.  So probabilities are formed and summed in 64 bits, which
// takes 17 instructions a logit, near what reading one takes.
//
// A row is cut into pieces of 64 lanes' values.  One launch reads all rows, a wave a piece, and leaves the
// pieces' maxima and sums; a second one walks, a workgroup a stream, and draws: it finds the piece that u falls into by
// the pieces' sums, and reads that one piece again.  What is drawn from (p - q)+ needs that row's two sums first: there the
// second launch has workgroups for all pieces of a stream, each of which walks by itself, and a third one draws.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxPieces = 512;  // of a row
constexpr double kLog2e = 1.4426950408889634074;

// Of a piece of a row, or of a row: the largest logit, where it is first, and sum of e^{(x - m) / T}.  Nothing
// above -inf: s is 0; a NaN or +inf among them: s is NaN.
struct Stat {
    float m;
    int best;  // -1: none
    double s;
};

// 2^a for a <= 0, as 2^n 2^f with a polynomial through Chebyshev's nodes of |f| <= 1/2, within 2^-45; under
// 2^-1000 it is 2^-1000.  n comes out of the low bits of a + 1.5 * 2^52 and goes into the exponent as an integer.
__device__ __forceinline__ double exp2_64(double a) {
    constexpr double magic = 6755399441055744.0;
    a = a < -1000.0 ? -1000.0 : a;
    const double t = a + magic, f = a - (t - magic);
    double y = 1.0205905320493103e-07;
    y = fma(y, f, 1.3259645243929057e-06);
    y = fma(y, f, 1.5252672925346873e-05);
    y = fma(y, f, 0.00015403433751254997);
    y = fma(y, f, 0.0013333558200793719);
    y = fma(y, f, 0.009618129193934304);
    y = fma(y, f, 0.05550410866465168);
    y = fma(y, f, 0.2402265069564034);
    y = fma(y, f, 0.6931471805599462);
    y = fma(y, f, 1.0);
    return __hiloint2double(__double2hiint(y) + (__double2loint(t) << 20), __double2loint(y));
}
// e^{(x - m) / T}, k = log2(e) / T.  The difference first: logits may be far from 0.
__device__ __forceinline__ double raw_weight(float x, float m, double k) { return exp2_64(((double)x - (double)m) * k); }
// The same with 0 for what is under 2^-1000, -inf among it.
__device__ __forceinline__ double weight(float x, float m, double k) {
    const double a = ((double)x - (double)m) * k;
    return a >= -1000.0 ? exp2_64(a) : 0.0;
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

// The workspace: statistics [streams][max_rows][pieces] of the target, then of the draft; then of draws from
// (p - q)+ the mass of each piece [streams][pieces], and [streams] what is drawn from.
struct Draw {
    Stat p, q;  // of the row
    int row, mode;
};
enum { DRAW_NONE = 0, DRAW_P = 1, DRAW_REST = 2 };
struct VerifyWs {
    Stat *p, *q;
    double *mass;
    Draw *draw;
};
__host__ __device__ __forceinline__ VerifyWs verify_ws(int streams, int max_rows, int pieces, bool draft, void *ws) {
    VerifyWs w;
    const size_t n = (size_t)streams * max_rows * pieces;
    w.p = (Stat *)ws;
    w.q = w.p + n;
    w.mass = (double *)(w.q + (draft ? n : 0));
    w.draw = (Draw *)(w.mass + (draft ? (size_t)streams * pieces : 0));
    return w;
}

// Rows of stream s: first and how many take part.
__device__ __forceinline__ int2 nodes_of(const VerifyArgs &a, int s) {
    const int r0 = a.row_start[s], r1 = a.row_start[s + 1];
    return r0 >= 0 && r1 >= r0 && r1 <= a.rows ? make_int2(r0, min(r1 - r0, a.max_rows)) : make_int2(0, 0);
}

// One piece of one row of the target (blockIdx.y 0) or the draft (1), a wave each: EPT values a lane, read V at a time.
template <class T, int EPT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void stat_kernel(VerifyArgs a, int pieces) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    const int lane = threadIdx.x & 63;
    const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const int at = unit / pieces, c = unit - at * pieces;
    const int s = at / a.max_rows, node = at - s * a.max_rows;
    if (s >= a.streams) return;
    const bool of_draft = blockIdx.y == 1;
    const int2 rows = nodes_of(a, s);
    if (node >= rows.y - of_draft) return;  // (nothing was drawn behind the last row)
    const T *p = of_draft ? (const T *)a.y + (rows.x + node) * a.y_row : (const T *)a.x + (rows.x + node) * a.x_row;
    const int base = c * EPT * 64 + lane * V;
    float x[EPT / V][V];
#pragma unroll
    for (int i = 0; i < EPT / V; ++i) load_logits<T, V>(p, base + i * 64 * V, a.vocab, x[i]);
    float m = -INFINITY;
    int best = 0x7fffffff;
    double sum = 0.0;
    if constexpr (GREEDY) {
#pragma unroll
        for (int i = 0; i < EPT / V; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (x[i][j] > m) {
                    m = x[i][j];
                    best = base + i * 64 * V + j;
                }
        wave_argmax(m, best);
    } else {
#pragma unroll
        for (int i = 0; i < EPT / V; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) m = fmaxf(m, x[i][j]);
        m = wave_max(m);
        if (m > -INFINITY) {
            const double k = (double)(of_draft ? a.draft_inv_t : a.inv_t) * kLog2e;
            bool bad = !(m < INFINITY);
            double more[2] = {};
#pragma unroll
            for (int i = 0; i < EPT / V; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    bad |= x[i][j] != x[i][j];
                    more[j & 1] += raw_weight(x[i][j], m, k);
                }
            sum = wave_sum64(bad ? __builtin_nan("") : more[0] + more[1]);
        } else {  // nothing but -inf, or NaN
            bool bad = false;
#pragma unroll
            for (int i = 0; i < EPT / V; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) bad |= x[i][j] != x[i][j];
            if (__any(bad)) sum = __builtin_nan("");
        }
    }
    if (lane == 0) {
        const VerifyWs ws = verify_ws(a.streams, a.max_rows, pieces, a.y != nullptr, a.ws);
        (of_draft ? ws.q : ws.p)[(size_t)at * pieces + c] = Stat{m, m > -INFINITY ? best : -1, sum};
    }
}

// The pieces of a row together, by one wave; every lane has the result.
template <bool GREEDY>
__device__ __forceinline__ Stat row_stat(const Stat *c, int pieces, double k) {
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    int best = 0x7fffffff;
    for (int i = lane; i < pieces; i += 64) {
        const Stat o = c[i];
        if (o.m > m) {
            m = o.m;
            best = o.best;
        }
    }
    if constexpr (GREEDY) {
        wave_argmax(m, best);
        return Stat{m, m > -INFINITY ? best : -1, 0.0};
    } else {
        m = wave_max(m);
        double s = 0.0;
        for (int i = lane; i < pieces; i += 64) {
            const Stat o = c[i];
            if (!(o.s == 0.0)) s += o.s * weight(o.m, m, k);
        }
        return Stat{m, -1, wave_sum64(s)};
    }
}

// Inclusive sums over the workgroup in 64 bits: what earlier threads hold, this thread's among them.
__device__ __forceinline__ double scan64(double v, double *lds, double &all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
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
    double mass[kMaxPieces];
    double scan[kWaves];
    double before;
    int found, last;
};

// Of values in order, N a thread: the first whose cumulative sum, on top of `before`, passes u of `whole` (or, whole < 0, of
// their own sum), else the last above 0; -1 where there is none.  `before` becomes the sum in front of it, whole theirs.
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
    double run = before + scan64(sum, lds.scan, all) - sum;
    if (whole < 0.0) whole = all;
    const double aim = u * whole;
    int found = -1, last = -1;
    double front[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        front[i] = run;
        run += v[i];
        if (v[i] > 0.0) last = t * N + i;
        if (v[i] > 0.0 && run > aim && found < 0) found = t * N + i;
    }
    if (found >= 0) atomicMin(&lds.found, found);
    if (last >= 0) atomicMax(&lds.last, last);
    __syncthreads();
    const int got = lds.found != 0x7fffffff ? lds.found : lds.last;
    if (got >= 0 && got / N == t) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (got % N == i) lds.before = front[i];
    }
    __syncthreads();
    before = lds.before;
    return got;
}

// What the tokens of a row weigh, up to a factor of the row.
template <class T>
struct Weights {
    const T *x, *y;
    float pm, qm;
    double kp, kq, ps, qs;  // ps, qs: 1 / sum
    bool rest;              // (p - q)+
    __device__ __forceinline__ Weights(const VerifyArgs &a, const Draw &d)
        : x((const T *)a.x + d.row * a.x_row), y((const T *)a.y + d.row * a.y_row), pm(d.p.m), qm(d.q.m), kp((double)a.inv_t * kLog2e),
          kq((double)a.draft_inv_t * kLog2e), ps(1.0 / d.p.s), qs(1.0 / d.q.s), rest(d.mode == DRAW_REST) {}
    // of N tokens from e on
    template <int N>
    __device__ __forceinline__ void of(int e, int vocab, double (&v)[N]) const {
        float lx[N];
        load_logits<T, N>(x, e, vocab, lx);
        if (rest) {
            float ly[N];
            load_logits<T, N>(y, e, vocab, ly);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const double d = weight(lx[i], pm, kp) * ps - weight(ly[i], qm, kq) * qs;
                v[i] = d > 0.0 ? d : 0.0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = weight(lx[i], pm, kp);
        }
    }
};

// The token drawn with u; lds.mass holds the pieces' masses, -1 where there are none.  drop(first, v) leaves tokens out.
template <class T, int EPT, class Drop>
__device__ __forceinline__ int pick(const Weights<T> &w, int vocab, int pieces, double u, PickLds &lds, Drop &&drop) {
    constexpr int N = EPT * 64 / kThreads, NP = kMaxPieces / kThreads;
    const int t = threadIdx.x;
    double mass[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) mass[i] = t * NP + i < pieces ? lds.mass[t * NP + i] : 0.0;
    double before = 0.0, whole = -1.0;
    const int c = pick_of<NP>(mass, u, before, whole, lds);
    if (c < 0) return -1;
    const int first = c * EPT * 64 + t * N;
    double v[N];
    w.template of<N>(first, vocab, v);
    drop(first, v);
    const int got = pick_of<N>(v, u, before, whole, lds);
    return got < 0 ? -1 : c * EPT * 64 + got;
}
struct KeepAll {
    template <int N>
    __device__ __forceinline__ void operator()(int, double (&)[N]) const {}
};

__device__ __forceinline__ double uniform(double u) { return u < 1.0 ? (u > 0.0 ? u : 0.0) : 1.0; }  // (NaN: 1)

struct WalkLds {
    Stat p[kTreeMax], q[kTreeMax];
    Draw draw;
    int gone[kTreeMax], n_gone;  // the children of the last node, all rejected
    double gone_weight[kTreeMax];
};

// The walk of one stream, by one workgroup: the rows' sums by all waves, then a lane a node.  `writes`: whether this
// workgroup leaves the outputs.  A barrier follows.
template <class T, bool GREEDY>
__device__ __forceinline__ void walk(const VerifyArgs &a, int s, int2 rows, const VerifyWs &ws, int pieces, bool writes, WalkLds &lds) {
    const int t = threadIdx.x, n = rows.y;
    const bool drafted = a.y != nullptr;
    const double kp = (double)a.inv_t * kLog2e, kq = (double)a.draft_inv_t * kLog2e;
    // what a lane needs of its node, asked for early
    const bool in = t < n;
    const int tok = in ? a.tokens[rows.x + t] : -1;
    int parent = t - 1;
    if (in && a.row_mask != nullptr) {
        const uint64_t mask = a.row_mask[rows.x + t], up = mask & ((1ull << t) - 1);
        parent = (mask >> t & 1) && up ? 63 - __builtin_clzll(up) : -1;
    }
    if (!in || t == 0) parent = -1;
    const int of = max(parent, 0);
    const bool known = tok >= 0 && tok < a.vocab && parent >= 0;
    double u = 0.0;
    float lx = -INFINITY, ly = -INFINITY;
    if (!GREEDY && known) {
        u = uniform(a.uniforms[rows.x + t]);
        lx = logit((const T *)a.x + (rows.x + of) * a.x_row + tok);
        if (drafted) ly = logit((const T *)a.y + (rows.x + of) * a.y_row + tok);
    }
    for (int i = t >> 6; i < n; i += kWaves) {
        const Stat p = row_stat<GREEDY>(ws.p + ((size_t)s * a.max_rows + i) * pieces, pieces, kp);
        if ((t & 63) == 0) lds.p[i] = p;
        if (!GREEDY && drafted && i < n - 1) {
            const Stat q = row_stat<GREEDY>(ws.q + ((size_t)s * a.max_rows + i) * pieces, pieces, kq);
            if ((t & 63) == 0) lds.q[i] = q;
        }
    }
    __syncthreads();
    if (t < 64) {
        bool accept = false;
        const Stat p = lds.p[of];
        double prob = 0.0;
        if constexpr (GREEDY) {
            accept = known && tok == p.best;
        } else {
            const bool fine = known && p.s > 0.0;  // (not NaN)
            if (fine) prob = weight(lx, p.m, kp) / p.s;
            if (drafted) {
                const Stat q = lds.q[of];
                if (fine && q.s > 0.0) accept = u * (weight(ly, q.m, kq) / q.s) < prob;
            } else {
                double left = 1.0;
                bool again = false;  // an elder sibling is the same token
                if (a.row_mask != nullptr)
                    for (int j = 1; j < n; ++j) {
                        const int pj = __builtin_amdgcn_readlane(parent, j), tj = __builtin_amdgcn_readlane(tok, j);
                        const bool aj = __builtin_amdgcn_readlane((int)again, j);
                        const double bj = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(prob), j), __builtin_amdgcn_readlane(__double2loint(prob), j));
                        if (t > j && parent == pj && pj >= 0) {
                            again |= tok == tj;
                            if (!aj) left -= bj;
                        }
                    }
                accept = !again && known && u * (left > 0.0 ? left : 0.0) < prob;
            }
        }
        // from node to node by the first child that is accepted
        int cur = 0;
        uint64_t on = 1;
        while (true) {
            const uint64_t next = __ballot(accept && parent == cur);
            if (!next) break;
            cur = __builtin_ctzll(next);
            on |= 1ull << cur;
        }
        if (in && writes) {  // entry j of the path is the j-th node on it
            const int taken = __popcll(on);
            if (on >> t & 1) a.path[rows.x + __popcll(on & ((1ull << t) - 1))] = t;
            if (t >= taken) a.path[rows.x + t] = -1;
        }
        const bool child = !GREEDY && !drafted && parent == cur && known;
        const uint64_t children = __ballot(child);
        if (child) {
            const int i = __popcll(children & ((1ull << t) - 1));
            lds.gone[i] = tok;
            lds.gone_weight[i] = weight(lx, p.m, kp);
        }
        if (t == 0) {
            const Stat pl = lds.p[cur];
            Stat ql{};
            if (drafted && cur < n - 1) ql = lds.q[cur];
            lds.n_gone = __popcll(children);
            lds.draw = Draw{pl, ql, rows.x + cur, !(pl.s > 0.0) ? DRAW_NONE : (ql.s > 0.0 ? DRAW_REST : DRAW_P)};
            if (writes) {
                a.accepted[s] = __popcll(on) - 1;
                if (GREEDY) a.next[s] = pl.best;
            }
        }
    }
    __syncthreads();
}

// The pieces' masses of the row, relative to its largest logit.
__device__ __forceinline__ void masses_of(const Stat *row, int pieces, float m, double k, PickLds &lds) {
    for (int c = threadIdx.x; c < pieces; c += kThreads) lds.mass[c] = row[c].s == 0.0 ? 0.0 : row[c].s * weight(row[c].m, m, k);
}

// One workgroup a stream of tokens picked outright: the walk and the draw.
template <class T, int EPT, bool GREEDY>
__global__ __launch_bounds__(kThreads) void walk_kernel(VerifyArgs a, int pieces) {
    __shared__ PickLds lds;
    __shared__ WalkLds wl;
    const int s = blockIdx.x, t = threadIdx.x;
    const int2 rows = nodes_of(a, s);
    if (rows.y == 0) {
        if (t == 0) {
            a.accepted[s] = 0;
            a.next[s] = -1;
        }
        return;
    }
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, pieces, false, a.ws);
    walk<T, GREEDY>(a, s, rows, ws, pieces, true, wl);
    if constexpr (!GREEDY) {
        if (wl.draw.mode == DRAW_NONE) {
            if (t == 0) a.next[s] = -1;
            return;
        }
        constexpr int PIECE = EPT * 64, N = PIECE / kThreads;
        const Weights<T> w(a, wl.draw);
        const Stat *row = ws.p + ((size_t)s * a.max_rows + (wl.draw.row - rows.x)) * pieces;
        const int n_gone = wl.n_gone;
        const double u = uniform(a.uniforms[rows.x]);
        auto drop = [&](int first, double(&v)[N]) {
            for (int i = 0; i < n_gone; ++i) {
                const unsigned d = (unsigned)(wl.gone[i] - first);
                if (d < (unsigned)N)
#pragma unroll
                    for (int j = 0; j < N; ++j) v[j] = (int)d == j ? 0.0 : v[j];
            }
        };
        masses_of(row, pieces, wl.draw.p.m, w.kp, lds);
        __syncthreads();
        if (n_gone > 0) {
            // The rejected tokens' weights come off their pieces' sums, each token once.  Where less than 2^-12 is left, the
            // difference would be coarser than 2^-40 of it, and the piece is summed again.
            for (int c = t; c < pieces; c += kThreads) {
                const double all = lds.mass[c];
                double off = 0.0;
                for (int i = 0; i < n_gone; ++i) {
                    if (wl.gone[i] / PIECE != c) continue;
                    bool seen = false;
                    for (int j = 0; j < i; ++j) seen |= wl.gone[j] == wl.gone[i];
                    if (!seen) off += wl.gone_weight[i];
                }
                if (off > 0.0) lds.mass[c] = all - off >= all * 0x1p-12 ? all - off : -1.0;
            }
            __syncthreads();
            for (int i = 0; i < n_gone; ++i) {
                const int c = wl.gone[i] / PIECE;
                if (!(lds.mass[c] < 0.0)) continue;  // (of the whole workgroup)
                double v[N], sum = 0.0, all;
                w.template of<N>(c * PIECE + t * N, a.vocab, v);
                drop(c * PIECE + t * N, v);
#pragma unroll
                for (int j = 0; j < N; ++j) sum += v[j];
                scan64(sum, lds.scan, all);
                if (t == 0) lds.mass[c] = all;
                __syncthreads();
            }
        }
        int got = pick<T, EPT>(w, a.vocab, pieces, u, lds, drop);
        if (got < 0) {  // nothing is left: p itself
            __syncthreads();
            masses_of(row, pieces, wl.draw.p.m, w.kp, lds);
            __syncthreads();
            got = pick<T, EPT>(w, a.vocab, pieces, u, lds, KeepAll());
        }
        if (t == 0) a.next[s] = got;
    }
}

// Chains with the draft's logits: every workgroup of a stream walks; where a token is rejected, each wave has the mass of
// (p - q)+ in one piece of the row in front of it.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void walk_draft_kernel(VerifyArgs a, int pieces, int parts) {
    __shared__ WalkLds wl;
    const int s = blockIdx.x / parts, part = blockIdx.x - s * parts, t = threadIdx.x;
    const int2 rows = nodes_of(a, s);
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, pieces, true, a.ws);
    if (rows.y == 0) {
        if (t == 0 && part == 0) {
            a.accepted[s] = 0;
            ws.draw[s].mode = DRAW_NONE;
        }
        return;
    }
    walk<T, false>(a, s, rows, ws, pieces, part == 0, wl);
    if (t == 0 && part == 0) ws.draw[s] = wl.draw;
    const int c = part * kWaves + (t >> 6);
    if (wl.draw.mode != DRAW_REST || c >= pieces) return;
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    const Weights<T> w(a, wl.draw);
    double sum = 0.0;
#pragma unroll 2
    for (int i = 0; i < EPT / V; ++i) {
        double v[V];
        w.template of<V>(c * EPT * 64 + (i * 64 + (t & 63)) * V, a.vocab, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += v[j];
    }
    sum = wave_sum64(sum);
    if ((t & 63) == 0) ws.mass[(size_t)s * pieces + c] = sum;
}

// Their draw.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void draw_kernel(VerifyArgs a, int pieces) {
    __shared__ PickLds lds;
    const int s = blockIdx.x, t = threadIdx.x;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, pieces, true, a.ws);
    const Draw d = ws.draw[s];
    if (d.mode == DRAW_NONE) {
        if (t == 0) a.next[s] = -1;
        return;
    }
    const int2 rows = nodes_of(a, s);
    const double u = uniform(a.uniforms[rows.x]);
    Weights<T> w(a, d);
    int got = -1;
    if (w.rest) {
        for (int c = t; c < pieces; c += kThreads) lds.mass[c] = ws.mass[(size_t)s * pieces + c];
        __syncthreads();
        got = pick<T, EPT>(w, a.vocab, pieces, u, lds, KeepAll());
        __syncthreads();
    }
    if (got < 0) {  // all were accepted, or nothing is left over: from p itself
        w.rest = false;
        masses_of(ws.p + ((size_t)s * a.max_rows + (d.row - rows.x)) * pieces, pieces, d.p.m, w.kp, lds);
        __syncthreads();
        got = pick<T, EPT>(w, a.vocab, pieces, u, lds, KeepAll());
    }
    if (t == 0) a.next[s] = got;
}

// Values of a lane of a piece: few while that fills the chip, many where the pieces' sums would be much work themselves.
int ept_of(int rows, int vocab) {
    const int small = (vocab + 255) / 256;
    if (small <= 64 && (long long)rows * small <= 4096) return 4;
    return vocab <= 64 * 1024 ? 16 : 32;
}
int pieces_of(int rows, int vocab) {
    const int n = ept_of(rows, vocab) * 64;
    return (vocab + n - 1) / n;
}
static_assert(kMaxPieces * 32 * 64 >= kVocabMax, "a row's pieces");

template <class T, int EPT>
hipError_t verify_e(const VerifyArgs &a, hipStream_t s) {
    const int pieces = pieces_of(a.streams * a.max_rows, a.vocab);
    const dim3 grid((unsigned)(((long long)a.streams * a.max_rows * pieces + kWaves - 1) / kWaves), a.y != nullptr ? 2 : 1);
    (void)hipGetLastError();
    if (a.greedy) {
        hipLaunchKernelGGL((stat_kernel<T, EPT, true>), grid, dim3(kThreads), 0, s, a, pieces);
        hipLaunchKernelGGL((walk_kernel<T, EPT, true>), dim3(a.streams), dim3(kThreads), 0, s, a, pieces);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((stat_kernel<T, EPT, false>), grid, dim3(kThreads), 0, s, a, pieces);
    if (a.y != nullptr) {
        const int parts = (pieces + kWaves - 1) / kWaves;
        hipLaunchKernelGGL((walk_draft_kernel<T, EPT>), dim3((unsigned)a.streams * parts), dim3(kThreads), 0, s, a, pieces, parts);
        hipLaunchKernelGGL((draw_kernel<T, EPT>), dim3(a.streams), dim3(kThreads), 0, s, a, pieces);
    } else {
        hipLaunchKernelGGL((walk_kernel<T, EPT, false>), dim3(a.streams), dim3(kThreads), 0, s, a, pieces);
    }
    return hipGetLastError();
}

template <class T>
hipError_t verify_t(const VerifyArgs &a, hipStream_t s) {
    switch (ept_of(a.streams * a.max_rows, a.vocab)) {
        case 4: return verify_e<T, 4>(a, s);
        case 16: return verify_e<T, 16>(a, s);
        default: return verify_e<T, 32>(a, s);
    }
}

}  // namespace

size_t verify_workspace(int streams, int max_rows, int vocab, bool draft) {
    const VerifyWs w = verify_ws(streams, max_rows, pieces_of(streams * max_rows, vocab), draft, nullptr);
    return (size_t)(uintptr_t)(w.draw + (draft ? streams : 0));
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) { return a.dtype == ELEM_F16 ? verify_t<__half>(a, s) : verify_t<float>(a, s); }

}  // namespace mh
