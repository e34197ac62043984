// verify.hip -- drafted tokens against the target's probabilities, from given random numbers (gfx950).
//
// p = softmax(x / T) after each node, q the draft's.  A chain whose tokens were drawn from q accepts node i
// where u_i q(t_i) < p(t_i), and draws the token behind the first one that it rejects from (p - q)+.  Tokens
// that were picked outright are point masses: of a node's children, in order, c is accepted where
// u_c (1 - the rejected ones' p) < p(t_c), and the token behind them is drawn from p without them.  Both leave the
// target's own distribution.  A draw with u is the first token whose cumulative sum passes u times the whole.
//
// A draw compares u with as many borders as the vocabulary has tokens, and sums of 32 bits move each by up to
// 2^-24: one draw in a hundred over 2^17 tokens.  So probabilities are formed and summed in 64 bits; that is about
// 20 instructions a logit, near what reading one takes.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxChunks = 128;  // of a row
constexpr double kLog2e = 1.4426950408889634074;

// Of a chunk of a row, or of a row: the largest logit, where it is first, and sum of e^{(x - m) / T}.  Nothing
// above -inf: s is 0; a NaN or +inf among them: s is NaN.
struct Stat {
    float m;
    int best;  // -1: none
    double s;
};

// 2^x for x <= 0, or NaN: the series of 2^f, |f| <= 1/2, to f^12 (2^-52 of the result).
__device__ __forceinline__ double exp2_64(double x) {
    x = x < -1100.0 ? -1100.0 : x;
    const double n = rint(x), f = (x - n) * 0.69314718055994530942;
    double y = 1.0 / 479001600;
    y = fma(y, f, 1.0 / 39916800);
    y = fma(y, f, 1.0 / 3628800);
    y = fma(y, f, 1.0 / 362880);
    y = fma(y, f, 1.0 / 40320);
    y = fma(y, f, 1.0 / 5040);
    y = fma(y, f, 1.0 / 720);
    y = fma(y, f, 1.0 / 120);
    y = fma(y, f, 1.0 / 24);
    y = fma(y, f, 1.0 / 6);
    y = fma(y, f, 0.5);
    y = fma(y, f, 1.0);
    y = fma(y, f, 1.0);
    return ldexp(y, (int)n);
}
// e^{(x - m) / T}, k = log2(e) / T
__device__ __forceinline__ double weight(float x, float m, double k) { return exp2_64(((double)x - (double)m) * k); }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}

template <class T>
__device__ __forceinline__ float logit(const T *p) {
    if constexpr (sizeof(T) == 2)
        return __half2float(*(const __half *)p);
    else
        return *p;
}

// The workspace: statistics [streams][max_rows][chunks] of the target, then of the draft; then of draws from
// (p - q)+ the mass of each chunk [streams][chunks], and [streams] what is drawn from.
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
__host__ __device__ __forceinline__ VerifyWs verify_ws(int streams, int max_rows, int chunks, bool draft, void *ws) {
    VerifyWs w;
    const size_t n = (size_t)streams * max_rows * chunks;
    w.p = (Stat *)ws;
    w.q = w.p + n;
    w.mass = (double *)(w.q + (draft ? n : 0));
    w.draw = (Draw *)(w.mass + (size_t)streams * chunks);
    return w;
}

// Rows of stream s: first and how many take part.
__device__ __forceinline__ int2 nodes_of(const VerifyArgs &a, int s) {
    const int r0 = a.row_start[s], r1 = a.row_start[s + 1];
    return r0 >= 0 && r1 >= r0 && r1 <= a.rows ? make_int2(r0, min(r1 - r0, a.max_rows)) : make_int2(0, 0);
}

// One chunk of one row of the target (y: 0) or the draft (1); EPT values a thread, read V at a time.
template <class T, int EPT, int V, bool GREEDY>
__global__ __launch_bounds__(kThreads) void stat_kernel(VerifyArgs a, int chunks) {
    __shared__ float lm[kWaves];
    __shared__ int li[kWaves];
    __shared__ double ls[kWaves];
    const int at = blockIdx.x / chunks, c = blockIdx.x - at * chunks;
    const int s = at / a.max_rows, node = at - s * a.max_rows;
    const bool of_draft = blockIdx.y == 1;
    const int2 rows = nodes_of(a, s);
    if (node >= rows.y - of_draft) return;  // (nothing was drawn behind the last row)
    const T *p = of_draft ? (const T *)a.y + (rows.x + node) * a.y_row : (const T *)a.x + (rows.x + node) * a.x_row;
    const int base = c * EPT * kThreads, t = threadIdx.x, w = t >> 6;
    float x[EPT];
#pragma unroll
    for (int i = 0; i < EPT; i += V) {
        const int e = base + i * kThreads + t * V;
        if (e + V <= a.vocab) {
            T raw[V];  // (16 bytes at any address that a logit may have)
            uint32_t u[V * sizeof(T) / 4];
            __builtin_memcpy(u, p + e, sizeof(u));
            __builtin_memcpy(raw, u, sizeof(u));
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = logit(raw + j);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = e + j < a.vocab ? logit(p + e + j) : -INFINITY;
        }
    }
    float m = -INFINITY;
    int best = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
        if (x[i] > m) {
            m = x[i];
            best = base + (i / V) * V * kThreads + t * V + i % V;
        }
    if constexpr (GREEDY) {
        wave_argmax(m, best);
    } else {
        m = wave_max(m);
    }
    if ((t & 63) == 0) {
        lm[w] = m;
        li[w] = best;
    }
    __syncthreads();
    for (int v = 0; v < kWaves; ++v)
        if (lm[v] > m || (lm[v] == m && li[v] < best)) {
            m = lm[v];
            best = li[v];
        }
    double sum = 0.0;
    if constexpr (!GREEDY) {
        const double k = (double)(of_draft ? a.draft_inv_t : a.inv_t) * kLog2e;
        const float m0 = m == -INFINITY ? 0.0f : m;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            bad |= !(x[i] < INFINITY);
            sum += weight(x[i], m0, k);
        }
        sum = wave_sum64(bad ? __builtin_nan("") : sum);
        if ((t & 63) == 0) ls[w] = sum;
        __syncthreads();
        sum = 0.0;
        for (int v = 0; v < kWaves; ++v) sum += ls[v];
    }
    if (t == 0) {
        const VerifyWs ws = verify_ws(a.streams, a.max_rows, chunks, a.y != nullptr, a.ws);
        (of_draft ? ws.q : ws.p)[(size_t)at * chunks + c] = Stat{m, m > -INFINITY ? best : -1, sum};
    }
}

// The chunks of a row together.
__device__ __forceinline__ Stat row_stat(const Stat *c, int chunks, double k) {
    Stat r{-INFINITY, -1, 0.0};
    for (int i = 0; i < chunks; ++i) {
        const Stat o = c[i];
        if (o.m > r.m) {  // (the first of equal ones stays)
            r.m = o.m;
            r.best = o.best;
        }
    }
    const float m0 = r.m == -INFINITY ? 0.0f : r.m;
    for (int i = 0; i < chunks; ++i) {
        const Stat o = c[i];
        r.s += o.s == 0.0 ? 0.0 : o.s * weight(o.m, m0, k);
    }
    return r;
}
__device__ __forceinline__ bool fine(const Stat &s) { return s.s > 0.0; }  // (not of NaN)

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
    for (int i = 0; i < kWaves; ++i) {
        if (i < w) before += lds[i];
        all += lds[i];
    }
    return before + v;
}

struct PickLds {
    double mass[kMaxChunks];
    double scan[kWaves];
    uint32_t gone[32 * kThreads / 32];  // a bit per token of one chunk: rejected
    int found, last;
};

// What token e of the row weighs, up to a factor of the row.
template <class T>
struct Weights {
    const T *x, *y;
    Stat p, q;
    double kp, kq;
    bool rest;  // (p - q)+
    __device__ __forceinline__ double of(int e) const {
        const double wp = weight(logit(x + e), p.m, kp);
        if (!rest) return wp;
        const double d = wp / p.s - weight(logit(y + e), q.m, kq) / q.s;
        return d > 0.0 ? d : 0.0;
    }
};

// The token drawn with u: lds.mass holds the chunks' masses.  `rejected` says of a token whether it is left out.
template <class T, int EPT, class Gone>
__device__ int pick(const Weights<T> &w, int vocab, int chunks, double u, PickLds &lds, Gone &&gone) {
    const int t = threadIdx.x;
    double all = 0.0;
    for (int c = 0; c < chunks; ++c) all += lds.mass[c];
    if (!(all > 0.0)) return -1;
    const double aim = u * all;
    double before = 0.0;
    int at = -1;
    for (int c = 0; c < chunks; ++c) {  // the first that passes it; where rounding lets none, the last with any mass
        if (!(lds.mass[c] > 0.0)) continue;
        if (at >= 0) before += lds.mass[at];
        at = c;
        if (before + lds.mass[c] > aim) break;
    }
    const int first = at * EPT * kThreads + t * EPT;  // neighbouring tokens of a thread
    double sum = 0.0;
    for (int i = 0; i < EPT; ++i)
        if (first + i < vocab && !gone(first + i)) sum += w.of(first + i);
    double total;
    double run = before + scan64(sum, lds.scan, total) - sum;
    if (t == 0) {
        lds.found = 0x7fffffff;
        lds.last = -1;
    }
    __syncthreads();
    int found = -1, last = -1;
    if (sum > 0.0)
        for (int i = 0; i < EPT; ++i) {
            if (first + i >= vocab || gone(first + i)) continue;
            const double v = w.of(first + i);
            run += v;
            if (v > 0.0) last = first + i;
            if (v > 0.0 && run > aim && found < 0) found = first + i;
        }
    if (found >= 0) atomicMin(&lds.found, found);
    if (last >= 0) atomicMax(&lds.last, last);
    __syncthreads();
    return lds.found < vocab ? lds.found : lds.last;
}

__device__ __forceinline__ double uniform(double u) { return u < 1.0 ? (u > 0.0 ? u : 0.0) : 1.0; }  // (NaN: 1)

// One workgroup a stream: the walk, by its first wave, a lane a node; and, but for draws from (p - q)+, the draw.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void walk_kernel(VerifyArgs a, int chunks) {
    __shared__ PickLds lds;
    __shared__ Draw draw;
    __shared__ int gone[kTreeMax], n_gone;
    const int s = blockIdx.x, t = threadIdx.x;
    const int2 rows = nodes_of(a, s);
    const int n = rows.y;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, chunks, a.y != nullptr, a.ws);
    const bool drafted = a.y != nullptr;
    const double kp = (double)a.inv_t * kLog2e, kq = (double)a.draft_inv_t * kLog2e;
    if (n == 0) {
        if (t == 0) {
            a.accepted[s] = 0;
            a.next[s] = -1;
            if (drafted) ws.draw[s].mode = DRAW_NONE;
        }
        return;
    }
    if (t < 64) {
        const bool in = t < n;
        Stat p{-INFINITY, -1, 0.0}, q = p;
        if (in) p = row_stat(ws.p + ((size_t)s * a.max_rows + t) * chunks, chunks, kp);
        if (drafted && t < n - 1) q = row_stat(ws.q + ((size_t)s * a.max_rows + t) * chunks, chunks, kq);
        int parent = t - 1;
        if (in && a.row_mask != nullptr) {
            const uint64_t mask = a.row_mask[rows.x + t], up = mask & ((1ull << t) - 1);
            parent = (mask >> t & 1) && up ? 63 - __builtin_clzll(up) : -1;
        }
        if (!in || t == 0) parent = -1;
        const int of = max(parent, 0);
        const int tok = in ? a.tokens[rows.x + t] : -1;
        const bool known = tok >= 0 && tok < a.vocab && parent >= 0;
        const double u = in && a.uniforms != nullptr ? uniform(a.uniforms[rows.x + t]) : 0.0;
        bool accept = false;
        if (a.greedy) {
            const int best = __shfl(p.best, of);  // (by all lanes: a parent need not have a token itself)
            accept = known && tok == best;
        } else {
            const float pm = __shfl(p.m, of), qm = __shfl(q.m, of);
            const double psum = __shfl(p.s, of), qsum = __shfl(q.s, of);
            const bool p_fine = psum > 0.0;
            double prob = 0.0;
            if (known && p_fine) prob = weight(logit((const T *)a.x + (rows.x + of) * a.x_row + tok), pm, kp) / psum;
            if (drafted) {
                if (known && p_fine && qsum > 0.0)
                    accept = u * (weight(logit((const T *)a.y + (rows.x + of) * a.y_row + tok), qm, kq) / qsum) < prob;
            } else {
                double left = 1.0;
                bool again = false;  // an elder sibling is the same token
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
        if (in) {  // entry j of the path is the j-th node on it
            const int taken = __popcll(on);
            if (on >> t & 1) a.path[rows.x + __popcll(on & ((1ull << t) - 1))] = t;
            if (t >= taken) a.path[rows.x + t] = -1;
        }
        const int best = __shfl(p.best, cur);
        const Stat pl{__shfl(p.m, cur), 0, __shfl(p.s, cur)}, ql{__shfl(q.m, cur), 0, __shfl(q.s, cur)};
        const bool child = parent == cur && known && !drafted;
        const uint64_t children = __ballot(child);
        if (child) gone[__popcll(children & ((1ull << t) - 1))] = tok;
        if (t == 0) {
            n_gone = __popcll(children);
            a.accepted[s] = __popcll(on) - 1;
            if (a.greedy) a.next[s] = best;
            draw.p = pl;
            draw.q = ql;
            draw.row = rows.x + cur;
            draw.mode = !fine(pl) ? DRAW_NONE : (drafted && cur < n - 1 && fine(ql) ? DRAW_REST : DRAW_P);
            if (drafted) ws.draw[s] = draw;
        }
    }
    if (a.greedy || drafted) return;
    __syncthreads();
    if (draw.mode == DRAW_NONE) {
        if (t == 0) a.next[s] = -1;
        return;
    }
    const T *x = (const T *)a.x + draw.row * a.x_row;
    const Weights<T> w{x, nullptr, draw.p, draw.q, kp, kq, false};
    const Stat *row = ws.p + ((size_t)s * a.max_rows + (draw.row - rows.x)) * chunks;
    auto masses = [&] {
        __syncthreads();
        for (int c = t; c < chunks; c += kThreads) lds.mass[c] = row[c].s == 0.0 ? 0.0 : row[c].s * weight(row[c].m, draw.p.m, kp);
        __syncthreads();
    };
    auto bits_of = [&](int c) {  // those of chunk c that were rejected
        for (int i = t; i < EPT * kThreads / 32; i += kThreads) lds.gone[i] = 0;
        __syncthreads();
        if (t < n_gone && gone[t] / (EPT * kThreads) == c) {
            const int b = gone[t] - c * EPT * kThreads;
            atomicOr(&lds.gone[b / 32], 1u << (b % 32));
        }
        __syncthreads();
    };
    auto is_gone = [&](int e) {
        const int b = e % (EPT * kThreads);
        return (lds.gone[b / 32] >> (b % 32) & 1) != 0;
    };
    masses();
    // chunks that lose tokens are summed again (a difference of sums would lose what little is left)
    for (int i = 0; i < n_gone; ++i) {
        const int c = gone[i] / (EPT * kThreads);
        bool seen = false;
        for (int j = 0; j < i; ++j) seen |= gone[j] / (EPT * kThreads) == c;
        if (seen) continue;
        bits_of(c);
        double sum = 0.0, all;
        for (int e = c * EPT * kThreads + t; e < min(a.vocab, (c + 1) * EPT * kThreads); e += kThreads)
            if (!is_gone(e)) sum += w.of(e);
        scan64(sum, lds.scan, all);
        if (t == 0) lds.mass[c] = all;
        __syncthreads();
    }
    double all = 0.0;
    for (int c = 0; c < chunks; ++c) all += lds.mass[c];
    const double u = uniform(a.uniforms[rows.x]);
    int got;
    if (all > 0.0) {
        // the chunk's bits depend on which chunk the draw falls into: all rejected tokens are looked up there
        got = pick<T, EPT>(w, a.vocab, chunks, u, lds, [&](int e) {
            for (int i = 0; i < n_gone; ++i)
                if (gone[i] == e) return true;
            return false;
        });
    } else {
        masses();
        got = pick<T, EPT>(w, a.vocab, chunks, u, lds, [](int) { return false; });
    }
    if (t == 0) a.next[s] = got;
}

// The mass of (p - q)+ in one chunk of the row behind a rejected token.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void rest_kernel(VerifyArgs a, int chunks) {
    __shared__ double lds[kWaves];
    const int s = blockIdx.x / chunks, c = blockIdx.x - s * chunks;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, chunks, true, a.ws);
    const Draw d = ws.draw[s];
    if (d.mode != DRAW_REST) return;
    const Weights<T> w{(const T *)a.x + d.row * a.x_row, (const T *)a.y + d.row * a.y_row, d.p, d.q, (double)a.inv_t * kLog2e,
                       (double)a.draft_inv_t * kLog2e, true};
    double sum = 0.0, all;
    for (int e = c * EPT * kThreads + (int)threadIdx.x; e < min(a.vocab, (c + 1) * EPT * kThreads); e += kThreads) sum += w.of(e);
    scan64(sum, lds, all);
    if (threadIdx.x == 0) ws.mass[(size_t)s * chunks + c] = all;
}

// The draw of a chain with the draft's logits.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void draw_kernel(VerifyArgs a, int chunks) {
    __shared__ PickLds lds;
    const int s = blockIdx.x, t = threadIdx.x;
    const VerifyWs ws = verify_ws(a.streams, a.max_rows, chunks, true, a.ws);
    const Draw d = ws.draw[s];
    if (d.mode == DRAW_NONE) {
        if (t == 0) a.next[s] = -1;
        return;
    }
    const int2 rows = nodes_of(a, s);
    const double kp = (double)a.inv_t * kLog2e, u = uniform(a.uniforms[rows.x]);
    Weights<T> w{(const T *)a.x + d.row * a.x_row, (const T *)a.y + d.row * a.y_row, d.p, d.q, kp, (double)a.draft_inv_t * kLog2e,
                 d.mode == DRAW_REST};
    int got = -1;
    if (w.rest) {
        for (int c = t; c < chunks; c += kThreads) lds.mass[c] = ws.mass[(size_t)s * chunks + c];
        __syncthreads();
        got = pick<T, EPT>(w, a.vocab, chunks, u, lds, [](int) { return false; });
        __syncthreads();
    }
    if (got < 0) {  // nothing was left over: from p itself
        w.rest = false;
        const Stat *row = ws.p + ((size_t)s * a.max_rows + (d.row - rows.x)) * chunks;
        for (int c = t; c < chunks; c += kThreads) lds.mass[c] = row[c].s == 0.0 ? 0.0 : row[c].s * weight(row[c].m, d.p.m, kp);
        __syncthreads();
        got = pick<T, EPT>(w, a.vocab, chunks, u, lds, [](int) { return false; });
    }
    if (t == 0) a.next[s] = got;
}

// Values of a thread of a chunk: few while that fills the chip.
int ept_of(int rows, int vocab) {
    for (const int ept : {4, 16}) {
        const int chunks = (vocab + ept * kThreads - 1) / (ept * kThreads);
        if (chunks <= (ept == 4 ? 16 : 32) && (chunks == 1 || (long long)rows * chunks <= 2048)) return ept;
    }
    return 32;
}
int chunks_of(int rows, int vocab) {
    const int n = ept_of(rows, vocab) * kThreads;
    return (vocab + n - 1) / n;
}
static_assert(kMaxChunks * 32 * kThreads >= kVocabMax, "a row's chunks");

template <class T, int EPT>
hipError_t verify_e(const VerifyArgs &a, hipStream_t s) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    const int chunks = chunks_of(a.streams * a.max_rows, a.vocab);
    const dim3 grid((unsigned)a.streams * a.max_rows * chunks, a.y != nullptr ? 2 : 1);
    (void)hipGetLastError();
    if (a.greedy)
        hipLaunchKernelGGL((stat_kernel<T, EPT, V, true>), grid, dim3(kThreads), 0, s, a, chunks);
    else
        hipLaunchKernelGGL((stat_kernel<T, EPT, V, false>), grid, dim3(kThreads), 0, s, a, chunks);
    hipLaunchKernelGGL((walk_kernel<T, EPT>), dim3(a.streams), dim3(kThreads), 0, s, a, chunks);
    if (a.y != nullptr && !a.greedy) {
        hipLaunchKernelGGL((rest_kernel<T, EPT>), dim3((unsigned)a.streams * chunks), dim3(kThreads), 0, s, a, chunks);
        hipLaunchKernelGGL((draw_kernel<T, EPT>), dim3(a.streams), dim3(kThreads), 0, s, a, chunks);
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
    const VerifyWs w = verify_ws(streams, max_rows, chunks_of(streams * max_rows, vocab), draft, nullptr);
    return (size_t)(uintptr_t)(w.draw + streams);
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) { return a.dtype == ELEM_F16 ? verify_t<__half>(a, s) : verify_t<float>(a, s); }

}  // namespace mh
