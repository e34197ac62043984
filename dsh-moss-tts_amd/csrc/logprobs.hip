// logprobs.hip -- log probabilities of given tokens, the entropy and the top alternatives of rows of
// logits (gfx950).
//
// Of a row z = x / T: with m = max z, S = sum e^(z - m) and U = sum e^(z - m) (z - m),
//   log p(t) = z_t - m - log S,     entropy = -sum p log p = log S - U / S,
// and the k largest x, of equal values the lowest index first.  One pass: a workgroup takes a
// chunk of a row into registers, so memory is read once; m, S, U and the alternatives all come
// from there.  A row of more than one chunk leaves (m, S, U) and its k best per chunk in the
// workspace, and a second, small launch joins them in chunk order (fixed, no atomics).
//
// The k best of a chunk: each wave sorts its 64 lanes' maxima (21 exchange steps).  At least k values
// reach the k-th of a wave's, and at least k reach the least of the four waves' (k / 4)-th, so only
// values at or above the larger of those are candidates -- in practice a few more than k of
// thousands.  A candidate's rank is the number of better ones.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxChunks = 128;  // of a row: with 32 alternatives each, 16 values a thread of the join
static_assert(kMaxChunks * kTopMax <= 16 * kThreads && kMaxChunks * 32 * kThreads >= kVocabMax, "the join holds all chunks' best");

// A row in the workspace: (m, S, U, -) of each chunk, then the chunks' k values each, then their indices; whole
// 16-byte pieces.
__host__ __device__ constexpr size_t row_words(int chunks, int k) { return ((size_t)chunks * (4 + 2 * k) + 3) / 4 * 4; }

// fp32 as an unsigned integer of the same order; -0 counts as +0, and -inf and NaN as 0, below all
// others: neither is an alternative.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ ((b & 0x80000000u) ? 0xffffffffu : 0x80000000u);
    return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }

// v of the 64 lanes in descending order
template <int M>
__device__ __forceinline__ uint32_t exchange(uint32_t v, bool descending) {
    const uint32_t o = (uint32_t)xshfl<M>((int)v);
    const bool low = (__lane_id() & M) == 0;
    return low == descending ? max(v, o) : min(v, o);
}
__device__ __forceinline__ uint32_t sort64(uint32_t v) {
    const int l = __lane_id();
    v = exchange<1>(v, (l & 2) == 0);
    v = exchange<2>(v, (l & 4) == 0);
    v = exchange<1>(v, (l & 4) == 0);
    v = exchange<4>(v, (l & 8) == 0);
    v = exchange<2>(v, (l & 8) == 0);
    v = exchange<1>(v, (l & 8) == 0);
    v = exchange<8>(v, (l & 16) == 0);
    v = exchange<4>(v, (l & 16) == 0);
    v = exchange<2>(v, (l & 16) == 0);
    v = exchange<1>(v, (l & 16) == 0);
    v = exchange<16>(v, (l & 32) == 0);
    v = exchange<8>(v, (l & 32) == 0);
    v = exchange<4>(v, (l & 32) == 0);
    v = exchange<2>(v, (l & 32) == 0);
    v = exchange<1>(v, (l & 32) == 0);
    v = exchange<32>(v, true);
    v = exchange<16>(v, true);
    v = exchange<8>(v, true);
    v = exchange<4>(v, true);
    v = exchange<2>(v, true);
    v = exchange<1>(v, true);
    return v;
}

// Candidates one wave can have: values above the k-th lane maximum lie in at most k - 1 lanes, and
// equal ones are taken only until k of them are held, one step of V * 64 at a time.
template <int EPT, int V>
constexpr int cand_max() {
    return (kTopMax - 1) * EPT + kTopMax + 64 * V;
}

template <int CAP>
struct TopLds {
    uint2 cand[kWaves][CAP];  // key, position
    int n[kWaves];
    uint32_t kth[kWaves], quarter[kWaves];
};

// First half: the waves' sorted maxima (a barrier must follow).
template <int EPT, int CAP>
__device__ __forceinline__ void top_floor(const float (&x)[EPT], int k, TopLds<CAP> &lds) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) best = max(best, key_of(x[i]));
    const uint32_t sorted = sort64(best);
    const int w = threadIdx.x >> 6;
    // read before the branch: inside it the other lanes' last exchange need not have happened
    const uint32_t kth = __builtin_amdgcn_readlane(sorted, k - 1);
    const uint32_t quarter = __builtin_amdgcn_readlane(sorted, (k + kWaves - 1) / kWaves - 1);
    if ((threadIdx.x & 63) == 0) {
        lds.kth[w] = kth;
        lds.quarter[w] = quarter;
    }
}

// The k best of the workgroup's values x[i], element i of thread t at position
// ((i / V) * kThreads + t) * V + i % V: put(rank, key, position) is called once for each rank
// that exists.
template <int EPT, int V, int CAP, class Put>
__device__ __forceinline__ int top_of(const float (&x)[EPT], int k, TopLds<CAP> &lds, Put &&put) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const uint32_t least = min(min(lds.quarter[0], lds.quarter[1]), min(lds.quarter[2], lds.quarter[3]));
    const uint32_t floor_key = max(least, max(max(lds.kth[0], lds.kth[1]), max(lds.kth[2], lds.kth[3])));
    int n = 0, equal = 0;  // of the wave
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i0 = 0; i0 < EPT; i0 += V) {
        const bool more = equal < k;
#pragma unroll
        for (int i = i0; i < i0 + V; ++i) {
            const uint32_t key = key_of(x[i]);
            const bool eq = key == floor_key && key != 0 && more;
            const bool take = key > floor_key || eq;
            const uint64_t who = __ballot(take);
            if (who == 0) continue;
            if (take) lds.cand[w][n + __popcll(who & below)] = make_uint2(key, ((i / V) * kThreads + t) * V + i % V);
            n += __popcll(who);
            equal += __popcll(__ballot(eq));
        }
    }
    if (lane == 0) lds.n[w] = n;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) total += lds.n[v];
    for (int c = lane; c < n; c += 64) {
        const uint2 me = lds.cand[w][c];
        int rank = 0;
        for (int v = 0; v < kWaves; ++v) {
            const int nv = lds.n[v];
#pragma unroll 4
            for (int j = 0; j < nv; ++j) {
                const uint2 o = lds.cand[v][j];
                rank += o.x > me.x || (o.x == me.x && o.y < me.y);
            }
        }
        if (rank < k) put(rank, me.x, (int)me.y);
    }
    return total;
}

struct Sums {
    float m, s, u;
};

// m, S and U of a chunk, and the first half of its k best; -inf contributes nothing, NaN and +inf make the
// sums NaN.
template <int EPT, int CAP>
__device__ __forceinline__ Sums sums_of(const float (&x)[EPT], float inv_t, int k, float (*red)[kWaves], TopLds<CAP> &lds) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) m = fmaxf(m, x[i] * inv_t);
    m = wave_max(m);
    if (lane == 0) red[0][w] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float m0 = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const float z = x[i] * inv_t - m0;
        const float e = __builtin_amdgcn_exp2f(z * 1.44269504088896341f);
        s += e;
        u += e == 0.0f ? 0.0f : e * z;
    }
    s = wave_sum(s);
    u = wave_sum(u);
    if (lane == 0) {
        red[1][w] = s;
        red[2][w] = u;
    }
    if (k > 0) top_floor(x, k, lds);
    __syncthreads();
    return Sums{m, (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]), (red[2][0] + red[2][1]) + (red[2][2] + red[2][3])};
}

template <class T>
__device__ __forceinline__ float logit(const T *p) {
    if constexpr (sizeof(T) == 2)
        return __half2float(*(const __half *)p);
    else
        return *p;
}

// What a row's sums give: the token's log probability and the entropy (thread 0), and the log
// probability of an alternative.
template <class T>
__device__ __forceinline__ void finish_row(const LogprobArgs &a, int r, const Sums &q) {
    const float log_s = logf(q.s);
    const int tok = a.tokens[r];
    float lp = __uint_as_float(0x7fc00000u);
    if (tok >= 0 && tok < a.vocab) {
        const float z = logit((const T *)a.x + r * a.row + tok) * a.inv_t;
        lp = q.s == 0.0f ? -INFINITY : z - q.m - log_s;  // no token is allowed at all
    }
    a.logprob[r] = lp;
    if (a.entropy != nullptr) a.entropy[r] = q.s == 0.0f ? 0.0f : log_s - q.u / q.s;
}
__device__ __forceinline__ float alt_lp(const LogprobArgs &a, const Sums &q, uint32_t key) {
    return of_key(key) * a.inv_t - q.m - logf(q.s);
}
__device__ __forceinline__ void no_alternatives(const LogprobArgs &a, int r, int from) {
    for (int i = from + (int)threadIdx.x; i < a.top_k; i += kThreads) {
        a.top_ids[(size_t)r * a.top_k + i] = -1;
        a.top_lp[(size_t)r * a.top_k + i] = -INFINITY;
    }
}

// One chunk of one row: EPT values a thread, read V at a time.
template <class T, int EPT, int V>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobArgs a, int chunks) {
    __shared__ float red[3][kWaves];
    __shared__ TopLds<cand_max<EPT, V>()> lds;
    const int r = blockIdx.x / chunks, c = blockIdx.x - r * chunks, t = threadIdx.x;
    const int base = c * EPT * kThreads;
    const T *p = (const T *)a.x + r * a.row;
    float x[EPT];
#pragma unroll
    for (int i = 0; i < EPT; i += V) {
        const int e = base + (i * kThreads) + t * V;
        if (V > 1 && e + V <= a.vocab) {
            uint4 raw = *(const uint4 *)(p + e);
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = logit((const T *)&raw + j);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = e + j < a.vocab ? logit(p + e + j) : -INFINITY;
        }
    }
    const Sums q = sums_of(x, a.inv_t, a.top_k, red, lds);
    if (chunks == 1) {
        if (t == 0) finish_row<T>(a, r, q);
        if (a.top_k > 0) {
            const int n = top_of<EPT, V>(x, a.top_k, lds, [&](int rank, uint32_t key, int at) {
                a.top_ids[(size_t)r * a.top_k + rank] = at;
                a.top_lp[(size_t)r * a.top_k + rank] = alt_lp(a, q, key);
            });
            no_alternatives(a, r, n);
        }
        return;
    }
    float *row = (float *)a.ws + r * row_words(chunks, a.top_k);
    if (t == 0) *(float4 *)(row + 4 * c) = make_float4(q.m, q.s, q.u, 0.0f);
    if (a.top_k > 0) {
        float *o = row + 4 * chunks + c * a.top_k;
        const int n = top_of<EPT, V>(x, a.top_k, lds, [&](int rank, uint32_t key, int at) {
            o[rank] = of_key(key);
            ((int *)o)[chunks * a.top_k + rank] = base + at;
        });
        for (int i = n + t; i < a.top_k; i += kThreads) o[i] = -INFINITY;
    }
}

// The chunks of one row joined; EPT values a thread hold all chunks' best.
template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobArgs a, int chunks) {
    __shared__ TopLds<cand_max<EPT, 1>()> lds;
    const int r = blockIdx.x, t = threadIdx.x, n = chunks * a.top_k;
    const float *w = (const float *)a.ws + r * row_words(chunks, a.top_k), *best = w + 4 * chunks;
    // position c * k + j: equal values of a lower index come first, as chunks and ranks do
    float x[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) x[i] = i * kThreads + t < n ? best[i * kThreads + t] : -INFINITY;
    Sums q{-INFINITY, 0.0f, 0.0f};
    float4 part[2];  // every wave joins all chunks, at most 128
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = (t & 63) + 64 * i;
        part[i] = c < chunks ? *(const float4 *)(w + 4 * c) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        q.m = fmaxf(q.m, part[i].x);
    }
    q.m = wave_max(q.m);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (part[i].x == -INFINITY && part[i].y == 0.0f) continue;  // nothing allowed in this chunk
        const float d = part[i].x - q.m, f = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
        q.s += f * part[i].y;
        q.u += f == 0.0f ? 0.0f : f * (part[i].z + part[i].y * d);
    }
    q.s = wave_sum(q.s);
    q.u = wave_sum(q.u);
    if (t == 0) finish_row<T>(a, r, q);
    if (a.top_k == 0) return;
    top_floor(x, a.top_k, lds);
    __syncthreads();
    const int got = top_of<EPT, 1>(x, a.top_k, lds, [&](int rank, uint32_t key, int at) {
        a.top_ids[(size_t)r * a.top_k + rank] = ((const int *)best)[n + at];
        a.top_lp[(size_t)r * a.top_k + rank] = alt_lp(a, q, key);
    });
    no_alternatives(a, r, got);
}

// Values a thread holds.
int ept_of(int rows, int vocab) {
    if (vocab <= 4 * kThreads) return 4;
    const int chunks8 = (vocab + 8 * kThreads - 1) / (8 * kThreads);
    return chunks8 <= kMaxChunks && (long long)rows * chunks8 <= 4096 ? 8 : 32;
}
int chunks_of(int rows, int vocab) {
    const int n = ept_of(rows, vocab) * kThreads;
    return (vocab + n - 1) / n;
}

template <class T, int EPT>
void launch_chunks(const LogprobArgs &a, int chunks, hipStream_t s) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    const dim3 grid((unsigned)a.rows * chunks);
    if (V * sizeof(T) == 16 && (uintptr_t)a.x % 16 == 0 && a.row % V == 0)
        hipLaunchKernelGGL((logprobs_kernel<T, EPT, V>), grid, dim3(kThreads), 0, s, a, chunks);
    else
        hipLaunchKernelGGL((logprobs_kernel<T, EPT, 1>), grid, dim3(kThreads), 0, s, a, chunks);
}

template <class T>
hipError_t logprobs_t(const LogprobArgs &a, hipStream_t s) {
    const int chunks = chunks_of(a.rows, a.vocab), ept = ept_of(a.rows, a.vocab);
    (void)hipGetLastError();
    if (ept == 4)
        launch_chunks<T, 4>(a, chunks, s);
    else if (ept == 8)
        launch_chunks<T, 8>(a, chunks, s);
    else
        launch_chunks<T, 32>(a, chunks, s);
    if (chunks > 1 && chunks * a.top_k <= 2 * kThreads)
        hipLaunchKernelGGL((logprobs_join_kernel<T, 2>), dim3(a.rows), dim3(kThreads), 0, s, a, chunks);
    else if (chunks > 1)
        hipLaunchKernelGGL((logprobs_join_kernel<T, 16>), dim3(a.rows), dim3(kThreads), 0, s, a, chunks);
    return hipGetLastError();
}

}  // namespace

size_t logprobs_workspace(int rows, int vocab, int top_k) {
    const int chunks = chunks_of(rows, vocab);
    return chunks == 1 ? 0 : rows * row_words(chunks, top_k) * sizeof(float);
}

hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s) {
    return a.dtype == ELEM_F16 ? logprobs_t<__half>(a, s) : logprobs_t<float>(a, s);
}

}  // namespace mh
