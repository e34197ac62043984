// logprobs.hip -- log probabilities of given tokens, the entropy and the top alternatives of rows of
// logits (gfx950).
//
// Of a row: with m = max x, z = (x - m) / T, S = sum e^z and U = sum e^z z,
//   log p(t) = z_t - log S,     entropy = -sum p log p = log S - U / S,
// the differences first, so that a row of the type's lowest value does not leave its range when it is scaled, and as half
// of themselves (z / 2 = (x / 2 - m / 2) / T, exact but for subnormal x), so that those of the type's two ends do not either;
// and the k largest x, of equal values the lowest index first.  One pass: a workgroup takes a
// chunk of a row into registers, so memory is read once; m, S, U and the alternatives all come
// from there.  A row of more than one chunk leaves (m, S, U) and its k best per chunk in the
// workspace, and a second, small launch joins them in chunk order (fixed, no atomics).
//
// The k best of a chunk: each wave sorts its 64 lanes' maxima (21 exchange steps).  At least k values
// reach the k-th of a wave's, and at least k reach the least of the four waves' (k / 4)-th, so only
// values at or above the larger of those are candidates -- in practice a few more than k of
// thousands.  A candidate's rank is the number of better ones.
//
// 16 rows of 1024 with 5 alternatives 5.0 us; 181 of 16384 with 20 12.2 us, of which the sums alone take 5.8 (2.0 TB/s) and
// the rest is the chain of sort, marks, second reads and ranks; 3 fp16 rows of 130001 with 8 6.1 and 4.8 of the join.
// Few rows are a chain of dependent steps, not memory.
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

// v of the 64 lanes in descending order: a bitonic sort.  Step M of runs of RUN: the lower lane of a pair keeps
// the larger value where its run descends; which lanes those are is a constant.
__host__ __device__ constexpr uint64_t keep_larger(int run, int m) {
    uint64_t mask = 0;
    for (int l = 0; l < 64; ++l) mask |= (uint64_t)(((l & m) == 0) == ((l & run) == 0)) << l;
    return mask;
}
template <int RUN, int M>
__device__ __forceinline__ uint32_t exchange(uint32_t v) {
    constexpr uint64_t mask = keep_larger(RUN, M);
    const uint32_t o = (uint32_t)xshfl<M>((int)v);
    return __builtin_amdgcn_inverse_ballot_w64(mask) ? max(v, o) : min(v, o);
}
template <int RUN, int M = RUN / 2>
__device__ __forceinline__ uint32_t merge_runs(uint32_t v) {
    v = exchange<RUN, M>(v);
    if constexpr (M > 1) v = merge_runs<RUN, M / 2>(v);
    return v;
}
__device__ __forceinline__ uint32_t sort64(uint32_t v) {
    return merge_runs<64>(merge_runs<32>(merge_runs<16>(merge_runs<8>(merge_runs<4>(merge_runs<2>(v))))));
}

// Candidates one wave can have: values above the k-th lane maximum lie in at most k - 1 lanes, and
// equal ones are taken only until k of them are held, one step of V * 64 at a time.
template <int EPT, int V>
constexpr int cand_max() {
    return (kTopMax - 1) * EPT + kTopMax + 64 * V;
}

constexpr int kFastCand = 512;  // candidates that are all taken
template <int CAP>
struct TopLds {
    static_assert(kWaves * CAP >= kFastCand, "room for them");
    uint2 cand[kWaves * CAP];  // key, position, in any order
    int n;                     // how many (cleared in the first half)
    uint32_t kth[kWaves], quarter[kWaves];
};

// First half: the waves' sorted maxima, `best` being the lane's (a barrier must follow).
template <int CAP>
__device__ __forceinline__ void top_floor(float best, int k, TopLds<CAP> &lds) {
    const uint32_t sorted = sort64(key_of(best));
    const int w = threadIdx.x >> 6;
    if (threadIdx.x == 0) lds.n = 0;
    // read before the branch: inside it the other lanes' last exchange need not have happened
    const uint32_t kth = __builtin_amdgcn_readlane(sorted, k - 1);
    const uint32_t quarter = __builtin_amdgcn_readlane(sorted, (k + kWaves - 1) / (kWaves) - 1);
    if ((threadIdx.x & 63) == 0) {
        lds.kth[w] = kth;
        lds.quarter[w] = quarter;
    }
}

// The k best of the workgroup's values x[i], element i of thread t at position
// ((i / V) * kThreads + t) * V + i % V: put(rank, key, position) is called once for each rank
// that exists.  What reaches the floor is marked with a bit each, and read once more by position, again(position),
// by loops of few instructions: taken out of the registers where they are found, in straight code of EPT branches
// whose instructions are fetched for the first time, 20 of 16384 took 11 us of 16.
template <int EPT, int V, int CAP, class Again, class Put>
__device__ __forceinline__ int top_of(const float (&x)[EPT], int k, TopLds<CAP> &lds, Again &&again, Put &&put) {
    const int t = threadIdx.x, lane = t & 63;
    uint32_t floor_key = 0, least = 0xffffffffu;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        floor_key = max(floor_key, lds.kth[v]);
        least = min(least, lds.quarter[v]);
    }
    floor_key = max(floor_key, least);
    const float floor = floor_key == 0 ? -3.40282347e38f : of_key(floor_key);  // comparisons leave NaN out, and -inf below
    uint64_t bits = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) bits |= x[i] >= floor ? 1ull << i : 0;
    auto place = [&](int i) { return ((i / V) * kThreads + t) * V + i % V; };
    int at = 0;
    if (bits) at = atomicAdd(&lds.n, __popcll(bits));
    __syncthreads();
    int total = lds.n;
    if (total <= kFastCand) {
        while (bits) {
            const int p = place(__builtin_ctzll(bits));
            bits &= bits - 1;
            lds.cand[at++] = make_uint2(key_of(again(p)), p);
        }
    } else {  // hundreds at the floor itself: each wave's first k of those will do, in the order of their positions
        __syncthreads();
        if (t == 0) lds.n = 0;
        __syncthreads();
        int equal = 0;  // of the wave
        const uint64_t below = (1ull << lane) - 1;
#pragma unroll 1
        for (int i0 = 0; i0 < EPT; i0 += V) {
            const bool more = floor_key != 0 && equal < k;
#pragma unroll 1
            for (int i = i0; i < i0 + V; ++i) {
                const bool has = (bits >> i) & 1;
                if (!__any(has)) continue;
                const uint32_t key = has ? key_of(again(place(i))) : 0;
                const bool eq = has && key == floor_key && more, take = key > floor_key || eq;
                const uint64_t who = __ballot(take);
                int to = 0;
                if (lane == 0) to = atomicAdd(&lds.n, __popcll(who));
                to = __builtin_amdgcn_readfirstlane(to);
                if (take) lds.cand[to + __popcll(who & below)] = make_uint2(key, place(i));
                equal += __popcll(__ballot(eq));
            }
        }
        __syncthreads();
        total = lds.n;
    }
    __syncthreads();
    for (int c = t; c < total; c += kThreads) {
        const uint2 me = lds.cand[c];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < total; ++j) {
            const uint2 o = lds.cand[j];
            rank += o.x > me.x || (o.x == me.x && o.y < me.y);
        }
        if (rank < k) put(rank, me.x, (int)me.y);
    }
    return total;
}

struct Sums {
    float m, s, u;
};

__device__ __forceinline__ float half_diff(float x, float m) { return fmaf(x, 0.5f, -0.5f * m); }

// m, S and U of a chunk, and the first half of its k best; -inf contributes nothing, NaN and +inf make the
// sums NaN.
template <int EPT, int CAP>
__device__ __forceinline__ Sums sums_of(const float (&x)[EPT], float inv_t, int k, float (*red)[kWaves], TopLds<CAP> &lds) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) best = fmaxf(best, x[i]);
    float m = wave_max(best);
    if (lane == 0) red[0][w] = m;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) m = fmaxf(m, red[0][v]);
    const float m0 = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const float z = half_diff(x[i], m0) * inv_t;
        const float e = __builtin_amdgcn_exp2f(z * (2.0f * 1.44269504088896341f));
        s += e;
        u += e == 0.0f ? 0.0f : e * z;
    }
    s = wave_sum(s);
    u = wave_sum(u);
    if (lane == 0) {
        red[1][w] = s;
        red[2][w] = u;
    }
    if (k > 0) top_floor(best, k, lds);
    __syncthreads();
    Sums q{m, 0.0f, 0.0f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
        q.s += red[1][v];
        q.u += red[2][v];
    }
    q.u *= 2.0f;
    return q;
}

template <class T>
__device__ __forceinline__ float logit(const T *p) {
    if constexpr (sizeof(T) == 2)
        return __half2float(*(const __half *)p);
    else
        return *p;
}

// The logit of a row's token, asked for early; NaN for a token outside the vocabulary.
template <class T>
__device__ __forceinline__ float token_logit(const LogprobArgs &a, int r) {
    const int tok = a.tokens[r];
    return tok >= 0 && tok < a.vocab ? logit((const T *)a.x + r * a.row + tok) : __uint_as_float(0x7fc00000u);
}
// What a row's sums give: the token's log probability and the entropy (one thread), and the log
// probability of an alternative.
__device__ __forceinline__ void finish_row(const LogprobArgs &a, int r, float x, const Sums &q) {
    const float log_s = logf(q.s);
    a.logprob[r] = q.s == 0.0f && x == x ? -INFINITY : 2.0f * (half_diff(x, q.m) * a.inv_t) - log_s;  // (sum 0: no token is allowed at all)
    if (a.entropy != nullptr) a.entropy[r] = q.s == 0.0f ? 0.0f : log_s - q.u / q.s;
}
__device__ __forceinline__ float alt_lp(const LogprobArgs &a, const Sums &q, uint32_t key) {
    return 2.0f * (half_diff(of_key(key), q.m) * a.inv_t) - logf(q.s);
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
    float token = 0.0f;
    if (chunks == 1 && t == 0) token = token_logit<T>(a, r);
    float x[EPT];
#pragma unroll
    for (int i = 0; i < EPT; i += V) {
        const int e = base + i * kThreads + t * V;
        if (e + V <= a.vocab) {
            T raw[V];  // (16 bytes at any address that a logit may have: the hardware takes them unaligned)
            uint32_t w[V * sizeof(T) / 4];
            __builtin_memcpy(w, p + e, sizeof(w));
            __builtin_memcpy(raw, w, sizeof(w));
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = logit(raw + j);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = e + j < a.vocab ? logit(p + e + j) : -INFINITY;
        }
    }
    const Sums q = sums_of(x, a.inv_t, a.top_k, red, lds);
    if (chunks == 1) {
        if (t == 0) finish_row(a, r, token, q);
        if (a.top_k > 0) {
            const int n = top_of<EPT, V>(x, a.top_k, lds, [&](int at) { return logit(p + base + at); }, [&](int rank, uint32_t key, int at) {
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
        const int n = top_of<EPT, V>(x, a.top_k, lds, [&](int at) { return logit(p + base + at); }, [&](int rank, uint32_t key, int at) {
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
    float token = 0.0f;
    if (t == 0) token = token_logit<T>(a, r);
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
        const float d = 2.0f * (half_diff(part[i].x, q.m) * a.inv_t), f = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
        q.s += f * part[i].y;
        q.u += f == 0.0f ? 0.0f : f * (part[i].z + part[i].y * d);
    }
    q.s = wave_sum(q.s);
    q.u = wave_sum(q.u);
    if (t == 0) finish_row(a, r, token, q);
    if (a.top_k == 0) return;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; ++i) most = fmaxf(most, x[i]);
    top_floor(most, a.top_k, lds);
    __syncthreads();
    const int got = top_of<EPT, 1>(x, a.top_k, lds, [&](int at) { return best[at]; }, [&](int rank, uint32_t key, int at) {
        a.top_ids[(size_t)r * a.top_k + rank] = ((const int *)best)[n + at];
        a.top_lp[(size_t)r * a.top_k + rank] = alt_lp(a, q, key);
    });
    no_alternatives(a, r, got);
}

// Values a thread holds.  Up to 16384 logits a row is one chunk: one launch and no join.  A longer one is cut finely
// while there are few, so that they fill the chip (3 rows of 130001: 10.6 us, in chunks of 8192 11.9).
int ept_of(int rows, int vocab) {
    for (int ept = 4; ept <= 64; ept *= 2)
        if (vocab <= ept * kThreads) return ept;
    const int chunks8 = (vocab + 8 * kThreads - 1) / (8 * kThreads);
    return chunks8 <= kMaxChunks && (long long)rows * chunks8 <= 1024 ? 8 : 32;
}
int chunks_of(int rows, int vocab) {
    const int n = ept_of(rows, vocab) * kThreads;
    return (vocab + n - 1) / n;
}

template <class T, int EPT>
void launch_chunks(const LogprobArgs &a, int chunks, hipStream_t s) {
    constexpr int V = std::min<int>(16 / (int)sizeof(T), EPT);
    hipLaunchKernelGGL((logprobs_kernel<T, EPT, V>), dim3((unsigned)a.rows * chunks), dim3(kThreads), 0, s, a, chunks);
}

template <class T>
hipError_t logprobs_t(const LogprobArgs &a, hipStream_t s) {
    const int chunks = chunks_of(a.rows, a.vocab);
    (void)hipGetLastError();
    switch (ept_of(a.rows, a.vocab)) {
        case 4: launch_chunks<T, 4>(a, chunks, s); break;
        case 8: launch_chunks<T, 8>(a, chunks, s); break;
        case 16: launch_chunks<T, 16>(a, chunks, s); break;
        case 32: launch_chunks<T, 32>(a, chunks, s); break;
        default: launch_chunks<T, 64>(a, chunks, s); break;
    }
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
