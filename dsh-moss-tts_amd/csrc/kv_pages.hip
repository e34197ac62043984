// kv_pages.hip -- the pages of a paged K/V cache: streams that share them, room for new rows, and
// accepted rows moved to their final positions (gfx950).
//
// A page is held by the table entries that name it, and refs[page] counts those (and whatever holds the
// caller adds); a page with 0 is free.  Everything is decided on the device, by rules whose outcome does
// not depend on the order in which workgroups run: sums of counts, and prefix sums in the order of streams.
// What a table or a list names outside its range is never followed.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256;
constexpr int kBookThreads = 1024;  // of the workgroup that keeps the books

// ---------------------------------------------------------------- fork

// Entry (s, j) afterwards: the parent's, where it lies within the length.
__device__ __forceinline__ int forked(const ForkArgs &a, int s, int j) {
    const int p = a.parent[s];
    if (p < 0 || p >= a.p.streams) return -1;
    if (a.len != nullptr && (long long)j * a.p.page_size >= a.len[s]) return -1;
    const int e = a.p.table[(size_t)p * a.p.table_stride + j];
    return e >= 0 && e < a.p.n_pages ? e : -1;
}
__device__ __forceinline__ void count_change(const PagesArgs &p, int from, int to) {
    if (from == to) return;
    if (from >= 0 && from < p.n_pages) atomicAdd(p.refs + from, -1);
    if (to >= 0) atomicAdd(p.refs + to, 1);
}

// Tables of up to N * 1024 entries: one workgroup holds all of them, so the old ones are read before
// the first new one is written.
template <int N>
__global__ __launch_bounds__(kBookThreads) void fork_kernel(ForkArgs a) {
    const int n = a.p.streams * a.p.table_stride;
    int from[N], to[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = i * kBookThreads + (int)threadIdx.x;
        if (e >= n) break;
        const int s = e / a.p.table_stride;
        from[i] = a.p.table[e];
        to[i] = forked(a, s, e - s * a.p.table_stride);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = i * kBookThreads + (int)threadIdx.x;
        if (e >= n) break;
        if (from[i] != to[i]) a.p.table[e] = to[i];
        count_change(a.p, from[i], to[i]);
    }
}

// Larger ones by two launches, the new table in the workspace between them.
__global__ __launch_bounds__(kThreads) void fork_read_kernel(ForkArgs a, long long n) {
    const long long e = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (e >= n) return;
    const int s = (int)(e / a.p.table_stride);
    const int to = forked(a, s, (int)(e - (long long)s * a.p.table_stride));
    a.ws[e] = to;
    count_change(a.p, a.p.table[e], to);
}
__global__ __launch_bounds__(kThreads) void fork_write_kernel(ForkArgs a, long long n) {
    const long long e = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (e < n) a.p.table[e] = a.ws[e];
}

constexpr int kForkEntries = 16;  // of a thread of the one workgroup

// ---------------------------------------------------------------- reserve

// Pages j0 .. j1 are those that stream s writes (none where j1 < j0); ok: its rows have places at all.
struct Range {
    int j0, j1;
    bool ok;
};
__device__ __forceinline__ Range range_of(const ReserveArgs &a, int s) {
    const long long n = (long long)a.row_start[s + 1] - a.row_start[s], ctx = a.ctx_len[s];
    Range r{0, -1, ctx >= 0 && n >= 0 && n <= a.max_rows && ctx + n <= (long long)a.p.table_stride * a.p.page_size};
    if (r.ok && n > 0) {
        r.j0 = (int)(ctx / a.p.page_size);
        r.j1 = (int)((ctx + n - 1) / a.p.page_size);
    }
    return r;
}

// What becomes of an entry: it is missing, it is shared and gets a page of its own, it stays, or (from 0 on) it
// stays if every earlier holder, up to that stream, takes another page.
enum { MISSING = -3, SHARED = -2, STAYS = -1 };

// Streams are served one after the other: an earlier stream of this call that writes the same page has
// given it up by then, so the last of a page's holders keeps it.  By one wave, its lanes an earlier stream each.
__device__ __forceinline__ int fate_of(const ReserveArgs &a, int s, int j) {
    const int e = a.p.table[(size_t)s * a.p.table_stride + j];
    if (e < 0 || e >= a.p.n_pages) return MISSING;
    const int held = a.p.refs[e];
    if (held <= 1) return STAYS;
    int earlier = 0, last = 0;
    for (int o0 = 0; o0 < s; o0 += 64) {
        const int o = o0 + ((int)threadIdx.x & 63);
        bool same = false;
        if (o < s) {
            const int theirs = a.p.table[(size_t)o * a.p.table_stride + j];  // (asked for together with the range)
            const Range r = range_of(a, o);
            same = j >= r.j0 && j <= r.j1 && theirs == e;
        }
        const uint64_t who = __ballot(same);
        earlier += __popcll(who);
        if (who) last = o0 + 63 - __builtin_clzll(who);
    }
    return held - earlier > 1 ? SHARED : last;
}

// Pages that one stream's rows can touch: those that max_rows positions can lie on, and no more than a stream has.
int pages_of(const PagesArgs &p, int max_rows) { return (int)std::min<long long>(((long long)max_rows + p.page_size - 2) / p.page_size + 1, p.table_stride); }

__global__ __launch_bounds__(kThreads) void fate_kernel(ReserveArgs a, int n, int per) {
    for (int e = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)); e < n; e += gridDim.x * (kThreads / 64)) {
        const int s = e / per, r = e - s * per;
        const Range g = range_of(a, s);
        const int f = g.j0 + r <= g.j1 ? fate_of(a, s, g.j0 + r) : STAYS;
        if ((threadIdx.x & 63) == 0) a.fate[e] = f;
    }
}

// Sum over the workgroup's earlier threads, and over all of them.
__device__ __forceinline__ int2 block_scan(int v, int *lds) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
    }
    __syncthreads();
    if (lane == 63) lds[w] = sum;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < kBookThreads / 64; ++i) {
        if (i < w) before += lds[i];
        all += lds[i];
    }
    return make_int2(before + sum - v, all);
}

// The lowest free pages, as many as are wanted, into `list`: how many there are.  A barrier has to follow.
__device__ __forceinline__ int lowest_free(const PagesArgs &p, int wanted, int *list, int *lds) {
    const int t = threadIdx.x;
    int found = 0;
    for (int p0 = 0; p0 < p.n_pages && found < wanted; p0 += 4 * kBookThreads) {
        bool is[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int page = p0 + 4 * t + i;
            is[i] = page < p.n_pages && p.refs[page] == 0;
            n += is[i];
        }
        const int2 at = block_scan(n, lds);
        int k = found + at.x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (is[i]) {
                if (k < wanted) list[k] = p0 + 4 * t + i;
                ++k;
            }
        found += at.y;
    }
    return found;
}

// An entry's new page.
__device__ __forceinline__ int4 take_page(const ReserveArgs &a, int s, int j, int j0, int fate, int page) {
    int *entry = a.p.table + (size_t)s * a.p.table_stride + j;
    int4 copy = make_int4(0, 0, 0, 0);
    if (fate == SHARED) {
        const int old = *entry;
        atomicAdd(a.p.refs + old, -1);
        if (j == j0) copy = make_int4(old, page, a.ctx_len[s] - j * a.p.page_size, 0);
    }
    a.p.refs[page] = 1;
    *entry = page;
    return copy;
}

// The books of one call of up to 1024 entries (streams times the pages that one of them can touch), by one workgroup, a thread
// an entry: a chain of a few dependent loads.
__global__ __launch_bounds__(kBookThreads) void reserve_small_kernel(ReserveArgs a, int per) {
    __shared__ int lds[kBookThreads / 64], unserved, free_pages[kBookThreads], bad[kBookThreads];
    __shared__ int2 entries[kBookThreads];  // page, place in the table
    const int t = threadIdx.x, s = t / per, r = t - s * per;
    const bool in = s < a.p.streams;
    Range g{0, -1, false};
    if (in) g = range_of(a, s);
    const int j = g.j0 + r;
    int e = -1, held = 0;
    if (j <= g.j1) e = a.p.table[(size_t)s * a.p.table_stride + j];
    if (e < 0 || e >= a.p.n_pages) e = -1;
    if (e >= 0) held = a.p.refs[e];
    entries[t] = make_int2(e, j);
    bad[t] = 0;
    if (t == 0) unserved = a.p.streams;
    __syncthreads();
    int fate = STAYS;
    if (j <= g.j1 && e < 0) fate = MISSING;
    if (held > 1) {
        int earlier = 0, last = 0;
        for (int o = 0; o < s * per; ++o)
            if (entries[o].x == e && entries[o].y == j) {
                ++earlier;
                last = o;
            }
        fate = held - earlier > 1 ? SHARED : last / per;
    }
    const bool need = fate <= SHARED;
    const int2 at = block_scan(need, lds);
    const int found = lowest_free(a.p, at.y, free_pages, lds);
    if (need && at.x >= found) atomicMin(&unserved, s);
    __syncthreads();
    if (in && (!g.ok || fate >= unserved || (need && s >= unserved))) bad[s] = 1;
    __syncthreads();
    if (!in) return;
    const bool ok = !bad[s];
    int4 copy = make_int4(0, 0, 0, 0);
    if (ok && need) copy = take_page(a, s, j, g.j0, fate, free_pages[at.x]);
    if (r == 0) {
        a.ok[s] = ok;
        a.copies[s] = copy;
    }
}

// The same for more entries: what becomes of them is in the workspace, a thread a stream.
__global__ __launch_bounds__(kBookThreads) void reserve_kernel(ReserveArgs a, int per) {
    __shared__ int lds[kBookThreads / 64], unserved;
    const int t = threadIdx.x;
    if (t == 0) unserved = a.p.streams;
    // how many pages are wanted
    int mine = 0;
    for (long long e = t; e < (long long)a.p.streams * per; e += kBookThreads) mine += a.fate[e] <= SHARED;
    const int wanted = block_scan(mine, lds).y;
    const int found = lowest_free(a.p, wanted, a.free_pages, lds);
    __syncthreads();  // (the list is read by other threads of this workgroup)
    // Streams in their order: those before the first that finds too few are served.
    int given = 0;
    for (int s0 = 0; s0 < a.p.streams; s0 += kBookThreads) {
        const int s = s0 + t;
        int need = 0, left = -1;
        if (s < a.p.streams)
            for (int r = 0; r < per; ++r) {
                const int f = a.fate[(size_t)s * per + r];
                need += f <= SHARED;
                left = max(left, f);
            }
        const int2 at = block_scan(need, lds);
        if (need > 0 && given + at.x + need > found) atomicMin(&unserved, s);
        __syncthreads();
        if (s < a.p.streams) {
            const Range g = range_of(a, s);
            const bool ok = g.ok && left < unserved && (need == 0 || s < unserved);
            int4 copy = make_int4(0, 0, 0, 0);
            if (ok && need > 0) {
                int k = given + at.x;
                for (int j = g.j0; j <= g.j1; ++j) {
                    const int f = a.fate[(size_t)s * per + (j - g.j0)];
                    if (f > SHARED) continue;
                    const int4 c = take_page(a, s, j, g.j0, f, a.free_pages[k++]);
                    if (c.z > 0) copy = c;
                }
            }
            a.ok[s] = ok;
            a.copies[s] = copy;
        }
        given += at.y;
    }
}

// The first `slots` positions of one head of a page in one of the layers' K's and V's.  Memory bound: 32 streams' copies of half a
// page of 32 layers x 8 heads x 128 int8, 69 MB, 31 us (4.4 TB/s), a load of a thread at a time.  Where nothing is copied the workgroups
// still start: 32768 at 64 streams of 32 layers x 8 heads, 8.5 us.  A workgroup of all heads, whose pieces then lie at steps of a power
// of two, took 50.
template <bool SCALES>
__global__ __launch_bounds__(kThreads) void copy_kernel(ReserveArgs a, KvLayers l) {
    // Neighbouring workgroups, which go to the 8 XCDs in turn, have one stream's pools: streams differ in what there is to do, and
    // 64 of them side by side left some XCDs with nothing (50 us).
    const int s = blockIdx.x / (2 * a.layers), pool = blockIdx.x - s * 2 * a.layers, layer = pool >> 1;
    const int4 c = a.copies[s];
    if (c.z <= 0) return;
    const bool is_v = pool & 1;
    const size_t from = ((size_t)c.x * a.heads + blockIdx.y) * a.p.page_size, to = ((size_t)c.y * a.heads + blockIdx.y) * a.p.page_size;
    char *data = (char *)(is_v ? l.v[layer] : l.k[layer]);
    const uint4 *x = (const uint4 *)(data + from * a.vec_bytes);
    uint4 *y = (uint4 *)(data + to * a.vec_bytes);
    const int units = c.z * a.vec_bytes / 16;
#pragma unroll 4
    for (int u = threadIdx.x; u < units; u += kThreads) y[u] = x[u];
    if constexpr (SCALES) {
        float *scale = is_v ? l.v_scale[layer] : l.k_scale[layer];
        for (int u = threadIdx.x; u < c.z; u += kThreads) scale[to + u] = scale[from + u];
    }
}

// ---------------------------------------------------------------- compact

constexpr int kMovesPerThread = 8;  // 16-byte pieces, all of which are loaded before the first is stored

// One workgroup: the rows of one stream in pools_each of the layers' K's and V's, heads_each heads.  The list of moves is made
// once; then, pool by pool and a group of heads at a time, all rows of a head are in registers before the first is
// stored, so any row may take any other's place.  64 streams, 12 rows each of 32 layers x 8 heads x 128 bytes and scales: 36 us,
// 2.3 TB/s in pieces of 128 bytes whose heads lie at steps of a power of two.  The pieces lie in scratch memory (144 bytes a lane), so a
// thread has one load in flight at a time.
template <bool SCALES>
__global__ __launch_bounds__(kThreads) void compact_kernel(CompactArgs a, KvLayers l, int pools_each, int heads_each) {
    __shared__ size_t from[kTreeMax], to[kTreeMax];  // vectors of head 0
    __shared__ int moves;
    const int of_stream = (2 * a.layers + pools_each - 1) / pools_each;  // (neighbours have one stream's pools, as above)
    const int s = blockIdx.x / of_stream, first_pool = (blockIdx.x - s * of_stream) * pools_each, t = threadIdx.x;
    if (t < 64) {
        const int r0 = a.row_start[s], r1 = a.row_start[s + 1], ctx = a.ctx_len[s];
        bool move = false;
        size_t src = 0, dst = 0;
        if (r0 >= 0 && r1 >= r0 && r1 <= a.rows && ctx >= 0 && t < min(r1 - r0, a.max_rows)) {  // (no difference leaves 32 bits)
            const int k = a.kept[r0 + t];
            if (k >= 0 && k < r1 - r0 && k != t) {
                const unsigned ps = (unsigned)ctx + k, pd = (unsigned)ctx + t;  // (below 2^31 + 2^23)
                const unsigned js = ps / (unsigned)a.c.page_size, jd = pd / (unsigned)a.c.page_size;
                if (js < (unsigned)a.c.table_stride && jd < (unsigned)a.c.table_stride) {
                    const int *row = a.c.table + (size_t)s * a.c.table_stride;
                    const int pf = row[js], pt = row[jd];
                    move = pf >= 0 && pf < a.c.n_pages && pt >= 0 && pt < a.c.n_pages;
                    src = (size_t)pf * a.c.heads * a.c.page_size + (ps - js * a.c.page_size);
                    dst = (size_t)pt * a.c.heads * a.c.page_size + (pd - jd * a.c.page_size);
                }
            }
        }
        const uint64_t who = __ballot(move);
        if (move) {
            const int at = __popcll(who & ((1ull << t) - 1));
            from[at] = src;
            to[at] = dst;
        }
        if (t == 0) moves = __popcll(who);
    }
    __syncthreads();
    const int m = moves;
    if (m == 0) return;
    const int shift = __builtin_ctz(a.vec_bytes) - 4, per = 1 << shift, of_head = m << shift;  // 16-byte pieces
    const int first = blockIdx.y * heads_each, last = min(first + heads_each, a.c.heads);
    const int group = max(1, kMovesPerThread * kThreads / of_head);  // heads at a time
    for (int pool = first_pool; pool < min(first_pool + pools_each, 2 * a.layers); ++pool) {
        char *data = (char *)(pool & 1 ? l.v[pool >> 1] : l.k[pool >> 1]);
        float *scale = pool & 1 ? l.v_scale[pool >> 1] : l.k_scale[pool >> 1];
        for (int h0 = first; h0 < last; h0 += group) {
            const int units = min(group, last - h0) * of_head;
            uint4 x[kMovesPerThread];
            float d[kMovesPerThread];
            size_t at[kMovesPerThread];
#pragma unroll
            for (int i = 0; i < kMovesPerThread; ++i) {
                const int u = i * kThreads + t;
                if (u >= units) break;
                const int hr = u >> shift, h = hr / m, r = hr - h * m, e = u & (per - 1);
                const size_t head = (size_t)(unsigned)((h0 + h) * a.c.page_size);
                x[i] = *(const uint4 *)(data + (from[r] + head) * a.vec_bytes + 16 * e);
                if (SCALES && e == 0) d[i] = scale[from[r] + head];
                at[i] = to[r] + head;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kMovesPerThread; ++i) {
                const int u = i * kThreads + t;
                if (u >= units) break;
                const int e = u & (per - 1);
                *(uint4 *)(data + at[i] * a.vec_bytes + 16 * e) = x[i];
                if (SCALES && e == 0) scale[at[i]] = d[i];
            }
        }
    }
}

}  // namespace

size_t fork_workspace(const PagesArgs &p) {
    const size_t n = (size_t)p.streams * p.table_stride;
    return n <= kForkEntries * kBookThreads ? 0 : n * sizeof(int);
}

hipError_t launch_kv_fork(const ForkArgs &a, hipStream_t s) {
    const long long n = (long long)a.p.streams * a.p.table_stride;
    (void)hipGetLastError();
    if (n <= kBookThreads) {
        hipLaunchKernelGGL(fork_kernel<1>, dim3(1), dim3(kBookThreads), 0, s, a);
    } else if (n <= kForkEntries * kBookThreads) {
        hipLaunchKernelGGL(fork_kernel<kForkEntries>, dim3(1), dim3(kBookThreads), 0, s, a);
    } else {
        const unsigned blocks = (unsigned)((n + kThreads - 1) / kThreads);
        hipLaunchKernelGGL(fork_read_kernel, dim3(blocks), dim3(kThreads), 0, s, a, n);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;  // (what follows trusts what it leaves)
        hipLaunchKernelGGL(fork_write_kernel, dim3(blocks), dim3(kThreads), 0, s, a, n);
    }
    return hipGetLastError();
}

// The workspace: copies [streams] (from page, to page, slots); the lowest free pages, and what becomes of each entry
// [streams][pages of a stream].
size_t reserve_workspace(const PagesArgs &p, int max_rows) {
    const size_t n = (size_t)p.streams * pages_of(p, max_rows);
    return p.streams * sizeof(int4) + (n <= kBookThreads ? 0 : 2 * sizeof(int) * n);
}

hipError_t launch_kv_reserve(ReserveArgs a, const KvLayers &l, hipStream_t s) {
    const int per = pages_of(a.p, a.max_rows), n = a.p.streams * per;  // (within 2^26, as the table)
    a.copies = (int4 *)a.ws;
    a.free_pages = (int *)(a.copies + a.p.streams);
    a.fate = a.free_pages + n;
    (void)hipGetLastError();
    if (n <= kBookThreads) {
        hipLaunchKernelGGL(reserve_small_kernel, dim3(1), dim3(kBookThreads), 0, s, a, per);
    } else {
        // A wave an entry, of up to 2^26: those of 65536 workgroups take them in turn, as a grid holds fewer than 2^32 threads.
        hipLaunchKernelGGL(fate_kernel, dim3(std::min((n + 3) / 4, 1 << 16)), dim3(kThreads), 0, s, a, n, per);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;  // (what follows trusts what it leaves)
        hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kBookThreads), 0, s, a, per);
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const dim3 grid(a.p.streams * 2 * a.layers, a.heads);
    if (a.scales)
        hipLaunchKernelGGL(copy_kernel<true>, grid, dim3(kThreads), 0, s, a, l);
    else
        hipLaunchKernelGGL(copy_kernel<false>, grid, dim3(kThreads), 0, s, a, l);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const CompactArgs &a, const KvLayers &l, hipStream_t s) {
    (void)hipGetLastError();
    // As many heads as one pass takes, and two pools where that leaves 2048 workgroups (64 streams of 32 layers x 8 heads: 36 us, one pool
    // 42, twice the heads 42, half of them 39); fewer heads where streams are few.
    const int pools = 2 * a.layers;
    int heads_each = std::max(1, std::min(a.c.heads, kMovesPerThread * kThreads * 16 / (a.max_rows * a.vec_bytes)));
    auto parts = [&] { return (a.c.heads + heads_each - 1) / heads_each; };
    const int pools_each = (long long)a.c.streams * pools * parts() >= 4096 ? 2 : 1;
    while (heads_each > 1 && (long long)a.c.streams * pools * parts() < 512) heads_each /= 2;
    const dim3 grid(a.c.streams * ((pools + pools_each - 1) / pools_each), parts());
    if (quantised(a.c.dtype))
        hipLaunchKernelGGL(compact_kernel<true>, grid, dim3(kThreads), 0, s, a, l, pools_each, heads_each);
    else
        hipLaunchKernelGGL(compact_kernel<false>, grid, dim3(kThreads), 0, s, a, l, pools_each, heads_each);
    return hipGetLastError();
}

}  // namespace mh
