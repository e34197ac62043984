// paged_ops.h -- launchers of the operators of a caller's own decoding loop: rotary positions, a
// paged K/V cache in fp32, fp16, int8 or e4m3 and its pages, attention of drafted rows over it, token
// log probabilities, verification of drafted tokens, and adapters beside a projection (internal C++
// API; the C entry points check the arguments).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mh_device.h"

namespace mh {

// Element types, the values of the C enum MOSS_HIP_F32 ...
enum ElemType : int { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_I8 = 2, ELEM_E4M3 = 3 };
constexpr bool quantised(int t) { return t == ELEM_I8 || t == ELEM_E4M3; }
constexpr int elem_size(int t) { return t == ELEM_F32 ? 4 : (t == ELEM_F16 ? 2 : 1); }

struct RopeArgs {
    const double *freqs = nullptr;  // rot / 2 angles per position (device); null: no rotation
    int rot = 0;
    int halves = 0;  // pairs (i, i + rot / 2) rather than (2i, 2i + 1)
    float mscale = 1.0f;
};

struct RopeRowsArgs {
    const void *x = nullptr;
    void *y = nullptr;
    int dtype = ELEM_F32;
    int rows = 0, heads = 0, dim = 0;
    int64_t x_row = 0, x_head = 0, y_row = 0, y_head = 0;  // strides in elements
    const int *pos = nullptr;
    RopeArgs rope;
};
hipError_t launch_rope_rows(const RopeRowsArgs &a, hipStream_t s);

// Pools [page][kv_heads][page_size][dim]; scales [page][kv_heads][page_size] of the 8-bit types.
struct KvCacheArgs {
    void *k = nullptr, *v = nullptr;
    float *k_scale = nullptr, *v_scale = nullptr;
    int dtype = ELEM_F16;
    int heads = 0, dim = 0;
    int page_size = 0, n_pages = 0;
    const int *table = nullptr;
    int table_stride = 0, streams = 0;
};

struct KvRowsArgs {
    KvCacheArgs c;
    const void *k = nullptr, *v = nullptr;  // write: the rows
    void *k_out = nullptr, *v_out = nullptr;  // read: where they go
    int64_t k_row = 0, v_row = 0;  // row strides in elements; a row's heads are contiguous
    int dtype = ELEM_F32;
    int rows = 0;
    const int *stream = nullptr, *pos = nullptr;
    RopeArgs rope;  // write: applied to the keys
    const int *rope_pos = nullptr;
};
hipError_t launch_kv_write(const KvRowsArgs &a, hipStream_t s);
hipError_t launch_kv_read(const KvRowsArgs &a, hipStream_t s);

struct LogprobArgs {
    const void *x = nullptr;  // logits [rows][vocab], fp32 or fp16
    int dtype = ELEM_F32;
    int64_t row = 0;  // row stride in elements
    int rows = 0, vocab = 0;
    const int *tokens = nullptr;
    float inv_t = 1.0f;
    float *logprob = nullptr, *entropy = nullptr;
    int top_k = 0;
    int *top_ids = nullptr;
    float *top_lp = nullptr;
    void *ws = nullptr;
};
constexpr int kTopMax = 32;           // alternatives of one row
constexpr int kVocabMax = 1 << 20;
size_t logprobs_workspace(int rows, int vocab, int top_k);
hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s);

struct TreeArgs {
    KvCacheArgs c;
    const void *q = nullptr;
    int q_dtype = ELEM_F32;
    int64_t q_row = 0, out_row = 0;  // row strides in elements; a row's heads are contiguous
    int heads = 0;
    const int *row_start = nullptr, *ctx_len = nullptr;
    const uint64_t *row_mask = nullptr;
    int rows = 0, max_rows = 0, max_keys = 0;
    float scale = 0.0f;
    void *out = nullptr;
    int out_dtype = ELEM_F32;
    float *lse = nullptr;
    void *ws = nullptr;
    bool q_vec = false, out_vec = false;  // 16-byte accesses are aligned (set at the launch)
};
constexpr int kTreeMax = 64;  // drafted rows of a stream
constexpr int kTreeKeysMax = 1 << 28, kTreePageMax = 1 << 15;
size_t tree_workspace(const KvCacheArgs &c, int heads, int rows, int max_rows, int max_keys);
hipError_t launch_attn_tree(const TreeArgs &a, hipStream_t s);

// ---- pages of the cache

// The pools of all layers, by value: what one launch works on.
constexpr int kLayersMax = 64;
struct KvLayers {
    void *k[kLayersMax], *v[kLayersMax];
    float *k_scale[kLayersMax], *v_scale[kLayersMax];
};
struct PagesArgs {
    int *table = nullptr;  // [streams][table_stride]
    int table_stride = 0, streams = 0;
    int *refs = nullptr;  // [n_pages]
    int n_pages = 0, page_size = 0;
};
struct ForkArgs {
    PagesArgs p;
    const int *parent = nullptr, *len = nullptr;
    int *ws = nullptr;
};
size_t fork_workspace(const PagesArgs &p);
hipError_t launch_kv_fork(const ForkArgs &a, hipStream_t s);

struct ReserveArgs {
    PagesArgs p;
    int layers = 0, heads = 0, vec_bytes = 0;  // vec_bytes: of one head of one position
    bool scales = false;
    const int *row_start = nullptr, *ctx_len = nullptr;
    int max_rows = 0;
    int *ok = nullptr;
    void *ws = nullptr;
    int4 *copies = nullptr;  // parts of the workspace (set at the launch)
    int *free_pages = nullptr, *fate = nullptr;
};
size_t reserve_workspace(const PagesArgs &p, int max_rows);
hipError_t launch_kv_reserve(ReserveArgs a, const KvLayers &l, hipStream_t s);

struct CompactArgs {
    KvCacheArgs c;  // of one layer: its shape and the table
    int layers = 0, vec_bytes = 0;
    const int *row_start = nullptr, *ctx_len = nullptr, *kept = nullptr;
    int rows = 0, max_rows = 0;
};
hipError_t launch_kv_compact(const CompactArgs &a, const KvLayers &l, hipStream_t s);

// ---- verification of drafted tokens

struct VerifyArgs {
    const void *x = nullptr, *y = nullptr;  // logits [rows][vocab] of the target, and of the draft or null
    int dtype = ELEM_F32;
    int64_t x_row = 0, y_row = 0;  // row strides in elements
    int rows = 0, vocab = 0;
    const int *tokens = nullptr, *row_start = nullptr;
    const uint64_t *row_mask = nullptr;
    int streams = 0, max_rows = 0;
    const double *uniforms = nullptr;
    float inv_t = 1.0f, draft_inv_t = 1.0f;
    bool greedy = false;
    int *accepted = nullptr, *path = nullptr, *next = nullptr;
    void *ws = nullptr;
};
size_t verify_need(int streams, int max_rows, int vocab, bool draft);       // of a call
size_t verify_workspace(int streams, int max_rows, int vocab, bool draft);  // of any call of no more streams and rows
hipError_t launch_verify(const VerifyArgs &a, hipStream_t s);

// ---- low-rank adapters beside a projection

struct AdapterArgs {
    const void *a = nullptr, *b = nullptr;  // packed weights of n adapters
    const float *scale = nullptr;  // [n], null: 1
    int n = 0, max_rank = 0, cols = 0, out = 0;
    const void *x = nullptr, *base = nullptr;
    void *y = nullptr;
    int x_dtype = ELEM_F32, y_dtype = ELEM_F32;
    int64_t x_row = 0, base_row = 0, y_row = 0;  // row strides in elements
    const int *which = nullptr;  // [rows]
    int rows = 0;
};
constexpr int kAdapterRankMax = 128;
void adapter_sizes(const AdapterArgs &a, size_t *a_bytes, size_t *b_bytes);  // of the packed weights
hipError_t launch_adapter_rows(const AdapterArgs &a, hipStream_t s);

struct AdapterPackArgs {
    const void *a = nullptr, *b = nullptr;  // fp16 [count][max_rank][cols], [count][out][max_rank]
    const int *rank = nullptr;  // [count], null: max_rank
    int count = 0, first = 0;
    int max_rank = 0, cols = 0, out = 0;
    void *to_a = nullptr, *to_b = nullptr;
};
hipError_t launch_adapter_pack(const AdapterPackArgs &p, hipStream_t s);

}  // namespace mh
