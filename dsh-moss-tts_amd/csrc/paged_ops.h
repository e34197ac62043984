// paged_ops.h -- launchers of the operators of a caller's own decoding loop: rotary positions, a
// paged K/V cache in fp32, fp16, int8 or e4m3, attention of drafted rows over it, and token
// log probabilities (internal C++ API; the C entry points check the arguments).
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

}  // namespace mh
