// Launch interface of the sequence operators: attention over packed
// sequences, the 8-bit paged key / value cache (append, read, single-token
// attention) and the logit rules.  Every launcher enqueues on `stream` and
// returns the launch error; none allocates, synchronises or keeps state, so
// any of them can be captured into a graph or run on several streams at once.
//
// Strides are in elements; the last axis of every tensor is contiguous.
// Offsets, lengths and block tables live on the device.  The kernels clamp
// them to the tensors' extents, so a bad one reads and writes nothing out of
// bounds, and set *bad to 1 (for the C ABI page-locked host memory, which the
// host reads and raises; null: not reported).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace ppocr {

struct SeqTensor {
    void* ptr = nullptr;
    long long token_stride = 0, head_stride = 0;
};

// out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j of query i's
// sequence; causal: j <= i + (keys - queries of the sequence); no key: zeros.
struct PackedAttentionParams {
    SeqTensor q, k, v, out;              // [total][heads][d]
    const int32_t* q_offsets = nullptr;  // [sequences + 1]; null: `uniform` tokens per sequence
    const int32_t* k_offsets = nullptr;
    int uniform = 0;
    int sequences = 0, total_q = 0, total_k = 0;
    int heads = 0, kv_heads = 0, d = 0;
    int causal = 0;
    float scale = 1.f;                   // > 0
    DType dtype = DT_F32;
    int* bad = nullptr;
    // tcgen05 kernel: a pipeline wait that runs out stores its code in *err (null:
    // not reported) after wait_ns (0: 2 s); skip_load = 1 (self-test only) leaves
    // block 0's second stage unloaded so that the waits on it run out.
    int* err = nullptr;
    uint64_t wait_ns = 0;
    int skip_load = 0;
};
constexpr int kPackedMaxD = 128;
cudaError_t launch_attention_packed(const PackedAttentionParams& p, cudaStream_t stream);
cudaError_t launch_attention_packed_f32(const PackedAttentionParams& p, cudaStream_t stream);   // DT_F32, not empty

// Its tcgen05 kernel (attention_tc.cu): BF16, 16-byte aligned rows, d a multiple
// of 8 and at most 128 query heads to a KV head.
bool attention_tc_supported(const PackedAttentionParams& p);
cudaError_t launch_attention_tc(const PackedAttentionParams& p, cudaStream_t stream);

// 8-bit cache: values[page][head][slot][d] with one FP32 scale per (page, head).
struct PagedCacheView {
    int8_t* k = nullptr;
    int8_t* v = nullptr;
    float* k_scales = nullptr;
    float* v_scales = nullptr;
    int pages = 0, kv_heads = 0, page = 0, d = 0;   // page: 16, 32, 64 or 128 tokens; d: a multiple of 8 up to 128
};

struct BlockTable {
    const int32_t* pages = nullptr;      // [sequences][width]: the page of each block of `page` tokens
    int sequences = 0, width = 0;
    long long stride = 0;
};

struct CacheAppendParams {
    PagedCacheView cache;
    BlockTable table;
    SeqTensor k, v;                      // [total][kv_heads][d]
    const int32_t* offsets = nullptr;    // [sequences + 1] into the new tokens
    const int32_t* held = nullptr;       // [sequences] tokens already in the cache
    int total = 0;
    DType dtype = DT_F32;
    int* bad = nullptr;
};
cudaError_t launch_cache_append(const CacheAppendParams& p, cudaStream_t stream);

struct CacheReadParams {
    PagedCacheView cache;
    BlockTable table;
    SeqTensor k, v;                      // outputs [total][kv_heads][d]
    const int32_t* offsets = nullptr;    // [sequences + 1] into the outputs
    const int32_t* first = nullptr;      // [sequences] position of each sequence's first token read
    int total = 0;
    DType dtype = DT_F32;
    int* bad = nullptr;
};
cudaError_t launch_cache_read(const CacheReadParams& p, cudaStream_t stream);

struct CachedAttentionParams {
    PagedCacheView cache;
    BlockTable table;
    SeqTensor q, out;                    // [sequences][heads][d]
    const int32_t* lengths = nullptr;    // [sequences] tokens attended to
    int heads = 0;
    float scale = 1.f;                   // > 0
    DType dtype = DT_F32;
    int* bad = nullptr;
};
cudaError_t launch_attention_cached(const CachedAttentionParams& p, cudaStream_t stream);

// out = the row's logits after, in this order: the repetition penalty (ids in
// the row's history: x / r where x > 0, else x r), - frequency count -
// presence [count > 0], + bias, and -infinity where the row's mask has a 0 bit.
struct LogitRulesParams {
    const void* logits = nullptr;
    void* out = nullptr;                 // may be `logits`
    long long ld = 0, out_ld = 0;
    int rows = 0, vocab = 0;
    const int32_t* history = nullptr;    // packed ids
    const int32_t* history_offsets = nullptr;   // [rows + 1], null: no history
    int history_total = 0;
    const float* repetition = nullptr;   // [rows] or null
    const float* presence = nullptr;
    const float* frequency = nullptr;
    const float* bias = nullptr;         // [vocab] or null
    const uint32_t* mask = nullptr;      // [states][words], bit v % 32 of word v / 32: class v allowed
    long long mask_ld = 0;
    int states = 0;
    const int32_t* mask_index = nullptr; // [rows] state of each row, -1: unmasked; null: state 0 for all
    DType dtype = DT_F32;
    int* bad = nullptr;
};
cudaError_t launch_logit_rules(const LogitRulesParams& p, cudaStream_t stream);

}  // namespace ppocr
