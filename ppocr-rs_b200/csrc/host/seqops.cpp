// extern "C" boundary of the sequence operators: checks of what the host can
// see, then one launch on the caller's stream.  The calls keep nothing in the
// handle (its mutex is not taken) and restore the caller's current device.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../kernels/seq.h"
#include "handles.hpp"
#include "seq_status.hpp"

using namespace ppocr;

namespace {

void require(bool ok, const char* message) {
    if (!ok) fail(PPOCR_ERR_INVALID_INPUT, std::string("invalid input: ") + message);
}

[[noreturn]] void refuse(const char* name, const char* what) {
    fail(PPOCR_ERR_INVALID_INPUT, std::string("invalid input: ") + name + what);
}

// The handle's device current for a call; the caller's afterwards.
class OnDevice {
public:
    explicit OnDevice(const ppocr_gpu* gpu) {
        cuda_check(cudaGetDevice(&before_), "cudaGetDevice");
        if (gpu->poisoned || before_ != gpu->device) gpu->bind();
    }
    ~OnDevice() {
        int now = before_;
        if (cudaGetDevice(&now) == cudaSuccess && now != before_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

private:
    int before_ = 0;
};

cudaStream_t stream_of(const ppocr_gpu* gpu, void* stream) { return stream ? static_cast<cudaStream_t>(stream) : gpu->stream; }

DType dtype_of(int dtype) {
    require(dtype == PPOCR_DTYPE_F32 || dtype == PPOCR_DTYPE_BF16, "dtype must be 0 (F32) or 1 (BF16)");
    return dtype == PPOCR_DTYPE_F32 ? DT_F32 : DT_BF16;
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

SeqTensor tensor_of(const ppocr_tokens& t, int64_t tokens, DType dtype, const char* name) {
    if (!t.data && tokens > 0) refuse(name, " pointer is null");
    if (!aligned(t.data, dtype_size(dtype))) refuse(name, " is not aligned to its type");
    // Every byte offset of a tensor stays far from the ends of 64 bits.
    const int64_t most = INT64_C(1) << 30;
    if (t.token_stride < 0 || t.head_stride < 0 || t.token_stride > most || t.head_stride > most)
        refuse(name, "'s strides must be 0..2^30");
    SeqTensor s;
    s.ptr = t.data;
    s.token_stride = t.token_stride;
    s.head_stride = t.head_stride;
    return s;
}

// An output's elements may not share memory: a token holds its heads apart and
// a token's heads lie within its stride (or the other way round).
void require_distinct(const ppocr_tokens& t, int64_t tokens, int heads, int d, const char* name) {
    const bool token_major = (heads == 1 || t.head_stride >= d) &&
                             (tokens <= 1 || t.token_stride >= (heads - 1) * t.head_stride + d);
    const bool head_major = (tokens <= 1 || t.token_stride >= d) &&
                            (heads == 1 || t.head_stride >= (tokens - 1) * t.token_stride + d);
    if (!token_major && !head_major) refuse(name, "'s strides make elements share memory");
}

// Counts leave room for a tile of tokens past the last one.
int count_of(int64_t n, const char* what) {
    require(n >= 0 && n < INT_MAX - 65536, what);
    return (int)n;
}

// Device arrays of 32-bit words (offsets, lengths, ids, floats).
void require_words(std::initializer_list<const void*> arrays) {
    for (const void* p : arrays) require(aligned(p, 4), "an array of 32-bit words is not aligned to them");
}

float scale_of(float scale, int d) {
    require(scale >= 0.f && scale <= 1e30f, "scale must be 0 (d^-1/2) or positive, up to 1e30");
    return scale == 0.f ? 1.f / std::sqrt((float)d) : scale;
}

void check_heads(int heads, int kv_heads) {
    require(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "heads must be a multiple of kv_heads, both positive");
    require(heads <= 65535, "more than 65535 heads");
}

PagedCacheView cache_of(const ppocr_paged_cache& c) {
    require(c.page == 16 || c.page == 32 || c.page == 64 || c.page == 128, "a page holds 16, 32, 64 or 128 tokens");
    require(c.d >= 8 && c.d <= 128 && c.d % 8 == 0, "the cache's head size must be a multiple of 8 up to 128");
    require(c.kv_heads >= 1 && c.kv_heads <= 65535, "the cache's heads must be 1..65535");
    require(c.pages >= 0, "the cache's pages must not be negative");
    require(c.pages == 0 || (c.k && c.v && c.k_scales && c.v_scales), "a cache pointer is null");
    require(aligned(c.k, 16) && aligned(c.v, 16), "the cache's pages must be 16-byte aligned");
    require(aligned(c.k_scales, 4) && aligned(c.v_scales, 4), "the cache's scales must be aligned to their type");
    PagedCacheView v;
    v.k = c.k;
    v.v = c.v;
    v.k_scales = c.k_scales;
    v.v_scales = c.v_scales;
    v.pages = c.pages;
    v.kv_heads = c.kv_heads;
    v.page = c.page;
    v.d = c.d;
    return v;
}

BlockTable table_of(const ppocr_block_table& t, const PagedCacheView& cache) {
    require(t.sequences >= 0 && t.width >= 0, "the block table's extents must not be negative");
    require(t.stride >= t.width || t.sequences <= 1, "the block table's stride is smaller than its width");
    require(t.pages || t.sequences == 0 || t.width == 0, "block table pointer is null");
    require_words({t.pages});
    // Positions stay below 2^31 with room for a tile behind the last one.
    require((int64_t)t.width * cache.page <= INT_MAX - 4096, "the block table spans 2^31 tokens or more");
    require((int64_t)t.sequences * cache.kv_heads <= (1 << 30), "more than 2^30 sequences x heads");
    BlockTable b;
    b.pages = t.pages;
    b.sequences = t.sequences;
    b.width = t.width;
    b.stride = t.stride;
    return b;
}

}  // namespace

extern "C" {

int ppocr_gpu_synchronize(ppocr_gpu* gpu, void* stream, int timeout_ms) {
    return guard([&] {
        if (!gpu) fail(PPOCR_ERR_INVALID_INPUT, "gpu handle is null");
        OnDevice on(gpu);
        // The caller's stream may hold work of its own that takes longer than it cares to
        // wait here: only the handle's own stream condemns the handle.
        wait_stream(stream_of(gpu, stream), timeout_ms, stream ? nullptr : gpu);
        const int bad = take_status(gpu->seq_status), wait = take_status(gpu->seq_status + 1);
        if (wait)
            fail(PPOCR_ERR_GPU, "GPU error: a tensor-core pipeline wait ran out (code " + std::to_string(wait) +
                                    "); the results are incomplete");
        if (bad) fail(PPOCR_ERR_INVALID_INPUT, "invalid input: an offset, length, table entry, id or state is out of range");
    });
}

int ppocr_attention_packed(ppocr_gpu* gpu, const ppocr_attention_packed_args* args, void* stream) {
    return guard([&] {
        if (!gpu || !args) fail(PPOCR_ERR_INVALID_INPUT, "null argument");
        const ppocr_attention_packed_args& a = *args;
        PackedAttentionParams p;
        p.dtype = dtype_of(a.dtype);
        check_heads(a.heads, a.kv_heads);
        require(a.d >= 1 && a.d <= kPackedMaxD, "the head size must be 1..128");
        require(a.causal == 0 || a.causal == 1, "causal must be 0 or 1");
        p.heads = a.heads;
        p.kv_heads = a.kv_heads;
        p.d = a.d;
        p.causal = a.causal;
        p.scale = scale_of(a.scale, a.d);
        p.sequences = count_of(a.sequences, "sequences is negative or near 2^31");
        p.total_q = count_of(a.total_q, "total_q is negative or near 2^31");
        p.total_k = count_of(a.total_k, "total_k is negative or near 2^31");
        require(p.sequences == 0 || (a.q_offsets && a.k_offsets), "offsets pointer is null");
        require_words({a.q_offsets, a.k_offsets});
        // The grid: one block per 64 rows of queries and group heads at most.
        require((int64_t)p.total_q * p.heads / 64 + ((int64_t)p.sequences + 1) * p.kv_heads <= INT_MAX,
                "too many query rows for one call");
        p.q = tensor_of(a.q, a.total_q, p.dtype, "q");
        p.k = tensor_of(a.k, a.total_k, p.dtype, "k");
        p.v = tensor_of(a.v, a.total_k, p.dtype, "v");
        p.out = tensor_of(a.out, a.total_q, p.dtype, "out");
        require_distinct(a.out, a.total_q, a.heads, a.d, "out");
        p.q_offsets = a.q_offsets;
        p.k_offsets = a.k_offsets;
        p.bad = gpu->seq_status;
        p.err = gpu->seq_status + 1;
        OnDevice on(gpu);
        cuda_check(launch_attention_packed(p, stream_of(gpu, stream)), "packed attention");
    });
}

int ppocr_cache_append(ppocr_gpu* gpu, const ppocr_cache_append_args* args, void* stream) {
    return guard([&] {
        if (!gpu || !args) fail(PPOCR_ERR_INVALID_INPUT, "null argument");
        const ppocr_cache_append_args& a = *args;
        CacheAppendParams p;
        p.dtype = dtype_of(a.dtype);
        p.cache = cache_of(a.cache);
        p.table = table_of(a.table, p.cache);
        p.total = count_of(a.total, "total is negative or near 2^31");
        require(p.table.sequences == 0 || (a.offsets && a.held), "offsets or held pointer is null");
        require_words({a.offsets, a.held});
        require((int64_t)p.total / p.cache.page + 2 * (int64_t)p.table.sequences <= INT_MAX, "too many tokens for one call");
        p.k = tensor_of(a.k, a.total, p.dtype, "k");
        p.v = tensor_of(a.v, a.total, p.dtype, "v");
        p.offsets = a.offsets;
        p.held = a.held;
        p.bad = gpu->seq_status;
        OnDevice on(gpu);
        cuda_check(launch_cache_append(p, stream_of(gpu, stream)), "cache append");
    });
}

int ppocr_cache_read(ppocr_gpu* gpu, const ppocr_cache_read_args* args, void* stream) {
    return guard([&] {
        if (!gpu || !args) fail(PPOCR_ERR_INVALID_INPUT, "null argument");
        const ppocr_cache_read_args& a = *args;
        CacheReadParams p;
        p.dtype = dtype_of(a.dtype);
        p.cache = cache_of(a.cache);
        p.table = table_of(a.table, p.cache);
        p.total = count_of(a.total, "total is negative or near 2^31");
        require(p.table.sequences == 0 || (a.offsets && a.first), "offsets or first pointer is null");
        require_words({a.offsets, a.first});
        p.k = tensor_of(a.k, a.total, p.dtype, "k");
        p.v = tensor_of(a.v, a.total, p.dtype, "v");
        require_distinct(a.k, a.total, p.cache.kv_heads, p.cache.d, "k");
        require_distinct(a.v, a.total, p.cache.kv_heads, p.cache.d, "v");
        p.offsets = a.offsets;
        p.first = a.first;
        p.bad = gpu->seq_status;
        OnDevice on(gpu);
        cuda_check(launch_cache_read(p, stream_of(gpu, stream)), "cache read");
    });
}

int ppocr_attention_cached(ppocr_gpu* gpu, const ppocr_attention_cached_args* args, void* stream) {
    return guard([&] {
        if (!gpu || !args) fail(PPOCR_ERR_INVALID_INPUT, "null argument");
        const ppocr_attention_cached_args& a = *args;
        CachedAttentionParams p;
        p.dtype = dtype_of(a.dtype);
        p.cache = cache_of(a.cache);
        p.table = table_of(a.table, p.cache);
        check_heads(a.heads, p.cache.kv_heads);
        // The grid: sequences x up to 16 parts of a sequence.
        require(p.table.sequences <= INT_MAX / 16, "too many sequences for one call");
        p.heads = a.heads;
        p.scale = scale_of(a.scale, p.cache.d);
        require(p.table.sequences == 0 || a.lengths, "lengths pointer is null");
        require_words({a.lengths});
        p.q = tensor_of(a.q, p.table.sequences, p.dtype, "q");
        p.out = tensor_of(a.out, p.table.sequences, p.dtype, "out");
        require_distinct(a.out, p.table.sequences, a.heads, p.cache.d, "out");
        p.lengths = a.lengths;
        p.bad = gpu->seq_status;
        OnDevice on(gpu);
        cuda_check(launch_attention_cached(p, stream_of(gpu, stream)), "cached attention");
    });
}

int ppocr_logit_rules(ppocr_gpu* gpu, const ppocr_logit_rules_args* args, void* stream) {
    return guard([&] {
        if (!gpu || !args) fail(PPOCR_ERR_INVALID_INPUT, "null argument");
        const ppocr_logit_rules_args& a = *args;
        LogitRulesParams p;
        p.dtype = dtype_of(a.dtype);
        count_of(a.rows, "rows is negative or near 2^31");
        count_of(a.vocab, "vocab is negative or near 2^31");
        const bool some = a.rows > 0 && a.vocab > 0;
        require(!some || (a.logits && a.out), "logits or out pointer is null");
        require(aligned(a.logits, dtype_size(p.dtype)) && aligned(a.out, dtype_size(p.dtype)), "logits or out is not aligned to its type");
        require(a.rows <= 1 || (a.stride >= a.vocab && a.out_stride >= a.vocab), "a row stride is smaller than vocab");
        require(a.stride >= 0 && a.out_stride >= 0 && a.stride <= INT64_C(1) << 40 && a.out_stride <= INT64_C(1) << 40,
                "a row stride is negative or beyond 2^40");
        require(a.logits != a.out || a.rows <= 1 || a.stride == a.out_stride, "in place, both row strides must be the same");
        require(!(a.repetition || a.presence || a.frequency) || a.history_offsets, "the penalties need a history");
        p.history_total = count_of(a.history_total, "history_total is negative or near 2^31");
        require(!a.history_offsets || a.history || p.history_total == 0, "history pointer is null");
        require(!a.mask_index || a.mask, "mask_index needs a mask");
        require(!a.mask || (a.states >= 1 && a.mask_stride >= ((int64_t)a.vocab + 31) / 32),
                "a mask needs at least one row of ceil(vocab / 32) words");
        require_words({a.history, a.history_offsets, a.repetition, a.presence, a.frequency, a.bias, a.mask, a.mask_index});
        p.logits = a.logits;
        p.out = a.out;
        p.ld = a.stride;
        p.out_ld = a.out_stride;
        p.rows = a.rows;
        p.vocab = a.vocab;
        p.history = a.history;
        p.history_offsets = a.history_offsets;
        p.repetition = a.repetition;
        p.presence = a.presence;
        p.frequency = a.frequency;
        p.bias = a.bias;
        p.mask = a.mask;
        p.mask_ld = a.mask_stride;
        p.states = a.states;
        p.mask_index = a.mask_index;
        p.bad = gpu->seq_status;
        OnDevice on(gpu);
        cuda_check(launch_logit_rules(p, stream_of(gpu, stream)), "logit rules");
    });
}

}  // extern "C"
