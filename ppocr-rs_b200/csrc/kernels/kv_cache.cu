// The 8-bit paged key / value cache: appending tokens and reading them back.
//
// A page holds `page` consecutive tokens of one sequence for every head, as
// integers in [-127, 127]; the values they stand for are integer x scale with
// one FP32 scale per (page, head), the largest magnitude the page's head has
// seen / 127.  Appending to a part-filled page whose scale grows rounds the
// integers that it held again: q' = round(q s_before / s).  Every rounding to
// an integer is that of the exact quotient (ties to even), so the cache's
// contents depend on the values alone.
//
// Both kernels are bound by HBM: values are read once in their own type (the
// second look at a page's new values, after its maximum is known, hits
// registers or L1) and written once in 8 bits, or the reverse.
#include "seq_common.cuh"

namespace ppocr {

namespace {

constexpr int kThreads = 128;

// Eight consecutive values, as one or two 16-byte loads when `vec`.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
    if (vec) {
        const float4 a = load4(p), b = load4(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = to_f(p[j]);
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, bool vec, float (&x)[8]) {
    if (vec) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = to_f(p[j]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8]) {
    if (vec) {
        store4(p, make_float4(x[0], x[1], x[2], x[3]));
        store4(p + 4, make_float4(x[4], x[5], x[6], x[7]));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = from_f<T>(x[j]);
    }
}

// round(a / s) of the exact quotient, ties to even, clamped to +-127; 0 for a
// scale of 0 or a quotient that is no number.  t = a (1 / s) in FP32 is within
// 2^-15 of the quotient (|a / s| <= 128, three roundings of 2^-24), so unless
// t lies that near to a half it rounds as the quotient does; the few that do
// are divided in FP64, which is exact at a tie.
__device__ __forceinline__ int round_quotient(float a, float s, float inv) {
    if (!(s > 0.f)) return 0;
    const float t = a * inv;
    float r = rintf(t);
    if (!(fabsf(fabsf(t - r) - 0.5f) > 1.f / 8192.f) || !(fabsf(t) < 256.f)) {
        const double d = (double)a / (double)s;
        if (!(fabs(d) < 1e9)) return 0;
        r = (float)rint(d);
    }
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}

__device__ __forceinline__ uint2 pack8(const int (&q)[8]) {
    uint2 u;
    u.x = (q[0] & 0xff) | (q[1] & 0xff) << 8 | (q[2] & 0xff) << 16 | (uint32_t)q[3] << 24;
    u.y = (q[4] & 0xff) | (q[5] & 0xff) << 8 | (q[6] & 0xff) << 16 | (uint32_t)q[7] << 24;
    return u;
}

// One block per (touched page, head, K or V).
template <typename T>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(CacheAppendParams p, bool vec) {
    __shared__ uint32_t top[kThreads / 32];
    // A sequence's n new tokens touch at most n / page + 2 pages.
    const int page = p.cache.page, d8 = p.cache.d / 8, head = blockIdx.y;
    const int page_shift = 31 - __clz(page), id = blockIdx.x;
    auto first_id = [&](int i) { return (seq_offset(p.offsets, 0, i, p.total) >> page_shift) + 2 * i; };
    const int seq = find_owner(p.table.sequences, id, first_id);
    const int index = id - first_id(seq);   // of the pages this sequence's new tokens touch
    const Span span = seq_span(p.offsets, 0, seq, p.total, p.status);
    const int held = p.held[seq];
    if (span.len == 0 || index < 0) return;
    if (held < 0 || (long long)held + span.len > (long long)p.table.width * page) {
        if (threadIdx.x == 0) seq_bad_index(p.status);
        return;
    }
    const int old = index == 0 ? held % page : 0;                      // slots filled before
    const int first = index == 0 ? 0 : index * page - held % page;     // new token in slot `old`
    const int fresh = min(page - old, span.len - first);
    if (fresh <= 0) return;
    const int block = held / page + index;
    const int where = p.table.pages[seq * p.table.stride + block];
    if (where < 0 || where >= p.cache.pages) {
        if (threadIdx.x == 0) seq_bad_index(p.status);
        return;
    }
    const SeqTensor& src = blockIdx.z ? p.v : p.k;
    const T* in = static_cast<const T*>(src.ptr) + (span.begin + first) * src.token_stride + head * src.head_stride;
    const long long cell = (long long)where * p.cache.kv_heads + head;
    int8_t* out = (blockIdx.z ? p.cache.v : p.cache.k) + cell * page * p.cache.d;
    float* scale = (blockIdx.z ? p.cache.v_scales : p.cache.k_scales) + cell;
    const float before = old ? *scale : 0.f;

    // The largest magnitude, compared as bit patterns: those of non-negative
    // floats order as the floats do, with infinity and NaN on top, so a NaN
    // marks its page's scale instead of getting lost.
    constexpr int KEEP = 4;
    float kept[KEEP][8];
    const int items = fresh * d8;
    uint32_t amax = 0;
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
        const int i = threadIdx.x + n * kThreads;
        if (i < items) {
            load8(in + (i / d8) * src.token_stride + (i % d8) * 8, vec, kept[n]);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(kept[n][j]) & 0x7fffffffu);
        }
    }
    for (int i = threadIdx.x + KEEP * kThreads; i < items; i += kThreads) {
        float x[8];
        load8(in + (i / d8) * src.token_stride + (i % d8) * 8, vec, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(x[j]) & 0x7fffffffu);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = amax;
    __syncthreads();   // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = max(amax, top[w]);
    const float mine = __uint_as_float(amax) * (1.f / 127.f);
    const float now = __uint_as_float(max(__float_as_uint(mine) & 0x7fffffffu, __float_as_uint(before) & 0x7fffffffu));
    const float inv = 1.f / now;
    if (threadIdx.x == 0) *scale = now;

    if (old && now > before) {
        const int again = old * d8;
        for (int i = threadIdx.x; i < again; i += kThreads) {
            uint2* cellp = reinterpret_cast<uint2*>(out) + i;
            const uint2 u = *cellp;
            int q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int v = (int8_t)((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
                // q s_before has at most 32 bits: the quotient goes through FP64 only, two roundings away from exact ties.
                q[j] = (int)rint((double)v * (double)before / (double)now);
            }
            *cellp = pack8(q);
        }
    }
    uint2* dst = reinterpret_cast<uint2*>(out + (long long)old * p.cache.d);
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
        const int i = threadIdx.x + n * kThreads;
        if (i < items) {
            int q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = round_quotient(kept[n][j], now, inv);
            dst[i] = pack8(q);
        }
    }
    for (int i = threadIdx.x + KEEP * kThreads; i < items; i += kThreads) {
        float x[8];
        load8(in + (i / d8) * src.token_stride + (i % d8) * 8, vec, x);
        int q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = round_quotient(x[j], now, inv);
        dst[i] = pack8(q);
    }
}

// Tokens per block of the read kernel.
constexpr int kReadTokens = 8;

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(CacheReadParams p, bool vec) {
    __shared__ int where[kReadTokens], slot[kReadTokens];
    const int t0 = blockIdx.x * kReadTokens;
    const int tokens = min(kReadTokens, p.total - t0);
    if (threadIdx.x < tokens) {
        // The sequence of the token: the last one whose offset is not past it.
        const int t = t0 + threadIdx.x;
        int lo = 0, hi = p.table.sequences;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.offsets[mid] <= t) lo = mid; else hi = mid;
        }
        where[threadIdx.x] = -1;
        if (t >= p.offsets[lo] && t < p.offsets[lo + 1]) {
            const long long at = (long long)p.first[lo] + (t - p.offsets[lo]);
            if (p.first[lo] >= 0 && at < (long long)p.table.width * p.cache.page) {
                const int w = p.table.pages[lo * p.table.stride + at / p.cache.page];
                if (w >= 0 && w < p.cache.pages) where[threadIdx.x] = w;
                slot[threadIdx.x] = (int)(at % p.cache.page);
            }
            if (where[threadIdx.x] < 0) seq_bad_index(p.status);
        }
    }
    __syncthreads();
    const int d8 = p.cache.d / 8, per = p.cache.kv_heads * d8;
    const int8_t* pages = blockIdx.y ? p.cache.v : p.cache.k;
    const float* scales = blockIdx.y ? p.cache.v_scales : p.cache.k_scales;
    const SeqTensor& dst = blockIdx.y ? p.v : p.k;
    for (int i = threadIdx.x; i < tokens * per; i += kThreads) {
        const int t = i / per, head = (i % per) / d8, c = i % d8;
        if (where[t] < 0) continue;
        const long long cell = (long long)where[t] * p.cache.kv_heads + head;
        const float s = __ldg(scales + cell);
        const uint2 u = __ldcs(reinterpret_cast<const uint2*>(pages + (cell * p.cache.page + slot[t]) * p.cache.d) + c);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)((j < 4 ? u.x : u.y) >> (8 * (j & 3))) * s;
        store8(static_cast<T*>(dst.ptr) + (t0 + t) * dst.token_stride + head * dst.head_stride + c * 8, vec, x);
    }
}

// Whether every group of eight values of a tensor starts on a 16-byte boundary
// (8 bytes for the BF16 stores, which go out in two halves, would do as well).
bool vec8(const SeqTensor& t, int esize) {
    return ((reinterpret_cast<uintptr_t>(t.ptr) | (uintptr_t)(t.token_stride * esize) | (uintptr_t)(t.head_stride * esize)) & 15) == 0;
}

}  // namespace

cudaError_t launch_cache_append(const CacheAppendParams& p, cudaStream_t stream) {
    if (p.total == 0 || p.table.sequences == 0) return cudaSuccess;
    const int esize = (int)dtype_size(p.dtype);
    const bool vec = vec8(p.k, esize) && vec8(p.v, esize);
    const dim3 grid((unsigned)(p.total / p.cache.page + 2ll * p.table.sequences), p.cache.kv_heads, 2);
    if (p.dtype == DT_F32) cache_append_kernel<float><<<grid, kThreads, 0, stream>>>(p, vec);
    else cache_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, vec);
    return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheReadParams& p, cudaStream_t stream) {
    if (p.total == 0 || p.table.sequences == 0) return cudaSuccess;
    const int esize = (int)dtype_size(p.dtype);
    const bool vec = vec8(p.k, esize) && vec8(p.v, esize);
    const dim3 grid((p.total + kReadTokens - 1) / kReadTokens, 2);
    if (p.dtype == DT_F32) cache_read_kernel<float><<<grid, kThreads, 0, stream>>>(p, vec);
    else cache_read_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, vec);
    return cudaGetLastError();
}

}  // namespace ppocr
