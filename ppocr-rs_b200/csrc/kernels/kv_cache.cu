// The 8-bit paged key / value cache: appending tokens and reading them back.
//
// A page holds `page` consecutive tokens of one sequence for every head, as
// integers in [-127, 127]; the values they stand for are integer x scale with
// one FP32 scale per (page, head), the largest magnitude the page's head has
// seen x FP32's 1 / 127.  Appending to a part-filled page whose scale grows rounds the
// integers that it held again: q' = round(q s_before / s).  Every rounding to
// an integer is that of the exact quotient (ties to even), so the cache's
// contents depend on the values alone.
//
// Both kernels are bound by HBM: values are read once in their own type (the
// second look at a page's new values, after its maximum is known, hits
// registers or L1) and written once in 8 bits, or the reverse.  9,096 tokens of 8
// heads of 128 in BF16, pages of 32: append 20 us (2.8 TB/s), read 16 us (3.6); the
// dozen instructions per value of the exact rounding (a branch to 64-bit
// arithmetic for near ties: 33 us) and one wave of loads are what is left.  256
// single tokens of 4 heads of 64 in FP32: 9.7 us, a launch and three dependent
// reads (offsets, table, page).
#include "seq_common.cuh"

namespace ppocr {

namespace {

constexpr int kThreads = 128;

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

// The integers of eight values of a page with scale s: round(a / s) of the exact
// quotient, ties to even.  With r = round(a inv), inv = 1 / s, the remainder
// a - r s is a multiple of half the last place of s and not much above s / 2,
// so a fused multiply-add gives it exactly; r moves by one towards it where it
// is more than s / 2, or just that and r is odd (as integers the bit patterns of
// positive floats compare as the floats do).  No branch: values of half a page's
// largest are common, and their quotient is 63.5.  Adding 1.5 x 2^23 rounds to
// an integer whose low byte is the sum's.
template <typename T>
__device__ __forceinline__ uint2 round8(const Pack<T, 8>& x, float s, float inv) {
    constexpr float kMagic = 12582912.f;
    const int half = __float_as_int(0.5f * s);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = x.get(j);
        y[j] = fmaf(a, inv, kMagic);
        const int e = __float_as_int(fmaf(kMagic - y[j], s, a));
        if ((e & 0x7fffffff) + (__float_as_int(y[j]) & 1) > half) y[j] += __int_as_float((e & 0x80000000) | 0x3f800000);
    }
    auto low = [&](int j) {
        const uint32_t a = __byte_perm(__float_as_uint(y[j]), __float_as_uint(y[j + 1]), 0x0040);
        const uint32_t b = __byte_perm(__float_as_uint(y[j + 2]), __float_as_uint(y[j + 3]), 0x0040);
        return __byte_perm(a, b, 0x5410);
    };
    return make_uint2(low(0), low(4));
}

// The same for a scale without an ordinary reciprocal, in FP64; 0 for a scale of
// 0 or a quotient that is no number.
template <typename T>
__device__ __noinline__ uint2 round8_odd(const T* p, float s) {
    uint2 u = make_uint2(0, 0);
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
        const double d = s > 0.f ? (double)to_f(p[j]) / (double)s : 0.0;
        const int q = fabs(d) < 1e9 ? (int)fmin(fmax(rint(d), -127.0), 127.0) : 0;
        const uint32_t byte = (uint32_t)(q & 0xff) << (8 * (j & 3));
        if (j < 4) u.x |= byte; else u.y |= byte;
    }
    return u;
}

__device__ __forceinline__ uint2 pack8(const int (&q)[8]) {
    uint2 u;
    u.x = (q[0] & 0xff) | (q[1] & 0xff) << 8 | (q[2] & 0xff) << 16 | (uint32_t)q[3] << 24;
    u.y = (q[4] & 0xff) | (q[5] & 0xff) << 8 | (q[6] & 0xff) << 16 | (uint32_t)q[7] << 24;
    return u;
}

// One block per (touched page, head, K or V).
template <typename T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 7) cache_append_kernel(CacheAppendParams p, bool vec) {
    __shared__ uint32_t top[kThreads / 32];
    // A sequence's n new tokens touch at most n / page + 2 pages.
    const int page = p.cache.page, d8 = p.cache.d / 8;
    const int page_shift = 31 - __clz(page), id = blockIdx.x;
    check_offsets(p.offsets, p.table.sequences, p.total, p.bad);
    auto first_id = [&](int i) { return (seq_offset(p.offsets, 0, i, p.total) >> page_shift) + 2 * i; };
    const int seq = find_owner(p.table.sequences, id, first_id);
    const int index = id - first_id(seq);   // of the pages this sequence's new tokens touch
    const Span span = seq_span(p.offsets, 0, seq, p.total, p.bad);
    const int held = p.held[seq];
    if (span.len == 0 || index < 0) return;
    if (held < 0 || (long long)held + span.len > (long long)p.table.width * page) {
        if (threadIdx.x == 0) seq_bad_index(p.bad);
        return;
    }
    const int old = index == 0 ? held % page : 0;                      // slots filled before
    const int first = index == 0 ? 0 : index * page - held % page;     // new token in slot `old`
    const int fresh = min(page - old, span.len - first);
    if (fresh <= 0) return;
    const int block = held / page + index;
    const int where = p.table.pages[seq * p.table.stride + block];
    if (where < 0 || where >= p.cache.pages) {
        if (threadIdx.x == 0) seq_bad_index(p.bad);
        return;
    }
    const SeqTensor& src = blockIdx.z ? p.v : p.k;
    // Item i is eights i % d8 of token i / d8; a thread's items are kThreads apart.
    constexpr int KEEP = 4;
    const int step_row = kThreads / d8, step_col = kThreads % d8, row0 = threadIdx.x / d8, col0 = threadIdx.x % d8;
    auto next = [&](int& row, int& col) {
        row += step_row;
        col += step_col;
        if (col >= d8) {
            col -= d8;
            ++row;
        }
    };
    const int head = blockIdx.y;
    const T* in = static_cast<const T*>(src.ptr) + (long long)(span.begin + first) * src.token_stride + head * src.head_stride;
    const long long cell = (long long)where * p.cache.kv_heads + head;
    int8_t* out = (blockIdx.z ? p.cache.v : p.cache.k) + cell * page * p.cache.d;
    float* scale = (blockIdx.z ? p.cache.v_scales : p.cache.k_scales) + cell;
    const float before = old ? *scale : 0.f;

    // The largest magnitude, compared as bit patterns: those of non-negative
    // floats order as the floats do, with infinity and NaN on top, so a NaN
    // marks its page's scale instead of getting lost.
    Pack<T, 8> kept[KEEP];
    auto load = [&](Pack<T, 8>& x, int r, int c) {
        const T* p8 = in + r * src.token_stride + c * 8;
        if (vec) x.load(p8);
        else x.load_some(p8, 8);
    };
    uint32_t amax = 0;
    int row = row0, col = col0;
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
        if (row < fresh) load(kept[n], row, col);
        next(row, col);
    }
    row = row0;
    col = col0;
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
        if (row < fresh) {
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(kept[n].get(j)) & 0x7fffffffu);
        }
        next(row, col);
    }
    for (int r = row, c = col; r < fresh; next(r, c)) {
        Pack<T, 8> x;
        load(x, r, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(x.get(j)) & 0x7fffffffu);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = amax;
    __syncthreads();   // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = max(amax, top[w]);
    const float mine = __uint_as_float(amax) * (1.f / 127.f);
    const float now = __uint_as_float(max(__float_as_uint(mine) & 0x7fffffffu, __float_as_uint(before) & 0x7fffffffu));
    const float inv = now > 1e-30f && now < 1e30f ? 1.f / now : 0.f;
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
    auto store = [&](int r, int c, const Pack<T, 8>& x) {
        const uint2 u = inv != 0.f ? round8(x, now, inv) : round8_odd(in + r * src.token_stride + c * 8, now);
        dst[r * d8 + c] = u;
    };
    row = row0;
    col = col0;
#pragma unroll
    for (int n = 0; n < KEEP; ++n) {
        if (row < fresh) store(row, col, kept[n]);
        next(row, col);
    }
    for (; row < fresh; next(row, col)) {
        Pack<T, 8> x;
        load(x, row, col);
        store(row, col, x);
    }
}

// Tokens per block of the read kernel, and values in flight per thread.
constexpr int kReadTokens = 16, kReadThreads = 256, kReadAhead = 4;

template <typename T>
__global__ void __launch_bounds__(kReadThreads) cache_read_kernel(CacheReadParams p, bool vec) {
    __shared__ int where[kReadTokens], slot[kReadTokens];
    const int t0 = blockIdx.x * kReadTokens, lane = threadIdx.x & 31;
    const int tokens = min(kReadTokens, p.total - t0);
    check_offsets(p.offsets, p.table.sequences, p.total, p.bad);
    for (int i = threadIdx.x / 32; i < tokens; i += kReadThreads / 32) {
        const int t = t0 + i, seq = find_owner(p.table.sequences, t, [&](int s) { return seq_offset(p.offsets, 0, s, p.total); });
        // Sequences without tokens start where the next one does: the last one is the owner.
        const Span span = seq_span(p.offsets, 0, seq, p.total, p.bad);
        const int first = p.first[seq];
        int w = -1, at = 0;
        if (t >= span.begin && t - span.begin < span.len) {
            const long long pos = (long long)first + (t - span.begin);
            if (first >= 0 && pos < (long long)p.table.width * p.cache.page) {
                w = p.table.pages[seq * p.table.stride + pos / p.cache.page];
                at = (int)(pos % p.cache.page);
            }
            if (w < 0 || w >= p.cache.pages) {
                w = -1;
                if (lane == 0) seq_bad_index(p.bad);
            }
        }
        if (lane == 0) {
            where[i] = w;
            slot[i] = at;
        }
    }
    __syncthreads();
    // A thread keeps its place in a token (head and eight) and takes every n-th
    // token; places beyond the threads' number in further rounds.
    const int d8 = p.cache.d / 8, per = p.cache.kv_heads * d8;
    const int8_t* pages = blockIdx.y ? p.cache.v : p.cache.k;
    const float* scales = blockIdx.y ? p.cache.v_scales : p.cache.k_scales;
    const SeqTensor& dst = blockIdx.y ? p.v : p.k;
    const int every = max(1, kReadThreads / per), mine = every > 1 ? threadIdx.x / per : 0;
    if (mine >= every) return;
    for (int place = every > 1 ? threadIdx.x % per : threadIdx.x; place < per; place += kReadThreads) {
        const int head = place / d8, c = place % d8;
        const long long in_at = (long long)head * p.cache.page * p.cache.d + c * 8, out_at = head * dst.head_stride + c * 8;
        for (int i0 = mine; i0 < tokens; i0 += every * kReadAhead) {
            uint2 u[kReadAhead];
            float s[kReadAhead];
#pragma unroll
            for (int n = 0; n < kReadAhead; ++n) {
                const int i = i0 + n * every;
                if (i >= tokens || where[i] < 0) continue;
                s[n] = __ldg(scales + (long long)where[i] * p.cache.kv_heads + head);
                u[n] = __ldcs(reinterpret_cast<const uint2*>(
                    pages + ((long long)where[i] * p.cache.kv_heads * p.cache.page + slot[i]) * p.cache.d + in_at));
            }
#pragma unroll
            for (int n = 0; n < kReadAhead; ++n) {
                const int i = i0 + n * every;
                if (i >= tokens || where[i] < 0) continue;
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)((j < 4 ? u[n].x : u[n].y) >> (8 * (j & 3))) * s[n];
                store8(static_cast<T*>(dst.ptr) + (t0 + i) * dst.token_stride + out_at, vec, x);
            }
        }
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
    // A sequence's ids are two more than the pages it fills.
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
    if (p.dtype == DT_F32) cache_read_kernel<float><<<grid, kReadThreads, 0, stream>>>(p, vec);
    else cache_read_kernel<__nv_bfloat16><<<grid, kReadThreads, 0, stream>>>(p, vec);
    return cudaGetLastError();
}

}  // namespace ppocr
