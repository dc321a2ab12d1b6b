// Shared by the packed attention kernels: the row of queries a tile row
// stands for, and the careful row.
#pragma once

#include "seq_common.cuh"

namespace ppocr {

// One row, one warp, from its definition: no key past `keys` is read.  The
// tiled kernels multiply the zero weights of masked keys with those keys'
// values, so an infinity or NaN among masked values of a tile spoils rows that
// must not see it; a row that came out non-finite is computed again here, and so
// is one whose scores are too large for its kernel's weights.
template <typename T>
__device__ __noinline__ void attend_row(const T* q, const T* k, long long k_stride, const T* v, long long v_stride, int d,
                                        int keys, float scale_log2, T* out) {
    const int lane = threadIdx.x & 31;
    // Both passes compute a score in the same steps: where its rounding is worth
    // more than a power of two, the largest one's weight is 1 all the same.
    auto score = [&](int j) {
        float s = 0.f;
        for (int x = 0; x < d; ++x) s = fmaf(to_f(q[x]), to_f(k[j * k_stride + x]), s);
        return __fmul_rn(s, scale_log2);
    };
    float top = -INFINITY;
    bool nan = false;
    for (int j = lane; j < keys; j += 32) {
        const float s = score(j);
        nan |= isnan(s);
        top = fmaxf(top, s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    nan = __any_sync(0xffffffffu, nan) || top == INFINITY;
    float acc[kPackedMaxD / 32] = {}, sum = 0.f;
    if (!nan && top != -INFINITY) {
        for (int j0 = 0; j0 < keys; j0 += 32) {
            const float w = j0 + lane < keys ? exp2_hw(score(j0 + lane) - top) : 0.f;
            for (int j = j0; j < min(j0 + 32, keys); ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j - j0);
                sum += wj;
#pragma unroll
                for (int i = 0; i < kPackedMaxD / 32; ++i)
                    if (lane + 32 * i < d) acc[i] = fmaf(wj, to_f(v[j * v_stride + lane + 32 * i]), acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPackedMaxD / 32; ++i)
        if (lane + 32 * i < d) out[lane + 32 * i] = from_f<T>(nan ? NAN : sum == 0.f ? 0.f : acc[i] / sum);
}

// Kernels that take the scale in the exponent's multiply-add hold weights relative
// to the rounded product of largest score and scale, so a row's weights share a
// factor of 2^(that rounding's error).  Up to a product of 2^24 it is at most 2^1;
// near 2^31 it can pass FP32's range either way, where a finite result may be
// wrong.  Rows beyond 2^24 are computed again from their definition.
__device__ __forceinline__ bool rounding_spoils(float top) { return top != -INFINITY && fabsf(top) > 16777216.f; }

// A block's piece of the mma.sync kernels: up to ROWS rows (row = query token x
// group + head) of one (sequence, KV head).
template <int ROWS>
struct PackedPiece {
    Span qs, ks;
    int kv, group, rows;       // rows <= 0: nothing to do
    int token0, part0, shift;  // row n is query token0 + (part0 + n) / group; causal: query i sees keys j <= i + shift
    bool causal;

    __device__ __forceinline__ explicit PackedPiece(const PackedAttentionParams& p) {
        group = p.heads / p.kv_heads;
        kv = blockIdx.x % p.kv_heads;
        causal = p.causal;
        if ((long long)blockIdx.x * blockDim.x < p.sequences) {
            check_offsets(p.q_offsets, p.sequences, p.total_q, p.bad);
            check_offsets(p.k_offsets, p.sequences, p.total_k, p.bad);
        }
        // The longest rows of a causal sequence are dealt first.
        const long long pieces = gridDim.x / p.kv_heads, at_id = blockIdx.x / p.kv_heads;
        const long long id = causal ? pieces - 1 - at_id : at_id;
        auto first_id = [&](int i) { return (long long)seq_offset(p.q_offsets, p.uniform, i, p.total_q) * group / ROWS + i; };
        const int seq = find_owner(p.sequences, id, first_id);
        qs = seq_span(p.q_offsets, p.uniform, seq, p.total_q, p.bad);
        ks = seq_span(p.k_offsets, p.uniform, seq, p.total_k, p.bad);
        const long long row0 = (id - first_id(seq)) * ROWS, all = (long long)qs.len * group;
        rows = row0 < 0 ? 0 : (int)max(min((long long)ROWS, all - row0), 0ll);
        shift = ks.len - qs.len;
        // Divisions of 64 bits cost as much as a tile of keys.
        token0 = (int)(group == 1 ? row0 : row0 >> 32 ? row0 / group : (unsigned)row0 / (unsigned)group);
        part0 = (int)(row0 - (long long)token0 * group);
    }
    __device__ __forceinline__ int token_of(int n) const { return group == 1 ? n : (part0 + n) / group; }
    __device__ __forceinline__ int keys_of(int n) const {
        return causal ? min(max(token0 + token_of(n) + shift + 1, 0), ks.len) : ks.len;
    }
    template <typename T>
    __device__ __forceinline__ T* queries(const SeqTensor& t) const {
        return static_cast<T*>(t.ptr) + (qs.begin + (long long)token0) * t.token_stride + (long long)kv * group * t.head_stride;
    }
    template <typename T>
    __device__ __forceinline__ const T* keys(const SeqTensor& t) const {
        return static_cast<const T*>(t.ptr) + (long long)ks.begin * t.token_stride + kv * t.head_stride;
    }
    __device__ __forceinline__ long long row_at(const SeqTensor& t, int n) const {
        const int token = token_of(n);   // strides are at most 2^30: products of 32 bits
        return (long long)token * (int)t.token_stride + (long long)(part0 + n - token * group) * (int)t.head_stride;
    }
    // Blocks of a launch: sequence i owns the ids from floor(offset_i group / ROWS) + i, at least its number of pieces.
    static long long blocks(const PackedAttentionParams& p) {
        return ((long long)p.total_q * (p.heads / p.kv_heads) / ROWS + p.sequences) * p.kv_heads;
    }
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool live) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool live) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}

// Whether pairs of a tensor's values are aligned to their size.
inline bool pairs_aligned(const SeqTensor& t, int esize) {
    return ((reinterpret_cast<uintptr_t>(t.ptr) | (uintptr_t)(t.token_stride * esize) | (uintptr_t)(t.head_stride * esize)) %
            (2 * esize)) == 0;
}

// Whether every row of a tensor starts on a 16-byte boundary.
inline bool rows16(const SeqTensor& t, int esize) {
    return ((reinterpret_cast<uintptr_t>(t.ptr) | (uintptr_t)(t.token_stride * esize) | (uintptr_t)(t.head_stride * esize)) & 15) == 0;
}

}  // namespace ppocr
