// Logit rules: penalties over each row's history, a bias per class and a
// grammar mask, in one pass over the logits.
//
// Bound: HBM, the logits read and written once (2 x element size per class).
// Without a history a thread owns VEC neighbouring columns and walks a group
// of rows, so the bias (and a mask shared by all rows) is read once per group
// and stays in registers; with a history a block owns one chunk of one row and
// counts the chunk's ids in shared memory first (integer counts, so the order
// of the atomics does not matter).
#include "seq_common.cuh"

namespace ppocr {

namespace {

constexpr int kThreads = 256;

template <typename T, int VEC> struct VecType;
template <> struct VecType<float, 4> { using type = uint4; };
template <> struct VecType<float, 2> { using type = uint2; };
template <> struct VecType<float, 1> { using type = uint32_t; };
template <> struct VecType<__nv_bfloat16, 8> { using type = uint4; };
template <> struct VecType<__nv_bfloat16, 4> { using type = uint2; };
template <> struct VecType<__nv_bfloat16, 2> { using type = uint32_t; };
template <> struct VecType<__nv_bfloat16, 1> { using type = uint16_t; };

// The mask bits of columns [v, v + VEC) (v a multiple of VEC, so they lie in
// one word), bit 0 first.
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* words, int v) { return __ldg(words + (v >> 5)) >> (v & 31); }

// The mask row of `row`: null when every class is allowed.
__device__ __forceinline__ const uint32_t* mask_row(const LogitRulesParams& p, int row) {
    if (!p.mask) return nullptr;
    const int state = p.mask_index ? p.mask_index[row] : 0;
    if (state < 0) {
        if (state != -1) seq_bad_index(p.status);
        return nullptr;
    }
    if (state >= p.states) {
        seq_bad_index(p.status);
        return nullptr;
    }
    return p.mask + (long long)state * p.mask_ld;
}

// Rows are independent and without a history: block (x, y) holds columns
// [x, x + 1) x kThreads x VEC and rows y, y + gridDim.y, ...; four rows are in
// flight per thread so that each SM has enough loads outstanding.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) logit_rules_rows_kernel(LogitRulesParams p) {
    using V = typename VecType<T, VEC>::type;
    constexpr int ROWS = 4;
    const int v = (blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (v >= p.vocab) return;
    const int live = min(VEC, p.vocab - v);
    float bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) bias[j] = p.bias && j < live ? __ldg(p.bias + v + j) : 0.f;
    const bool shared = !p.mask_index;
    const uint32_t bits0 = p.mask && shared ? mask_bits(p.mask, v) : ~0u;
    const T* in = static_cast<const T*>(p.logits) + v;
    T* out = static_cast<T*>(p.out) + v;
    for (int r0 = blockIdx.y; r0 < p.rows; r0 += ROWS * gridDim.y) {
        V x[ROWS];
        uint32_t bits[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = r0 + i * gridDim.y;
            bits[i] = bits0;
            if (r >= p.rows) continue;
            const T* src = in + r * p.ld;
            if (live == VEC) {
                x[i] = __ldcs(reinterpret_cast<const V*>(src));
            } else {
                T* e = reinterpret_cast<T*>(&x[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j < live) e[j] = src[j];
            }
            if (!shared) {
                const uint32_t* m = mask_row(p, r);
                if (m) bits[i] = mask_bits(m, v);
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = r0 + i * gridDim.y;
            if (r >= p.rows) continue;
            T* e = reinterpret_cast<T*>(&x[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float y = to_f(e[j]) + bias[j];
                e[j] = from_f<T>((bits[i] >> j) & 1u ? y : -INFINITY);
            }
            T* dst = out + r * p.out_ld;
            if (live == VEC) {
                __stcs(reinterpret_cast<V*>(dst), x[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (j < live) dst[j] = e[j];
            }
        }
    }
}

// One chunk of one row with a history.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) logit_rules_history_kernel(LogitRulesParams p, int chunk) {
    using V = typename VecType<T, VEC>::type;
    extern __shared__ uint32_t counts[];
    const int row = blockIdx.y, lo = blockIdx.x * chunk, hi = min(lo + chunk, p.vocab);
    const Span h = seq_span(p.history_offsets, 0, row, p.history_total, p.status);
    const bool any = h.len > 0;
    if (any) {
        for (int i = threadIdx.x; i < hi - lo; i += kThreads) counts[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < h.len; i += kThreads) {
            const int id = __ldg(p.history + h.begin + i);
            if (id >= lo && id < hi) atomicAdd(&counts[id - lo], 1u);
            else if (id < 0 || id >= p.vocab) seq_bad_index(p.status);
        }
        __syncthreads();
    }
    const float rep = p.repetition ? p.repetition[row] : 1.f;
    const float pres = p.presence ? p.presence[row] : 0.f;
    const float freq = p.frequency ? p.frequency[row] : 0.f;
    const uint32_t* mask = mask_row(p, row);
    const T* in = static_cast<const T*>(p.logits) + row * p.ld;
    T* out = static_cast<T*>(p.out) + row * p.out_ld;
    for (int v = lo + threadIdx.x * VEC; v < hi; v += kThreads * VEC) {
        const int live = min(VEC, hi - v);
        V x;
        T* e = reinterpret_cast<T*>(&x);
        if (live == VEC) {
            x = __ldcs(reinterpret_cast<const V*>(in + v));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < live) e[j] = in[v + j];
        }
        const uint32_t bits = mask ? mask_bits(mask, v) : ~0u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (j >= live) continue;
            float y = to_f(e[j]);
            const uint32_t n = any ? counts[v - lo + j] : 0u;
            if (n) {
                y = y > 0.f ? y / rep : y * rep;
                y = y - freq * (float)n - pres;
            }
            if (p.bias) y += __ldg(p.bias + v + j);
            e[j] = from_f<T>((bits >> j) & 1u ? y : -INFINITY);
        }
        if (live == VEC) {
            __stcs(reinterpret_cast<V*>(out + v), x);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < live) out[v + j] = e[j];
        }
    }
}

template <typename T, int VEC>
cudaError_t launch_vec(const LogitRulesParams& p, cudaStream_t stream) {
    if (!p.history_offsets) {
        const int gx = (p.vocab + kThreads * VEC - 1) / (kThreads * VEC);
        // About eight blocks per SM in all, and no more than one row group each.
        const int gy = max(1, min((p.rows + 3) / 4, (148 * 8 + gx - 1) / gx));
        logit_rules_rows_kernel<T, VEC><<<dim3(gx, gy), kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    // A chunk's counts fit 16 KB, so the blocks of an SM are bound by threads.
    const int chunk = 4096;
    for (int r0 = 0; r0 < p.rows; r0 += 65535) {
        LogitRulesParams q = p;
        q.rows = min(65535, p.rows - r0);
        q.logits = static_cast<const T*>(p.logits) + r0 * p.ld;
        q.out = static_cast<T*>(p.out) + r0 * p.out_ld;
        q.history_offsets = p.history_offsets + r0;
        if (p.repetition) q.repetition = p.repetition + r0;
        if (p.presence) q.presence = p.presence + r0;
        if (p.frequency) q.frequency = p.frequency + r0;
        if (p.mask_index) q.mask_index = p.mask_index + r0;
        logit_rules_history_kernel<T, VEC><<<dim3((p.vocab + chunk - 1) / chunk, q.rows), kThreads,
                                             chunk * sizeof(uint32_t), stream>>>(q, chunk);
    }
    return cudaGetLastError();
}

// Bytes every row's start is aligned to, in input and output.
int row_alignment(const LogitRulesParams& p, int esize) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.out) |
                           (uintptr_t)(p.ld * esize) | (uintptr_t)(p.out_ld * esize) | 16;
    return (int)(bits & (~bits + 1));
}

}  // namespace

cudaError_t launch_logit_rules(const LogitRulesParams& p, cudaStream_t stream) {
    if (p.rows == 0 || p.vocab == 0) return cudaSuccess;
    if (p.dtype == DT_F32) {
        switch (row_alignment(p, 4)) {
            case 16: return launch_vec<float, 4>(p, stream);
            case 8: return launch_vec<float, 2>(p, stream);
            default: return launch_vec<float, 1>(p, stream);
        }
    }
    switch (row_alignment(p, 2)) {
        case 16: return launch_vec<__nv_bfloat16, 8>(p, stream);
        case 8: return launch_vec<__nv_bfloat16, 4>(p, stream);
        case 4: return launch_vec<__nv_bfloat16, 2>(p, stream);
        default: return launch_vec<__nv_bfloat16, 1>(p, stream);
    }
}

}  // namespace ppocr
