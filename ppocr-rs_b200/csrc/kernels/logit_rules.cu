// Logit rules: penalties over each row's history, a bias per class and a
// grammar mask, in one pass over the logits.
//
// Bound: HBM, the logits read and written once (2 x element size per class).
// Without a history a thread owns VEC neighbouring columns and walks a group
// of rows, so the bias (and a mask shared by all rows) is read once per group
// and stays in registers; with a history a block owns one chunk of one row and
// counts the chunk's ids in shared memory first (integer counts, so the order
// of the atomics does not matter).
//
// Measured: 10,240 x 6,906 in FP32, bias and one mask: 113 us (5.0 TB/s; one row in
// flight per thread: 142); 64 x 128,000 in BF16 with histories of up to 4,000 ids:
// 20 us (1.7 TB/s; scalar reads of bias and counts: 26), where clearing, filling
// and reading the counts stand before and between the loads.
#include "seq_common.cuh"

namespace ppocr {

namespace {

constexpr int kThreads = 256;

// The mask bits of columns [v, v + VEC) (v a multiple of VEC, so they lie in
// one word), bit 0 first.
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* words, int v) { return __ldg(words + (v >> 5)) >> (v & 31); }

// The mask row of `row`: null when every class is allowed.
__device__ __forceinline__ const uint32_t* mask_row(const LogitRulesParams& p, int row) {
    if (!p.mask) return nullptr;
    const int state = p.mask_index ? p.mask_index[row] : 0;
    if (state < 0) {
        if (state != -1) seq_bad_index(p.bad);
        return nullptr;
    }
    if (state >= p.states) {
        seq_bad_index(p.bad);
        return nullptr;
    }
    return p.mask + (long long)state * p.mask_ld;
}

// Rows without a history: a block holds COLS vectors of columns per thread
// and rows y, y + gridDim.y, ...; kRowsAhead rows of them are in flight per
// thread, so that each SM has enough loads outstanding and what a row costs
// besides (its mask's state, addresses) is shared by the vectors.
constexpr int kRowsAhead = 4;
template <int VEC> constexpr int kRowCols = VEC == 8 ? 1 : 2;   // more would not fit the registers

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 5) logit_rules_rows_kernel(LogitRulesParams p) {
    constexpr int COLS = kRowCols<VEC>;
    const int v0 = (blockIdx.x * kThreads * COLS + threadIdx.x) * VEC;
    float bias[COLS][VEC];
    uint32_t bits0[COLS];
    const bool shared = !p.mask_index;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const int v = v0 + c * kThreads * VEC;
        bits0[c] = p.mask && shared && v < p.vocab ? mask_bits(p.mask, v) : ~0u;
#pragma unroll
        for (int j = 0; j < VEC; ++j) bias[c][j] = p.bias && v + j < p.vocab ? __ldg(p.bias + v + j) : 0.f;
    }
    for (int r0 = blockIdx.y; r0 < p.rows; r0 += kRowsAhead * (int)gridDim.y) {
        Pack<T, VEC> x[kRowsAhead][COLS];
        uint32_t bits[kRowsAhead][COLS];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
            const int r = r0 + i * (int)gridDim.y;
            if (r >= p.rows) continue;
            const T* in = static_cast<const T*>(p.logits) + r * p.ld;
            const uint32_t* m = shared ? nullptr : mask_row(p, r);
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const int v = v0 + c * kThreads * VEC;
                bits[i][c] = shared ? bits0[c] : m && v < p.vocab ? mask_bits(m, v) : ~0u;
                if (v + VEC <= p.vocab) x[i][c].load(in + v);
                else x[i][c].load_some(in + v, p.vocab - v);
            }
        }
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
            const int r = r0 + i * (int)gridDim.y;
            if (r >= p.rows) continue;
            T* out = static_cast<T*>(p.out) + r * p.out_ld;
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const int v = v0 + c * kThreads * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[i][c].put(j, (bits[i][c] >> j) & 1u ? x[i][c].get(j) + bias[c][j] : -INFINITY);
                if (v + VEC <= p.vocab) x[i][c].store(out + v);
                else x[i][c].store_some(out + v, p.vocab - v);
            }
        }
    }
}

// One chunk of one row with a history.  The first kAhead vectors of logits are
// on their way while the history is counted.
constexpr int kRowThreads = 512, kAhead = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads) logit_rules_history_kernel(LogitRulesParams p, int chunk) {
    extern __shared__ uint4 counts4[];
    uint32_t* counts = reinterpret_cast<uint32_t*>(counts4);
    const int row = blockIdx.y, lo = blockIdx.x * chunk, hi = min(lo + chunk, p.vocab);
    const T* in = static_cast<const T*>(p.logits) + row * p.ld;
    T* out = static_cast<T*>(p.out) + row * p.out_ld;
    auto load = [&](int v) {
        Pack<T, VEC> x;
        if (v + VEC <= hi) x.load(in + v);
        else x.load_some(in + v, hi - v);
        return x;
    };
    Pack<T, VEC> ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = load(lo + (threadIdx.x + i * kRowThreads) * VEC);
    const Span h = seq_span(p.history_offsets, 0, row, p.history_total, p.bad);
    const bool any = h.len > 0;
    if (any) {
        for (int i = threadIdx.x; i < (hi - lo + 3) / 4; i += kRowThreads) counts4[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < h.len; i += kRowThreads) {
            const int id = __ldg(p.history + h.begin + i);
            if (id >= lo && id < hi) atomicAdd(&counts[id - lo], 1u);
            else if (id < 0 || id >= p.vocab) seq_bad_index(p.bad);
        }
        __syncthreads();
    }
    const float rep = p.repetition ? p.repetition[row] : 1.f;
    const float pres = p.presence ? p.presence[row] : 0.f;
    const float freq = p.frequency ? p.frequency[row] : 0.f;
    const uint32_t* mask = mask_row(p, row);
    const bool bias4 = (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
    auto apply = [&](int v, Pack<T, VEC> x) {
        const int live = min(VEC, hi - v);
        const uint32_t bits = mask ? mask_bits(mask, v) : ~0u;
        // Bias and counts by fours where VEC has fours: a lane's neighbours are
        // VEC words on, so single words would meet in the same banks and sectors.
        float bias[VEC];
        uint32_t n[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            bias[j] = 0.f;
            n[j] = 0;
        }
        bool fours = false;
        if constexpr (VEC >= 4) {
            fours = live == VEC && bias4;
            if (fours) {
#pragma unroll
                for (int q = 0; q < VEC; q += 4) {
                    if (p.bias) {
                        const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + v + q));
                        bias[q] = b.x; bias[q + 1] = b.y; bias[q + 2] = b.z; bias[q + 3] = b.w;
                    }
                    if (any) {
                        const uint4 c = counts4[(v - lo + q) / 4];
                        n[q] = c.x; n[q + 1] = c.y; n[q + 2] = c.z; n[q + 3] = c.w;
                    }
                }
            }
        }
        if (!fours) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (j >= live) continue;
                if (p.bias) bias[j] = __ldg(p.bias + v + j);
                if (any) n[j] = counts[v - lo + j];
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float y = x.get(j);
            if (n[j]) {
                y = y > 0.f ? y / rep : y * rep;
                y = y - freq * (float)n[j] - pres;
            }
            x.put(j, (bits >> j) & 1u ? y + bias[j] : -INFINITY);
        }
        if (live == VEC) x.store(out + v);
        else x.store_some(out + v, live);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int v = lo + (threadIdx.x + i * kRowThreads) * VEC;
        if (v < hi) apply(v, ahead[i]);
    }
    for (int v = lo + (threadIdx.x + kAhead * kRowThreads) * VEC; v < hi; v += kRowThreads * VEC) apply(v, load(v));
}

template <typename T, int VEC>
cudaError_t launch_vec(const LogitRulesParams& p, cudaStream_t stream) {
    if (!p.history_offsets) {
        const int width = kThreads * VEC * kRowCols<VEC>, gx = (p.vocab + width - 1) / width;
        // One wave of five blocks per SM (a second, short one would double the
        // time), and no more than one group of rows each.
        const int gy = max(1, min((p.rows + kRowsAhead - 1) / kRowsAhead, 148 * 5 / gx));
        logit_rules_rows_kernel<T, VEC><<<dim3(gx, gy), kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    // Every block of a row reads the row's whole history, so a row is cut into
    // as few chunks as give about three blocks per SM, of 1,024 to 16,384
    // classes (64 KB of counts).
    const int parts = max((p.vocab + 16383) / 16384, min((p.vocab + 1023) / 1024, max(1, 148 * 3 / p.rows)));
    const int chunk = ((p.vocab + parts - 1) / parts + 63) / 64 * 64, smem = chunk * (int)sizeof(uint32_t);
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(logit_rules_history_kernel<T, VEC>), 16384 * 4);
    if (e != cudaSuccess) return e;
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
        logit_rules_history_kernel<T, VEC><<<dim3((p.vocab + chunk - 1) / chunk, q.rows), kRowThreads, smem, stream>>>(q, chunk);
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
