// Shared by the packed attention kernels: the row of queries a tile row
// stands for, and the careful row.
#pragma once

#include "seq_common.cuh"

namespace ppocr {

// One row, one warp, from its definition: no key past `keys` is read.  The
// tiled kernels multiply the zero weights of masked keys with those keys'
// values, so an infinity or NaN among masked values of a tile spoils rows that
// must not see it; a row that came out non-finite is computed again here.
template <typename T>
__device__ __noinline__ void attend_row(const T* q, const T* k, long long k_stride, const T* v, long long v_stride, int d,
                                        int keys, float scale_log2, T* out) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY;
    bool nan = false;
    for (int j = lane; j < keys; j += 32) {
        float s = 0.f;
        for (int x = 0; x < d; ++x) s = fmaf(to_f(q[x]), to_f(k[j * k_stride + x]), s);
        s *= scale_log2;
        nan |= isnan(s);
        top = fmaxf(top, s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    nan = __any_sync(0xffffffffu, nan) || top == INFINITY;
    float acc[kPackedMaxD / 32] = {}, sum = 0.f;
    if (!nan && top != -INFINITY) {
        for (int j = 0; j < keys; ++j) {
            float s = 0.f;
            for (int x = lane; x < d; x += 32) s = fmaf(to_f(q[x]), to_f(k[j * k_stride + x]), s);
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const float w = exp2_hw(s * scale_log2 - top);
            sum += w;
#pragma unroll
            for (int i = 0; i < kPackedMaxD / 32; ++i)
                if (lane + 32 * i < d) acc[i] = fmaf(w, to_f(v[j * v_stride + lane + 32 * i]), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPackedMaxD / 32; ++i)
        if (lane + 32 * i < d) out[lane + 32 * i] = from_f<T>(nan ? NAN : sum == 0.f ? 0.f : acc[i] / sum);
}

// Whether every row of a tensor starts on a 16-byte boundary.
inline bool rows16(const SeqTensor& t, int esize) {
    return ((reinterpret_cast<uintptr_t>(t.ptr) | (uintptr_t)(t.token_stride * esize) | (uintptr_t)(t.head_stride * esize)) & 15) == 0;
}

}  // namespace ppocr
