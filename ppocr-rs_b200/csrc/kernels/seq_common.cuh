// Device helpers shared by the sequence operators: clamped offsets, the
// search for a block's sequence, error reporting.
#pragma once

#include "common.cuh"
#include "seq.h"

namespace ppocr {

__device__ __forceinline__ void seq_bad_index(int* status) {
    if (status) *reinterpret_cast<volatile int*>(status) = SEQ_BAD_INDEX;
}

struct Span {
    int begin, len;
};

// Tokens [begin, begin + len) of sequence i, clamped to [0, total); a negative,
// decreasing or too large offset is reported.
__device__ __forceinline__ Span seq_span(const int32_t* offsets, int uniform, int i, int total, int* status) {
    if (!offsets) return Span{i * uniform, uniform};
    const int b = offsets[i], e = offsets[i + 1];
    if (b < 0 || e < b || e > total) seq_bad_index(status);
    const int cb = min(max(b, 0), total);
    return Span{cb, min(max(e, cb), total) - cb};
}

// Deals ids to the sequences without a prefix sum: sequence i owns the ids
// [first(i), first(i + 1)), where first() needs i's offset alone and grows with
// i by at least i's number of pieces (some ids then own no piece).  A converged
// warp finds the owner of `id`, 32 sequences a round: one round trip to memory
// for up to 32 sequences, two for 1,024.
template <typename Id, typename First>
__device__ __forceinline__ int find_owner(int sequences, Id id, First first) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = sequences;   // the owner is one of [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const unsigned mask = __ballot_sync(0xffffffffu, at < n && first(lo + at) <= id) | 1u;
        const int skip = (31 - __clz(mask)) * step;
        lo += skip;
        n = min(step, n - skip);
    }
    return lo;
}

// Offset i, clamped to [0, total].
__device__ __forceinline__ int seq_offset(const int32_t* offsets, int uniform, int i, int total) {
    return offsets ? min(max(__ldg(offsets + i), 0), total) : i * uniform;
}

// 2^x by the hardware unit (relative error about 2^-22; 0 for -infinity).
__device__ __forceinline__ float exp2_hw(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ppocr
