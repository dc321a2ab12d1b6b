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
// i by at least i's number of pieces (some ids then own no piece).  The owner
// of `id` is found by bisection; every thread gets the answer.
template <typename First>
__device__ __forceinline__ int find_owner(int sequences, long long id, First first) {
    int lo = 0, hi = sequences;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first(mid) <= id) lo = mid; else hi = mid;
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
