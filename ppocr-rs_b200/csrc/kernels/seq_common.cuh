// Device helpers shared by the sequence operators: clamped offsets, the
// search for a block's sequence, error reporting.
#pragma once

#include "common.cuh"
#include "seq.h"

namespace ppocr {

__device__ __forceinline__ void seq_bad_index(int* bad) {
    if (bad) *reinterpret_cast<volatile int*>(bad) = 1;
}

struct Span {
    int begin, len;
};

// Tokens [begin, begin + len) of sequence i, clamped to [0, total); a negative,
// decreasing or too large offset is reported.
__device__ __forceinline__ Span seq_span(const int32_t* offsets, int uniform, int i, int total, int* bad) {
    if (!offsets) return Span{i * uniform, uniform};
    const int b = offsets[i], e = offsets[i + 1];
    if (b < 0 || e < b || e > total) seq_bad_index(bad);
    const int cb = min(max(b, 0), total);
    return Span{cb, min(max(e, cb), total) - cb};
}

// Reports bad offsets of any sequence: with offsets that fall inside a longer
// list, find_owner passes over sequences, whose blocks then look at no offset.
// The grid's first blocks take the sequences by turns; nothing waits for it.
__device__ __forceinline__ void check_offsets(const int32_t* offsets, int sequences, int total, int* bad) {
    if ((long long)blockIdx.x * blockDim.x >= sequences || (blockIdx.y | blockIdx.z) != 0 || !offsets) return;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < sequences; i += (long long)gridDim.x * blockDim.x) {
        const int b = __ldg(offsets + i), e = __ldg(offsets + i + 1);
        if (b < 0 || e < b || e > total) seq_bad_index(bad);
    }
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

// VEC values of T as 32-bit words (a lone BF16 in the low half of one), read and
// written 2, 4, 8 or 16 bytes at a time, 32 in two halves.  Words, so that they
// stay in registers: an array of T seen through a pointer goes to local memory.
template <typename T, int VEC>
struct Pack {
    static constexpr int kBytes = VEC * (int)sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p) {   // aligned to its size (16 at most), streamed
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
            }
        } else if constexpr (kBytes == 8) {
            const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
            w[0] = u.x; w[1] = u.y;
        } else if constexpr (kBytes == 4) {
            w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
        } else {
            w[0] = __ldcs(reinterpret_cast<const uint16_t*>(p));
        }
    }
    // The first `live` values one by one, zeros behind them.
    __device__ __forceinline__ void load_some(const T* p, int live) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) put(j, j < live ? to_f(p[j]) : 0.f);
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i)
                __stcs(reinterpret_cast<uint4*>(p) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
        } else if constexpr (kBytes == 8) {
            __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
        } else if constexpr (kBytes == 4) {
            __stcs(reinterpret_cast<uint32_t*>(p), w[0]);
        } else {
            __stcs(reinterpret_cast<uint16_t*>(p), (uint16_t)w[0]);
        }
    }
    __device__ __forceinline__ void store_some(T* p, int live) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (j < live) p[j] = from_f<T>(get(j));
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
    __device__ __forceinline__ void put(int j, float x) {
        if constexpr (sizeof(T) == 4) {
            w[j] = __float_as_uint(x);
        } else {
            const uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rn(x));
            w[j / 2] = j & 1 ? __byte_perm(w[j / 2], b, 0x5410) : __byte_perm(b, w[j / 2], 0x7610);   // the other half stays
        }
    }
};

__device__ __forceinline__ float power(int e) { return __int_as_float((127 + e) << 23); }   // 2^e, -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return (__float_as_int(x) >> 23) - 127; }   // of x >= 0

// 2^x by the hardware unit (relative error about 2^-22; 0 for -infinity).
__device__ __forceinline__ float exp2_hw(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ppocr
