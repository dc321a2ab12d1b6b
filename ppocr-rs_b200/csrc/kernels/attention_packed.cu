// Attention over packed sequences on mma.sync (BF16): every head size up to
// 128, stride and length; the kernel of the short sequences, whose tiles are
// too small to fill a tcgen05 tile (128 rows) or to pay for its set-up.
//
// A block owns 64 rows of one (sequence, KV head): the `group` query heads
// that share the KV head are rows too (row = token x group + head), so K and V
// are read once per group.  Keys pass through shared memory in tiles, double
// buffered with cp.async, with the running maximum and sum of the softmax in
// registers; scores and weights never leave them.  Weights are rounded to BF16
// for the second product (2^-8 of a weight at most, averaged over the keys; the
// sum uses the unrounded ones).  Rows with no key give zeros; a non-finite row
// and one of scores beyond 2^24 is computed again from its definition (attend_row).
//
// Short lines are bound by latency: a block waits for its sequence's offsets,
// then for its tiles, and computes for a short while, so what counts is how
// many blocks an SM holds.  256 lines of 20 to 160 tokens, 8 heads of 24
// (35 MB, 5.4 us at the copy rate): 45.7 us with six blocks per SM, 48.9 with
// five, 57.9 with eight (registers spilled).  The issue slots are then 70 % busy, so
// instructions count next: with the scale in the exponent's multiply-add, masks only
// where a tile needs them and 32-bit divisions and strides, 41.8 us.
#include "attention_packed.cuh"

namespace ppocr {

namespace {

using T = __nv_bfloat16;

constexpr int kThreads = 128, kRows = 64, kKeys = 64, kPad = 8;
using Piece = PackedPiece<kRows>;

__device__ __forceinline__ void mma_bf16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Rows [0, rows) of `src` into shared memory at pitch DP + pad, zeros past
// them and past column d; row n of the tile is at src + at(n).
template <int DP, typename At>
__device__ __forceinline__ void load_tile(T* dst, const T* src, At at, int tile_rows, int rows, int d, bool vec) {
    constexpr int P = DP + kPad;
    if (vec) {
        constexpr int E = 16 / sizeof(T), C = DP / E;
        for (int i = threadIdx.x; i < tile_rows * C; i += kThreads) {
            const int n = i / C, x = (i % C) * E;
            const bool live = n < rows && x < d;
            cp_async16(dst + n * P + x, live ? src + at(n) + x : src, live);
        }
    } else {
        for (int i = threadIdx.x; i < tile_rows * DP; i += kThreads) {
            const int n = i / DP, x = i % DP;
            dst[n * P + x] = n < rows && x < d ? src[at(n) + x] : from_f<T>(0.f);
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads, DP > 64 ? 3 : DP > 32 ? 4 : 6)
    attention_packed_kernel(PackedAttentionParams p, bool vec, bool vec_out) {
    constexpr int BN = kKeys, P = DP + kPad, NT = BN / 8, DT = DP / 8;
    extern __shared__ uint4 smem16[];
    T* sq = reinterpret_cast<T*>(smem16);
    T* sk = sq + kRows * P;              // two stages
    T* sv = sk + 2 * BN * P;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const Piece at(p);
    const int rows = at.rows, d = p.d;
    if (rows <= 0) return;
    const int keys = at.keys_of(rows - 1);
    const int tiles = (keys + BN - 1) / BN;

    const T* q = at.queries<T>(p.q);
    const T* k = at.keys<T>(p.k);
    const T* v = at.keys<T>(p.v);
    load_tile<DP>(sq, q, [&](int n) { return at.row_at(p.q, n); }, kRows, rows, d, vec);
    auto load_keys = [&](int j) {
        const int n = min(BN, keys - j * BN);
        const T* kt = k + (long long)j * BN * p.k.token_stride;
        const T* vt = v + (long long)j * BN * p.v.token_stride;
        load_tile<DP>(sk + (j & 1) * BN * P, kt, [&](int i) { return (long long)i * (int)p.k.token_stride; }, BN, n, d, vec);
        load_tile<DP>(sv + (j & 1) * BN * P, vt, [&](int i) { return (long long)i * (int)p.v.token_stride; }, BN, n, d, vec);
    };
    if (tiles > 0) load_keys(0);
    cp_async_commit();

    const float scale = p.scale * 1.4426950408889634f;
    const int n0 = warp * 16 + r;                  // this lane's rows: n0 and n0 + 8
    const int keys0 = at.keys_of(min(n0, rows - 1)), keys1 = at.keys_of(min(n0 + 8, rows - 1));
    const int sure = __reduce_min_sync(0xffffffffu, (unsigned)min(keys0, keys1));   // keys every row of the warp sees
    const int most = n0 - r < rows ? (int)__reduce_max_sync(0xffffffffu, (unsigned)max(keys0, keys1)) : 0;
    float o[DT][4];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    uint32_t qf[DP / 16][4];

    for (int j = 0; j < tiles; ++j) {
        if (j + 1 < tiles) load_keys(j + 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        const T* kt = sk + (j & 1) * BN * P;
        const T* vt = sv + (j & 1) * BN * P;
        // Eights of keys that some row of the warp sees (0 for a warp without
        // rows): lines are short, and tiles seldom full.
        const int seen = min(NT, (most - j * BN + 7) / 8);
        if (seen <= 0) {
            __syncthreads();
            continue;
        }
        float s[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[i][x] = 0.f;
        if (j == 0) {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) ldmatrix4(qf[i], sq + (warp * 16 + (lane & 15)) * P + i * 16 + (lane >> 4) * 8);
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            if (n >= seen) break;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                uint32_t b[4];
                ldmatrix4(b, kt + (n * 8 + (lane & 7) + (lane >> 4) * 8) * P + i * 16 + ((lane >> 3) & 1) * 8);
                mma_bf16_16816(s[n], qf[i], b[0], b[1]);
                mma_bf16_16816(s[n + 1], qf[i], b[2], b[3]);
            }
        }
        // Mask, running maximum (of the products; the scale, which is positive,
        // comes with the exponent's subtraction).
        float t0 = -INFINITY, t1 = -INFINITY;
        if ((j + 1) * BN > sure) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n >= (seen + 1) / 2 * 2) break;   // they come in pairs
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int key = j * BN + n * 8 + 2 * c + x;
                    if (key >= keys0) s[n][x] = -INFINITY;
                    if (key >= keys1) s[n][x + 2] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n >= (seen + 1) / 2 * 2) break;
            t0 = fmaxf(t0, fmaxf(s[n][0], s[n][1]));
            t1 = fmaxf(t1, fmaxf(s[n][2], s[n][3]));
        }
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(m0, fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)));
        t1 = fmaxf(m1, fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2)));
        const float b0 = t0 == -INFINITY ? 0.f : __fmul_rn(t0, scale), b1 = t1 == -INFINITY ? 0.f : __fmul_rn(t1, scale);
        // 0 while the maximum is -infinity; the products as they were rounded for the weights so far.
        const float g0 = exp2_hw(__fmul_rn(m0, scale) - b0), g1 = exp2_hw(__fmul_rn(m1, scale) - b1);
        m0 = t0;
        m1 = t1;
        l0 *= g0;
        l1 *= g1;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            o[i][0] *= g0; o[i][1] *= g0;
            o[i][2] *= g1; o[i][3] *= g1;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n >= (seen + 1) / 2 * 2) break;
            s[n][0] = exp2_hw(fmaf(s[n][0], scale, -b0)); s[n][1] = exp2_hw(fmaf(s[n][1], scale, -b0));
            s[n][2] = exp2_hw(fmaf(s[n][2], scale, -b1)); s[n][3] = exp2_hw(fmaf(s[n][3], scale, -b1));
            l0 += s[n][0] + s[n][1];
            l1 += s[n][2] + s[n][3];
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            if (n >= seen) break;
            uint32_t a[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(s[n + (x >> 1)][2 * (x & 1)], s[n + (x >> 1)][2 * (x & 1) + 1]);
                a[x] = *reinterpret_cast<const uint32_t*>(&h);
            }
#pragma unroll
            for (int i = 0; i < DT; i += 2) {
                uint32_t b[4];
                ldmatrix4_trans(b, vt + (n * 8 + (lane & 15)) * P + i * 8 + (lane >> 4) * 8);
                mma_bf16_16816(o[i], a, b[0], b[1]);
                mma_bf16_16816(o[i + 1], a, b[2], b[3]);
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const float i0 = m0 == -INFINITY ? 0.f : 1.f / l0, i1 = m1 == -INFINITY ? 0.f : 1.f / l1;
    T* out = at.queries<T>(p.out);
    bool bad[2] = {false, false};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int n = n0 + 8 * half;
        if (n >= rows) continue;
        T* dst = out + at.row_at(p.out, n);
        float odd = 0.f;   // stays 0, or becomes NaN
        const float inv = half ? i1 : i0;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int x = i * 8 + 2 * c;
            const float a = o[i][2 * half] * inv, b = o[i][2 * half + 1] * inv;
            odd = fmaf(a, 0.f, fmaf(b, 0.f, odd));   // columns past d hold zeros
            if (vec_out && x + 1 < d) {
                *reinterpret_cast<__nv_bfloat162*>(dst + x) = __floats2bfloat162_rn(a, b);
            } else {
                if (x < d) dst[x] = from_f<T>(a);
                if (x + 1 < d) dst[x + 1] = from_f<T>(b);
            }
        }
        bad[half] = odd != 0.f || rounding_spoils((half ? m1 : m0) * scale);
    }
    // Rows with a non-finite value or too large scores again, by their definition,
    // after the warp's own stores above.  A row is shared by four lanes.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const unsigned again = __ballot_sync(0xffffffffu, bad[half]);
        for (int rr = 0; again && rr < 8; ++rr) {
            if (!(again >> (4 * rr) & 0xfu)) continue;
            const int n = warp * 16 + rr + 8 * half;
            __syncwarp();
            attend_row<T>(q + at.row_at(p.q, n), k, p.k.token_stride, v, p.v.token_stride, d, at.keys_of(n), scale,
                          out + at.row_at(p.out, n));
        }
    }
}

template <int DP>
cudaError_t launch_dp(const PackedAttentionParams& p, cudaStream_t stream) {
    const int esize = sizeof(T);
    const bool vec = rows16(p.q, esize) && rows16(p.k, esize) && rows16(p.v, esize) && p.d * esize % 16 == 0;
    constexpr int smem = (kRows + 4 * kKeys) * (DP + kPad) * (int)sizeof(T);
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(attention_packed_kernel<DP>), smem);
    if (e != cudaSuccess) return e;
    attention_packed_kernel<DP><<<(unsigned)Piece::blocks(p), kThreads, smem, stream>>>(p, vec, pairs_aligned(p.out, esize));
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_packed(const PackedAttentionParams& p, cudaStream_t stream) {
    if (p.total_q == 0 || p.sequences == 0) return cudaSuccess;
    if (p.dtype == DT_F32) return launch_attention_packed_f32(p, stream);
    // tcgen05 from 16,384 keys x (padded) values per sequence on, 24,576 where its
    // 64 values to a row are half empty.  Measured on 16,384 tokens in causal
    // sequences of equal length, mma.sync / tcgen05 in us:
    //   8 heads of 24           length 384: 38 / 57, 512: 47 / 55, 1,024: 78 / 67
    //   16 of 64, 4 KV heads    length 128: 64 / 72, 192: 74 / 73, 256: 85 / 74
    //   8 of 128                length 96: 78 / 84, 128: 67 / 68, 512: 131 / 64
    //   32 of 128, 8 KV heads   length 64: 216 / 171, 128: 252 / 158
    const int padded = p.d <= 16 ? 16 : p.d <= 32 ? 32 : p.d <= 64 ? 64 : 128;
    const long long least = padded <= 32 ? 24576 : 16384;
    if ((long long)p.total_k * padded >= least * p.sequences && attention_tc_supported(p)) return launch_attention_tc(p, stream);
    if (p.d <= 16) return launch_dp<16>(p, stream);
    if (p.d <= 32) return launch_dp<32>(p, stream);
    if (p.d <= 64) return launch_dp<64>(p, stream);
    return launch_dp<128>(p, stream);
}

}  // namespace ppocr
