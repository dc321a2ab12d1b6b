// Attention over packed sequences in FP32, on mma.sync m16n8k16 with FP16
// operands: every head size up to 128, stride and length.
//
// Every value is carried as two FP16 pieces (22 bits) of the value times a
// power of two, and a product as its three leading ones: FP32-class, at half
// the tensor-core time of TF32 pieces (whose MMAs hold half the values).  FP16's
// range is met by one power of two per row of Q, K and V, the one that takes the
// row's largest magnitude into [2^14, 2^15): Q's and K's multiply the scores, and
// V's the weights before these are split in turn.  A row's own power, and not a
// tile's, so that a key which a query must not see cannot touch its precision.
// Second pieces are held times 2^11 and their products summed apart: so FP16's
// least step cuts a value at 2^-50 of its row's largest, and one down to 2^-28 of
// it, a channel next to a far larger one, has its 22 bits.  (With both pieces in
// the same power that ended at 2^-16, and 2^-30 kept four bits.)
//
// A block owns 64 rows of one (sequence, KV head): the `group` query heads
// that share the KV head are rows too, so K and V are read once per group.
// Keys come in tiles of 32: cp.async brings the FP32 values, each thread splits
// those that it fetched itself (once per block, where the warps would otherwise
// each split what they read) into FP16 planes in shared memory, and the copies
// of the next tile run while the warps work on the planes.
//
// The tensor cores truncate when they add to an accumulator, so chains are
// short: two steps of 16 for the leading products, and their sums are added
// with rounding.
//
// Bound: the tensor cores (three products) together with splitting, 1 us of
// every 4 where it stood between two barriers; with eight warps one half of
// them splits the next tile while the other half multiplies (95 -> 89 us).
// Chunks of 3 requests, 16 heads of 64, 4 KV heads: 80 to 85 us (second pieces in
// the first ones' power: 1 us less; TF32 pieces split by each warp: 165).  64 lines
// of 4 to 200 tokens, 8 heads of 15: 28 us, latency.
//
// Softmax: weights are relative to the maximum + 4 (in log2) when it last moved,
// and it moves when a score passes that, so most tiles need no reduction; likewise
// the power of two that weight x V's power is taken relative to.
#include <cuda_fp16.h>

#include "attention_packed.cuh"

namespace ppocr {

namespace {

constexpr int kKeys = 32, kPad = 8;
constexpr float kSlack = 4.f;   // log2 of what weights leave above the maximum: at most 1, they may meet any V row's power

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same onto zeros: the first step of a chain.
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// a and b as FP16 pairs: the values rounded, and what is left times 2^11 (no more
// than the value, so it is never out of range, and 2^-11 of FP16's least step counts).
constexpr float kSecond = 2048.f;
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn((a - f.x) * kSecond, (b - f.y) * kSecond);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// ROWS rows on their way to FP16 planes by a block of WARPS warps.  kLanes threads
// share a row; a thread's pieces of 16 bytes lie at raw[piece x kThreads + thread],
// for it alone.
template <int DP, int WARPS, int ROWS>
struct Rows {
    static constexpr int kThreads = 32 * WARPS, kPitch = DP + kPad;
    static constexpr int kLanes = DP >= 32 ? 8 : 4, kPieces = DP / 4 / kLanes, kPerPass = kThreads / kLanes;
    static constexpr int kPasses = ROWS / kPerPass;
    static constexpr int kRawBytes = ROWS * DP * 4, kPlaneBytes = ROWS * kPitch * 2;
    static_assert(kPasses * kPerPass == ROWS, "whole passes");

    // row(n): row n's values, null for zeros; `any` is readable.
    template <typename Row>
    static __device__ __forceinline__ void fetch(float4* raw, Row row, const float* any, int d, bool vec) {
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const float* src = row(tid / kLanes + kPerPass * i);
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                const int x = (tid % kLanes + kLanes * j) * 4;
                float4* dst = raw + (i * kPieces + j) * kThreads + tid;
                if (vec) {
                    const bool live = src && x < d;
                    cp_async16(dst, live ? src + x : any, live);
                } else {
                    const int n = src ? d - x : 0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) cp_async4(&dst->x + u, n > u ? src + x + u : any, n > u);
                }
            }
        }
    }
    // The rows' planes, and done(n, top, e) by one thread for row n, which holds
    // its values times 2^(14 - e); top is its largest magnitude.
    template <typename Done>
    static __device__ __forceinline__ void split(const float4* raw, __half* hi, __half* lo, Done done) {
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            float4 x[kPieces];
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                x[j] = raw[(i * kPieces + j) * kThreads + tid];
                top = fmaxf(fmaxf(top, fmaxf(fabsf(x[j].x), fabsf(x[j].y))), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
            }
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = min(max(exponent(top), -100), 127), n = tid / kLanes + kPerPass * i;
            const float up = power(14 - e);
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                uint2 h, l;
                split2(x[j].x * up, x[j].y * up, h.x, l.x);
                split2(x[j].z * up, x[j].w * up, h.y, l.y);
                const int at = n * kPitch + (tid % kLanes + kLanes * j) * 4;
                *reinterpret_cast<uint2*>(hi + at) = h;
                *reinterpret_cast<uint2*>(lo + at) = l;
            }
            if (tid % kLanes == 0) done(n, top, e);
        }
    }
};

// What a row of Q or K was divided by.  Rows of 2^60 and more are left to
// attend_row: the factors' product might overflow where the score does not.
__device__ __forceinline__ float score_factor(float top, int e) { return top < power(60) ? power(e - 14) : NAN; }

// What a block of WARPS warps, 16 rows each, keeps in shared memory.  With two
// buffers of planes the next tile is split while this one is worked on.
template <int DP, int WARPS>
struct Plan {
    static constexpr int kRows = 16 * WARPS, kBuffers = DP > 64 && WARPS == 4 ? 1 : 2;
    using Q = Rows<DP, WARPS, kRows>;
    using KV = Rows<DP, WARPS, 2 * kKeys>;   // a tile's K rows, then its V rows
    static constexpr int kPlanes = 2 * KV::kPlaneBytes, kFactors = 2 * kKeys * 4;
    static constexpr int kBytes = KV::kRawBytes + 2 * Q::kPlaneBytes + kBuffers * (kPlanes + kFactors) + kRows * 4;
    static_assert(Q::kRawBytes <= kBuffers * kPlanes, "Q is staged where the planes will be");
};

template <int DP, int WARPS, int BLOCKS>
__global__ void __launch_bounds__(32 * WARPS, BLOCKS)
    attention_packed_f32_kernel(PackedAttentionParams p, bool vec, bool vec_out) {
    using L = Plan<DP, WARPS>;
    using R = typename L::KV;
    constexpr int P = R::kPitch, NT = kKeys / 8, KS = DP / 16, DT = DP / 8, kRows = L::kRows;
    extern __shared__ uint4 smem16[];
    float4* raw = reinterpret_cast<float4*>(smem16);
    __half* qh = reinterpret_cast<__half*>(reinterpret_cast<char*>(smem16) + R::kRawBytes);
    __half* ql = qh + kRows * P;
    __half* planes = ql + kRows * P;     // per buffer the first pieces, then the second
    float* fq = reinterpret_cast<float*>(reinterpret_cast<char*>(planes) + L::kBuffers * L::kPlanes);   // factors of Q's rows
    float* factors = fq + kRows;         // per buffer those of K's rows, then the powers of V's
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const PackedPiece<kRows> at(p);
    const int rows = at.rows, d = p.d;
    if (rows <= 0) return;
    const int keys = at.keys_of(rows - 1);
    const int tiles = (keys + kKeys - 1) / kKeys;

    const float* q = at.template queries<float>(p.q);
    const float* k = at.template keys<float>(p.k);
    const float* v = at.template keys<float>(p.v);
    auto fetch_keys = [&](int j) {
        R::fetch(raw, [&](int n) {
            const int key = j * kKeys + n % kKeys;
            const float* src = n < kKeys ? k + (long long)key * (int)p.k.token_stride : v + (long long)key * (int)p.v.token_stride;
            return key < keys ? src : nullptr;
        }, q, d, vec);
    };
    float4* raw_q = reinterpret_cast<float4*>(planes);   // until the first tile's planes
    L::Q::fetch(raw_q, [&](int n) { return n < rows ? q + at.row_at(p.q, n) : nullptr; }, q, d, vec);
    if (tiles > 0) fetch_keys(0);
    cp_async_commit();
    cp_async_wait<0>();
    L::Q::split(raw_q, qh, ql, [&](int n, float top, int e) { fq[n] = score_factor(top, e); });
    __syncthreads();
    // Tile j, whose copies are the last that were started, into its planes; starts the next one's.
    auto split_keys = [&](int j) {
        cp_async_wait<0>();
        const int at_buffer = j % L::kBuffers;
        __half* hi = planes + at_buffer * (L::kPlanes / 2);
        float* f = factors + at_buffer * (2 * kKeys);
        R::split(raw, hi, hi + 2 * kKeys * P,
                 [&](int n, float top, int e) { f[n] = n < kKeys ? score_factor(top, e) : power(e); });
        if (j + 1 < tiles) fetch_keys(j + 1);
        cp_async_commit();
    };

    const float scale = p.scale * 1.4426950408889634f;
    const int n0 = warp * 16 + r;                  // this lane's rows: n0 and n0 + 8
    const int keys0 = at.keys_of(min(n0, rows - 1)), keys1 = at.keys_of(min(n0 + 8, rows - 1));
    const int sure = __reduce_min_sync(0xffffffffu, (unsigned)min(keys0, keys1));   // keys every row of the warp sees
    const int most = n0 - r < rows ? (int)__reduce_max_sync(0xffffffffu, (unsigned)max(keys0, keys1)) : 0;
    // Rows whose factor, scale and a key's factor might overflow are left to attend_row too.
    auto factor = [&](int n) { return fq[n] * scale < power(82) ? fq[n] * scale : NAN; };
    const float f0 = factor(n0), f1 = factor(n0 + 8);
    float o[DT][4];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, b0 = 0.f, b1 = 0.f, l0 = 0.f, l1 = 0.f;   // b: m, 0 while it is -infinity
    int e0 = -100, e1 = -100;            // o holds sums of weight x V, times 2^(22 - e)
    float unit0 = power(108), unit1 = power(108);   // 2^(8 - e)

    if (tiles > 0) {
        split_keys(0);
        __syncthreads();
    }
    for (int j = 0; j < tiles; ++j) {
        const __half* hi = planes + j % L::kBuffers * (L::kPlanes / 2);
        const __half* lo = hi + 2 * kKeys * P;
        const float* fk = factors + j % L::kBuffers * (2 * kKeys);
        const float* fv = fk + kKeys;
        // With eight warps one half splits the next tile before its work on this
        // one and the other after it, so that both kinds of work are at hand.
        const bool late = WARPS == 8 && warp >= 4;
        if (L::kBuffers > 1 && !late && j + 1 < tiles) split_keys(j + 1);
        if (j * kKeys < most) {
            float s[NT][4], rest[NT][4];
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t ah[4], al[4];
                const int qa = (warp * 16 + (lane & 15)) * P + i * 16 + (lane >> 4) * 8;
                ldmatrix4(ah, qh + qa);
                ldmatrix4(al, ql + qa);
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t bh[4], bl[4];
                    const int kb = (n * 8 + (lane & 7) + (lane >> 4) * 8) * P + i * 16 + ((lane >> 3) & 1) * 8;
                    ldmatrix4(bh, hi + kb);
                    ldmatrix4(bl, lo + kb);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float part[4];
                        if (i == 0) mma_first(rest[n + u], al, bh[2 * u], bh[2 * u + 1]);
                        else mma(rest[n + u], al, bh[2 * u], bh[2 * u + 1]);
                        mma(rest[n + u], ah, bl[2 * u], bl[2 * u + 1]);
                        if (i == 0) {
                            mma_first(s[n + u], ah, bh[2 * u], bh[2 * u + 1]);
                        } else {
                            mma_first(part, ah, bh[2 * u], bh[2 * u + 1]);
#pragma unroll
                            for (int x = 0; x < 4; ++x) s[n + u][x] += part[x];
                        }
                    }
                }
            }
            // Scale, mask; the maximum, where a score passes it by far.
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 f = *reinterpret_cast<const float2*>(fk + n * 8 + 2 * c);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float fx = x ? f.y : f.x;
                    s[n][x] = fmaf(rest[n][x], 1.f / kSecond, s[n][x]) * (f0 * fx);
                    s[n][x + 2] = fmaf(rest[n][x + 2], 1.f / kSecond, s[n][x + 2]) * (f1 * fx);
                }
            }
            if ((j + 1) * kKeys > sure) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int key = j * kKeys + n * 8 + 2 * c + x;
                        if (key >= keys0) s[n][x] = -INFINITY;
                        if (key >= keys1) s[n][x + 2] = -INFINITY;
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                t0 = fmaxf(t0, fmaxf(s[n][0], s[n][1]));
                t1 = fmaxf(t1, fmaxf(s[n][2], s[n][3]));
            }
            if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1)) {
                auto raise = [&](float t, float& m, float& b, float& l, int& e, float& unit, int half) {
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                    if (t > m) {   // the whole row's four lanes; a row's steps depend on its own scores alone
                        t += kSlack;
                        // What the sums hold shrinks with the weights, so their power may fall as far.
                        const float fall = m - t;   // -infinity for the first keys
                        const int next = max(e + (int)fmaxf(ceilf(fall), -300.f), -100);
                        const float back = exp2_hw(fall + (float)(e - next));
                        l *= exp2_hw(fall);
#pragma unroll
                        for (int i = 0; i < DT; ++i) {
                            o[i][half] *= back;
                            o[i][half + 1] *= back;
                        }
                        e = next;
                        unit = power(8 - e);
                        b = m = t;
                    }
                };
                raise(t0, m0, b0, l0, e0, unit0, 0);
                raise(t1, m1, b1, l1, e1, unit1, 2);
            }
            // Weights, times the powers of the V rows.
            float y0 = 0.f, y1 = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 f = *reinterpret_cast<const float2*>(fv + n * 8 + 2 * c);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    s[n][x] = exp2_hw(s[n][x] - b0);
                    s[n][x + 2] = exp2_hw(s[n][x + 2] - b1);
                    l0 += s[n][x];
                    l1 += s[n][x + 2];
                    s[n][x] *= x ? f.y : f.x;
                    s[n][x + 2] *= x ? f.y : f.x;
                    y0 = fmaxf(y0, s[n][x]);
                    y1 = fmaxf(y1, s[n][x + 2]);
                }
            }
            if (__any_sync(0xffffffffu, y0 * unit0 > 32768.f || y1 * unit1 > 32768.f)) {
                auto raise = [&](float y, int& e, float& unit, int half) {
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
                    if (y * unit > 32768.f) {
                        const int next = min(max(e, exponent(y) + 1), 126);
                        const float back = power(max(e - next, -126));   // what 2^-126 leaves of a sum counts for nothing
#pragma unroll
                        for (int i = 0; i < DT; ++i) {
                            o[i][half] *= back;
                            o[i][half + 1] *= back;
                        }
                        e = next;
                        unit = power(8 - e);
                    }
                };
                raise(y0, e0, unit0, 0);
                raise(y1, e1, unit1, 2);
            }
            uint32_t wh[NT / 2][4], wl[NT / 2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                split2(s[n][0] * unit0, s[n][1] * unit0, wh[n / 2][n % 2 * 2], wl[n / 2][n % 2 * 2]);
                split2(s[n][2] * unit1, s[n][3] * unit1, wh[n / 2][n % 2 * 2 + 1], wl[n / 2][n % 2 * 2 + 1]);
            }
#pragma unroll
            for (int i = 0; i < DT; i += 2) {
                uint32_t bh[NT / 2][4], bl[NT / 2][4];
#pragma unroll
                for (int n = 0; n < NT / 2; ++n) {
                    const int vb = (kKeys + n * 16 + (lane & 15)) * P + i * 8 + (lane >> 4) * 8;
                    ldmatrix4_trans(bh[n], hi + vb);
                    ldmatrix4_trans(bl[n], lo + vb);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float sum[4], small[4];
                    mma_first(small, wl[0], bh[0][2 * u], bh[0][2 * u + 1]);
                    mma_first(sum, wh[0], bh[0][2 * u], bh[0][2 * u + 1]);
                    mma(small, wh[0], bl[0][2 * u], bl[0][2 * u + 1]);
#pragma unroll
                    for (int n = 1; n < NT / 2; ++n) {
                        mma(small, wl[n], bh[n][2 * u], bh[n][2 * u + 1]);
                        mma(sum, wh[n], bh[n][2 * u], bh[n][2 * u + 1]);
                        mma(small, wh[n], bl[n][2 * u], bl[n][2 * u + 1]);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[i + u][x] += fmaf(small[x], 1.f / kSecond, sum[x]);
                }
            }
        }
        if (L::kBuffers > 1 && late && j + 1 < tiles) split_keys(j + 1);
        __syncthreads();
        if (L::kBuffers == 1 && j + 1 < tiles) {
            split_keys(j + 1);
            __syncthreads();
        }
    }

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
    const float u0 = power(e0 - 22), u1 = power(e1 - 22);
    float* out = at.template queries<float>(p.out);
    bool bad[2] = {false, false};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int n = n0 + 8 * half;
        if (n >= rows) continue;
        float* dst = out + at.row_at(p.out, n);
        float odd = 0.f;   // stays 0, or becomes NaN
        const float inv = half ? i1 : i0, unit = half ? u1 : u0;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int x = i * 8 + 2 * c;
            const float a = o[i][2 * half] * inv * unit, b = o[i][2 * half + 1] * inv * unit;
            odd = fmaf(a, 0.f, fmaf(b, 0.f, odd));   // columns past d hold zeros
            if (vec_out && x + 1 < d) {
                *reinterpret_cast<float2*>(dst + x) = make_float2(a, b);
            } else {
                if (x < d) dst[x] = a;
                if (x + 1 < d) dst[x + 1] = b;
            }
        }
        bad[half] = odd != 0.f;
    }
    // Rows with a non-finite value again, by their definition, after the
    // warp's own stores above.  A row is shared by four lanes.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const unsigned again = __ballot_sync(0xffffffffu, bad[half]);
        for (int rr = 0; again && rr < 8; ++rr) {
            if (!(again >> (4 * rr) & 0xfu)) continue;
            const int n = warp * 16 + rr + 8 * half;
            __syncwarp();
            attend_row<float>(q + at.row_at(p.q, n), k, p.k.token_stride, v, p.v.token_stride, d, at.keys_of(n), scale,
                              out + at.row_at(p.out, n));
        }
    }
}

template <int DP, int WARPS, int BLOCKS>
cudaError_t launch(const PackedAttentionParams& p, cudaStream_t stream) {
    const bool vec = rows16(p.q, 4) && rows16(p.k, 4) && rows16(p.v, 4) && p.d % 4 == 0;
    using L = Plan<DP, WARPS>;
    const auto kernel = attention_packed_f32_kernel<DP, WARPS, BLOCKS>;
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kBytes);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)PackedPiece<L::kRows>::blocks(p), 32 * WARPS, L::kBytes, stream>>>(p, vec, pairs_aligned(p.out, 4));
    return cudaGetLastError();
}

// Blocks of eight warps (128 rows, K and V split half as often) where sequences
// fill them.  Measured on 8,192 tokens in causal sequences of equal length, four
// / eight warps in us (rows per sequence: length x heads per KV head):
//   8 heads of 15          length 64: 20 / 28, 96: 23 / 27, 128: 25 / 25, 1,024: 97 / 85
//   16 of 32, 4 KV heads   length 64: 36 / 38, 96: 42 / 42, 128: 48 / 46, 1,024: 190 / 164
//   8 of 64                length 64: 40 / 47, 96: 52 / 45, 128: 49 / 40, 1,024: 184 / 161
//   16 of 64, 4 KV heads   length 32: 50 / 45, 64: 62 / 50
//   32 of 128, 8 KV heads  length 32: 180 / 175, 64: 230 / 193, 1,024: 1,061 / 836
// For d = 64, where two blocks on an SM have to share its registers, a block has
// an SM to itself up to 1.5 x 148 blocks: each is faster, and the last ones, the
// shortest of causal sequences, start where others end.  16 heads, 4 KV heads,
// alone / two per SM in us:
//   1,024 tokens (128 blocks)  length 128: 15 / 18, 512: 38 / 39
//   1,480 tokens (185)         length 92: 20 / 18, 185: 26 / 27, 370: 35 / 44, 740: 51 / 64
//   2,220 tokens (277)         length 138: 31 / 25, 277: 42 / 36, 555: 64 / 64, 1,110: 78 / 116
//   2,960 tokens (370)         length 185: 42 / 37, 370: 59 / 54, 740: 91 / 77, 1,480: 142 / 146
template <int DP>
cudaError_t launch_dp(const PackedAttentionParams& p, cudaStream_t stream) {
    const long long rows = (long long)p.total_q * (p.heads / p.kv_heads);
    const bool full = DP > 32 ? rows >= 96ll * p.sequences : rows >= 128ll * p.sequences && p.total_k >= 128ll * p.sequences;
    if (!full) return launch<DP, 4, (DP > 64 ? 2 : DP > 32 ? 3 : 5)>(p, stream);
    if constexpr (DP == 64) {
        if (rows * p.kv_heads <= 128ll * 222) return launch<DP, 8, 1>(p, stream);
    }
    return launch<DP, 8, (DP > 64 ? 1 : 2)>(p, stream);
}

}  // namespace

cudaError_t launch_attention_packed_f32(const PackedAttentionParams& p, cudaStream_t stream) {
    if (p.d <= 16) return launch_dp<16>(p, stream);
    if (p.d <= 32) return launch_dp<32>(p, stream);
    if (p.d <= 64) return launch_dp<64>(p, stream);
    return launch_dp<128>(p, stream);
}

}  // namespace ppocr
