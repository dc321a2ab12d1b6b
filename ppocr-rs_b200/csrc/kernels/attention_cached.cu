// Single-token attention over the 8-bit paged cache.
//
//   out[h] = sum_t softmax_t(scale q[h] . k_t) v_t,  k_t = s_k int8, v_t = s_v int8
//
// Bound: HBM, the cache's bytes (2 d + 8 / page per token and KV head).  A
// byte is worth 2 multiply-adds per query head, so grouped heads would keep
// CUDA cores busier than the memory; the products run on mma.m16n8k16 with 16
// tokens (or 16 values of d) as M and the up to eight query heads of a group
// as N, so a tile of 16 tokens costs two MMAs per 16 values of d whatever the
// group.  (tcgen05 would want 128 rows of M, and operands of its own types in
// shared memory, where the integers are bytes.)
//
// Integers are exact in FP16.  q is scaled by a power of two per head to fit
// FP16; FP32 inputs are carried as two FP16 pieces (22 bits), as are their
// softmax weights, so their products are FP32-class.  A page's K scale
// multiplies its scores; its V scale multiplies its weights, and the product is
// taken relative to a power of two per head that follows the largest one: up
// when a product would pass FP16's range, down with the weights when the maximum
// moves.  So pages of large values and no weight cost the others no bits.  (A
// power of the V scales alone does: at 2^27 between two pages the weights of the
// smaller one had three bits left.)  Second pieces are held times 2^11
// and their products summed apart, which keeps 22 bits of weights down to 2^-20 of
// the largest product and of q's values down to 2^-28 of the head's largest.
//
// A warp owns every fourth pair of tiles of its block's token range, fetches
// them with cp.async into a ring of its own in shared memory (two pairs; no
// barrier of the block is involved) and keeps its own softmax state; weights are
// relative to the maximum + 6 (in log2) when it last moved, and it moves when a
// score passes that, so most tiles need no reduction at all.  The two tiles of a pair are two
// independent chains of products.  The range of a sequence is split over the
// blocks of a cluster (1 to 16) when there are few sequences and heads; warps
// join through shared memory, blocks through distributed shared memory, both in
// a fixed order: one launch, no workspace.  The longest sequences start first.
//
// Measured: 64 sequences of 1 to 4,100 tokens, 32 heads on 8 KV heads of 128, pages
// of 32, BF16: 70 us (4.0 TB/s; 68 with weights relative to the V scales alone, then
// 115 with the loads straight to registers, 75 without the order of sequences).  Two
// of up to 65,000 tokens, 24 heads, FP32: 89 us (2.6 TB/s).  One of 101 tokens: 4.8 us.  The instructions between the loads
// and the MMAs (a byte_perm and a subtraction per two values, and the softmax:
// 470 per 16 tokens of d = 128) keep the issue slots 56 % busy while four of eight
// columns of N are live, and are what is left above the bytes.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <climits>

#include "seq_common.cuh"

namespace ppocr {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kHeads = 8, kMaxSplits = 16;
constexpr int kTile = 16;             // tokens per tile: within one page, whatever its size
constexpr int kPair = 2;              // tiles that a warp takes at a time: two independent chains of products
constexpr float kSlack = 6.f;         // log2 of what weights leave above the maximum: they are at most 1
constexpr float kMost = 65000.f;      // of a weight x V scale x unit, in FP16
constexpr int kLeast = -119;          // of the power that these products are relative to; 2^(7 - it) and 2^(it - 7) are numbers
constexpr float kSecond = 2048.f;     // what second pieces are held times

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Two bytes of `u` (integers + 128, at byte selectors of `sel`) as FP16: the
// byte under 0x64 is 1024 + byte, and 1152 less is the integer, exactly.
__device__ __forceinline__ uint32_t bytes_to_h2(uint32_t u, uint32_t sel) {
    const uint32_t w = __byte_perm(u, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));
    return h2_bits(h);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same onto zeros: the first step of a chain.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void add4(float (&a)[4], const float (&b)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += b[i];
}

// Transposes an 8 x 8 matrix of FP16 held two columns per lane (row lane / 4).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// A warp's ring of pairs of tiles in shared memory: per tile the 16 K rows, the
// 16 V rows (DP bytes each, zeros past d) and the page's two scales.  16-byte
// chunks are permuted within a row so that the reads below, which take
// different rows at the same bytes, spread over the banks.
template <int DP, bool FULL>
struct Ring {
    static constexpr int kStages = 2, kChunks = DP / 16, kRows = kTile * DP, kOne = 2 * kRows + 16, kStage = kPair * kOne;
    static constexpr int kBytes = kStages * kStage;
    static __device__ __forceinline__ int k_chunk(int row, int chunk) { return DP == 128 ? chunk ^ (row & 1) << 2 : chunk; }
    static __device__ __forceinline__ int v_chunk(int row, int chunk) {
        return DP == 128 ? chunk ^ (row >> 1 & 3) << 1 : DP == 64 ? chunk ^ (row >> 1 & 3) : chunk;
    }

    // Starts the copies of slots slot0 .. slot0 + 15 of `head` of page `where`.
    static __device__ __forceinline__ void fetch(const CachedAttentionParams& p, uint32_t stage, int where, int head, int slot0,
                                                 int page_bytes, int lane) {
        const int d = FULL ? DP : p.cache.d;
        const long long cell = (long long)where * p.cache.kv_heads + head, at0 = cell * page_bytes + slot0 * d;
        const int8_t* kp = p.cache.k + at0;
        const int8_t* vp = p.cache.v + at0;
#pragma unroll
        for (int i = 0; i < kTile * kChunks / 32; ++i) {
            const int row = (lane + 32 * i) / kChunks, chunk = (lane + 32 * i) % kChunks, from = row * d + chunk * 16;
            const uint32_t to = stage + row * DP;
            copy(to + k_chunk(row, chunk) * 16, kp + from, d - chunk * 16, kp);
            copy(to + kRows + v_chunk(row, chunk) * 16, vp + from, d - chunk * 16, vp);
        }
        if (lane < 2) copy4(stage + 2 * kRows + 4 * lane, (lane ? p.cache.v_scales : p.cache.k_scales) + cell);
    }
    // 16 bytes of a row with `live` of them (a multiple of 8; FULL: all) in it.
    static __device__ __forceinline__ void copy(uint32_t to, const int8_t* from, int live, const int8_t* base) {
        if constexpr (FULL) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = live > 8 * h ? 8 : 0;
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to + 8 * h), "l"(n ? from + 8 * h : base), "r"(n) : "memory");
            }
        }
    }
    static __device__ __forceinline__ void copy4(uint32_t to, const float* from) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
    }
};

// BYTES (4, 8 or 16) bytes of shared memory.
template <int BYTES>
__device__ __forceinline__ void read_words(uint32_t at, uint32_t* w) {
    if constexpr (BYTES == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at));
    else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    else asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
}

template <typename T, int DP, bool FULL>
__global__ void __launch_bounds__(kThreads, 3) attention_cached_kernel(CachedAttentionParams p, int splits) {
    constexpr bool SPLIT = sizeof(T) == 4;   // FP32: two FP16 pieces
    constexpr int KS = DP / 16;              // 16-wide steps over d
    // A lane holds, of a token of K, the bytes at c PK (and, for d 128, 64
    // further), of a token of V the bytes at r DP / 8.
    constexpr int PK = DP == 32 ? 8 : 16, PV = DP / 8;
    using Tiles = Ring<DP, FULL>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    int seq = blockIdx.x / splits;
    const int split = blockIdx.x % splits;
    const int group = p.heads / p.cache.kv_heads, parts = (group + kHeads - 1) / kHeads;
    const int kv = blockIdx.y / parts, part = blockIdx.y % parts;
    const int head0 = kv * group + part * kHeads, live_heads = min(kHeads, group - part * kHeads);
    const int page = p.cache.page, d = p.cache.d;

    if (p.table.sequences <= kThreads) {
        // Blocks start in the order of their numbers: the longest sequences come
        // first, so that none is begun when the others are nearly done.  Thread i
        // counts the sequences that come before sequence i.
        int* lengths = reinterpret_cast<int*>(smem);
        const int mine = threadIdx.x < p.table.sequences ? p.lengths[threadIdx.x] : INT_MIN;
        lengths[threadIdx.x] = mine;
        __syncthreads();
        int before = 0;
        for (int i = 0; i < p.table.sequences; ++i) {
            const int other = lengths[i];
            before += other > mine || (other == mine && i < threadIdx.x);
        }
        __syncthreads();
        if (threadIdx.x < p.table.sequences && before == seq) lengths[0] = threadIdx.x;
        __syncthreads();
        seq = lengths[0];
        __syncthreads();   // the rings take its place
    }
    int len = p.lengths[seq];
    const long long room = (long long)p.table.width * page;
    if (len < 0 || len > room) {
        if (threadIdx.x == 0) seq_bad_index(p.bad);
        len = len < 0 ? 0 : (int)room;
    }
    // Pairs of tiles, dealt to the splits in ranges and to a block's warps by turns.
    const int tiles = (len + kTile - 1) / kTile, pairs = (tiles + kPair - 1) / kPair, per = (pairs + splits - 1) / splits;
    const int t_end = min(pairs, (split + 1) * per);
    const int32_t* pages = p.table.pages + seq * p.table.stride;
    const int page_shift = 31 - __clz(page) - 4;   // log2 of the tiles in a page
    auto page_of = [&](int pair, int half) {
        const int tile = pair * kPair + half;
        if (pair >= t_end || tile >= tiles) return -1;
        const int w = __ldg(pages + (tile >> page_shift));
        if ((unsigned)w >= (unsigned)p.cache.pages) {
            seq_bad_index(p.bad);
            return -1;
        }
        return w;
    };
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * Tiles::kBytes;
    int t = split * per + warp;      // the pair at hand
    int ahead = t, stage = 0, stage_ahead = 0, w_ahead[kPair];   // the next pair to fetch and its pages
    unsigned missing = 0;            // bit kPair s + h: half h of stage s holds no tile
#pragma unroll
    for (int h = 0; h < kPair; ++h) w_ahead[h] = page_of(ahead, h);
    auto fetch = [&] {
        missing &= ~(((1u << kPair) - 1) << kPair * stage_ahead);
#pragma unroll
        for (int h = 0; h < kPair; ++h) {
            if (w_ahead[h] >= 0)
                Tiles::fetch(p, ring + stage_ahead * Tiles::kStage + h * Tiles::kOne, w_ahead[h], kv,
                             (ahead * kPair + h) * kTile & (page - 1), page * d, lane);
            else
                missing |= 1u << (kPair * stage_ahead + h);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += kWarps;
#pragma unroll
        for (int h = 0; h < kPair; ++h) w_ahead[h] = page_of(ahead, h);
        stage_ahead = stage_ahead + 1 == Tiles::kStages ? 0 : stage_ahead + 1;
    };
#pragma unroll
    for (int i = 0; i < Tiles::kStages - 1; ++i) fetch();

    // B operand of the scores: head r's values of d, in the order in which the
    // lane's K bytes come; b0 holds bytes 4s, 4s + 1 and b1 bytes 4s + 2, 4s + 3.
    uint32_t qh[KS][2], ql[SPLIT ? KS : 1][2];
    // Scores are divided by a head's power, times its K scale and the call's: a scale
    // above 1 last, since its product with the power may overflow where the score does not.
    const float scale = p.scale * 1.4426950408889634f, first = fminf(scale, 1.f), last = fmaxf(scale, 1.f);
    float qscale;
    {
        float x[DP / 4];
        float top = 0.f;
        const T* q = static_cast<const T*>(p.q.ptr) + seq * p.q.token_stride + (head0 + r) * p.q.head_stride;
#pragma unroll
        for (int i = 0; i < DP / 4; ++i) {
            const int at = 64 * (i / PK) + c * PK + i % PK;
            x[i] = r < live_heads && at < d ? to_f(q[at]) : 0.f;
            top = fmaxf(top, fabsf(x[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // Power of two that takes the head's largest value into [2^14, 2^15).
        const int e = max(exponent(top), -100);
        const float up = power(14 - e);
        qscale = first * power(e - 14);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = x[4 * s + 2 * h] * up, b = x[4 * s + 2 * h + 1] * up;
                const __half2 hi = __floats2half2_rn(a, b);
                qh[s][h] = h2_bits(hi);
                if constexpr (SPLIT) {
                    const float2 f = __half22float2(hi);
                    ql[s][h] = h2_bits(__floats2half2_rn(isinf(f.x) ? 0.f : (a - f.x) * kSecond, isinf(f.y) ? 0.f : (b - f.y) * kSecond));
                }
            }
    }
    // The scores' columns are heads 2c and 2c + 1: their factors.
    const float f0 = __shfl_sync(0xffffffffu, qscale, 8 * c), f1 = __shfl_sync(0xffffffffu, qscale, 8 * c + 4);

    float o[KS][4];
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    // Weights are relative to m (once a score was seen); o holds sums of weight x V
    // times 2^(7 - e) = unit.
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, unit0 = power(7 - kLeast), unit1 = unit0, units = unit0;   // the larger
    int e0 = kLeast, e1 = kLeast;

    const uint32_t k_at = r * DP, v_at = Tiles::kRows + 2 * c * DP;
    for (; t < t_end; t += kWarps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(Tiles::kStages - 2) : "memory");
        __syncwarp();   // the pair is there, and every lane has read the one that the next copies replace
        fetch();
        const uint32_t at = ring + stage * Tiles::kStage;
        const unsigned none = missing >> kPair * stage;
        stage = stage + 1 == Tiles::kStages ? 0 : stage + 1;

        // Scores: [tokens][heads] of each tile.  The tensor cores truncate when
        // they add to an accumulator, so FP32 sums take few steps each: the
        // second pieces apart (they are 2^-11 of the first), the first in
        // chains of two steps.
        float s[kPair][4], sv[kPair];
#pragma unroll
        for (int h = 0; h < kPair; ++h) {
            uint32_t k[2][DP / 16];
            float sk, rest[4], part[4];
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(sk), "=f"(sv[h]) : "r"(at + h * Tiles::kOne + 2 * Tiles::kRows));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DP / 4 / PK; ++j)
                    read_words<PK>(at + h * Tiles::kOne + k_at + 8 * i * DP + Tiles::k_chunk(r, (c * PK >> 4) + 4 * j) * 16 +
                                       (c * PK & 15),
                                   &k[i][j * PK / 4]);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t u0 = k[0][i] ^ 0x80808080u, u1 = k[1][i] ^ 0x80808080u;
                const uint32_t a0 = bytes_to_h2(u0, 0x4140), a1 = bytes_to_h2(u1, 0x4140);
                const uint32_t a2 = bytes_to_h2(u0, 0x4342), a3 = bytes_to_h2(u1, 0x4342);
                if constexpr (SPLIT) {
                    if (i == 0) mma_f16_first(rest, a0, a1, a2, a3, ql[i][0], ql[i][1]);
                    else mma_f16(rest, a0, a1, a2, a3, ql[i][0], ql[i][1]);
                    float (&sum)[4] = i < 2 ? s[h] : part;
                    if (i % 2 == 0) mma_f16_first(sum, a0, a1, a2, a3, qh[i][0], qh[i][1]);
                    else mma_f16(sum, a0, a1, a2, a3, qh[i][0], qh[i][1]);
                    if (i > 2 && i % 2 == 1) add4(s[h], part);
                } else if (i == 0) {
                    mma_f16_first(s[h], a0, a1, a2, a3, qh[i][0], qh[i][1]);
                } else {
                    mma_f16(s[h], a0, a1, a2, a3, qh[i][0], qh[i][1]);
                }
            }
            if constexpr (SPLIT) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][i] = fmaf(rest[i], 1.f / kSecond, s[h][i]);
            }
            const float k0 = f0 * sk * last, k1 = f1 * sk * last;
            s[h][0] *= k0; s[h][1] *= k1;
            s[h][2] *= k0; s[h][3] *= k1;
            // Past the sequence's end, or on a page that is none.
            const int left = none >> h & 1 ? 0 : len - (t * kPair + h) * kTile;
            if (left < kTile) {
                if (r >= left) s[h][0] = s[h][1] = -INFINITY;
                if (r + 8 >= left) s[h][2] = s[h][3] = -INFINITY;
                if (left <= 0) sv[h] = 0.f;   // what the stage holds is older
            }
        }
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int h = 0; h < kPair; ++h) {
            t0 = fmaxf(t0, fmaxf(s[h][0], s[h][2]));
            t1 = fmaxf(t1, fmaxf(s[h][1], s[h][3]));
        }
        auto weigh = [&] {
            const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
            for (int h = 0; h < kPair; ++h) {
                float* x = s[h];
                x[0] = exp2_hw(x[0] - b0); x[1] = exp2_hw(x[1] - b1);
                x[2] = exp2_hw(x[2] - b0); x[3] = exp2_hw(x[3] - b1);
                l0 += x[0] + x[2];
                l1 += x[1] + x[3];
            }
        };
        // A new maximum, or a V scale whose product with a weight of 1 would pass FP16.
        if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1 || fmaxf(fabsf(sv[0]), fabsf(sv[1])) * units > kMost)) {
            auto rescale = [&](int head, float& unit, int& e, int next, float back) {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    o[j][head] *= back;
                    o[j][head + 2] *= back;
                }
                e = next;
                unit = power(7 - e);
            };
            auto raise = [&](float t, float& m, float& l, int& e, float& unit, int head) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                if (t > m) {   // the whole head's eight lanes
                    // What the sums hold shrinks with the weights, so their power may fall as far.
                    const float fall = m - (t + kSlack);   // -infinity for the first tokens
                    const int next = max(e + (int)fmaxf(ceilf(fall), -300.f), kLeast);
                    rescale(head, unit, e, next, exp2_hw(fall + (float)(e - next)));
                    l *= exp2_hw(fall);
                    m = t + kSlack;
                }
            };
            raise(t0, m0, l0, e0, unit0, 0);
            raise(t1, m1, l1, e1, unit1, 1);
            weigh();
            auto cover = [&](float y, int& e, float& unit, int head) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, x));
                // To between 2^6 and 2^7, although FP16 holds more: weights of up to 1 come
                // without a look at them as long as the V scales stay near this one.
                const int next = min(max(e, exponent(y) + 1), 126);
                if (next > e) rescale(head, unit, e, next, power(max(e - next, -126)));   // what 2^-126 leaves of a sum counts for nothing
            };
            static_assert(kPair == 2, "the largest products of two tiles");
            cover(fmaxf(fmaxf(s[0][0], s[0][2]) * fabsf(sv[0]), fmaxf(s[1][0], s[1][2]) * fabsf(sv[1])), e0, unit0, 0);
            cover(fmaxf(fmaxf(s[0][1], s[0][3]) * fabsf(sv[0]), fmaxf(s[1][1], s[1][3]) * fabsf(sv[1])), e1, unit1, 1);
            units = fmaxf(unit0, unit1);
#pragma unroll
            for (int h = 0; h < kPair; ++h) {
                // The unit first: the V scale's product with it may pass FP32's range.
                s[h][0] = s[h][0] * unit0 * sv[h]; s[h][1] = s[h][1] * unit1 * sv[h];
                s[h][2] = s[h][2] * unit0 * sv[h]; s[h][3] = s[h][3] * unit1 * sv[h];
            }
        } else {
            weigh();
#pragma unroll
            for (int h = 0; h < kPair; ++h) {
                const float w0 = sv[h] * unit0, w1 = sv[h] * unit1;
                s[h][0] *= w0; s[h][1] *= w1;
                s[h][2] *= w0; s[h][3] *= w1;
            }
        }
        // Weights, as the B operand of the second product.
        uint32_t p0[kPair], p1[kPair], r0[kPair], r1[kPair], v[kPair][4][DP / 32];
#pragma unroll
        for (int h = 0; h < kPair; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (i & 1) + 8 * (i >> 1);
                read_words<PV>(at + h * Tiles::kOne + v_at + row * DP + Tiles::v_chunk(2 * c, r * PV >> 4) * 16 + (r * PV & 15),
                               v[h][i]);
            }
            const float* x = s[h];
            const __half2 h0 = __floats2half2_rn(x[0], x[1]), h1 = __floats2half2_rn(x[2], x[3]);
            p0[h] = transpose8(h2_bits(h0));
            p1[h] = transpose8(h2_bits(h1));
            if constexpr (SPLIT) {
                const float2 y = __half22float2(h0), z = __half22float2(h1);
                r0[h] = transpose8(h2_bits(__floats2half2_rn((x[0] - y.x) * kSecond, (x[1] - y.y) * kSecond)));
                r1[h] = transpose8(h2_bits(__floats2half2_rn((x[2] - z.x) * kSecond, (x[3] - z.y) * kSecond)));
            }
        }
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float sum[4], rest[4];
#pragma unroll
                for (int h = 0; h < kPair; ++h) {
                    // Bytes 2b and 2b + 1 of two tokens, interleaved by value of d.
                    const uint32_t x = __byte_perm(v[h][0][i], v[h][1][i], b ? 0x7362 : 0x5140) ^ 0x80808080u;
                    const uint32_t y = __byte_perm(v[h][2][i], v[h][3][i], b ? 0x7362 : 0x5140) ^ 0x80808080u;
                    const uint32_t a0 = bytes_to_h2(x, 0x4140), a1 = bytes_to_h2(x, 0x4342);
                    const uint32_t a2 = bytes_to_h2(y, 0x4140), a3 = bytes_to_h2(y, 0x4342);
                    if constexpr (SPLIT) {   // a pair's sum apart, added to the running one with rounding
                        if (h == 0) {
                            mma_f16_first(rest, a0, a1, a2, a3, r0[h], r1[h]);
                            mma_f16_first(sum, a0, a1, a2, a3, p0[h], p1[h]);
                        } else {
                            mma_f16(rest, a0, a1, a2, a3, r0[h], r1[h]);
                            mma_f16(sum, a0, a1, a2, a3, p0[h], p1[h]);
                        }
                    } else {
                        mma_f16(o[2 * i + b], a0, a1, a2, a3, p0[h], p1[h]);
                    }
                }
                if constexpr (SPLIT) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[2 * i + b][x] += fmaf(rest[x], 1.f / kSecond, sum[x]);
                }
            }
    }

    // Join the block's warps, where the rings were: warp w's sums at sm_o[w],
    // then their sum at sm_o[0], all taken relative to the block's maximum.
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float (*sm_o)[kHeads][DP] = reinterpret_cast<float (*)[kHeads][DP]>(smem);
    float (*sm_m)[kHeads] = reinterpret_cast<float (*)[kHeads]>(sm_o + kWarps);
    float (*sm_l)[kHeads] = sm_m + kWarps;
    float* top = reinterpret_cast<float*>(sm_l + kWarps);   // [kHeads], the block's maximum
    float* sum = top + kHeads;                              // [kHeads], and sum
    float* share = sum + kHeads;                            // [splits][kHeads]
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, x);
        l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (r == 0) {
        sm_m[warp][2 * c] = m0; sm_m[warp][2 * c + 1] = m1;
        sm_l[warp][2 * c] = l0; sm_l[warp][2 * c + 1] = l1;
    }
    const float back0 = power(e0 - 7), back1 = power(e1 - 7);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
        const int x = r * (DP / 8) + 2 * j;
        *reinterpret_cast<float2*>(&sm_o[warp][2 * c][x]) = make_float2(o[j][0] * back0, o[j][2] * back0);
        *reinterpret_cast<float2*>(&sm_o[warp][2 * c + 1][x]) = make_float2(o[j][1] * back1, o[j][3] * back1);
    }
    __syncthreads();
    auto factor = [](float m, float most) { return m == -INFINITY ? 0.f : exp2_hw(m - most); };
    for (int i = threadIdx.x; i < live_heads * DP; i += kThreads) {
        const int h = i / DP, x = i % DP;
        float most = sm_m[0][h];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) most = fmaxf(most, sm_m[w][h]);
        float a = 0.f, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float g = factor(sm_m[w][h], most);
            a = fmaf(g, sm_o[w][h][x], a);
            l = fmaf(g, sm_l[w][h], l);
        }
        if (splits == 1) {
            T* out = static_cast<T*>(p.out.ptr) + seq * p.out.token_stride + (head0 + h) * p.out.head_stride;
            if (x < d) out[x] = from_f<T>(l == 0.f ? 0.f : a / l);
        } else {
            sm_o[0][h][x] = a;
            if (x == 0) {
                top[h] = most;
                sum[h] = l;
            }
        }
    }
    if (splits == 1) return;

    // Join the cluster's blocks: each one's share in a head's output, then the
    // outputs, dealt to the cluster's threads, each summed in the blocks' order.
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < live_heads) {
        const int h = threadIdx.x;
        float most = -INFINITY, l = 0.f;
        for (int b = 0; b < splits; ++b) most = fmaxf(most, *cluster.map_shared_rank(top + h, b));
        for (int b = 0; b < splits; ++b) {
            const float g = factor(*cluster.map_shared_rank(top + h, b), most);
            share[b * kHeads + h] = g;
            l = fmaf(g, *cluster.map_shared_rank(sum + h, b), l);
        }
        for (int b = 0; b < splits; ++b) share[b * kHeads + h] = l == 0.f ? 0.f : share[b * kHeads + h] / l;
    }
    __syncthreads();
    for (int i = (int)cluster.block_rank() * kThreads + threadIdx.x; i < live_heads * DP; i += splits * kThreads) {
        const int h = i / DP, x = i % DP;
        float a = 0.f;
        for (int b = 0; b < splits; ++b) a = fmaf(share[b * kHeads + h], *cluster.map_shared_rank(&sm_o[0][h][x], b), a);
        T* out = static_cast<T*>(p.out.ptr) + seq * p.out.token_stride + (head0 + h) * p.out.head_stride;
        if (x < d) out[x] = from_f<T>(a);
    }
    cluster.sync();   // no block leaves while another reads its shared memory
}

template <typename T, int DP, bool FULL>
cudaError_t launch_one(const CachedAttentionParams& p, int splits, dim3 grid, cudaStream_t stream) {
    constexpr int join = (kWarps * kHeads * (DP + 2) + (2 + kMaxSplits) * kHeads) * (int)sizeof(float);
    constexpr int rings = kWarps * Ring<DP, FULL>::kBytes, smem = join > rings ? join : rings;
    const void* kernel = reinterpret_cast<const void*>(attention_cached_kernel<T, DP, FULL>);
    cudaError_t e = allow_dynamic_smem(kernel, smem);
    if (e == cudaSuccess && splits > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = kThreads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attention_cached_kernel<T, DP, FULL>, p, splits);
}

template <typename T>
cudaError_t launch_type(const CachedAttentionParams& p, int splits, dim3 grid, cudaStream_t stream) {
    const int d = p.cache.d;
    if (d <= 32) return d == 32 ? launch_one<T, 32, true>(p, splits, grid, stream) : launch_one<T, 32, false>(p, splits, grid, stream);
    if (d <= 64) return d == 64 ? launch_one<T, 64, true>(p, splits, grid, stream) : launch_one<T, 64, false>(p, splits, grid, stream);
    return d == 128 ? launch_one<T, 128, true>(p, splits, grid, stream) : launch_one<T, 128, false>(p, splits, grid, stream);
}

}  // namespace

cudaError_t launch_attention_cached(const CachedAttentionParams& p, cudaStream_t stream) {
    if (p.table.sequences == 0) return cudaSuccess;
    const int group = p.heads / p.cache.kv_heads, parts = (group + kHeads - 1) / kHeads;
    const long long rows = (long long)p.table.sequences * p.cache.kv_heads * parts;
    // Blocks per sequence and head: enough for three on each SM, as long as a
    // block keeps 16 tiles of the longest sequence the table holds.
    const long long tiles = (long long)p.table.width * p.cache.page / kTile;
    int splits = 1;
    while (splits < kMaxSplits && rows * splits < 148 * 3 && tiles / (2 * splits) >= 16) splits *= 2;
    const dim3 grid((unsigned)(p.table.sequences * (long long)splits), (unsigned)(p.cache.kv_heads * parts));
    return p.dtype == DT_F32 ? launch_type<float>(p, splits, grid, stream)
                             : launch_type<__nv_bfloat16>(p, splits, grid, stream);
}

}  // namespace ppocr
