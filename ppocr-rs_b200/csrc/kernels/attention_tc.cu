// Attention over packed sequences on tcgen05 (BF16): the kernel of long
// sequences.
//
// A CTA owns two tiles of 128 rows of one (sequence, KV head); the query heads
// that share the KV head are rows too (row = token x group + head), so K and V
// are read once per 256 rows.  Roles (384 threads):
//   warp 8            TMA: both Q tiles, then K and V tiles of 128 keys into a
//                     ring (128-byte swizzled, 64 values of d per row chunk);
//   warp 9            MMA: S = Q K^T (both operands in shared memory, K-major)
//                     into TMEM, and O += P V with P read from TMEM and V
//                     MN-major as it lies;
//   warps 0-3, 4-7    softmax of tile 0 and 1, one row per thread: scores from
//                     TMEM to registers, running maximum and sum, weights back
//                     as BF16 over the scores' columns, in two halves so that
//                     the product of the first runs while the second is made.
// While one tile's softmax runs, the tensor cores work on the other tile's
// products.  The maximum that weights are relative to moves only when a score
// passes it by more than 8 (in log2: weights up to 2^8), so the output
// accumulator in TMEM is rarely rescaled.
//
// Bound: the tensor cores, but for the pipeline's gaps.  A prompt of 8,191 tokens,
// 16 heads on 2 KV heads of 128, causal: 257 us (1,070 TFLOP/s), 7 ragged prompts of up
// to 2,500, 32 heads on 8: 157 us; the products alone, without softmax, take 187 us
// of the 257, since S reads both operands from shared memory.  Tried: tiles of
// 64 keys with two buffers of S, 279 to 336 us (products of N = 64 wait for
// shared memory); two softmax warpgroups to a tile, 290; outputs staged through
// shared memory before they leave, slower by 2,000 cycles a tile.
//
// Every wait is bounded: on expiry the CTA records a code in *err, stops,
// lets its copies and MMAs land, frees its TMEM and returns.  Rows that come
// out non-finite and those of scores beyond 2^24 are computed again from their
// definition (attend_row).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "attention_packed.cuh"
#include "tcgen05.cuh"

namespace ppocr {

namespace {

constexpr int kRows = 128, kKeys = 128, kTiles = 2;
constexpr int kHalves = 2, kHalf = kKeys / kHalves;          // a tile's weights are handed over in halves
constexpr int kSoftmaxWarps = 4 * kTiles, kThreads = 32 * kSoftmaxWarps + 128;
constexpr int kQChunk = kRows * 128, kChunk = kKeys * 128;   // bytes of a tile's rows x 64 values
constexpr int kTmemCols = 512;
constexpr float kSlack = 8.f;
constexpr int kEmulated = 2;   // of every eight pairs of exponentials, on the FMA pipes (0: 263 us, 1: 256, 2: 257, 3: 279)

// 2^x of two values, x < 127, without the special function unit: x = n + f
// with n the nearest integer (by adding 1.5 x 2^23, whose last mantissa bit is
// 1), 2^f by the polynomial of degree 4 that is 1 at 0 with the least largest
// relative error on [-1/2, 1/2] (2.9e-6, a thousandth of the BF16 rounding that
// follows), and n added to the exponent.  From -127 down, -infinity (a masked
// score) among them, f is 0 and the exponent field of 1 less 127 leaves exactly
// 0; in between the result is some number below 2^-126.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.x));   // -127; a NaN stays one
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x.y));
    const float2 magic = make_float2(12582912.f, 12582912.f);
    const float2 t = __fadd2_rn(x, magic);
    const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
    const float2 f = __fadd2_rn(x, make_float2(-n.x, -n.y));
    float2 y = __ffma2_rn(f, make_float2(0.009585382f, 0.009585382f), make_float2(0.05590663f, 0.05590663f));
    y = __ffma2_rn(y, f, make_float2(0.24024038f, 0.24024038f));
    y = __ffma2_rn(y, f, make_float2(0.6931242f, 0.6931242f));
    y = __ffma2_rn(y, f, make_float2(1.f, 1.f));
    return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)));
}

template <int DC>   // chunks of 64 values of d
struct Layout {
    static constexpr int stages = DC == 1 ? 4 : 2;   // of a V and a K tile each
    static constexpr int q_bytes = kTiles * DC * kQChunk, tile_bytes = DC * kChunk, stage_bytes = 2 * tile_bytes;
    static constexpr int smem = q_bytes + stages * stage_bytes + 1024;
};

// Shared-memory matrix descriptors in two halves: the low one holds the address
// and the leading byte offset, both in units of 16 bytes, the high one is the
// same for all tiles (8-row groups 1,024 bytes apart, version 1, 128-byte
// swizzle).  K-major tiles do not use the leading offset; MN-major ones (rows
// of 64 values along MN, one per K index) have their 64-value atoms that far
// apart.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t leading) { return (saddr & 0x3FFFFu) >> 4 | (leading >> 4) << 16; }

// kind::f16, BF16 operands, FP32 accumulation: both from shared memory, or A
// (two values per column) from TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh));
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One lane of a converged warp.  The tcgen05 instructions take their operands
// from uniform registers: under elect.sync the compiler knows that one lane
// runs them, under `lane == 0` it loops over the lanes that might (an MMA then
// took 120 cycles to issue, 64 to execute).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(one));
    return one;
}

// tc::mbar_wait without its first read of the global timer, which takes longer
// than most waits here: the timer is read once in 4,096 tries.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, const volatile int* abort, uint64_t limit_ns) {
    const uint32_t addr = tc::smem_u32(bar);
    uint64_t start = 0;
    for (uint32_t i = 1;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity)
            : "memory");
        if (done) return true;
        if ((i & 63) == 0 && *abort) return false;
        if ((i & 4095) == 0) {
            const uint64_t now = tc::globaltimer_ns();
            if (start == 0) start = now;
            else if (now - start > limit_ns) return false;
        }
    }
}

// The work of one CTA, from its id.
struct Work {
    Span qs, ks;
    int seq, kv, group, per;        // per: tokens of a tile, kRows / group
    int token0;                     // first query of tile 0
    int rows[kTiles], keys[kTiles]; // live rows; keys that the last of them sees
};

__device__ __forceinline__ int keys_of(const PackedAttentionParams& p, const Work& w, int tile, int row) {
    if (!p.causal) return w.ks.len;
    const int token = w.token0 + tile * w.per + row / w.group;
    return min(max(token + (w.ks.len - w.qs.len) + 1, 0), w.ks.len);
}

__device__ __forceinline__ bool find_work(const PackedAttentionParams& p, Work& w) {
    w.group = p.heads / p.kv_heads;
    w.per = kRows / w.group;
    w.kv = blockIdx.x % p.kv_heads;
    const int step = kTiles * w.per;   // queries of a CTA
    const int pieces = gridDim.x / p.kv_heads, at = blockIdx.x / p.kv_heads;
    const int id = p.causal ? pieces - 1 - at : at;   // the longest rows first
    auto first_id = [&](int i) { return seq_offset(p.q_offsets, p.uniform, i, p.total_q) / step + i; };
    w.seq = find_owner(p.sequences, id, first_id);
    w.qs = seq_span(p.q_offsets, p.uniform, w.seq, p.total_q, p.bad);
    w.ks = seq_span(p.k_offsets, p.uniform, w.seq, p.total_k, p.bad);
    const int index = id - first_id(w.seq);
    if (index < 0 || index > w.qs.len / step) return false;
    w.token0 = index * step;
    const int left = w.qs.len - w.token0;
    if (left <= 0) return false;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        w.rows[t] = (left >= (t + 1) * w.per ? w.per : left > t * w.per ? left - t * w.per : 0) * w.group;
        w.keys[t] = w.rows[t] ? keys_of(p, w, t, w.rows[t] - 1) : 0;
    }
    return true;
}

template <int DC>
__global__ void __launch_bounds__(kThreads, 1) attention_tc_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                   const __grid_constant__ CUtensorMap map_k,
                                                                   const __grid_constant__ CUtensorMap map_v,
                                                                   PackedAttentionParams p, bool vec_out) {
    using L = Layout<DC>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t q_full, full[L::stages], empty[L::stages], s_full[kTiles], p_full[kTiles][kHalves], o_full[kTiles], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    Work w;
    check_offsets(p.q_offsets, p.sequences, p.total_q, p.bad);
    check_offsets(p.k_offsets, p.sequences, p.total_k, p.bad);
    if (!find_work(p, w)) return;   // the whole CTA
    uint8_t* smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sq = smem;
    uint8_t* ring = smem + L::q_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n[kTiles] = {(w.keys[0] + kKeys - 1) / kKeys, (w.keys[1] + kKeys - 1) / kKeys};
    const int steps = max(n[0], n[1]);

    // Stage 0 of the ring holds K of step 0, stage j + 1 V of step j and K of step
    // j + 1 (which the last stage lacks).  One lane of the copying warp.
    auto load_stage = [&](int i) {
        const int s = i % L::stages;
        tc::mbar_expect_tx(&full[s], (uint32_t)(i == 0 || i == steps ? L::tile_bytes : L::stage_bytes));
        uint8_t* to = ring + s * L::stage_bytes;
        for (int c = 0; i < steps && c < DC; ++c)
            tma_load_3d(to + L::tile_bytes + c * kChunk, &map_k, &full[s], c * 64, w.kv, w.ks.begin + i * kKeys);
        for (int c = 0; i > 0 && c < DC; ++c)
            tma_load_3d(to + c * kChunk, &map_v, &full[s], c * 64, w.kv, w.ks.begin + (i - 1) * kKeys);
    };
    if (warp == kSoftmaxWarps && elect_one()) {
        tc::mbar_init(&q_full, 1);
        for (int i = 0; i < L::stages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            tc::mbar_init(&s_full[t], 1);
            for (int h = 0; h < kHalves; ++h) tc::mbar_init(&p_full[t][h], 128);
            tc::mbar_init(&o_full[t], 1);
        }
        tc::mbar_init(&drain, 1);
        abort_flag = 0;
        tc::mbar_fence_init();
        if (steps > 0) {
            // The first copies start while the others set up.  A Q box is per x
            // group rows; rows past the tensor are zeros.
            const int q_tiles = 1 + (w.rows[1] > 0);
            tc::mbar_expect_tx(&q_full, (uint32_t)(q_tiles * DC * w.per * w.group * 128));
            for (int t = 0; t < q_tiles; ++t)
                for (int c = 0; c < DC; ++c)
                    tma_load_3d(sq + (t * DC + c) * kQChunk, &map_q, &q_full, c * 64, w.kv * w.group, w.qs.begin + w.token0 + t * w.per);
            load_stage(0);
        }
    }
    if (warp == kSoftmaxWarps + 1) tc::tmem_alloc(&tmem_slot, kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t tm_s[kTiles] = {tmem, tmem + kKeys}, tm_o[kTiles] = {tmem + 2 * kKeys, tmem + 2 * kKeys + 64 * DC};
    auto expired = [&](int code) {
        if (p.err) *reinterpret_cast<volatile int*>(p.err) = code;
        abort_flag = 1;
    };

    // The softmax warpgroups take the registers that the copying and issuing one
    // leaves: 2 x 208 + 88 of the 3 x 168 that the block is launched with.
    if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == kSoftmaxWarps && steps > 0) {
            int i = 1;
            for (; i <= steps; ++i) {
                if (i >= L::stages && !__all_sync(0xffffffffu, wait_phase(&empty[i % L::stages], (i / L::stages + 1) & 1, &abort_flag, p.wait_ns))) {
                    expired(1);
                    break;
                }
                const bool skip = p.skip_load && i == 1 && blockIdx.x == 0;
                if (!skip && elect_one()) load_stage(i);
                __syncwarp();
            }
            // No copy is in flight when the CTA ends, however it ends.
            tc::mbar_wait(&q_full, 0, false, p.wait_ns);
            for (int b = max(0, i - L::stages); b < i; ++b) tc::mbar_wait(&full[b % L::stages], (b / L::stages) & 1, false, p.wait_ns);
        } else if (warp == kSoftmaxWarps + 1 && steps > 0) {
            // An issued instruction costs this warp 30 to 50 cycles and a wait 200
            // although its phase is long complete, so there are as few as can be:
            // all 4 DC steps over d (past d both operands are zeros), one commit
            // per tile and step, one to release a stage, and barriers that are
            // waited for together on different lanes.
            const int n_out = (p.d + 15) / 16 * 16;
            const uint32_t id_s = tc::idesc_bf16(kRows, kKeys);
            const uint32_t id_o = tc::idesc_bf16(kRows, n_out) | (1u << 16);   // B MN-major
            const uint32_t q_desc = desc_low(tc::smem_u32(sq), 0), k_desc = desc_low(tc::smem_u32(ring) + L::tile_bytes, 0);
            const uint32_t v_desc = desc_low(tc::smem_u32(ring), kChunk);
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                if (ok && !__all_sync(0xffffffffu, wait_phase(bar, parity, &abort_flag, p.wait_ns))) {
                    expired(code);
                    ok = false;
                }
                tc::fence_after();
            };
            // One lane: the scores of tile t from the K tile at `k`.
            auto scores = [&](int t, uint32_t k) {
#pragma unroll
                for (int x = 0; x < 4 * DC; ++x)
                    mma_ss(tm_s[t], q_desc + (((t * DC + (x >> 2)) * kQChunk + (x & 3) * 32) >> 4),
                           k + (((x >> 2) * kChunk + (x & 3) * 32) >> 4), id_s, x > 0);
                tc::commit(&s_full[t]);
            };
            wait(lane ? &full[0] : &q_full, 0, 2);
            if (ok && elect_one()) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    if (n[t] > 0) scores(t, k_desc);
                tc::commit(&empty[0]);
            }
            __syncwarp();
            int s = 1, phase = 0;
            for (int j = 0; j < steps && ok; ++j) {
                // The stage, and tile 0's first weights.
                const bool own = lane && j < n[0];
                wait(own ? &p_full[0][0] : &full[s], own ? j & 1 : phase, 3);
                if (ok && (j + 1) * kKeys > w.ks.len) {
                    // The last tile's rows of V behind the sequence belong to others, and a
                    // weight of 0 times an infinity or NaN there would send every row of the
                    // CTA to the second computation (2,000 tokens with NaN behind them: 84 ms
                    // instead of 0.06).
                    __syncwarp();
                    for (int c = 0; c < DC; ++c)
                        for (int at = (w.ks.len - j * kKeys) * 128 + lane * 16; at < kChunk; at += 512)
                            *reinterpret_cast<uint4*>(ring + s * L::stage_bytes + c * kChunk + at) = make_uint4(0, 0, 0, 0);
                    tc::fence_proxy_async();
                    __syncwarp();
                }
                const uint32_t v = v_desc + s * (L::stage_bytes >> 4), k = k_desc + s * (L::stage_bytes >> 4);
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        if (t + h > 0 && j < n[t]) wait(&p_full[t][h], j & 1, 4);
                        if (!ok) break;
                        if (elect_one()) {
                            if (j < n[t]) {
#pragma unroll
                                for (int x = h * kHalf / 16; x < (h + 1) * kHalf / 16; ++x)
                                    mma_ts(tm_o[t], tm_s[t] + x * 8, v + x * (2048 >> 4), id_o, (j | x) > 0);
                                // The MMAs run in order: the next scores overwrite the weights
                                // that the product has read by then, and their commit covers it.
                                if (h + 1 == kHalves) {
                                    if (j + 1 < n[t]) scores(t, k);
                                    else tc::commit(&o_full[t]);
                                }
                            }
                            if (t + 1 == kTiles && h + 1 == kHalves) tc::commit(&empty[s]);
                        }
                        __syncwarp();
                    }
                }
                if (++s == L::stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
            // Every MMA this warp issued completes before TMEM is freed.
            if (elect_one()) tc::commit(&drain);
            __syncwarp();
            tc::mbar_wait(&drain, 0, false, tc::kWaitNs);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const int live = t ? w.rows[1] : w.rows[0], tiles = t ? n[1] : n[0];
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = (t ? tm_s[1] : tm_s[0]) + lanes, to = (t ? tm_o[1] : tm_o[0]) + lanes;
        const int n_out = (p.d + 15) / 16 * 16;
        const float scale = p.scale * 1.4426950408889634f;
        const int keys = live ? keys_of(p, w, t, min(row, live - 1)) : 0;
        const int sure = (int)__reduce_min_sync(0xffffffffu, (unsigned)keys);
        float top = -INFINITY, ref = 0.f, sum = 0.f;   // ref: top, 0 while it is -infinity
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
            ok = __all_sync(0xffffffffu, wait_phase(bar, parity, &abort_flag, p.wait_ns));
            if (!ok) expired(code);
            tc::fence_after();
        };
        for (int j = 0; j < tiles; ++j) {
            wait(&s_full[t], j & 1, 5);
            if (!ok) break;
            uint32_t r[kKeys];
            float* s = reinterpret_cast<float*>(r);
            // Each quarter's maximum while the next quarter is on its way.
            constexpr int Q = kKeys / 4;
            float m[4];
            auto load = [&](int c0) {
#pragma unroll
                for (int c = c0; c < c0 + Q; c += 16) tc::tmem_ld16_async(ts + c, r + c);
            };
            load(0);
#pragma unroll
            for (int c0 = 0; c0 < kKeys; c0 += Q) {
                tc::tmem_wait_ld();
#pragma unroll
                for (int c = c0; c < c0 + Q; ++c) asm volatile("" : "+r"(r[c]));
                if (c0 + Q < kKeys) load(c0 + Q);
                if ((j + 1) * kKeys > sure) {
                    const int left = keys - j * kKeys;
#pragma unroll
                    for (int c = c0; c < c0 + Q; ++c)
                        if (c >= left) s[c] = -INFINITY;
                }
#pragma unroll
                for (int c = c0; c < c0 + Q; c += 4)
#pragma unroll
                    for (int i = 0; i < 4; ++i) m[i] = c == 0 ? s[c + i] : fmaxf(m[i], s[c + i]);
            }
            const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * scale;
            if (__any_sync(0xffffffffu, most > top + kSlack)) {
                // The warp's branch, but each row by its own scores: a key that a row
                // must not see cannot move what its neighbour's rounding depends on.
                const float next = most > top + kSlack ? most : top;
                const float g = next == top ? 1.f : top == -INFINITY ? 0.f : exp2_hw(top - next);
                top = next;
                ref = top == -INFINITY ? 0.f : top;
                sum *= g;
                if (j > 0) {   // the scores' commit covers the product that wrote O
                    for (int c = 0; c < n_out; c += 16) {
                        uint32_t o[16];
                        tc::tmem_ld16(to + c, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * g);
                        tmem_st16(to + c, o);
                    }
                }
            }
            float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            const float2 a = make_float2(scale, scale), b = make_float2(-ref, -ref);
#pragma unroll
            for (int c = 0; c < kKeys; c += 2) {
                float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), a, b);
                x = c / 2 % 8 < kEmulated ? exp2_fma(x) : make_float2(exp2_hw(x.x), exp2_hw(x.y));
                part[(c >> 1) & 1] = __fadd2_rn(part[(c >> 1) & 1], x);
                const __nv_bfloat162 v = __floats2bfloat162_rn(x.x, x.y);
                r[c / 2] = *reinterpret_cast<const uint32_t*>(&v);
                if (c % 32 == 30) tmem_st16(ts + c / 32 * 16, r + c / 32 * 16);
                if ((c + 2) % kHalf == 0) {
                    tmem_wait_st();
                    tc::fence_before();
                    tc::mbar_arrive(&p_full[t][c / kHalf]);
                }
            }
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
        }
        if (ok && tiles > 0) wait(&o_full[t], 0, 6);
        if (ok && live) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int token = w.qs.begin + w.token0 + t * w.per + row / w.group, head = w.kv * w.group + row % w.group;
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out.ptr) + token * p.out.token_stride + head * p.out.head_stride;
            bool bad = row < live && rounding_spoils(top);
            // Straight from TMEM, a row per lane.  (Through shared memory, with 512
            // bytes to a store, it took 5,000 cycles instead of 3,000: the other
            // tile's scores keep shared memory busy.)
            for (int c = 0; c < n_out; c += 16) {
                uint32_t o[16] = {};
                __syncwarp();   // the load is the warp's; rows past the piece have skipped the stores
                if (tiles > 0) tc::tmem_ld16(to + c, o);
                if (row >= live) continue;
                uint32_t h[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = __uint_as_float(o[2 * i]) * inv, y = __uint_as_float(o[2 * i + 1]) * inv;
                    bad |= !isfinite(x) || !isfinite(y);
                    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
                    h[i] = *reinterpret_cast<const uint32_t*>(&v);
                }
                if (vec_out) {   // d is a multiple of 8
                    *reinterpret_cast<uint4*>(out + c) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (c + 8 < p.d) *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (c + i < p.d) out[c + i] = reinterpret_cast<const __nv_bfloat16*>(h)[i];
                }
            }
            __syncwarp();
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q.ptr);
            const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(p.k.ptr) + (long long)w.ks.begin * p.k.token_stride + w.kv * p.k.head_stride;
            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v.ptr) + (long long)w.ks.begin * p.v.token_stride + w.kv * p.v.head_stride;
            for (unsigned again = __ballot_sync(0xffffffffu, bad); again; again &= again - 1) {
                const int rr = (warp & 3) * 32 + __ffs(again) - 1;
                const int tk = w.qs.begin + w.token0 + t * w.per + rr / w.group, hd = w.kv * w.group + rr % w.group;
                __syncwarp();
                attend_row<__nv_bfloat16>(q + tk * p.q.token_stride + hd * p.q.head_stride, k, p.k.token_stride, v, p.v.token_stride,
                                          p.d, keys_of(p, w, t, rr), scale,
                                          static_cast<__nv_bfloat16*>(p.out.ptr) + tk * p.out.token_stride + hd * p.out.head_stride);
            }
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + 1) {
        tc::fence_after();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            ptr = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    }();
    return fn;
}

// [tokens][heads][d] as a 3D map (d, heads, tokens), boxes of 64 values.
bool make_map(CUtensorMap* map, const SeqTensor& t, int d, int heads, int tokens, int box_heads, int box_tokens) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens};
    // A single head's or token's stride is never used, but has to be a valid one.
    cuuint64_t strides[2] = {heads > 1 ? (cuuint64_t)t.head_stride * 2 : 16, tokens > 1 ? (cuuint64_t)t.token_stride * 2 : 16};
    cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, t.ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool mappable(const SeqTensor& t, int heads, int tokens) {
    return rows16(t, 2) && (heads == 1 || t.head_stride > 0) && (tokens == 1 || t.token_stride > 0);
}

template <int DC>
cudaError_t launch_dc(const PackedAttentionParams& p, cudaStream_t stream) {
    const int group = p.heads / p.kv_heads, per = kRows / group;
    PackedAttentionParams a = p;
    if (!a.wait_ns) a.wait_ns = tc::kWaitNs;
    CUtensorMap mq, mk, mv;
    if (!make_map(&mq, p.q, p.d, p.heads, p.total_q, group, per) || !make_map(&mk, p.k, p.d, p.kv_heads, p.total_k, 1, kKeys) ||
        !make_map(&mv, p.v, p.d, p.kv_heads, p.total_k, 1, kKeys))
        return cudaErrorInvalidValue;
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(attention_tc_kernel<DC>), Layout<DC>::smem);
    if (e != cudaSuccess) return e;
    const long long pieces = (long long)p.total_q / (kTiles * per) + p.sequences;
    attention_tc_kernel<DC><<<(unsigned)(pieces * p.kv_heads), kThreads, Layout<DC>::smem, stream>>>(mq, mk, mv, a, rows16(p.out, 2));
    return cudaGetLastError();
}

}  // namespace

bool attention_tc_supported(const PackedAttentionParams& p) {
    return p.dtype == DT_BF16 && p.d % 8 == 0 && p.d <= 128 && p.heads / p.kv_heads <= kRows && p.total_q > 0 && p.total_k > 0 &&
           mappable(p.q, p.heads, p.total_q) && mappable(p.k, p.kv_heads, p.total_k) && mappable(p.v, p.kv_heads, p.total_k);
}

cudaError_t launch_attention_tc(const PackedAttentionParams& p, cudaStream_t stream) {
    return p.d <= 64 ? launch_dc<1>(p, stream) : launch_dc<2>(p, stream);
}

}  // namespace ppocr
