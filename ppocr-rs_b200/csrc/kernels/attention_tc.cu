// Attention over packed sequences on tcgen05 (BF16): the kernel of long
// sequences.
//
// A CTA owns two tiles of 128 rows of one (sequence, KV head); the query heads
// that share the KV head are rows too (row = token x group + head), so K and V
// are read once per 256 rows.  Roles (320 threads):
//   warp 8 / lane 0   TMA: both Q tiles, then K and V tiles of 128 keys into a
//                     ring (128-byte swizzled, 64 values of d per row chunk);
//   warp 9 / lane 0   MMA: S = Q K^T (both operands in shared memory, K-major)
//                     into TMEM, and O += P V with P read from TMEM and V
//                     MN-major as it lies;
//   warps 0-3, 4-7    softmax of tile 0 and 1, one row per thread: scores from
//                     TMEM to registers, running maximum and sum, weights back
//                     as BF16 over the scores' columns.
// While one tile's softmax runs, the tensor cores work on the other's
// products.  The maximum that weights are relative to moves only when a score
// passes it by more than 8 (in log2: weights up to 2^8, exact in BF16's
// range), so the output accumulator in TMEM is rarely rescaled.
//
// Bound: per 128 x 128 tile and d = 128 the products take 1,024 cycles of the
// tensor cores and the 16,384 exponentials 1,024 cycles of the special
// function units (16 a cycle).
//
// Every wait is bounded: on expiry the CTA records a code in status[1], stops,
// lets its copies and MMAs land, frees its TMEM and returns.  Rows that come
// out non-finite are computed again from their definition (attend_row).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "attention_packed.cuh"
#include "tcgen05.cuh"

namespace ppocr {

namespace {

constexpr int kRows = 128, kKeys = 128, kTiles = 2, kThreads = 32 * (4 * kTiles + 2);
constexpr int kChunk = kKeys * 128;                  // bytes of 128 rows x 64 values
constexpr int kTmemCols = 512;
constexpr float kSlack = 8.f;

template <int DC>   // chunks of 64 values of d
struct Layout {
    static constexpr int slots = DC == 1 ? 6 : 4;
    static constexpr int q_bytes = kTiles * DC * kChunk, slot_bytes = DC * kChunk;
    static constexpr int smem = q_bytes + slots * slot_bytes + 1024;
};

// MN-major operand, 128-byte swizzle: rows of 64 values along MN, one per K
// index; 64-value atoms `atom_stride` bytes apart, groups of 8 K indices 1024.
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t atom_stride) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(atom_stride >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// A (BF16, two per column) from TMEM.
__device__ __forceinline__ void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate));
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
    const long long pieces = gridDim.x / p.kv_heads, at = blockIdx.x / p.kv_heads;
    const long long id = p.causal ? pieces - 1 - at : at;   // the longest rows first
    auto first_id = [&](int i) { return (long long)seq_offset(p.q_offsets, p.uniform, i, p.total_q) / step + i; };
    w.seq = find_owner(p.sequences, id, first_id);
    w.qs = seq_span(p.q_offsets, p.uniform, w.seq, p.total_q, p.status);
    w.ks = seq_span(p.k_offsets, p.uniform, w.seq, p.total_k, p.status);
    const long long first = (id - first_id(w.seq)) * step;
    if (first < 0 || first >= w.qs.len) return false;
    w.token0 = (int)first;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        w.rows[t] = min(max(w.qs.len - w.token0 - t * w.per, 0), w.per) * w.group;
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
    __shared__ __align__(8) uint64_t q_full, full[L::slots], empty[L::slots], s_full[kTiles], p_full[kTiles], o_full[kTiles], drain;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    Work w;
    if (!find_work(p, w)) return;   // the whole CTA
    uint8_t* smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sq = smem;
    uint8_t* ring = smem + L::q_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n[kTiles] = {(w.keys[0] + kKeys - 1) / kKeys, (w.keys[1] + kKeys - 1) / kKeys};
    const int steps = max(n[0], n[1]);

    if (threadIdx.x == 0) {
        tc::mbar_init(&q_full, 1);
        for (int i = 0; i < L::slots; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < kTiles; ++t) {
            tc::mbar_init(&s_full[t], 1);
            tc::mbar_init(&p_full[t], 128);
            tc::mbar_init(&o_full[t], 1);
        }
        tc::mbar_init(&drain, 1);
        abort_flag = 0;
        tc::mbar_fence_init();
    }
    if (warp == 4 * kTiles) tc::tmem_alloc(&tmem_slot, kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t tm_s[kTiles] = {tmem, tmem + kKeys}, tm_o[kTiles] = {tmem + 2 * kKeys, tmem + 2 * kKeys + 64 * DC};
    auto expired = [&](int code) {
        if (p.status) reinterpret_cast<volatile int*>(p.status)[1] = code;
        abort_flag = 1;
    };

    if (warp == 4 * kTiles) {
        if (lane == 0 && steps > 0) {
            int q_tiles = 0;
            for (int t = 0; t < kTiles; ++t) q_tiles += w.rows[t] > 0;
            // A Q box is per x group rows; rows past the tensor are zeros.
            tc::mbar_expect_tx(&q_full, (uint32_t)(q_tiles * DC * w.per * w.group * 128));
            for (int t = 0; t < q_tiles; ++t)
                for (int c = 0; c < DC; ++c)
                    tma_load_3d(sq + (t * DC + c) * kChunk, &map_q, &q_full, c * 64, w.kv * w.group, w.qs.begin + w.token0 + t * w.per);
            // Tile i of the ring: K of step i / 2, then V of it.
            int i = 0;
            for (; i < 2 * steps; ++i) {
                const int s = i % L::slots;
                if (i >= L::slots && !tc::mbar_wait(&empty[s], (i / L::slots + 1) & 1, false, tc::kWaitNs, &abort_flag)) {
                    expired(1);
                    break;
                }
                tc::mbar_expect_tx(&full[s], (uint32_t)L::slot_bytes);
                for (int c = 0; c < DC; ++c)
                    tma_load_3d(ring + s * L::slot_bytes + c * kChunk, i & 1 ? &map_v : &map_k, &full[s], c * 64, w.kv,
                                w.ks.begin + (i >> 1) * kKeys);
            }
            // No copy is in flight when the CTA ends, however it ends.
            tc::mbar_wait(&q_full, 0, false);
            for (int b = max(0, i - L::slots); b < i; ++b) tc::mbar_wait(&full[b % L::slots], (b / L::slots) & 1, false);
        }
    } else if (warp == 4 * kTiles + 1) {
        if (lane == 0 && steps > 0) {
            const int k_steps = (p.d + 15) / 16, n_out = k_steps * 16;
            const uint32_t id_s = tc::idesc_bf16(kRows, kKeys);
            const uint32_t id_o = tc::idesc_bf16(kRows, n_out) | (1u << 16);   // B MN-major
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                if (ok && !tc::mbar_wait(bar, parity, false, tc::kWaitNs, &abort_flag)) {
                    expired(code);
                    ok = false;
                }
                if (ok) tc::fence_after();
            };
            auto scores = [&](int t, int j) {
                const uint32_t q = tc::smem_u32(sq + t * DC * kChunk), k = tc::smem_u32(ring + (2 * j % L::slots) * L::slot_bytes);
                for (int x = 0; x < k_steps; ++x) {
                    const uint32_t at = (x >> 2) * kChunk + (x & 3) * 32;
                    tc::mma_bf16(tm_s[t], tc::sw128_desc(q + at), tc::sw128_desc(k + at), id_s, x > 0);
                }
                tc::commit(&s_full[t]);
            };
            wait(&q_full, 0, 2);
            wait(&full[0], 0, 3);
            if (ok) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    if (n[t] > 0) scores(t, 0);
                tc::commit(&empty[0]);
            }
            for (int j = 0; j < steps && ok; ++j) {
                const int v_at = 2 * j + 1, k_at = 2 * j + 2;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    if (!ok) break;
                    if (j < n[t]) {
                        wait(&p_full[t], j & 1, 4);
                        wait(&full[v_at % L::slots], (v_at / L::slots) & 1, 5);
                        if (!ok) break;
                        const uint32_t v = tc::smem_u32(ring + (v_at % L::slots) * L::slot_bytes);
#pragma unroll
                        for (int x = 0; x < kKeys / 16; ++x)
                            mma_bf16_ts(tm_o[t], tm_s[t] + x * 8, sw128_desc_mn(v + x * 2048, kChunk), id_o, (j | x) > 0);
                        if (j + 1 == n[t]) tc::commit(&o_full[t]);
                    }
                    if (t == kTiles - 1) tc::commit(&empty[v_at % L::slots]);
                    // The MMAs run in order: these scores overwrite the weights that
                    // the product above has read by then, and their commit covers it.
                    if (j + 1 < n[t]) {
                        wait(&full[k_at % L::slots], (k_at / L::slots) & 1, 6);
                        if (!ok) break;
                        scores(t, j + 1);
                    }
                }
                if (ok && j + 1 < steps) tc::commit(&empty[k_at % L::slots]);
            }
            // Every MMA this thread issued completes before TMEM is freed.
            tc::commit(&drain);
            tc::mbar_wait(&drain, 0, false);
        }
    } else {
        const int t = warp >> 2, row = (warp & 3) * 32 + lane, live = t ? w.rows[1] : w.rows[0], tiles = t ? n[1] : n[0];
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = (t ? tm_s[1] : tm_s[0]) + lanes, to = (t ? tm_o[1] : tm_o[0]) + lanes;
        const int n_out = (p.d + 15) / 16 * 16;
        const float scale = p.scale * 1.4426950408889634f;
        const int keys = live ? keys_of(p, w, t, min(row, live - 1)) : 0;
        const int sure = (int)__reduce_min_sync(0xffffffffu, (unsigned)keys);
        float top = -INFINITY, ref = 0.f, sum = 0.f;   // ref: top, 0 while it is -infinity
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&s_full[t], j & 1, false, tc::kWaitNs, &abort_flag));
            if (!ok) {
                if (lane == 0) expired(7);
                break;
            }
            tc::fence_after();
            uint32_t r[kKeys];
#pragma unroll
            for (int c = 0; c < kKeys; c += 16) tc::tmem_ld16_async(ts + c, r + c);
            tc::tmem_wait_ld_regs(r);
            float* s = reinterpret_cast<float*>(r);
            if ((j + 1) * kKeys > sure) {
                const int left = keys - j * kKeys;
#pragma unroll
                for (int c = 0; c < kKeys; ++c)
                    if (c >= left) s[c] = -INFINITY;
            }
            float m[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < kKeys; c += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i) m[i] = fmaxf(m[i], s[c + i]);
            const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * scale;
            if (__any_sync(0xffffffffu, most > top + kSlack)) {
                const float next = fmaxf(top, most);
                const float g = top == -INFINITY ? 0.f : exp2_hw(top - next);
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
                x = make_float2(exp2_hw(x.x), exp2_hw(x.y));
                part[(c >> 1) & 1] = __fadd2_rn(part[(c >> 1) & 1], x);
                const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
                r[c / 2] = *reinterpret_cast<const uint32_t*>(&h);
            }
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
#pragma unroll
            for (int c = 0; c < kKeys / 2; c += 16) tmem_st16(ts + c, r + c);
            tmem_wait_st();
            tc::fence_before();
            tc::mbar_arrive(&p_full[t]);
        }
        if (ok && tiles > 0) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&o_full[t], 0, false, tc::kWaitNs, &abort_flag));
            if (!ok && lane == 0) expired(8);
            tc::fence_after();
        }
        if (ok && live) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int token = w.token0 + t * w.per + row / w.group, head = w.kv * w.group + row % w.group;
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out.ptr) + (w.qs.begin + (long long)token) * p.out.token_stride +
                                 head * p.out.head_stride;
            bool bad = false;
            for (int c = 0; c < n_out; c += 16) {
                uint32_t o[16] = {};
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
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q.ptr);
            const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(p.k.ptr) + (long long)w.ks.begin * p.k.token_stride + w.kv * p.k.head_stride;
            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v.ptr) + (long long)w.ks.begin * p.v.token_stride + w.kv * p.v.head_stride;
            for (unsigned again = __ballot_sync(0xffffffffu, bad); again; again &= again - 1) {
                const int l = __ffs(again) - 1, rr = (warp & 3) * 32 + l;
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
    if (warp == 4 * kTiles) {
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
    CUtensorMap mq, mk, mv;
    if (!make_map(&mq, p.q, p.d, p.heads, p.total_q, group, per) || !make_map(&mk, p.k, p.d, p.kv_heads, p.total_k, 1, kKeys) ||
        !make_map(&mv, p.v, p.d, p.kv_heads, p.total_k, 1, kKeys))
        return cudaErrorInvalidValue;
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(attention_tc_kernel<DC>), Layout<DC>::smem);
    if (e != cudaSuccess) return e;
    const long long pieces = (long long)p.total_q / (kTiles * per) + p.sequences;
    attention_tc_kernel<DC><<<(unsigned)(pieces * p.kv_heads), kThreads, Layout<DC>::smem, stream>>>(mq, mk, mv, p, rows16(p.out, 2));
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
