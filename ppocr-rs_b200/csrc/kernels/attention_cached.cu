// Single-token attention over the 8-bit paged cache.
//
//   out[h] = sum_t softmax_t(scale q[h] . k_t) v_t,  k_t = s_k int8, v_t = s_v int8
//
// Bound: HBM, the cache's bytes (2 d + 8 / page per token and KV head).  A
// byte is worth 2 multiply-adds per query head, so grouped heads would keep
// CUDA cores busier than the memory; the products run on mma.m16n8k16 with 16
// tokens (or 16 values of d) as M and the up to eight query heads of a group
// as N, so a tile of 16 tokens costs two MMAs per 16 values of d whatever the
// group.  (tcgen05 would want 128 rows of M and the operands in shared memory;
// these tiles go from HBM to registers directly, in the layout that the MMA
// wants, and never touch shared memory.)
//
// Integers are exact in FP16.  q is scaled by a power of two per head to fit
// FP16; FP32 inputs are carried as two FP16 pieces (22 bits), as are their
// softmax weights, so their products are FP32-class.  A page's K scale
// multiplies its scores; its V scale multiplies its weights, taken relative to
// a running reference R so that they stay in FP16's range.
//
// A warp owns every fourth tile of its block's token range and keeps its own
// softmax state; the running maximum moves only when a score passes it by
// more than 8 (weights up to 2^8), so most tiles need no reduction at all.
// The range of a sequence is split over the blocks of a cluster (1 to 8) when
// there are few sequences and heads; warps join through shared memory, blocks
// through distributed shared memory, both in a fixed order: one launch, no
// workspace.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "seq_common.cuh"

namespace ppocr {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kHeads = 8;
constexpr int kTile = 16;             // tokens per tile
constexpr float kSlack = 8.f;         // log2 of the largest weight before the maximum moves
constexpr float kWeightScale = 64.f;  // weights are held times 64: a larger range above FP16's subnormals

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

// Transposes an 8 x 8 matrix of FP16 held two columns per lane (row lane / 4).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// BYTES bytes of a cache row into words; bytes at and past `live` (a multiple
// of 8) read as 0.  V16: rows are 16-byte aligned, else 8.
template <int BYTES, bool V16>
__device__ __forceinline__ void load_row(const int8_t* p, int live, uint32_t* w) {
    if constexpr (BYTES == 4) {
        w[0] = live > 0 ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
    } else if constexpr (BYTES == 16 && V16) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (live > 0) u = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) {
            uint2 u = make_uint2(0, 0);
            if (8 * i < live) u = __ldg(reinterpret_cast<const uint2*>(p) + i);
            w[2 * i] = u.x; w[2 * i + 1] = u.y;
        }
    }
}

// Bytes of K that a lane holds of one token, by piece: values of d
// [at, at + kPieceK) for piece 0, 64 further for piece 1.
template <int DP> constexpr int kPieceK = DP == 32 ? 8 : 16;
template <int DP> constexpr int kPiecesK = DP / 4 / kPieceK<DP>;

template <int DP, bool V16>
struct TileData {
    uint32_t k[2][DP / 16];   // tokens lane / 4 and lane / 4 + 8
    uint32_t v[4][DP / 32];   // tokens 2c, 2c + 1, 2c + 8, 2c + 9 with c = lane % 4
    float sk, sv;
    bool ok;

    __device__ __forceinline__ void load(const CachedAttentionParams& p, int where, int head, int slot0, int lane) {
        ok = where >= 0;
        if (!ok) return;
        const int d = p.cache.d, r = lane >> 2, c = lane & 3;
        const long long cell = (long long)where * p.cache.kv_heads + head;
        const int8_t* kp = p.cache.k + (cell * p.cache.page + slot0) * d;
        const int8_t* vp = p.cache.v + (cell * p.cache.page + slot0) * d;
        sk = __ldg(p.cache.k_scales + cell);
        sv = __ldg(p.cache.v_scales + cell);
        constexpr int PK = kPieceK<DP>;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < kPiecesK<DP>; ++i) {
                const int at = 64 * i + c * PK;
                load_row<PK, V16>(kp + (r + 8 * t) * d + at, d - at, &k[t][i * PK / 4]);
            }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int tok = 2 * c + (t & 1) + 8 * (t >> 1), at = r * (DP / 8);
            load_row<DP / 8, V16>(vp + tok * d + at, d - at, v[t]);
        }
    }
};

template <typename T, int DP, bool V16>
__global__ void __launch_bounds__(kThreads) attention_cached_kernel(CachedAttentionParams p, int splits) {
    constexpr bool SPLIT = sizeof(T) == 4;   // FP32: two FP16 pieces
    constexpr int KS = DP / 16;              // 16-wide steps over d
    constexpr int PK = kPieceK<DP>;
    __shared__ float sm_o[kWarps][kHeads][DP];
    __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int seq = blockIdx.x / splits, split = blockIdx.x % splits;
    const int group = p.heads / p.cache.kv_heads, parts = (group + kHeads - 1) / kHeads;
    const int kv = blockIdx.y / parts, part = blockIdx.y % parts;
    const int head0 = kv * group + part * kHeads, live_heads = min(kHeads, group - part * kHeads);
    const int page = p.cache.page, d = p.cache.d;

    int len = p.lengths[seq];
    const long long room = (long long)p.table.width * page;
    if (len < 0 || len > room) {
        if (threadIdx.x == 0) seq_bad_index(p.status);
        len = len < 0 ? 0 : (int)room;
    }
    const int tiles = (len + kTile - 1) / kTile, per = (tiles + splits - 1) / splits;
    const int t_end = min(tiles, (split + 1) * per);
    const int32_t* pages = p.table.pages + seq * p.table.stride;
    auto page_of = [&](int t) {
        if (t >= t_end) return -1;
        const int w = __ldg(pages + t * kTile / page);
        if (w < 0 || w >= p.cache.pages) {
            seq_bad_index(p.status);
            return -1;
        }
        return w;
    };
    TileData<DP, V16> cur, nxt;
    int t = split * per + warp;
    {
        const int w0 = page_of(t);
        cur.load(p, w0, kv, t * kTile % page, lane);
    }
    int w_next = page_of(t + kWarps);

    // B operand of the scores: head r's values of d, in the order in which the
    // lane's K bytes come; b0 holds bytes 4s, 4s + 1 and b1 bytes 4s + 2, 4s + 3.
    uint32_t qh[KS][2], ql[SPLIT ? KS : 1][2];
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
        // Power of two that takes the head's largest value into [2^8, 2^9).
        const int e = max((int)(__float_as_uint(top) >> 23) - 127, -100);
        const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
        qscale = p.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 8 + e) << 23);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = x[4 * s + 2 * h] * up, b = x[4 * s + 2 * h + 1] * up;
                const __half2 hi = __floats2half2_rn(a, b);
                qh[s][h] = h2_bits(hi);
                if constexpr (SPLIT) {
                    const float2 f = __half22float2(hi);
                    ql[s][h] = h2_bits(__floats2half2_rn(isinf(f.x) ? 0.f : a - f.x, isinf(f.y) ? 0.f : b - f.y));
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
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, ref = 0.f;

    for (; t < t_end; t += kWarps) {
        nxt.load(p, w_next, kv, (t + kWarps) * kTile % page, lane);
        w_next = page_of(t + 2 * kWarps);
        if (cur.ok) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t u0 = cur.k[0][i] ^ 0x80808080u, u1 = cur.k[1][i] ^ 0x80808080u;
                const uint32_t a0 = bytes_to_h2(u0, 0x4140), a1 = bytes_to_h2(u1, 0x4140);
                const uint32_t a2 = bytes_to_h2(u0, 0x4342), a3 = bytes_to_h2(u1, 0x4342);
                mma_f16(s, a0, a1, a2, a3, qh[i][0], qh[i][1]);
                if constexpr (SPLIT) mma_f16(s, a0, a1, a2, a3, ql[i][0], ql[i][1]);
            }
            const int tok = t * kTile + r;
            const float k0 = f0 * cur.sk, k1 = f1 * cur.sk;
            s[0] = tok < len ? s[0] * k0 : -INFINITY;
            s[1] = tok < len ? s[1] * k1 : -INFINITY;
            s[2] = tok + 8 < len ? s[2] * k0 : -INFINITY;
            s[3] = tok + 8 < len ? s[3] * k1 : -INFINITY;
            const float t0 = fmaxf(s[0], s[2]), t1 = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, t0 > m0 + kSlack || t1 > m1 + kSlack || cur.sv > 2.f * ref)) {
                float n0 = fmaxf(t0, m0), n1 = fmaxf(t1, m1);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
                    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
                }
                const float g0 = m0 == -INFINITY ? 0.f : exp2_hw(m0 - n0), g1 = m1 == -INFINITY ? 0.f : exp2_hw(m1 - n1);
                const float next = fmaxf(ref, cur.sv);
                const float back = next > ref ? ref / next : 1.f;
                m0 = n0; m1 = n1; ref = next;
                l0 *= g0; l1 *= g1;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    o[j][0] *= g0 * back; o[j][1] *= g1 * back;
                    o[j][2] *= g0 * back; o[j][3] *= g1 * back;
                }
            }
            const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
            s[0] = exp2_hw(s[0] - b0); s[1] = exp2_hw(s[1] - b1);
            s[2] = exp2_hw(s[2] - b0); s[3] = exp2_hw(s[3] - b1);
            l0 += s[0] + s[2];
            l1 += s[1] + s[3];
            // ref is 0 only while every V scale seen is 0: weights of zeros.
            const float w = ref > 0.f ? cur.sv * (kWeightScale / ref) : cur.sv;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] *= w;
            const __half2 h0 = __floats2half2_rn(s[0], s[1]), h1 = __floats2half2_rn(s[2], s[3]);
            const uint32_t p0 = transpose8(h2_bits(h0)), p1 = transpose8(h2_bits(h1));
            uint32_t e0 = 0, e1 = 0;
            if constexpr (SPLIT) {
                const float2 x = __half22float2(h0), y = __half22float2(h1);
                e0 = transpose8(h2_bits(__floats2half2_rn(s[0] - x.x, s[1] - x.y)));
                e1 = transpose8(h2_bits(__floats2half2_rn(s[2] - y.x, s[3] - y.y)));
            }
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const uint32_t u0 = cur.v[0][i] ^ 0x80808080u, u1 = cur.v[1][i] ^ 0x80808080u;
                const uint32_t u2 = cur.v[2][i] ^ 0x80808080u, u3 = cur.v[3][i] ^ 0x80808080u;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // Bytes 2h and 2h + 1 of two tokens, interleaved by value of d.
                    const uint32_t x = __byte_perm(u0, u1, h ? 0x7362 : 0x5140), y = __byte_perm(u2, u3, h ? 0x7362 : 0x5140);
                    const uint32_t a0 = bytes_to_h2(x, 0x4140), a1 = bytes_to_h2(x, 0x4342);
                    const uint32_t a2 = bytes_to_h2(y, 0x4140), a3 = bytes_to_h2(y, 0x4342);
                    mma_f16(o[2 * i + h], a0, a1, a2, a3, p0, p1);
                    if constexpr (SPLIT) mma_f16(o[2 * i + h], a0, a1, a2, a3, e0, e1);
                }
            }
        }
        cur = nxt;
    }

    // Join the warps, then the cluster's blocks.
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, x);
        l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (r == 0) {
        sm_m[warp][2 * c] = m0; sm_m[warp][2 * c + 1] = m1;
        sm_l[warp][2 * c] = l0; sm_l[warp][2 * c + 1] = l1;
    }
    const float unit = ref > 0.f ? ref / kWeightScale : 1.f;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
        const int at = r * (DP / 8) + 2 * j;
        sm_o[warp][2 * c][at] = o[j][0] * unit;
        sm_o[warp][2 * c + 1][at] = o[j][1] * unit;
        sm_o[warp][2 * c][at + 1] = o[j][2] * unit;
        sm_o[warp][2 * c + 1][at + 1] = o[j][3] * unit;
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (splits > 1) cluster.sync(); else __syncthreads();
    // Outputs are dealt to the cluster's threads; each sums the warps of all
    // blocks in order.
    const int rank = splits > 1 ? (int)cluster.block_rank() : 0;
    for (int i = rank * kThreads + threadIdx.x; i < live_heads * d; i += splits * kThreads) {
        const int h = i / d, x = i % d;
        float top = -INFINITY;
        for (int b = 0; b < splits; ++b) {
            const float* m = splits > 1 ? cluster.map_shared_rank(&sm_m[0][0], b) : &sm_m[0][0];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m[w * kHeads + h]);
        }
        float sum = 0.f, l = 0.f;
        for (int b = 0; b < splits; ++b) {
            const float* m = splits > 1 ? cluster.map_shared_rank(&sm_m[0][0], b) : &sm_m[0][0];
            const float* ls = splits > 1 ? cluster.map_shared_rank(&sm_l[0][0], b) : &sm_l[0][0];
            const float* os = splits > 1 ? cluster.map_shared_rank(&sm_o[0][0][0], b) : &sm_o[0][0][0];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = m[w * kHeads + h];
                const float g = mw == -INFINITY ? 0.f : exp2_hw(mw - top);
                l = fmaf(g, ls[w * kHeads + h], l);
                sum = fmaf(g, os[(w * kHeads + h) * DP + x], sum);
            }
        }
        T* out = static_cast<T*>(p.out.ptr) + seq * p.out.token_stride + (head0 + h) * p.out.head_stride;
        out[x] = from_f<T>(l == 0.f ? 0.f : sum / l);
    }
    if (splits > 1) cluster.sync();   // no block leaves while another reads its shared memory
}

template <typename T, int DP, bool V16>
cudaError_t launch_one(const CachedAttentionParams& p, int splits, dim3 grid, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = kThreads;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attention_cached_kernel<T, DP, V16>, p, splits);
}

template <typename T>
cudaError_t launch_type(const CachedAttentionParams& p, int splits, dim3 grid, cudaStream_t stream) {
    const int d = p.cache.d;
    if (d <= 32) return launch_one<T, 32, false>(p, splits, grid, stream);
    if (d <= 64) return d % 16 ? launch_one<T, 64, false>(p, splits, grid, stream) : launch_one<T, 64, true>(p, splits, grid, stream);
    return d % 16 ? launch_one<T, 128, false>(p, splits, grid, stream) : launch_one<T, 128, true>(p, splits, grid, stream);
}

}  // namespace

cudaError_t launch_attention_cached(const CachedAttentionParams& p, cudaStream_t stream) {
    if (p.table.sequences == 0) return cudaSuccess;
    const int group = p.heads / p.cache.kv_heads, parts = (group + kHeads - 1) / kHeads;
    const long long rows = (long long)p.table.sequences * p.cache.kv_heads * parts;
    // Blocks per sequence and head: enough for three blocks on each SM, as
    // long as a block keeps 16 tiles of the longest sequence the table holds.
    const long long tiles = (long long)p.table.width * p.cache.page / kTile;
    int splits = 1;
    while (splits < 8 && rows * splits < 148 * 3 && tiles / (2 * splits) >= 16) splits *= 2;
    const dim3 grid((unsigned)(p.table.sequences * (long long)splits), (unsigned)(p.cache.kv_heads * parts));
    return p.dtype == DT_F32 ? launch_type<float>(p, splits, grid, stream)
                             : launch_type<__nv_bfloat16>(p, splits, grid, stream);
}

}  // namespace ppocr
