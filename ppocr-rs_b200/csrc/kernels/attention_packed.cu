// Attention over packed sequences on mma.sync: every type, head size up to
// 128, stride and length; the kernel of the short sequences, whose tiles are
// too small to fill a tcgen05 tile (128 rows) or to pay for its set-up, and of
// FP32.
//
// A block owns 64 rows of one (sequence, KV head): the `group` query heads
// that share the KV head are rows too (row = token x group + head), so K and V
// are read once per group.  Keys pass through shared memory in tiles, double
// buffered with cp.async, with the running maximum and sum of the softmax in
// registers; scores and weights never leave them.
//   BF16: m16n8k16, weights rounded to BF16 for the second product (2^-9 of a
//         weight, averaged over the keys; the sum uses the unrounded ones).
//   FP32: m16n8k8 TF32 with both operands in two pieces (22 bits) and the
//         three leading products: FP32-class.
// Rows with no key give zeros; a non-finite row is computed again from its
// definition (attend_row).
#include "attention_packed.cuh"

namespace ppocr {

namespace {

constexpr int kThreads = 128, kRows = 64;

template <typename T> struct Traits;
template <> struct Traits<__nv_bfloat16> {
    static constexpr int keys = 64, pad = 8;
};
template <> struct Traits<float> {
    static constexpr int keys = 32, pad = 4;
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool live) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_bf16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32_1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
}

// x as a TF32 value (rounded to nearest) and the rest; the MMA ignores the low
// 13 bits, so the rest only needs its rounding added.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}

// Rows [0, rows) of `src` into shared memory at pitch DP + pad, zeros past
// them and past column d; row n of the tile is at src + at(n).
template <typename T, int DP, typename At>
__device__ __forceinline__ void load_tile(T* dst, const T* src, At at, int tile_rows, int rows, int d, bool vec) {
    constexpr int P = DP + Traits<T>::pad;
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

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, DP > 64 ? 3 : DP > 32 ? 4 : 5) attention_packed_kernel(PackedAttentionParams p, bool vec, bool vec_out) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int BN = Traits<T>::keys, P = DP + Traits<T>::pad, NT = BN / 8, DT = DP / 8;
    extern __shared__ uint4 smem16[];
    T* sq = reinterpret_cast<T*>(smem16);
    T* sk = sq + kRows * P;              // two stages
    T* sv = sk + 2 * BN * P;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int group = p.heads / p.kv_heads, d = p.d;
    const int kv = blockIdx.x % p.kv_heads;
    // The longest rows of a causal sequence are dealt first.
    const long long pieces = gridDim.x / p.kv_heads, at_id = blockIdx.x / p.kv_heads;
    const long long id = p.causal ? pieces - 1 - at_id : at_id;
    auto first_id = [&](int i) {
        return (long long)seq_offset(p.q_offsets, p.uniform, i, p.total_q) * group / kRows + i;
    };
    const int seq = find_owner(p.sequences, id, first_id);
    const Span qs = seq_span(p.q_offsets, p.uniform, seq, p.total_q, p.bad);
    const Span ks = seq_span(p.k_offsets, p.uniform, seq, p.total_k, p.bad);
    const long long row0 = (id - first_id(seq)) * kRows, all = (long long)qs.len * group;
    if (row0 < 0 || row0 >= all) return;
    const int rows = (int)min((long long)kRows, all - row0);
    const int shift = ks.len - qs.len;   // causal: query i sees keys j <= i + shift
    const int token0 = (int)(row0 / group), part0 = (int)(row0 % group);   // row n is query token0 + (part0 + n) / group
    auto keys_of = [&](int n) {
        return p.causal ? min(max(token0 + (part0 + n) / group + shift + 1, 0), ks.len) : ks.len;
    };
    const int keys = keys_of(rows - 1);
    const int tiles = (keys + BN - 1) / BN;

    const T* q = static_cast<const T*>(p.q.ptr) + (qs.begin + (long long)token0) * p.q.token_stride +
                 (long long)kv * group * p.q.head_stride;
    const T* k = static_cast<const T*>(p.k.ptr) + (long long)ks.begin * p.k.token_stride + kv * p.k.head_stride;
    const T* v = static_cast<const T*>(p.v.ptr) + (long long)ks.begin * p.v.token_stride + kv * p.v.head_stride;
    auto q_at = [&](int n) {
        const int x = part0 + n;
        return (long long)(x / group) * p.q.token_stride + (x % group) * p.q.head_stride;
    };
    load_tile<T, DP>(sq, q, q_at, kRows, rows, d, vec);
    auto load_keys = [&](int j) {
        const int n = min(BN, keys - j * BN);
        const T* kt = k + (long long)j * BN * p.k.token_stride;
        const T* vt = v + (long long)j * BN * p.v.token_stride;
        load_tile<T, DP>(sk + (j & 1) * BN * P, kt, [&](int i) { return i * p.k.token_stride; }, BN, n, d, vec);
        load_tile<T, DP>(sv + (j & 1) * BN * P, vt, [&](int i) { return i * p.v.token_stride; }, BN, n, d, vec);
    };
    if (tiles > 0) load_keys(0);
    cp_async_commit();

    const float scale = p.scale * 1.4426950408889634f;
    const int n0 = warp * 16 + r;                  // this lane's rows: n0 and n0 + 8
    const int keys0 = keys_of(min(n0, rows - 1)), keys1 = keys_of(min(n0 + 8, rows - 1));
    const int sure = __reduce_min_sync(0xffffffffu, (unsigned)min(keys0, keys1));   // keys every row of the warp sees
    const int most = n0 - r < rows ? (int)__reduce_max_sync(0xffffffffu, (unsigned)max(keys0, keys1)) : 0;
    float o[DT][4];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    uint32_t qf[F32 ? 1 : DP / 16][4];

    for (int j = 0; j < tiles; ++j) {
        if (j + 1 < tiles) load_keys(j + 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        const T* kt = sk + (j & 1) * BN * P;
        const T* vt = sv + (j & 1) * BN * P;
        // Eights of keys that some row of the warp sees (0 for a warp without
        // rows): lines are short, and tiles seldom full.
        const int left = min(NT, (most - j * BN + 7) / 8), seen = F32 && left > 0 ? NT : left;   // FP32: the whole tile is faster
        if (seen <= 0) {
            __syncthreads();
            continue;
        }
        float s[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[i][x] = 0.f;
        if constexpr (!F32) {
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
        } else {
            // The tensor cores truncate when they add to an accumulator: the small
            // cross products are summed apart, the leading ones in chains of two.
            float rest[NT][4], part[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) rest[n][x] = 0.f;
#pragma unroll 4
            for (int i = 0; i < DP / 8; ++i) {
                const float* qa = reinterpret_cast<const float*>(sq) + n0 * P + i * 8 + c;
                uint32_t ah[4], al[4];
                split_tf32(qa[0], ah[0], al[0]);
                split_tf32(qa[8 * P], ah[1], al[1]);
                split_tf32(qa[4], ah[2], al[2]);
                split_tf32(qa[8 * P + 4], ah[3], al[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n >= seen) break;
                    const float* kb = reinterpret_cast<const float*>(kt) + (n * 8 + r) * P + i * 8 + c;
                    uint32_t h0, e0, h1, e1;
                    split_tf32(kb[0], h0, e0);
                    split_tf32(kb[4], h1, e1);
                    if (i % 2 == 0) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f;
                    mma_tf32_1688(rest[n], al, h0, h1);
                    mma_tf32_1688(rest[n], ah, e0, e1);
                    mma_tf32_1688(part[n], ah, h0, h1);
                    if (i % 2 == 1) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[n][x] += part[n][x];
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[n][x] += rest[n][x];
        }
        // Scale, mask, running maximum.
        float t0 = -INFINITY, t1 = -INFINITY;
        const bool whole = (j + 1) * BN <= sure;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n >= (seen + 1) / 2 * 2) break;   // BF16 takes them in pairs
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int key = j * BN + n * 8 + 2 * c + x;
                s[n][x] = whole || key < keys0 ? s[n][x] * scale : -INFINITY;
                s[n][x + 2] = whole || key < keys1 ? s[n][x + 2] * scale : -INFINITY;
                t0 = fmaxf(t0, s[n][x]);
                t1 = fmaxf(t1, s[n][x + 2]);
            }
        }
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(m0, fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2)));
        t1 = fmaxf(m1, fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2)));
        const float b0 = t0 == -INFINITY ? 0.f : t0, b1 = t1 == -INFINITY ? 0.f : t1;
        const float g0 = exp2_hw(m0 - b0), g1 = exp2_hw(m1 - b1);   // 0 while the maximum is -infinity
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
            s[n][0] = exp2_hw(s[n][0] - b0); s[n][1] = exp2_hw(s[n][1] - b0);
            s[n][2] = exp2_hw(s[n][2] - b1); s[n][3] = exp2_hw(s[n][3] - b1);
            l0 += s[n][0] + s[n][1];
            l1 += s[n][2] + s[n][3];
        }
        if constexpr (!F32) {
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
        } else {
            // K index c stands for key 2c and c + 4 for key 2c + 1 of the eight,
            // so the scores are the A operand as they are.
            uint32_t ah[NT][4], al[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                split_tf32(s[n][0], ah[n][0], al[n][0]);
                split_tf32(s[n][2], ah[n][1], al[n][1]);
                split_tf32(s[n][1], ah[n][2], al[n][2]);
                split_tf32(s[n][3], ah[n][3], al[n][3]);
            }
            const float* vb = reinterpret_cast<const float*>(vt) + 2 * c * P + r;
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                float rest[4] = {0.f, 0.f, 0.f, 0.f}, part[4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (n >= (seen + 1) / 2 * 2) break;   // the sums' chains are of two
                    uint32_t h0, e0, h1, e1;
                    split_tf32(vb[n * 8 * P + i * 8], h0, e0);
                    split_tf32(vb[n * 8 * P + P + i * 8], h1, e1);
                    if (n % 2 == 0) part[0] = part[1] = part[2] = part[3] = 0.f;
                    mma_tf32_1688(rest, al[n], h0, h1);
                    mma_tf32_1688(rest, ah[n], e0, e1);
                    mma_tf32_1688(part, ah[n], h0, h1);
                    if (n % 2 == 1) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[i][x] += part[x];
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) o[i][x] += rest[x];
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();

    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;
    T* out = static_cast<T*>(p.out.ptr) + (qs.begin + (long long)token0) * p.out.token_stride +
             (long long)kv * group * p.out.head_stride;
    auto out_at = [&](int n) {
        const int x = part0 + n;
        return out + (long long)(x / group) * p.out.token_stride + (x % group) * p.out.head_stride;
    };
    bool bad[2] = {false, false};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int n = n0 + 8 * half;
        if (n >= rows) continue;
        T* dst = out_at(n);
        const float inv = half ? i1 : i0;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int x = i * 8 + 2 * c;
            const float a = o[i][2 * half] * inv, b = o[i][2 * half + 1] * inv;
            bad[half] |= (x < d && !isfinite(a)) || (x + 1 < d && !isfinite(b));
            if (vec_out && x + 1 < d) {
                if constexpr (F32) *reinterpret_cast<float2*>(dst + x) = make_float2(a, b);
                else *reinterpret_cast<__nv_bfloat162*>(dst + x) = __floats2bfloat162_rn(a, b);
            } else {
                if (x < d) dst[x] = from_f<T>(a);
                if (x + 1 < d) dst[x + 1] = from_f<T>(b);
            }
        }
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
            attend_row<T>(q + q_at(n), k, p.k.token_stride, v, p.v.token_stride, d, keys_of(n), scale, out_at(n));
        }
    }
}

template <typename T, int DP>
cudaError_t launch_dp(const PackedAttentionParams& p, cudaStream_t stream) {
    const int esize = sizeof(T), group = p.heads / p.kv_heads;
    const bool vec = rows16(p.q, esize) && rows16(p.k, esize) && rows16(p.v, esize) && p.d * esize % 16 == 0;
    // Pairs of outputs go out together when every pair is aligned.
    const uintptr_t ob = reinterpret_cast<uintptr_t>(p.out.ptr) | (uintptr_t)(p.out.token_stride * esize) |
                         (uintptr_t)(p.out.head_stride * esize);
    const bool vec_out = ob % (2 * esize) == 0;
    constexpr int pitch = DP + Traits<T>::pad;
    constexpr int smem = (kRows + 4 * Traits<T>::keys) * pitch * (int)sizeof(T);
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(attention_packed_kernel<T, DP>), smem);
    if (e != cudaSuccess) return e;
    // Sequence i owns the ids from floor(offset_i group / 64) + i: at least its number of 64-row pieces.
    const long long pieces = (long long)p.total_q * group / kRows + p.sequences;
    attention_packed_kernel<T, DP><<<(unsigned)(pieces * p.kv_heads), kThreads, smem, stream>>>(p, vec, vec_out);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const PackedAttentionParams& p, cudaStream_t stream) {
    if (p.d <= 16) return launch_dp<T, 16>(p, stream);
    if (p.d <= 32) return launch_dp<T, 32>(p, stream);
    if (p.d <= 64) return launch_dp<T, 64>(p, stream);
    return launch_dp<T, 128>(p, stream);
}

}  // namespace

cudaError_t launch_attention_packed(const PackedAttentionParams& p, cudaStream_t stream) {
    if (p.total_q == 0 || p.sequences == 0) return cudaSuccess;
    // tcgen05 from 16,384 keys x (padded) values per sequence on.  Measured on
    // 16,384 tokens in causal sequences of equal length, mma.sync / tcgen05 in us:
    //   8 heads of 24          length 384: 44 / 57, 512: 53 / 55, 1,024: 89 / 67
    //   16 of 64, 4 KV heads   length 128: 62 / 72, 192: 72 / 73, 256: 83 / 74
    //   8 of 128               length 96: 95 / 83, 128: 82 / 68, 512: 150 / 64
    const int padded = p.d <= 16 ? 16 : p.d <= 32 ? 32 : p.d <= 64 ? 64 : 128;
    if ((long long)p.total_k * padded >= 16384ll * p.sequences && attention_tc_supported(p)) return launch_attention_tc(p, stream);
    return p.dtype == DT_F32 ? launch_type<float>(p, stream) : launch_type<__nv_bfloat16>(p, stream);
}

}  // namespace ppocr
