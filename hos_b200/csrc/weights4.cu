// Products with weights in 4 bits: out[M, N] = x[M, K] . W[N, K]^T, W[n, k] = (c[n, k] - z[n, g]) s[n, g] with codes c of
// 4 bits and a scale s (bfloat16) and a zero code z (8 if there is none) for every `group` neighbouring weights of a row.
// Codes lie as blocks (fourbit.cuh) [N / 16][K / 64]; beside them, for every 16 rows and group, 8 records of the rows
// r and r + 8: their two scales, and where there are zero codes 128 + z of both, all in bfloat16.
//
// Few rows are bound by reading W once.  sum_k (c - z) s x = sum_g s_g sum_{k in g} (c - z) x: the integers c - z are exact in
// bfloat16, so a block's product runs on mma.sync without any rounding of the weights, and its 32-bit sum is multiplied by the
// scale, also in 32 bits.  A warp owns 16 features (with the gated epilogue 16 of gate and the same 16 of up, which share the
// rows of x) and a share of K; its blocks come through a ring of its own in shared memory by cp.async, kRing blocks ahead, so that
// nothing but its own copies is ever waited for.  The warps of a CTA share K; their sums are added in a fixed order, and how K is cut
// hangs on N and K alone, so that a row's bits hang on no other row.  Rows in 32 bits are three bfloat16 numbers each,
// x = x1 + x2 + x3 exactly (8 + 8 + 8 bits), and three products a block.
#include "common.cuh"
#include "fourbit.cuh"
#include "mma_utils.cuh"

namespace hos {

__device__ __forceinline__ float gate_times(int act, float gate, float up, float limit, bool fast) {
    if (fast) return act == 2 ? clamped_swish_fast(gate, up, limit) : (act == 0 ? gelu_tanh_fast(gate) : silu_fast(gate)) * up;
    if (act == 2) return clamped_swish(gate, up, limit);
    return (act == 0 ? gelu_tanh(gate) : gate / (1.f + expf(-gate))) * up;
}

// A lane's 16 numbers of a row of x, 8 from p on and 8 from p + 32 on, as operand registers: pair j holds the numbers 2 j and 2 j + 1.
struct Row16 { uint32_t v[8]; };
__device__ __forceinline__ void load_row(Row16 (&r)[1], const bf16* p, int left, bool vec) {
    if (vec) {                                   // whole 16-byte pieces: K is a multiple of 8 and the rows begin on 16 bytes
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 a = left > 0 ? __ldg((const uint4*)p) : zero, b = left > 32 ? __ldg((const uint4*)(p + 32)) : zero;
        r[0] = Row16{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        return;
    }
    const unsigned short* u = (const unsigned short*)p;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int at = 2 * j + (j < 4 ? 0 : 24);
        r[0].v[j] = (at < left ? (uint32_t)__ldg(u + at) : 0u) | (at + 1 < left ? (uint32_t)__ldg(u + at + 1) << 16 : 0u);
    }
}
__device__ __forceinline__ void load_row(Row16 (&r)[3], const float* p, int left, bool vec) {
    float f[16];
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 4 * i + (i < 2 ? 0 : 24);
            const float4 a = left > at ? __ldg((const float4*)(p + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
            f[4 * i] = a.x; f[4 * i + 1] = a.y; f[4 * i + 2] = a.z; f[4 * i + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int at = i + (i < 8 ? 0 : 24);
            f[i] = at < left ? __ldg(p + at) : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a = f[2 * j], b = f[2 * j + 1];
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            const uint32_t w = pack_bf16(a, b);
            r[t].v[j] = w;
            a -= bf16_lo(w);
            b -= bf16_hi(w);
        }
    }
}

// MT: tiles of 8 rows of x; T: tiles of 16 features a warp (2: gated); SUB: scales a block of 64 (2: groups of 32).
template <typename XT, typename OutT, int MT, int T, int SUB, bool ZEROS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS)
product4_kernel(const XT* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ records, OutT* __restrict__ out, int M, int N,
                int K, long long ldx, long long ldo, int group, int act, float limit, int vec) {
    constexpr int kTerms = sizeof(XT) == 4 ? 3 : 1;
    constexpr int kRing = T == 1 ? 8 : 5;
    constexpr int kRecord = ZEROS ? 64 : 32;                       // bytes of a tile's records of a group
    constexpr int kTile = kBlockBytes + SUB * kRecord, kStage = T * kTile;
    constexpr int kSums = T * MT * 16 * 9;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int tiles = (N + 15) / 16, k_blocks = (K + 63) / 64, groups = (k_blocks * 64 + group - 1) / group;
    const int per_way = (k_blocks + WARPS - 1) / WARPS, kb0 = min(k_blocks, warp * per_way), kb1 = min(k_blocks, kb0 + per_way);
    const int m0 = blockIdx.y * 8 * MT;
    uint8_t* ring = smem + warp * kRing * kStage;
    const uint32_t ring_at = smem_u32(ring);

    auto fetch = [&](int kb) {
        if (kb < kb1) {
            const uint32_t to = ring_at + (kb - kb0) % kRing * kStage;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const size_t tile = (size_t)t * tiles + blockIdx.x;
                copy16_async(to + t * kTile + lane * 16, codes + (tile * k_blocks + kb) * kBlockBytes + lane * 16);
                if (lane < SUB * kRecord / 16)
                    copy16_async(to + t * kTile + kBlockBytes + lane * 16, records + (tile * groups + (SUB == 2 ? 2 * kb : kb * 64 / group)) * kRecord + lane * 16);
            }
        }
        copies_commit();
    };
    // W is nothing that a kernel before this one writes
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fetch(kb0 + i);
    pdl_wait();
    pdl_launch_dependents();

    float acc[T][MT][4];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m][0] = acc[t][m][1] = acc[t][m][2] = acc[t][m][3] = 0.f;
    const XT* row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) row[m] = x + (size_t)min(m0 + 8 * m + g, M - 1) * ldx + 8 * t4;

    auto rows_of = [&](int kb, int m, Row16 (&r)[kTerms]) {
        const int left = m0 + 8 * m + g < M ? K - (kb * 64 + 8 * t4) : 0;
        load_row(r, row[m] + kb * 64, left, vec != 0);
    };
    Row16 next[kTerms];
    if (MT == 1 && kb0 < kb1) rows_of(kb0, 0, next);
    for (int kb = kb0; kb < kb1; ++kb) {
        copies_wait<kRing - 2>();
        __syncwarp();
        const uint32_t at = ring_at + (kb - kb0) % kRing * kStage;
        uint32_t a[T][4][4];
        float s[T][SUB][2];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const uint4 w = lds16(at + t * kTile + lane * 16);
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {                          // two MMA steps to a word
                uint32_t z0 = kZero8, z1 = kZero8;
                const uint8_t* rec = ring + (kb - kb0) % kRing * kStage + t * kTile + kBlockBytes + (SUB == 2 ? h : 0) * kRecord + g * (kRecord / 8);
                if (h < SUB) {
                    const uint32_t two = *(const uint32_t*)rec;
                    s[t][h][0] = bf16_lo(two);
                    s[t][h][1] = bf16_hi(two);
                }
                if (ZEROS) {
                    const uint32_t two = *(const uint32_t*)(rec + 4);
                    z0 = __byte_perm(two, 0, 0x1010);
                    z1 = __byte_perm(two, 0, 0x3232);
                }
                codes_to_bf16(h == 0 ? w.x : w.y, z0, lo);
                codes_to_bf16(h == 0 ? w.z : w.w, z1, hi);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    a[t][2 * h + e][0] = lo[2 * e];
                    a[t][2 * h + e][1] = hi[2 * e];
                    a[t][2 * h + e][2] = lo[2 * e + 1];
                    a[t][2 * h + e][3] = hi[2 * e + 1];
                }
            }
        }
        fetch(kb + kRing - 1);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            Row16 r[kTerms];
            if (MT == 1) {
#pragma unroll
                for (int i = 0; i < kTerms; ++i) r[i] = next[i];
                if (kb + 1 < kb1) rows_of(kb + 1, 0, next);
            } else {
                rows_of(kb, m, r);
            }
#pragma unroll
            for (int t = 0; t < T; ++t) {
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = kTerms - 1; i >= 0; --i)           // the small terms first
#pragma unroll
                        for (int st = 4 / SUB * sub; st < 4 / SUB * (sub + 1); ++st) mma_bf16(part, a[t][st], r[i].v[2 * st], r[i].v[2 * st + 1]);
                    acc[t][m][0] = fmaf(s[t][sub][0], part[0], acc[t][m][0]);
                    acc[t][m][1] = fmaf(s[t][sub][0], part[1], acc[t][m][1]);
                    acc[t][m][2] = fmaf(s[t][sub][1], part[2], acc[t][m][2]);
                    acc[t][m][3] = fmaf(s[t][sub][1], part[3], acc[t][m][3]);
                }
            }
        }
    }
    copies_wait<0>();
    __syncthreads();                             // the rings are done with: the sums go where they were
    float* sums = (float*)smem;
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float* p = sums + warp * kSums + (t * MT + m) * 144;
            p[g * 9 + 2 * t4] = acc[t][m][0];
            p[g * 9 + 2 * t4 + 1] = acc[t][m][1];
            p[(g + 8) * 9 + 2 * t4] = acc[t][m][2];
            p[(g + 8) * 9 + 2 * t4 + 1] = acc[t][m][3];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 8 * 16; i += WARPS * 32) {
        const int tok = i / 16, r = i % 16, n = blockIdx.x * 16 + r;      // consecutive threads: consecutive features
        if (m0 + tok >= M || n >= N) continue;
        float v[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            v[t] = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v[t] += sums[w * kSums + (t * MT + tok / 8) * 144 + r * 9 + tok % 8];
        }
        out[(size_t)(m0 + tok) * ldo + n] = from_float<OutT>(T == 2 ? gate_times(act, v[0], v[T - 1], limit, kTerms == 1) : v[0]);
    }
}

template <typename XT, typename OutT, int MT, int T, int SUB, bool ZEROS, int WARPS>
int launch_product4(const void* x, const void* codes, const void* records, void* out, int M, int N, int K, long long ldx, long long ldo, int group,
                    int act, float limit, int vec, cudaStream_t stream) {
    constexpr int ring = T == 1 ? 8 : 5, stage = T * (kBlockBytes + SUB * (ZEROS ? 64 : 32));
    constexpr int sums = T * MT * 144 * 4;
    constexpr int smem = WARPS * (ring * stage > sums ? ring * stage : sums);
    auto kernel = product4_kernel<XT, OutT, MT, T, SUB, ZEROS, WARPS>;
    if (smem > 48 * 1024) {
        static bool set = false;                 // once per kernel: the attribute stays
        if (!set) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return check_launch("product4");
            set = true;
        }
    }
    launch_pdl(kernel, dim3((unsigned)((N + 15) / 16), (unsigned)((M + 8 * MT - 1) / (8 * MT))), dim3(WARPS * 32), smem, stream, (const XT*)x,
               (const uint8_t*)codes, (const uint8_t*)records, (OutT*)out, M, N, K, ldx, ldo, group, act, limit, vec);
    return check_launch("product4");
}

}  // namespace hos

using namespace hos;

extern "C" const char* hos_last_error() { return error_buffer(); }

// Rows of x are ldx numbers apart, rows of out ldo; gated: W has 2 N rows, gate's 16-row tiles first, then up's.
extern "C" int hos_product4(const void* x, int x_dtype, long long ldx, const void* codes, const void* records, void* out, int out_dtype, long long ldo,
                            int M, int N, int K, int group, int zeros, int gated, int act, float limit, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) HOS_REFUSE("product4: K %d", K);
    if (group < 32 || (group != 32 && group % 64)) HOS_REFUSE("product4: groups of %d weights (32, or a multiple of 64)", group);
    if (M > 65535 * 8) HOS_REFUSE("product4: %d rows", M);
    if (x_dtype == kF32 ? out_dtype != kF32 : x_dtype != kBF16 || (out_dtype != kF32 && out_dtype != kBF16))
        HOS_REFUSE("product4: no product of type %d into type %d", x_dtype, out_dtype);
    const int piece = x_dtype == kF32 ? 4 : 8, vec = K % piece == 0 && ldx % piece == 0 && (uintptr_t)x % 16 == 0;
    const int sm = sm_count_cached(), ctas = (N + 15) / 16;
    // the warps that share a CTA's K: as few as fill the SMs with 16 warps each
    const int ways = ctas >= 4 * sm ? 4 : (ctas >= 2 * sm ? 8 : 16);
#define HOS_P4(X, O, MT, T, SUB, Z, W) return launch_product4<X, O, MT, T, SUB, Z, W>(x, codes, records, out, M, N, K, ldx, ldo, group, act, limit, vec, stream)
#define HOS_P4_W(X, O, MT, T, SUB, Z) do { if (ways == 4) HOS_P4(X, O, MT, T, SUB, Z, 4); else if (ways == 8) HOS_P4(X, O, MT, T, SUB, Z, 8); else HOS_P4(X, O, MT, T, SUB, Z, 16); } while (0)
#define HOS_P4_M(X, O, T, SUB, Z) do { if (M <= 8) HOS_P4_W(X, O, 1, T, SUB, Z); else if (M <= 16) HOS_P4_W(X, O, 2, T, SUB, Z); else HOS_P4_W(X, O, 4, T, SUB, Z); } while (0)
#define HOS_P4_S(X, O, T, Z) do { if (group == 32) HOS_P4_M(X, O, T, 2, Z); else HOS_P4_M(X, O, T, 1, Z); } while (0)
#define HOS_P4_G(X, O, Z) do { if (gated) HOS_P4_S(X, O, 2, Z); else HOS_P4_S(X, O, 1, Z); } while (0)
#define HOS_P4_Z(X, O) do { if (zeros) HOS_P4_G(X, O, true); else HOS_P4_G(X, O, false); } while (0)
    if (x_dtype == kF32) HOS_P4_Z(float, float);
    else if (out_dtype == kBF16) HOS_P4_Z(bf16, bf16);
    else HOS_P4_Z(bf16, float);
}
