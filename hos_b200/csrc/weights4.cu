// Products with weights in 4 bits: out[M, N] = x[M, K] . W[N, K]^T, W[n, k] = (c[n, k] - z[n, g]) s[n, g] with codes c of
// 4 bits and a scale s (bfloat16) and a zero code z (8 if there is none) for every `group` neighbouring weights of a row.
// Codes lie as blocks "by row" (fourbit.cuh) [N / 16][K / 64]; beside them, for every 16 rows and group, 8 records of the rows
// r and r + 8: their two scales, and where there are zero codes 128 + z of both, all in bfloat16.
#include "common.cuh"
#include "fourbit.cuh"

namespace hos {

__device__ __forceinline__ float gate_times(int act, float gate, float up, float limit) {
    if (act == 2) return clamped_swish(gate, up, limit);
    return (act == 0 ? gelu_tanh(gate) : gate / (1.f + expf(-gate))) * up;
}

// One warp per output feature, eight rows of x at a time; a lane takes a word of eight codes of every fourth block of 64.
template <typename T, typename OutT, bool ZEROS, bool GATED>
__global__ void __launch_bounds__(128)
product4_plain_kernel(const T* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, OutT* __restrict__ out,
                      int M, int N, int K, long long ldx, long long ldo, int group, int act, float limit) {
    pdl_enter();
    const int lane = threadIdx.x & 31, n = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (n >= N) return;
    const int k_blocks = (K + 63) / 64, groups = (k_blocks * 64 + group - 1) / group, tiles = (N + 15) / 16;
    constexpr int kRecord = ZEROS ? 8 : 4;
    for (int m0 = blockIdx.y * 8; m0 < min(M, (int)blockIdx.y * 8 + 8); m0 += 8) {
        float acc[GATED ? 2 : 1][8] = {};
        for (int half = 0; half < (GATED ? 2 : 1); ++half) {
            const size_t tile = (size_t)half * tiles + n / 16;
            for (int kb = lane >> 3; kb < k_blocks; kb += 4) {
                const int d = (lane & 7) * 8, k0 = kb * 64 + d;
                const uint32_t w = *(const uint32_t*)(codes + (tile * k_blocks + kb) * kBlockBytes + by_row_word(n & 15, d));
                const uint8_t* rec = scales + ((tile * groups + k0 / group) * 8 + (n & 7)) * kRecord;
                const float s = to_float(((const bf16*)rec)[(n >> 3) & 1]);
                const float z = ZEROS ? to_float(((const bf16*)rec)[2 + ((n >> 3) & 1)]) - 128.f : 8.f;
                for (int j = 0; j < 8; ++j) {
                    if (k0 + j >= K) break;
                    const float v = ((float)((w >> code_shift(j)) & 15u) - z) * s;
                    for (int m = 0; m < 8; ++m)
                        if (m0 + m < M) acc[half][m] = fmaf(v, to_float(x[(size_t)(m0 + m) * ldx + k0 + j]), acc[half][m]);
                }
            }
        }
        for (int m = 0; m < 8; ++m) {
            float v = warp_sum(acc[0][m]);
            if (GATED) v = gate_times(act, v, warp_sum(acc[GATED ? 1 : 0][m]), limit);
            if (lane == 0 && m0 + m < M) out[(size_t)(m0 + m) * ldo + n] = from_float<OutT>(v);
        }
    }
}

}  // namespace hos

using namespace hos;

extern "C" const char* hos_last_error() { return error_buffer(); }

// Rows of x are ldx numbers apart, rows of out ldo; gated: W has 2 N rows, gate's 16-row tiles first, then up's.
extern "C" int hos_product4(const void* x, int x_dtype, long long ldx, const void* codes, const void* scales, void* out, int out_dtype, long long ldo,
                            int M, int N, int K, int group, int zeros, int gated, int act, float limit, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) HOS_REFUSE("product4: K %d", K);
    if (group < 32 || (group != 32 && group % 64)) HOS_REFUSE("product4: groups of %d weights (32, or a multiple of 64)", group);
    const dim3 grid((unsigned)((N + 3) / 4), (unsigned)((M + 7) / 8));
#define HOS_P4(T, O, Z, G) launch_pdl(product4_plain_kernel<T, O, Z, G>, grid, dim3(128), 0, stream, (const T*)x, (const uint8_t*)codes, (const uint8_t*)scales, (O*)out, M, N, K, ldx, ldo, group, act, limit)
#define HOS_P4_G(T, O, Z) do { if (gated) HOS_P4(T, O, Z, true); else HOS_P4(T, O, Z, false); } while (0)
#define HOS_P4_Z(T, O) do { if (zeros) HOS_P4_G(T, O, true); else HOS_P4_G(T, O, false); } while (0)
    if (x_dtype == kF32 && out_dtype == kF32) HOS_P4_Z(float, float);
    else if (x_dtype == kBF16 && out_dtype == kBF16) HOS_P4_Z(bf16, bf16);
    else if (x_dtype == kBF16 && out_dtype == kF32) HOS_P4_Z(bf16, float);
    else HOS_REFUSE("product4: no product of type %d into type %d", x_dtype, out_dtype);
    return check_launch("product4");
}
