// Products of many rows with weights in 4 bits on the 5th-generation tensor cores: out[M, N] = x[M, K] . W[N, K]^T in bfloat16.
//
// The weights are formed in half precision on their way: (c - z) s, c - z exact and the product, of 12 bits, rounded once (2^-11 of a
// weight; in bfloat16 it would be 2^-8, as much as the result's own rounding), straight into the operand's place in shared memory, so
// that they cross memory in 4 bits however many rows there are.  Half precision has few exponents: a feature's scales are held times a
// power of two that brings the largest between 2^11 and 2^12 (parts/weights4.py; 15 of it are still a number, and scales down to 2^-25 of the
// largest keep all their bits, the last of them is lost below 2^-36), a row of x by one of its own to between 2^10 and 2^11 at its largest
// (rows_to_half_kernel; numbers below 2^-36 of that are lost), and the powers come back in the epilogue, exactly.
// A CTA takes 128 features (gated: 128 of gate and the same 128 of up) and up to 256 rows, tcgen05.mma with M = 128 features and N =
// rows.  Three groups of eight warps take the stages of 64 k in turn: each warp forms 16 features (its codes wait in
// registers, asked for a turn ahead); one more warp brings the rows of x by TMA, and one issues the products.  (With the rows
// brought by the makers' cp.async the fence behind what they form waited for those copies too: 2304 x 9216, 64 rows on one SM a tile 64 us.)
// Few tiles share K as a cluster, whose sums meet in shared memory.
// Bound by the products where rows fill the tile (2 clocks a row and stage), else by forming the weights: plan_tiles below chooses rows
// a tile and CTAs a cluster by these.
// Measured (B200, 14336 x 3584 gated, groups of 128 with zero codes): 64 rows 34 us, 512 rows 103 us (1.02 PFLOP/s), 2,048 rows 369 us (1.14).
#include "common.cuh"
#include "fourbit.cuh"
#include "mma_utils.cuh"
#include "tcgen05_one.cuh"
#include <cuda_fp16.h>

namespace hos {

constexpr int kTcFeatures = 128, kTcRows = 256, kTcGroup = 8, kTcGroups = 3, kTcMakers = kTcGroups * kTcGroup, kTcThreads = (kTcMakers + 2) * 32;
constexpr int kTcShared = 226 * 1024, kTcWeights = kTcFeatures * 128;            // bytes of a stage's 128 features
constexpr double kClocksForm = 500., kClocksRow = 1.5;      // of a stage: 128 features formed, and brought a row
constexpr long long kProductWaitCycles = 1ll << 31;
constexpr int kGiveUpProduct4 = 6;

__device__ int* g_product4_error_host = nullptr;            // a word in pinned host memory, if the host gave one

__device__ __forceinline__ void product4_give_up() {
    int* w = g_product4_error_host;
    if (w != nullptr) {
        atomicExch_system(w, kGiveUpProduct4);
        __threadfence_system();
    }
}

struct Product4Args {
    const uint8_t *codes, *records;      // scales, and 1024 + zero codes, in half precision
    const float *powers, *row_powers;    // of a feature (gate's, then up's), of a row
    void* out;
    long long ldo, wait_cycles;     // wait_cycles: the limit of every wait
    uint32_t group_magic;                // ceil(2^32 / blocks of 64 a group): the group of a block is a product's high half
    int out_f32, M, N, K, group_blocks, act, tile_rows, shares;
    int stop_stage;                      // for tests of the give-up path: the stage at which the products' warp takes its wait as run out (-1: none)
    float limit;
};

__host__ __device__ inline int stage_bytes(bool gated, int tile_rows) { return (gated ? 2 : 1) * kTcWeights + tile_rows * 128; }

// As mbar_wait_cycles, asleep for up to two microseconds at a time: a warp that polls takes issue slots from those that form weights.
__device__ __forceinline__ bool try_wait_asleep(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, long long limit) {
    if (try_wait_asleep(bar, parity)) return true;
    const long long t0 = clock64();
    while (!try_wait_asleep(bar, parity))
        if (clock64() - t0 > limit) return false;
    return true;
}

// Loads that stay where they are written, ahead of their use.
__device__ __forceinline__ uint4 load_now16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load_now8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t load_now4(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ float peer_value(uint32_t at, int rank) {
    uint32_t r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r));
    return v;
}
__device__ __forceinline__ void shares_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 16 columns of a warp's 32 lanes of tensor memory.
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}

__device__ __forceinline__ float gated_value(int act, float gate, float up, float limit) {
    return act == 2 ? clamped_swish_fast(gate, up, limit) : (act == 0 ? gelu_tanh_fast(gate) : silu_fast(gate)) * up;
}

// A sum times its feature's and its row's power of two.  Where one is as large as the other is small, the two first: the sum times one of
// them may pass the largest number.  Else one after the other, as the two together might, beside a sum of 0.
__device__ __forceinline__ float times_powers(float v, float feature, float row) {
    return (feature < 1.f) == (row < 1.f) ? v * feature * row : v * (feature * row);
}

// A row of x in half precision, its numbers times a power of two, padded to `width` with zeros; a block a row.
__global__ void __launch_bounds__(256) rows_to_half_kernel(const bf16* __restrict__ x, long long ldx, int K, int width, __half* __restrict__ y,
                                                           float* __restrict__ row_powers, int whole) {
    __shared__ float scratch[32];
    pdl_enter();
    const bf16* row = x + (size_t)blockIdx.x * ldx;
    __half* to = y + (size_t)blockIdx.x * width;
    constexpr int kHeld = 4;                                 // pieces of eight numbers that a thread holds between the two walks
    uint4 held[kHeld];
    float most = 0.f;
    auto load = [&](int i) {
        if (whole) return __ldg(reinterpret_cast<const uint4*>(row) + i);
        uint32_t w[4];
        const unsigned short* u = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = (8 * i + 2 * j < K ? (uint32_t)u[8 * i + 2 * j] : 0u) | (8 * i + 2 * j + 1 < K ? (uint32_t)u[8 * i + 2 * j + 1] << 16 : 0u);
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto look = [&](const uint4& v) {                        // infinities and NaN keep out of it
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = fabsf(bf16_lo(w[j])), b = fabsf(bf16_hi(w[j]));
            if (a < INFINITY) most = fmaxf(most, a);
            if (b < INFINITY) most = fmaxf(most, b);
        }
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int i = threadIdx.x + 256 * j;
        held[j] = 8 * i < width ? load(i) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < kHeld; ++j) look(held[j]);
    for (int i = threadIdx.x + 256 * kHeld; 8 * i < width; i += 256) look(load(i));
    most = block_max(most, scratch);
    // 2^e <= most < 2^(e+1): times 2^(10 - e), in two factors of which each is a normal number
    const int e = most > 0.f ? max(-126, min(127, (int)((__float_as_uint(most) >> 23) & 255u) - 127)) : 10;
    const float a = __uint_as_float((uint32_t)(127 + (10 - e) / 2) << 23), b = __uint_as_float((uint32_t)(127 + (10 - e) - (10 - e) / 2) << 23);
    if (threadIdx.x == 0) row_powers[blockIdx.x] = (1.f / a) * (1.f / b);
    auto put = [&](int i, const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 t = __floats2half2_rn(bf16_lo(w[j]) * a * b, bf16_hi(w[j]) * a * b);
            h[j] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(to + 8 * i) = make_uint4(h[0], h[1], h[2], h[3]);
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int i = threadIdx.x + 256 * j;
        if (8 * i < width) put(i, held[j]);
    }
    for (int i = threadIdx.x + 256 * kHeld; 8 * i < width; i += 256) put(i, load(i));
}

// The operand's registers of a word of codes: 1024 + c where a code's bits are the lowest of a half, 1024 + 16 c where they are the next,
// a sixteenth of which is 64 + c; minus 1024 + z or 64 + z, both exact, times s: the only rounding.
struct Scale16 { uint32_t s, z, z64; };                      // s, 1024 + z, -(64 + z)
__device__ __forceinline__ uint32_t half_weight(uint32_t w, bool upper, const Scale16& k) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(upper ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
    const __half2 h = *reinterpret_cast<const __half2*>(&v);
    const __half2 code = upper ? __hfma2(h, __float2half2_rn(0.0625f), *reinterpret_cast<const __half2*>(&k.z64)) : __hsub2(h, *reinterpret_cast<const __half2*>(&k.z));
    const __half2 c = __hmul2(code, *reinterpret_cast<const __half2*>(&k.s));
    return *reinterpret_cast<const uint32_t*>(&c);
}
__device__ __forceinline__ uint4 half_weights(uint32_t w, const Scale16& k) {
    const uint32_t up = w >> 8;
    return make_uint4(half_weight(w, false, k), half_weight(w, true, k), half_weight(up, false, k), half_weight(up, true, k));
}
template <bool ZEROS>
__device__ __forceinline__ Scale16 scale_of(uint32_t two, uint32_t zeros, uint32_t pick) {
    Scale16 k;
    k.s = __byte_perm(two, 0, pick);
    k.z = 0x64086408u;                                       // 1024 + 8
    k.z64 = 0xd480d480u;                                     // -(64 + 8)
    if (ZEROS) {
        k.z = __byte_perm(zeros, 0, pick);
        const __half2 z64 = __hsub2(__float2half2_rn(960.f), *reinterpret_cast<const __half2*>(&k.z));
        k.z64 = *reinterpret_cast<const uint32_t*>(&z64);
    }
    return k;
}

// S: stages of operands; SUB: scales a block of 64 (2: groups of 32).
template <int S, bool GATED, int SUB, bool ZEROS>
__global__ void __launch_bounds__(kTcThreads, 1) product4_tc_kernel(const __grid_constant__ CUtensorMap rows_map, Product4Args p) {
    constexpr int kAcc = GATED ? 2 : 1, kRecord = ZEROS ? 64 : 32;
    extern __shared__ unsigned char smem_unaligned[];
    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~(uintptr_t)1023);
    const int stage = stage_bytes(GATED, p.tile_rows);
    __shared__ uint64_t full[S], empty[S], done;
    __shared__ uint32_t tmem_base_smem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int columns = (p.tile_rows + 31) & ~31;           // of an accumulator
    int tmem_columns = 32;
    while (tmem_columns < kAcc * columns) tmem_columns *= 2;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) { mbar_init(&full[s], kTcGroup + 1); mbar_init(&empty[s], 1); }
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    if (warp == kTcMakers) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(tmem_columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_smem;
    pdl_enter();

    const int k_blocks = (p.K + 63) / 64, tiles = (p.N + 15) / 16, feature_tiles = (p.N + kTcFeatures - 1) / kTcFeatures;
    const int groups = SUB == 2 ? 2 * k_blocks : (k_blocks + p.group_blocks - 1) / p.group_blocks;
    const int share = blockIdx.x % p.shares, tile = blockIdx.x / p.shares, f0 = tile % feature_tiles * kTcFeatures, m0 = tile / feature_tiles * p.tile_rows;
    const int kb0 = (int)((long long)share * k_blocks / p.shares), n_k = (int)((long long)(share + 1) * k_blocks / p.shares) - kb0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_asleep(bar, parity, p.wait_cycles); };

    if (warp < kTcMakers) {
        const int group = warp / kTcGroup, mine = warp % kTcGroup;
        // where the codes of gate's, or of up's, block kb are: a tile beyond the last reads the last one, and its sums are dropped
        uint32_t code_at[kAcc], record_at[kAcc];
#pragma unroll
        for (int a = 0; a < kAcc; ++a) {
            const uint32_t t = a * tiles + min(f0 / 16 + mine, tiles - 1);
            code_at[a] = (t * k_blocks + kb0) * kBlockBytes + lane * 16;
            record_at[a] = t * groups * kRecord + g * (kRecord / 8);
        }
        uint4 codes[kAcc];
        uint32_t scale[kAcc][SUB], zero[kAcc][SUB];
        auto ask = [&](int a, int i) {                      // the codes of block i of this share
            if (i >= n_k) return;
            const uint32_t kb = kb0 + i, record = (SUB == 2 ? 2u * kb : (p.group_blocks == 1 ? kb : __umulhi(kb, p.group_magic))) * kRecord;
            codes[a] = load_now16(p.codes + (code_at[a] + i * kBlockBytes));
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const uint8_t* r = p.records + (record_at[a] + record + u * kRecord);
                if (ZEROS) {
                    const uint2 v = load_now8(r);
                    scale[a][u] = v.x;
                    zero[a][u] = v.y;
                } else {
                    scale[a][u] = load_now4(r);
                }
            }
        };
        auto form = [&](int a, int s) {                     // a block's weights into place s
            unsigned char* to = stages + s * stage + a * kTcWeights + mine * 2048 + g * 128;
            // the k below and from 32 on, in the other order for odd rows: eight lanes then fill all banks
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool upper = h != (g & 1);
                const uint32_t lo = upper ? codes[a].y : codes[a].x, hi = upper ? codes[a].w : codes[a].z;
                const uint32_t two = SUB == 2 && upper ? scale[a][SUB - 1] : scale[a][0];
                const uint32_t zz = !ZEROS ? 0u : (SUB == 2 && upper ? zero[a][SUB - 1] : zero[a][0]);
                const int chunk = (((upper ? 4 : 0) + t4) ^ g) << 4;
                *reinterpret_cast<uint4*>(to + chunk) = half_weights(lo, scale_of<ZEROS>(two, zz, 0x1010));
                *reinterpret_cast<uint4*>(to + 1024 + chunk) = half_weights(hi, scale_of<ZEROS>(two, zz, 0x3232));
            }
        };
#pragma unroll
        for (int a = 0; a < kAcc; ++a) ask(a, group);
        int s = group % S, round = group / S - 1;           // the block's place, and how often it was used before
        for (int i = group; i < n_k; i += kTcGroups) {
            if (i >= S) {
                ok = lane != 0 || wait(&empty[s], round & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
#pragma unroll
            for (int a = 0; a < kAcc; ++a) {
                form(a, s);
                ask(a, i + kTcGroups);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[s]);
            s += kTcGroups;
            if (s >= S) { s -= S; ++round; }
        }
    } else if (warp == kTcMakers + 1) {
        if (lane == 0) {
            for (int i = 0, s = 0, round = -1; i < n_k; ++i) {
                if (i >= S) ok = wait(&empty[s], round & 1);
                if (!ok) break;
                mbar_expect_tx(&full[s], p.tile_rows * 128);
                tc_tma_2d(stages + s * stage + kAcc * kTcWeights, &rows_map, (kb0 + i) * 64, m0, &full[s]);
                if (++s == S) { s = 0; ++round; }
            }
        }
    } else {
        // the warp walks together and one lane issues: what the products take is then in uniform registers; both operands in half precision
        const uint32_t idesc = tc_idesc(kTcFeatures, p.tile_rows, 0) & ~((1u << 7) | (1u << 10)), step = (uint32_t)stage >> 4;
        const uint64_t weights0 = desc_kmajor(smem_u32(stages)), rows0 = desc_kmajor(smem_u32(stages) + kAcc * kTcWeights);
        uint32_t leader;
        asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
        uint32_t off = 0;
        for (int i = 0, s = 0, round = 0; i < n_k; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait_cycles(&full[s], round & 1, p.wait_cycles)) && i != p.stop_stage;
            if (!ok) break;
            tc_fence_after_sync();
            if (leader) {
#pragma unroll
                for (int a = 0; a < kAcc; ++a)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma(tmem_base + a * columns, weights0 + off + a * (kTcWeights >> 4) + 2 * k, rows0 + off + 2 * k, idesc, (i > 0 || k > 0) ? 1u : 0u);
                tc_commit(&empty[s]);
            }
            __syncwarp();
            off += step;
            if (++s == S) { s = 0; off = 0; ++round; }
        }
        if (ok && leader) tc_commit(&done);
    }
    __syncwarp();
    if (warp < kTcMakers && ok) {
        ok = lane != 0 || wait(&done, 0);
        ok = __all_sync(0xffffffffu, ok);
    }
    tc_fence_after_sync();
    float* sums = reinterpret_cast<float*>(stages);          // [kAcc][tile_rows][128] of a share, over operands that are done with
    if (warp < kTcMakers && ok) {
        const int quarter = warp & 3, feature = quarter * 32 + lane, n = f0 + feature;
        const float power = n < p.N ? p.powers[n] : 0.f, up_power = GATED && n < p.N ? p.powers[p.N + n] : 0.f;
        const uint32_t from = tmem_base + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int c0 = (warp >> 2) * 16; c0 < p.tile_rows; c0 += kTcMakers * 4) {      // tile_rows is a multiple of 16
            uint32_t v[16], u[16];
            tc_ld16(from + c0, v);
            if (GATED) tc_ld16(from + columns + c0, u);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int c = c0 + j, m = m0 + c;
                if (p.shares > 1) {
                    sums[c * 128 + feature] = __uint_as_float(v[j]);
                    if (GATED) sums[(p.tile_rows + c) * 128 + feature] = __uint_as_float(u[j]);
                } else if (m < p.M && n < p.N) {
                    const float back = p.row_powers[m], gate = times_powers(__uint_as_float(v[j]), power, back);
                    const float y = GATED ? gated_value(p.act, gate, times_powers(__uint_as_float(u[j]), up_power, back), p.limit) : gate;
                    if (p.out_f32) ((float*)p.out)[(size_t)m * p.ldo + n] = y;
                    else ((bf16*)p.out)[(size_t)m * p.ldo + n] = __float2bfloat16_rn(y);
                }
            }
        }
    }
    if (!ok && lane == 0) product4_give_up();
    const bool gave_up = __syncthreads_or(!ok);
    if (gave_up) let_work_under_way_end();
    if (p.shares > 1) {
        shares_meet();
        if (warp < kTcMakers && !gave_up) {
            const int feature = threadIdx.x & 127, n = f0 + feature;
            const float power = n < p.N ? p.powers[n] : 0.f, up_power = GATED && n < p.N ? p.powers[p.N + n] : 0.f;
            const uint32_t at = smem_u32(sums);
            for (int c = kTcMakers / 4 * share + (threadIdx.x >> 7); c < p.tile_rows; c += kTcMakers / 4 * p.shares) {
                float v = 0.f, u = 0.f;
                for (int s = 0; s < p.shares; ++s) {
                    v += peer_value(at + (c * 128 + feature) * 4, s);
                    if (GATED) u += peer_value(at + ((p.tile_rows + c) * 128 + feature) * 4, s);
                }
                const int m = m0 + c;
                if (m < p.M && n < p.N) {
                    const float back = p.row_powers[m], gate = times_powers(v, power, back);
                    const float y = GATED ? gated_value(p.act, gate, times_powers(u, up_power, back), p.limit) : gate;
                    if (p.out_f32) ((float*)p.out)[(size_t)m * p.ldo + n] = y;
                    else ((bf16*)p.out)[(size_t)m * p.ldo + n] = __float2bfloat16_rn(y);
                }
            }
        }
        shares_meet();                                       // nobody leaves while its sums are read
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kTcMakers) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_columns));
}

template <int S, bool GATED, int SUB, bool ZEROS>
int launch_product4_tc(const CUtensorMap& rows_map, const Product4Args& p, int ctas, int smem, cudaStream_t stream) {
    auto kernel = product4_tc_kernel<S, GATED, SUB, ZEROS>;
    static bool set = false;                                 // once per kernel: the attribute stays
    if (!set) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcShared) != cudaSuccess) return check_launch("product4_tc");
        set = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)p.shares, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = p.shares > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, rows_map, p);
    return check_launch("product4_tc");
}

// Clusters of `shares` CTAs, one to an SM, that run at once (asked once).
static int clusters_at_once(int shares) {
    static int known[9] = {};
    if (known[shares] == 0) {
        auto kernel = product4_tc_kernel<4, false, 1, false>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(shares * 64));
        cfg.blockDim = dim3(kTcThreads);
        cfg.dynamicSmemBytes = 128 * 1024;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {(unsigned)shares, 1, 1};
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcShared) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = sm_count_cached() / shares / 2 + 1;
        }
        known[shares] = n;
    }
    return known[shares];
}

// Rows of a tile and CTAs that share a tile's K: the least of waves x (stages x clocks a stage + what a tile costs besides), in clocks.
// Sums of shares have to fit where the operands were.  Of 40 products of 33 to 2,048 rows and four shapes the plan chosen took the least time
// of those tried or up to 2% more, but for 200 and 256 rows of 4096 x 2048 (18.8 and 19.5 us, 17.8 with tiles of 64).
static void plan_tiles(int M, int N, int K, bool gated, int& tile_rows, int& shares) {
    const int sm = sm_count_cached(), acc = gated ? 2 : 1, feature_tiles = (N + kTcFeatures - 1) / kTcFeatures, k_blocks = (K + 63) / 64;
    double best = 0.;
    tile_rows = 0;
    for (int row_tiles = (M + kTcRows - 1) / kTcRows; row_tiles <= (M + 15) / 16; ++row_tiles) {
        const int rows = ((M + row_tiles - 1) / row_tiles + 15) / 16 * 16;
        const long long n = (long long)feature_tiles * ((M + rows - 1) / rows);
        for (int s = 1; s <= 8 && s <= k_blocks; s *= 2) {
            if (s > 1 && rows > 128) break;
            const int at_once = s == 1 ? sm : clusters_at_once(s);
            if (s > 1 && n > at_once) break;
            const double form = kClocksForm * acc + kClocksRow * rows, stage = rows * 2.1 * acc > form ? rows * 2.1 * acc : form;
            const double cost = (double)((n + at_once - 1) / at_once) * ((k_blocks + s - 1) / s * stage + 5000. + rows * acc * 12. + (s > 1 ? 3000. : 0.));
            if (tile_rows == 0 || cost < best) { best = cost; tile_rows = rows; shares = s; }
        }
        if (rows == 16) break;
    }
}

}  // namespace hos

using namespace hos;

extern "C" int hos_product4_tc_set_error_word(void* word) {
    return cudaMemcpyToSymbol(g_product4_error_host, &word, sizeof(word)) == cudaSuccess ? 0 : -1;
}

// As hos_product4 for bfloat16 rows.  half_rows: M * (K rounded up to 8) numbers of 16 bits on 16 bytes, and row_powers: M of 32, for the rows
// on their way.  tile_rows 0: chosen here, with shares.
extern "C" int hos_product4_tc(const void* x, long long ldx, const void* matrix, void* out, int out_dtype, long long ldo, int M, int act, float limit,
                               void* half_rows, float* row_powers, int tile_rows, int shares, long long wait_cycles, int stop_stage, cudaStream_t stream) {
    const Matrix4 w = *(const Matrix4*)matrix;
    if (M <= 0 || w.n <= 0) return 0;
    if (w.k < 64 || half_rows == nullptr || row_powers == nullptr || (uintptr_t)half_rows % 16) HOS_REFUSE("product4_tc: K %d (64 at least), or no place for the rows", w.k);
    if (w.group < 32 || (w.group != 32 && w.group % 64)) HOS_REFUSE("product4_tc: groups of %d weights (32, or a multiple of 64)", w.group);
    if (w.k > (1 << 21) || (long long)(w.gated ? 2 : 1) * ((w.n + 15) / 16) * ((w.k + 63) / 64) * kBlockBytes >= (1ll << 32))
        HOS_REFUSE("product4_tc: %d x %d weights are more than 4 GB of codes, or k more than %d", w.n, w.k, 1 << 21);
    const int width = (w.k + 7) / 8 * 8;
    if (out_dtype != kF32 && out_dtype != kBF16) HOS_REFUSE("product4_tc: no product into type %d", out_dtype);
    if (tile_rows == 0) plan_tiles(M, w.n, w.k, w.gated != 0, tile_rows, shares);
    const int k_blocks = (w.k + 63) / 64, sub = w.group == 32 ? 2 : 1;
    if (tile_rows < 16 || tile_rows > kTcRows || tile_rows % 16 || shares < 1 || shares > 8 || shares > k_blocks || (shares > 1 && tile_rows > 128))
        HOS_REFUSE("product4_tc: tiles of %d rows in %d shares", tile_rows, shares);
    Product4Args p = {};
    CUtensorMap rows_map;                                    // boxes of 64 numbers of tile_rows rows; what is beyond them reads as zeros
    if (int rc = tc_make_map(&rows_map, half_rows, M, width, width, tile_rows)) return rc;
    p.codes = w.codes; p.records = w.records16; p.powers = w.powers; p.row_powers = row_powers; p.out = out; p.ldo = ldo;
    p.wait_cycles = wait_cycles > 0 ? wait_cycles : kProductWaitCycles;
    p.out_f32 = out_dtype == kF32; p.M = M; p.N = w.n; p.K = w.k; p.group_blocks = w.group / 64;
    p.group_magic = p.group_blocks > 1 ? (uint32_t)(((1ull << 32) + p.group_blocks - 1) / p.group_blocks) : 0u; p.act = act; p.limit = limit;
    p.tile_rows = tile_rows; p.shares = shares; p.stop_stage = stop_stage;
    const long long ctas = (long long)((w.n + kTcFeatures - 1) / kTcFeatures) * ((M + tile_rows - 1) / tile_rows) * shares;
    if (ctas > 0x7fffffffll) HOS_REFUSE("product4_tc: %d rows", M);
    const int a_stage = stage_bytes(w.gated, tile_rows);
    const int S = 6 * a_stage + 1024 <= kTcShared ? 6 : (4 * a_stage + 1024 <= kTcShared ? 4 : 3), smem = S * a_stage + 1024;
    launch_pdl(rows_to_half_kernel, dim3((unsigned)M), dim3(256), 0, stream, (const bf16*)x, ldx, w.k, width, (__half*)half_rows, row_powers,
               w.k % 8 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 ? 1 : 0);
    if (int rc = check_launch("product4_tc: rows")) return rc;
#define HOS_PT(SS, G, U, Z) return launch_product4_tc<SS, G, U, Z>(rows_map, p, (int)ctas, smem, stream)
#define HOS_PT_S(G, U, Z) do { if (S == 6) HOS_PT(6, G, U, Z); else if (S == 4) HOS_PT(4, G, U, Z); else HOS_PT(3, G, U, Z); } while (0)
#define HOS_PT_U(G, Z) do { if (sub == 2) HOS_PT_S(G, 2, Z); else HOS_PT_S(G, 1, Z); } while (0)
#define HOS_PT_Z(G) do { if (w.zeros) HOS_PT_U(G, true); else HOS_PT_U(G, false); } while (0)
    if (w.gated) HOS_PT_Z(true);
    else HOS_PT_Z(false);
}
