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
// x = x1 + x2 + x3 exactly (8 + 8 + 8 bits), and three products a block.  A sum that is not finite is formed again number by number.
// Measured (B200): 8 rows of 36864 x 4608 gated 41.6 us (4.2 TB/s of codes and scales; no unit is full: ALU 58%, mma.sync 33%, an instruction
// issued in 57% of the clocks, by 14 warps an SM); 1 row of 2304 x 9216 6.8 us, 5 rows in 32 bits of 2051 x 1999 4.7 us (11 and 2 MB: launch,
// first bytes, sums).
#include "common.cuh"
#include "fourbit.cuh"
#include "mma_utils.cuh"

namespace hos {

struct TrueTag4 { static constexpr bool value = true; };
struct FalseTag4 { static constexpr bool value = false; };

__device__ __forceinline__ float gate_times(int act, float gate, float up, float limit, bool fast) {
    if (fast) return act == 2 ? clamped_swish_fast(gate, up, limit) : (act == 0 ? gelu_tanh_fast(gate) : silu_fast(gate)) * up;
    if (act == 2) return clamped_swish(gate, up, limit);
    return (act == 0 ? gelu_tanh(gate) : gate / (1.f + expf(-gate))) * up;
}

// d = a . b + c: not volatile and with sums of its own to start from, so that the products of several tiles may be woven into one
// another.
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// A lane's 16 numbers of a row of x, 8 from p on and 8 from p + 32 on, as operand registers: pair j holds the numbers 2 j and 2 j + 1.
// WHOLE: all of them are there and 16-byte pieces may be read; else `left` says how many numbers the row still has from p on.
struct Row16 { uint32_t v[8]; };
template <bool WHOLE>
__device__ __forceinline__ void load_row(Row16 (&r)[1], const bf16* p, int left) {
    if (WHOLE) {
        const uint4 a = __ldg((const uint4*)p), b = __ldg((const uint4*)(p + 32));
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
template <bool WHOLE>
__device__ __forceinline__ void load_row(Row16 (&r)[3], const float* p, int left) {
    float f[16];
    if (WHOLE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 4 * i + (i < 2 ? 0 : 24);
            const float4 a = __ldg((const float4*)(p + at));
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

// One number of the product by the definition, for sums that are not finite: an infinity of x, or numbers near the largest, meet 128 + c,
// an infinity's rest or a group's sum of bare codes on their way above, and give NaN where the result is an infinity or a number.  (c - z) s
// is exact in 32 bits, so nothing is larger here than the products themselves.  tile, records: of the feature's 16 rows, of which it is row r.
template <typename XT, int SUB, bool ZEROS>
__device__ float sum_by_definition(const XT* __restrict__ x, const uint8_t* __restrict__ tile, const uint8_t* __restrict__ records, int r, int K,
                                   int group_blocks) {
    constexpr int kRecord = ZEROS ? 64 : 32;
    float total = 0.f;
#pragma unroll 1
    for (int kb = 0; kb * 64 < K; ++kb) {
        float block = 0.f;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {                              // eight numbers to a word
            const uint8_t* rec = records + (size_t)(SUB == 2 ? 2 * kb + (e >> 2) : kb / group_blocks) * kRecord + (r & 7) * (kRecord / 8) + (r >> 3) * 2;
            const uint32_t w = *(const uint32_t*)(tile + (size_t)kb * kBlockBytes + ((r & 7) * 4 + (e & 3)) * 16 + ((r >> 3) * 2 + (e >> 2)) * 4);
            const float s = to_float(*(const bf16*)rec), z = ZEROS ? to_float(*(const bf16*)(rec + 4)) - 128.f : 8.f;
            const int k = kb * 64 + e * 8;
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < K) part = fmaf(((float)((w >> code_shift(j)) & 15u) - z) * s, to_float(x[k + j]), part);
            block += part;
        }
        total += block;
    }
    return total;
}

// MT: tiles of 8 rows of x; T: tiles of 16 features a warp (the first half of them gate's, the other up's, if GATED); SUB: scales a
// block of 64 (2: groups of 32); ring_of: blocks of T tiles that a warp's ring holds.
template <int T> struct ring_of { static constexpr int value = T == 1 ? 8 : (T == 2 ? 6 : 4); };
// The warps' sums (fixed order) and the epilogue.  AGAIN: sums that are not finite are formed by the definition.  That is a function of its
// own, so that what only it needs takes no registers from the walk; up to 16 rows it is called for such sums alone (a call costs 0.2 us of
// 4.5), above always, as the walk's registers are full and even the look at the sums beside it would spill more of them (24 rows of 14336 x
// 3584 gated, 41 us, 51).
template <typename XT, int MT, int T, bool GATED, int SUB, bool ZEROS, int WARPS, bool AGAIN>
__device__ __forceinline__ bool write_sums(const float* sums, const XT* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ records,
                                           void* __restrict__ out, int out_f32, int M, int N, int K, long long ldx, long long ldo, int group_blocks, int act,
                                           float limit) {
    constexpr int kWide = GATED ? T / 2 : T, kSums = T * MT * 16 * 9, kTerms = sizeof(XT) == 4 ? 3 : 1, kRecord = ZEROS ? 64 : 32;
    const int m0 = blockIdx.y * 8 * MT;
    bool finite = true;
    for (int i = threadIdx.x; i < MT * 8 * 16 * kWide; i += WARPS * 32) {
        const int tok = i / (16 * kWide), r = i % (16 * kWide), n = blockIdx.x * 16 * kWide + r;      // consecutive threads: consecutive features
        if (m0 + tok >= M || n >= N) continue;
        float v[GATED ? 2 : 1];
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h) {
            v[h] = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v[h] += sums[w * kSums + ((h * kWide + r / 16) * MT + tok / 8) * 144 + (r & 15) * 9 + tok % 8];
            if (!AGAIN) finite &= isfinite(v[h]);
            if (AGAIN && !isfinite(v[h])) {
                const int tiles = (N + 15) / 16, k_blocks = (K + 63) / 64, groups = SUB == 2 ? 2 * k_blocks : (k_blocks + group_blocks - 1) / group_blocks;
                const size_t tile = (size_t)h * tiles + blockIdx.x * kWide + r / 16;
                v[h] = sum_by_definition<XT, SUB, ZEROS>(x + (size_t)(m0 + tok) * ldx, codes + tile * k_blocks * kBlockBytes,
                                                         records + tile * groups * kRecord, r & 15, K, group_blocks);
            }
        }
        const float y = GATED ? gate_times(act, v[0], v[GATED ? 1 : 0], limit, kTerms == 1) : v[0];
        const size_t at = (size_t)(m0 + tok) * ldo + n;
        if (kTerms == 3 || out_f32) ((float*)out)[at] = y;
        else ((bf16*)out)[at] = __float2bfloat16_rn(y);
    }
    return finite;
}
template <typename XT, int MT, int T, bool GATED, int SUB, bool ZEROS, int WARPS>
__device__ __noinline__ void write_sums_again(const float* sums, const XT* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ records,
                                              void* __restrict__ out, int out_f32, int M, int N, int K, long long ldx, long long ldo, int group_blocks, int act,
                                              float limit) {
    write_sums<XT, MT, T, GATED, SUB, ZEROS, WARPS, true>(sums, x, codes, records, out, out_f32, M, N, K, ldx, ldo, group_blocks, act, limit);
}

template <typename XT, int MT, int T, bool GATED, int SUB, bool ZEROS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS)
product4_kernel(const XT* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ records, void* __restrict__ out, int out_f32,
                int M, int N, int K, long long ldx, long long ldo, int group_blocks, int act, float limit, int whole) {
    constexpr int kTerms = sizeof(XT) == 4 ? 3 : 1;
    // For rows in bfloat16 the codes go in as 128 + c and (128 + z) sum x, which a product with ones gives for all of the warp's tiles
    // at once, is where the sums start: a quarter of the instructions that form the operands.  The sums lose 2^-24 of 136 sum |x|, far
    // below the rounding of the result; 32-bit rows subtract first.
    constexpr bool kLate = kTerms == 1;
    constexpr int kRing = ring_of<T>::value;
    constexpr int kRecord = ZEROS ? 64 : 32;                       // bytes of a tile's records of a group
    constexpr int kTile = kBlockBytes + SUB * kRecord, kStage = T * kTile;
    constexpr int kSums = T * MT * 16 * 9;
    constexpr int kWide = GATED ? T / 2 : T;                       // tiles of features of the result
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int tiles = (N + 15) / 16, k_blocks = (K + 63) / 64;
    const int groups = SUB == 2 ? 2 * k_blocks : (k_blocks + group_blocks - 1) / group_blocks;
    const int per_way = (k_blocks + WARPS - 1) / WARPS, kb0 = min(k_blocks, warp * per_way), kb1 = min(k_blocks, kb0 + per_way);
    const int m0 = blockIdx.y * 8 * MT;
    uint8_t* ring = smem + warp * kRing * kStage;
    const uint32_t ring_at = smem_u32(ring);

    // where the next block to be fetched is; a tile beyond the last reads the last one, and its sums are dropped
    const uint8_t *code_at[T], *record_at[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const size_t tile = (size_t)(t / kWide) * tiles + min((int)blockIdx.x * kWide + t % kWide, tiles - 1);
        code_at[t] = codes + (tile * k_blocks + kb0) * kBlockBytes + lane * 16;
        record_at[t] = records + (tile * groups + (SUB == 2 ? 2 * kb0 : kb0 / group_blocks)) * kRecord + lane * 16;
    }
    int to_fetch = kb1 - kb0, in_group = SUB == 2 ? 1 : group_blocks - kb0 % group_blocks;
    auto fetch = [&](uint32_t to) {
        if (to_fetch > 0) {
            const bool has_record = lane < SUB * kRecord / 16;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                copy16_async(to + t * kTile + lane * 16, code_at[t]);
                if (has_record) copy16_async(to + t * kTile + kBlockBytes + lane * 16, record_at[t]);
                code_at[t] += kBlockBytes;
            }
            if (--in_group == 0) {
                in_group = SUB == 2 ? 1 : group_blocks;
#pragma unroll
                for (int t = 0; t < T; ++t) record_at[t] += SUB * kRecord;
            }
        }
        --to_fetch;
        copies_commit();
    };
    // W is nothing that a kernel before this one writes
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fetch(ring_at + i * kStage);
    pdl_wait();
    pdl_launch_dependents();

    float acc[T][MT][4];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m][0] = acc[t][m][1] = acc[t][m][2] = acc[t][m][3] = 0.f;
    const XT* row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) row[m] = x + (size_t)min(m0 + 8 * m + g, M - 1) * ldx + 8 * t4 + (size_t)kb0 * 64;   // rows beyond M: sums dropped
    int left = K - kb0 * 64 - 8 * t4;

    // One block: WHOLE as load_row's, AHEAD: the next block's rows may be asked for whole.
    Row16 next[kTerms];
    auto block = [&](uint32_t slot, auto whole_tag, int ahead) {
        constexpr bool kWhole = decltype(whole_tag)::value;
        // the rows of a tile of 8 with the sums of x over a group, columns 2 t and 2 t + 1 (kLate), where the products start
        auto rows_of = [&](int m, Row16 (&r)[kTerms], float (&start)[SUB][2]) {
            if (MT == 1) {
#pragma unroll
                for (int i = 0; i < kTerms; ++i) r[i] = next[i];
                if (ahead == 2) load_row<true>(next, row[0] + 64, 0);
                else if (ahead == 1) load_row<false>(next, row[0] + 64, left - 64);
            } else {
                load_row<kWhole>(r, row[m], left);
            }
            row[m] += 64;
            if (kLate) {
                const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int st = 4 / SUB * sub; st < 4 / SUB * (sub + 1); ++st) mma_from(sum, ones, r[0].v[2 * st], r[0].v[2 * st + 1], sum);
                    start[sub][0] = ZEROS ? sum[0] : -136.f * sum[0];
                    start[sub][1] = ZEROS ? sum[1] : -136.f * sum[1];
                }
            }
        };
        struct Tile { uint32_t a[4][4]; float s[SUB][2], z[SUB][2]; };
        auto operands_of = [&](int t, Tile& f) {
            const uint4 w = lds16(ring_at + slot + t * kTile + lane * 16);
            const uint8_t* rec = ring + slot + t * kTile + kBlockBytes + g * (kRecord / 8);
#pragma unroll
            for (int h = 0; h < 2; ++h) {                       // two MMA steps to a word
                const int sub = SUB == 2 ? h : 0;
                uint32_t z0 = kZero8, z1 = kZero8;
                if (h < SUB) {
                    const uint32_t two = *(const uint32_t*)(rec + sub * kRecord);
                    f.s[sub][0] = bf16_lo(two);
                    f.s[sub][1] = bf16_hi(two);
                }
                if (ZEROS) {
                    const uint32_t two = *(const uint32_t*)(rec + sub * kRecord + 4);
                    z0 = __byte_perm(two, 0, 0x1010);
                    z1 = __byte_perm(two, 0, 0x3232);
                    f.z[sub][0] = -bf16_lo(two);
                    f.z[sub][1] = -bf16_hi(two);
                }
                uint32_t lo[4], hi[4];
                codes_to_bf16<!kLate>(h == 0 ? w.x : w.y, z0, lo);
                codes_to_bf16<!kLate>(h == 0 ? w.z : w.w, z1, hi);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f.a[2 * h + e][0] = lo[2 * e];
                    f.a[2 * h + e][1] = hi[2 * e];
                    f.a[2 * h + e][2] = lo[2 * e + 1];
                    f.a[2 * h + e][3] = hi[2 * e + 1];
                }
            }
        };
        auto multiply = [&](int t, int m, const Tile& f, const Row16 (&r)[kTerms], const float (&start)[SUB][2]) {
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                if (kLate) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) part[c] = ZEROS ? f.z[sub][c >> 1] * start[sub][c & 1] : start[sub][c & 1];
                }
#pragma unroll
                for (int i = kTerms - 1; i >= 0; --i)           // the small terms first
#pragma unroll
                    for (int st = 4 / SUB * sub; st < 4 / SUB * (sub + 1); ++st) mma_from(part, f.a[st], r[i].v[2 * st], r[i].v[2 * st + 1], part);
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[t][m][c] = fmaf(f.s[sub][c >> 1], part[c], acc[t][m][c]);
            }
        };
        if (MT == 1) {                                          // the rows stay while the tiles go by
            Row16 r[kTerms];
            float start[SUB][2];
            rows_of(0, r, start);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                Tile f;
                operands_of(t, f);
                multiply(t, 0, f, r, start);
            }
        } else {                                                // and the other way round
            Tile f[T];
#pragma unroll
            for (int t = 0; t < T; ++t) operands_of(t, f[t]);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                Row16 r[kTerms];
                float start[SUB][2];
                rows_of(m, r, start);
#pragma unroll
                for (int t = 0; t < T; ++t) multiply(t, m, f[t], r, start);
            }
        }
        left -= 64;
    };
    // Blocks whose numbers are all there are read whole; a last one that is not, or all of them where rows are not made of 16-byte
    // pieces, number by number.
    const int n = kb1 - kb0, n_whole = !whole ? 0 : (kb1 * 64 > K ? n - 1 : n);
    if (MT == 1 && n > 0) {
        if (n_whole > 0) load_row<true>(next, row[0], 0);
        else load_row<false>(next, row[0], left);
    }
    uint32_t slot = 0, before = (kRing - 1) * kStage;              // this block's place in the ring, and the one before it
    int i = 0;
    for (; i < n_whole; ++i) {
        copies_wait<kRing - 2>();
        __syncwarp();
        fetch(ring_at + before);                                    // the place that the last block has left
        block(slot, TrueTag4{}, i + 1 < n_whole ? 2 : (i + 1 < n ? 1 : 0));
        before = slot;
        slot = slot == (kRing - 1) * kStage ? 0 : slot + kStage;
    }
    for (; i < n; ++i) {
        copies_wait<kRing - 2>();
        __syncwarp();
        fetch(ring_at + before);
        block(slot, FalseTag4{}, i + 1 < n ? 1 : 0);
        before = slot;
        slot = slot == (kRing - 1) * kStage ? 0 : slot + kStage;
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
    if (MT == 4 || !write_sums<XT, MT, T, GATED, SUB, ZEROS, WARPS, false>(sums, x, codes, records, out, out_f32, M, N, K, ldx, ldo, group_blocks, act, limit))
        write_sums_again<XT, MT, T, GATED, SUB, ZEROS, WARPS>(sums, x, codes, records, out, out_f32, M, N, K, ldx, ldo, group_blocks, act, limit);
}

template <typename XT, int MT, int T, bool GATED, int SUB, bool ZEROS, int WARPS>
int launch_product4(const void* x, const void* codes, const void* records, void* out, int out_f32, int M, int N, int K, long long ldx, long long ldo, int group,
                    int act, float limit, int whole, cudaStream_t stream) {
    constexpr int ring = ring_of<T>::value * T * (kBlockBytes + SUB * (ZEROS ? 64 : 32)), sums = T * MT * 144 * 4;
    constexpr int smem = WARPS * (ring > sums ? ring : sums), wide = 16 * (GATED ? T / 2 : T);
    auto kernel = product4_kernel<XT, MT, T, GATED, SUB, ZEROS, WARPS>;
    if (smem > 48 * 1024) {
        static bool set = false;                 // once per kernel: the attribute stays
        if (!set) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return check_launch("product4");
            set = true;
        }
    }
    launch_pdl(kernel, dim3((unsigned)((N + wide - 1) / wide), (unsigned)((M + 8 * MT - 1) / (8 * MT))), dim3(WARPS * 32), smem, stream, (const XT*)x,
               (const uint8_t*)codes, (const uint8_t*)records, out, out_f32, M, N, K, ldx, ldo, group / 64, act, limit, whole);
    return check_launch("product4");
}

}  // namespace hos

using namespace hos;

extern "C" const char* hos_last_error() { return error_buffer(); }

// Rows of x are ldx numbers apart, rows of out ldo.
extern "C" int hos_product4(const void* x, int x_dtype, long long ldx, const void* matrix, void* out, int out_dtype, long long ldo, int M, int act, float limit,
                            cudaStream_t stream) {
    const Matrix4 w = *(const Matrix4*)matrix;
    const int N = w.n, K = w.k, group = w.group, zeros = w.zeros, gated = w.gated;
    const void *codes = w.codes, *records = w.records;
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) HOS_REFUSE("product4: K %d", K);
    if (group < 32 || (group != 32 && group % 64)) HOS_REFUSE("product4: groups of %d weights (32, or a multiple of 64)", group);
    if (M > 65535 * 8) HOS_REFUSE("product4: %d rows", M);
    if (x_dtype == kF32 ? out_dtype != kF32 : x_dtype != kBF16 || (out_dtype != kF32 && out_dtype != kBF16))
        HOS_REFUSE("product4: no product of type %d into type %d", x_dtype, out_dtype);
    const int piece = x_dtype == kF32 ? 4 : 8, whole = K % piece == 0 && ldx % piece == 0 && (uintptr_t)x % 16 == 0;
    // How many tiles of 16 rows of W a warp takes (they share its rows of x), and how many warps of a CTA share K: what makes one wave of
    // CTAs with 16 warps an SM, more tiles before fewer warps.  Of rows of more than 8 a warp's sums leave room for two tiles.  (us, 8 rows,
    // with 16 features a warp and 8 or 16 warps / by this rule: 9216 x 2304 gated 10.4 / 9.3, 36864 x 4608 28.5 / 22.3, 4608 x 36864 32.9 / 28.9.)
    const int units = (N + 15) / 16 * (gated ? 2 : 1), sm = sm_count_cached();
    const int shape = units <= sm && !gated ? 0 : (units <= 2 * sm ? 1 : (units <= 4 * sm ? 2 : (units <= 8 * sm ? 3 : 4)));
#define HOS_P4(X, MT, T, G, SUB, Z, W) return launch_product4<X, MT, T, G, SUB, Z, W>(x, codes, records, out, out_dtype == kF32, M, N, K, ldx, ldo, group, act, limit, whole, stream)
#define HOS_P4_W(X, MT, G, SUB, Z)                                       \
    do {                                                                 \
        constexpr int kMost = MT == 1 ? 4 : 2;                           \
        if (shape == 4) HOS_P4(X, MT, kMost, G, SUB, Z, 4);              \
        else if (shape == 3) HOS_P4(X, MT, kMost, G, SUB, Z, 8);         \
        else if (shape == 2) HOS_P4(X, MT, kMost, G, SUB, Z, 16);        \
        else if (shape == 1) HOS_P4(X, MT, 2, G, SUB, Z, 16);            \
        else HOS_P4(X, MT, (G ? 2 : 1), G, SUB, Z, 16);                  \
    } while (0)
#define HOS_P4_M(X, G, SUB, Z) do { if (M <= 8) HOS_P4_W(X, 1, G, SUB, Z); else if (M <= 16) HOS_P4_W(X, 2, G, SUB, Z); else HOS_P4_W(X, 4, G, SUB, Z); } while (0)
#define HOS_P4_S(X, G, Z) do { if (group == 32) HOS_P4_M(X, G, 2, Z); else HOS_P4_M(X, G, 1, Z); } while (0)
#define HOS_P4_G(X, Z) do { if (gated) HOS_P4_S(X, true, Z); else HOS_P4_S(X, false, Z); } while (0)
#define HOS_P4_Z(X) do { if (zeros) HOS_P4_G(X, true); else HOS_P4_G(X, false); } while (0)
    if (x_dtype == kF32) HOS_P4_Z(float);
    else HOS_P4_Z(bf16);
}
