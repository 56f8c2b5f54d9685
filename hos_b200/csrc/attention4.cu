// Keys and values in 4 bits: rows put into the pages, and attention over them.
//
// For every 64 neighbouring numbers of a head a scale s and a middle m in bfloat16 and 64 codes c of 4 bits, -8..7:
//   s = bf16((max - min) / 15), m = bf16(min + 8 s), c = clamp(rint((x - m) / s), -8, 7); what is held is c s + m.
// All numbers alike (s 0 or below the smallest normal number): codes 0, the value m.  A NaN, an infinity or a range that
// overflows makes the 64 numbers NaN.  Divisions and roundings are IEEE's, so that a value is a function of its row alone.
// A page's tile of a kv head is laid out in fourbit.cuh: keys "by row", values "by column".
#include "attention4.cuh"

namespace hos {

// ---- rows into pages ---------------------------------------------------------------------------------------------------
// Four lanes hold 64 numbers of a row, 16 each.  Many rows are bound by instructions, 35 a number (the row's two sums with NaN kept in sight, a
// quotient that is IEEE's, two codes to a byte by column): they are issued in 73% of the clocks, memory runs at a quarter of its rate (B200:
// 8,192 rows of 16 kv heads of 128, 67 MB read and as many handed back, 49 us; 8 rows 3.2).
struct Numbers { float v[16]; };
__device__ __forceinline__ Numbers load16(const float* p, bool vec) {
    Numbers x;
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = *(const float4*)(p + 4 * i);
            x.v[4 * i] = f.x; x.v[4 * i + 1] = f.y; x.v[4 * i + 2] = f.z; x.v[4 * i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x.v[i] = p[i];
    }
    return x;
}
__device__ __forceinline__ Numbers load16(const bf16* p, bool vec) {
    Numbers x;
    if (vec) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = *(const uint4*)(p + 8 * i);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x.v[8 * i + 2 * j] = bf16_lo(u[j]);
                x.v[8 * i + 2 * j + 1] = bf16_hi(u[j]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x.v[i] = to_float(p[i]);
    }
    return x;
}
__device__ __forceinline__ void store16(float* p, const Numbers& x, bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(float4*)(p + 4 * i) = make_float4(x.v[4 * i], x.v[4 * i + 1], x.v[4 * i + 2], x.v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = x.v[i];
    }
}
__device__ __forceinline__ void store16(bf16* p, const Numbers& x, bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *(uint4*)(p + 8 * i) = make_uint4(pack_bf16(x.v[8 * i], x.v[8 * i + 1]), pack_bf16(x.v[8 * i + 2], x.v[8 * i + 3]),
                                              pack_bf16(x.v[8 * i + 4], x.v[8 * i + 5]), pack_bf16(x.v[8 * i + 6], x.v[8 * i + 7]));
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = from_float<bf16>(x.v[i]);
    }
}

// Scale and middle of 64 numbers that four lanes hold, their codes as words (eight codes each, as a word of keys holds them), and what
// is held in the numbers' place.  The quotient by Markstein's correction (IA-64 and Elementary Functions, 2000): with r = 1 / s rounded and
// q near y / s, q + (y - q s) r rounded once is y / s rounded, for numbers whose parts stay normal; others are divided.
__device__ __forceinline__ void quantise64(Numbers& x, uint32_t& scale_middle, uint32_t (&w)[2]) {
    float lo = x.v[0], hi = x.v[0], odd = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        lo = fminf(lo, x.v[i]);
        hi = fmaxf(hi, x.v[i]);
        odd = fmaf(x.v[i], 0.f, odd);                          // NaN after an infinity or a NaN
    }
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
    odd += __shfl_xor_sync(0xffffffffu, odd, 1);
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 2));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 2));
    odd += __shfl_xor_sync(0xffffffffu, odd, 2);
    float s = to_float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
    if (!(s >= 1.17549435e-38f)) s = 0.f;                      // subnormal or 0 (a NaN is caught below)
    float m = to_float(__float2bfloat16_rn(__fadd_rn(lo, 8.f * s)));
    if (odd != 0.f || !isfinite(s) || !isfinite(m)) s = m = __int_as_float(0x7fffffff);
    scale_middle = pack_bf16(s, m);
    const float magic = 12582912.f;                            // 1.5 2^23: a sum with it is rounded to a whole number, ties to even
    const int zero = 0x4b400000;                               // its bits
    const bool none = !(s > 0.f), rough = s < 0x1p-100f || s > 0x1p100f;
    const float r = none ? 0.f : __frcp_rn(s);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t word = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float& v = x.v[8 * half + i];
            const float y = __fsub_rn(v, m);
            float q = __fmul_rn(y, r);
            q = fmaf(fmaf(-q, s, y), r, q);
            if (rough) q = none ? 0.f : __fdiv_rn(y, s);
            q = none ? 0.f : fminf(fmaxf(q, -8.f), 7.f);
            const float whole = __fadd_rn(q, magic);
            word += (uint32_t)(__float_as_int(whole) - zero + 8) << code_shift(i);
            v = fmaf(whole - magic, s, m);
        }
        w[half] = word;
    }
}

// The eight bytes that 16 values of a row are by column: byte j holds the numbers j and j + 8.
__device__ __forceinline__ uint32_t column_byte(const uint32_t (&w)[2], int j) {
    return ((w[0] >> code_shift(j)) & 15u) | (((w[1] >> code_shift(j)) & 15u) << 4);
}

// A few rows: four lanes a row and 64 numbers, straight into the pages.  A row is n_kv_heads * head_dim numbers of keys, then as many of
// values.
template <typename T>
__global__ void __launch_bounds__(128)
store4_few_kernel(const T* rows, long long stride, T* held, long long held_stride, const int* __restrict__ token_pos, const int* __restrict__ token_seq,
                  const int* __restrict__ seq_slot, const int* __restrict__ seq_len_after, Paged4 c, int n_tokens, int vec) {
    pdl_enter();
    const int dim = c.head_dim, groups = dim / 64, per_row = 2 * c.n_kv_heads * groups;
    const long long item = (long long)blockIdx.x * 32 + (threadIdx.x >> 2);
    const bool live = item < (long long)n_tokens * per_row;
    const int n = live ? (int)(item / per_row) : 0, r = live ? (int)(item % per_row) : 0, l = threadIdx.x & 3, col = r * 64 + l * 16;
    const int seq = token_seq[n], pos = token_pos[n];
    Numbers x = load16(rows + (size_t)n * stride + col, vec & 1);
    uint32_t sm, w[2];
    quantise64(x, sm, w);
    if (!live) return;
    if (held != nullptr) store16(held + (size_t)n * held_stride + col, x, vec & 2);
    if (seq < 0) return;
    if (c.ring_pages > 0 && pos + c.ring_pages * kPageTokens < seq_len_after[seq]) return;     // the same step writes over it
    const bool value = r >= c.n_kv_heads * groups;
    const int head = (r - (value ? c.n_kv_heads * groups : 0)) / groups, g = r % groups, row = pos % kPageTokens;
    const int page = page4_of(c, seq_slot[seq], pos);
    uint8_t* tile = (value ? c.v_pages : c.k_pages) + ((size_t)page * c.n_kv_heads + head) * tile4_bytes(dim);
    uint8_t* block = tile + ((row >> 4) * groups + g) * kBlockBytes;
    if (!value) {
        *(uint2*)(block + by_row_word(row & 15, l * 16)) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) block[by_column_byte(row & 15, l * 16 + j)] = (uint8_t)column_byte(w, j);
    }
    if (l == 0) *(uint32_t*)(tile + tile4_codes(dim) + (row * groups + g) * 4) = sm;
}

// Many rows: a warp takes 64 numbers of the up to 16 rows whose positions make a block of the pages, forms the block's 512 bytes in shared
// memory and writes them at once (with positions missing, or written over by the same step, what is there only).  Blocks are the
// sequences' in order, and after them the padding rows, 16 at a time, which store nothing but are handed back.
template <typename T>
__global__ void __launch_bounds__(256)
store4_many_kernel(const T* rows, long long stride, T* held, long long held_stride, const int* __restrict__ token_pos, const int* __restrict__ cu_seqlens,
                   int row_base, int n_seqs, const int* __restrict__ seq_slot, const int* __restrict__ seq_len_after, int seq_base, Paged4 c, int n_tokens,
                   int vec) {
    __shared__ __align__(16) uint8_t blocks[8][kBlockBytes];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 3, quad = lane >> 2;
    const int dim = c.head_dim, groups = dim / 64, per_row = 2 * c.n_kv_heads * groups;
    const RowBlock found = find_rows(cu_seqlens, row_base, n_seqs, token_pos, n_tokens, blockIdx.x, 16, 15);
    const int seq = found.seq, row0 = found.row0, pos0 = found.pos0, count = found.count;
    if (count <= 0) return;
    const int r = blockIdx.y * 8 + warp;                       // which 64 numbers of a row
    if (r >= per_row) return;
    const bool value = r >= c.n_kv_heads * groups;
    const int head = (r - (value ? c.n_kv_heads * groups : 0)) / groups, g = r % groups, at0 = pos0 & 15, page_row = pos0 & (kPageTokens - 1) & ~15;
    uint8_t* tile = nullptr;
    int kept = 0;                                              // the rows before this one are written over by the same step
    if (seq >= 0) {
        const int slot = seq_slot[seq_base + seq];
        tile = (value ? c.v_pages : c.k_pages) + ((size_t)page4_of(c, slot, pos0) * c.n_kv_heads + head) * tile4_bytes(dim);
        if (c.ring_pages > 0) kept = max(0, seq_len_after[seq_base + seq] - c.ring_pages * kPageTokens - pos0);
    }
#pragma unroll
    for (int it = 0; it < 2; ++it) {
        const int i = it * 8 + quad;                           // eight rows at a time
        const T* from = rows + (size_t)(row0 + min(i, count - 1)) * stride + r * 64 + l * 16;
        Numbers x = load16(from, vec & 1);
        uint32_t sm, w[2];
        quantise64(x, sm, w);
        if (i < count) {
            if (held != nullptr) store16(held + (size_t)(row0 + i) * held_stride + r * 64 + l * 16, x, vec & 2);
            const int row = at0 + i;
            if (tile != nullptr && i >= kept) {
                if (l == 0) *(uint32_t*)(tile + tile4_codes(dim) + ((page_row + row) * groups + g) * 4) = sm;
                if (!value) {
                    *(uint2*)(blocks[warp] + by_row_word(row, l * 16)) = make_uint2(w[0], w[1]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) blocks[warp][by_column_byte(row, l * 16 + j)] = (uint8_t)column_byte(w, j);
                }
            }
        }
    }
    __syncwarp();
    if (tile == nullptr) return;
    uint8_t* to = tile + ((page_row >> 4) * groups + g) * kBlockBytes + lane * 16;
    const uint8_t* mine = blocks[warp] + lane * 16;
    if (count == 16 && kept == 0) {
        *(uint4*)to = *(const uint4*)mine;
        return;
    }
    auto there = [&](int row) { return row >= at0 + kept && row < at0 + count; };
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = value ? 2 * (lane & 3) + ((i >> 1) & 1) + 8 * (i & 1) : (lane >> 2) + 8 * (i >> 3);
        if (there(row)) to[i] = mine[i];
    }
}

// ---- attention of single rows --------------------------------------------------------------------------------------
// No unit is full (8 rows over 8,192 keys: reads at 29% of their rate, ALU 41%, mma.sync 14%, an instruction issued in 48% of the clocks, 850 for
// 16 keys of a kv head of 256): 14 warps an SM, which wait for their own results and, at the merge, for one another.  An infinity in a query
// gives NaN, as without a soft-cap the definition does.
//
// Scores: S^T = K Q^T with 16 keys as the MMA's rows and up to 8 query heads of a kv head as its columns (fewer heads: of several
// neighbouring rows of a sequence, each with its own mask).  The score of a key is
// sum_g (s_g (sum_{d in g} q c') - 136 s_g sum q + m_g sum q) over its groups of 64, c' = 128 + c + 8 the operand as codes_to_bf16 makes
// it without subtracting: a group's product starts at -136 sum q and is multiplied by the key's scale, in 32 bits; neither scale nor
// middle is rounded into an operand.  Values: O^T = V^T P^T with 16 numbers of a head as rows, P times the value's scale in half
// precision (attention4.cuh; in bfloat16, 2^-8 of a weight, long rows whose output is a small mean lost as much as the result's own
// rounding), the codes exact, and the middles' sum, one number a group and head, in 32 bits beside it.  The scores' registers,
// transposed eight by eight, are P's operand.
// Rows in 32 bits: q, and p times the scale, are three bfloat16 numbers each, exactly, and the codes are subtracted first.
//
// A CTA takes a share of the pages of one (row or neighbouring rows, kv head, 8 heads); its warps take 16 keys in turn, each through a ring of its own that
// cp.async fills, so that no barrier stands in the walk.  Running maxima are a warp's own and are raised when a score passes them by
// 2^8.  The warps merge through shared memory; 2, 4 or 8 shares may be a cluster and merge through its shared memory, others through a
// workspace and attend4_merge_kernel.
// Measured (B200): 8 rows over 8,192 keys, 8 heads over 4 of 256, 31 us (2.4 TB/s of pages); 48 rows over up to 8,000 keys, window
// 4,096, 32 heads over 16 of 128, 119 us; 1 row over 1,000 keys 9.7 us.
constexpr int kAttendWarps = 8, kMaxSharePages = 256, kClusterShares = 8;

template <int DIM> struct Attend4 {
    static constexpr int kGroups = DIM / 64;
    static constexpr int kCodes = kGroups * kBlockBytes, kMeta = 64 * kGroups;          // of 16 keys, or values
    static constexpr int kStage = 2 * (kCodes + kMeta);
    static constexpr int kRing = DIM == 256 ? 2 : (DIM == 192 ? 3 : (DIM == 128 ? 4 : 8));      // two CTAs to an SM
    static constexpr int kPitch = DIM + 4;                                              // floats of a head's sums in shared memory
    static constexpr int kRingBytes = kAttendWarps * kRing * kStage, kSumBytes = kAttendWarps * 8 * kPitch * 4;
    static constexpr int kShared = kRingBytes > kSumBytes ? kRingBytes : kSumBytes;
};

template <int GROUPS>
__device__ __forceinline__ void load_meta(uint32_t at, uint32_t (&m)[GROUPS]) {
    if (GROUPS == 4) {
        const uint4 v = lds16(at);
        m[0] = v.x; m[1 % GROUPS] = v.y; m[2 % GROUPS] = v.z; m[3 % GROUPS] = v.w;
    } else if (GROUPS == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(m[0]), "=r"(m[1 % GROUPS]) : "r"(at));
    } else {
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(m[i]) : "r"(at + 4 * i));
    }
}

__device__ __forceinline__ uint32_t peer_at(uint32_t at, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_float(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// GROUPS: a CTA takes up to 8 / (heads of a kv head) neighbouring rows of a sequence; without, column j is simply head h0 + j of a row.
template <typename T, int DIM, bool GROUPS>
__global__ void __launch_bounds__(kAttendWarps * 32, 2)
attend4_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const int* __restrict__ token_pos,
               const int* __restrict__ token_seq, const int* __restrict__ seq_slot, const int* __restrict__ token_slot, const int* __restrict__ cu_seqlens, int row_base,
               int n_seqs, int n_tokens, Paged4 c, int n_heads, float scale, float cap, int window, int share, int splits, float* __restrict__ part_o, float2* __restrict__ part_ml) {
    using A = Attend4<DIM>;
    constexpr int G = A::kGroups, kTerms = sizeof(T) == 4 ? 3 : 1, kTiles = DIM / 16;
    constexpr bool kExact = kTerms == 3;
    extern __shared__ __align__(16) uint8_t ring_bytes[];
    __shared__ __align__(16) uint4 q_frag[kTerms][G][2][32];
    __shared__ float q_sum[G][8];
    __shared__ int ids[kMaxSharePages];
    __shared__ float2 warp_ml[kAttendWarps][8];
    __shared__ float warp_f[kAttendWarps][8];
    __shared__ float2 cta_ml[8];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int split = blockIdx.x % splits;
    const int per = n_heads / c.n_kv_heads;
    RowBlock rows = {0, (int)blockIdx.x / splits, 0, 1};
    if (GROUPS) {
        rows = find_rows(cu_seqlens, row_base, n_seqs, token_pos, n_tokens, blockIdx.x / splits, 8 / per, 0);
        if (rows.count <= 0) return;                           // all of a cluster's CTAs alike
    }
    const int n = rows.row0, chunks = (per + 7) / 8, kvh = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
    const int h0 = kvh * per + chunk * 8, nh = min(8, per - chunk * 8), columns = nh * rows.count;
    auto row_at = [&](int column) { return GROUPS ? column / nh : 0; };                     // column j: head h0 + j % nh of row n + j / nh
    auto head_at = [&](int column) { return GROUPS ? column % nh : column; };
    const int seq = token_seq[n], known_slot = token_slot != nullptr ? token_slot[n] : -1;
    const int pos0 = token_pos[n], last = pos0 + rows.count - 1, first = window > 0 ? max(0, pos0 - window + 1) : 0;
    // the pages of the keys, from page0 to before page1; where there are more than planned a share is longer
    const int page0 = first / kPageTokens, page1 = last / kPageTokens + 1, pages = max(share, (page1 - page0 + splits - 1) / splits);
    const int p0 = page0 + split * pages, p1 = seq < 0 ? p0 : min(page1, p0 + pages);      // a padding row has no pages
    const bool clustered = splits > 1 && part_o == nullptr;
    float* sums = (float*)ring_bytes;                          // once the walk is over
    if (p0 >= p1) {                                            // a share without keys says so; a padding row becomes zeros
        if (splits == 1) {
            for (int i = threadIdx.x; i < columns * DIM; i += blockDim.x)
                out[(size_t)(n + row_at(i / DIM)) * out_stride + (size_t)(h0 + head_at(i / DIM)) * DIM + i % DIM] = from_float<T>(0.f);
            return;
        }
        if (threadIdx.x < 8) cta_ml[threadIdx.x] = make_float2(-INFINITY, 0.f);
        if (!clustered) {
            if (threadIdx.x < columns)
                part_ml[((size_t)(n + row_at(threadIdx.x)) * n_heads + h0 + head_at(threadIdx.x)) * splits + split] = make_float2(-INFINITY, 0.f);
            return;
        }
    } else {
    const int* table = c.page_table + (size_t)(token_slot != nullptr ? known_slot : seq_slot[seq]) * c.table_stride;
    auto page_of = [&](int p) { return table[c.ring_pages > 0 ? p % c.ring_pages : p]; };
    const int b0 = max(first, p0 * kPageTokens) >> 4, b1 = min(last, p1 * kPageTokens - 1) >> 4;      // blocks of 16 keys, b1 the last
    const uint32_t ring = smem_u32(ring_bytes) + warp * A::kRing * A::kStage;
    int to_fetch = b0 + warp;
    auto fetch = [&](uint32_t to, bool known) {
        if (to_fetch <= b1) {
            const int p = to_fetch >> 2, in = to_fetch & 3;
            const size_t tile = ((size_t)(known && p - p0 < kMaxSharePages ? ids[p - p0] : page_of(p)) * c.n_kv_heads + kvh) * tile4_bytes(DIM);
            const uint8_t *k = c.k_pages + tile, *v = c.v_pages + tile;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                copy16_async(to + i * kBlockBytes + lane * 16, k + (in * G + i) * kBlockBytes + lane * 16);
                copy16_async(to + A::kCodes + A::kMeta + i * kBlockBytes + lane * 16, v + (in * G + i) * kBlockBytes + lane * 16);
            }
            if ((lane & 15) < 4 * G) {
                const uint8_t* src = (lane < 16 ? k : v) + tile4_codes(DIM) + in * A::kMeta + (lane & 15) * 16;
                copy16_async(to + A::kCodes + (lane < 16 ? 0 : A::kCodes + A::kMeta) + (lane & 15) * 16, src);
            }
        }
        to_fetch += kAttendWarps;
        copies_commit();
    };
#pragma unroll
    for (int i = 0; i < A::kRing - 1; ++i) fetch(ring + i * A::kStage, false);      // before the page numbers are in shared memory
    for (int i = threadIdx.x; i < min(p1 - p0, kMaxSharePages); i += blockDim.x) ids[i] = page_of(p0 + i);
    // the columns' numbers as operands, and their sums over 64
    const T* q_row = q + (size_t)n * q_stride + (size_t)h0 * DIM;
    for (int i = threadIdx.x; i < G * 64; i += blockDim.x) {
        const int l = i & 31, half = (i >> 5) & 1, grp = i >> 6, head = l >> 2, d = grp * 64 + (l & 3) * 16 + half * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = head < columns ? to_float(q_row[row_at(head) * q_stride + head_at(head) * DIM + d + j]) : 0.f;
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                v[2 * j] -= bf16_lo(w[j]);
                v[2 * j + 1] -= bf16_hi(w[j]);
            }
            q_frag[term][grp][half][l] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    for (int i = warp; i < G * 8; i += kAttendWarps) {
        const int head = i & 7, grp = i >> 3;
        const T* from = q_row + row_at(head) * q_stride + head_at(head) * DIM + grp * 64 + lane;
        float v = head < columns ? to_float(from[0]) + to_float(from[32]) : 0.f;
        v = warp_sum(v);
        if (lane == 0) q_sum[grp][head] = v;
    }
    __syncthreads();

    float o[kTiles][4], mid[G][2], best[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    float into[G];                                              // of the weights in half precision
#pragma unroll
    for (int i = 0; i < G; ++i) into[i] = kIntoFirst;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) mid[i][0] = mid[i][1] = 0.f;
    const int row_of[2] = {row_at(2 * t4), row_at(2 * t4 + 1)};     // of a lane's columns
    const float scale2 = scale * 1.44269504f, cap2 = cap * 1.44269504f, in_cap = cap > 0.f ? 2.f * scale2 / cap : 0.f;
    uint32_t slot = ring, before = ring + (A::kRing - 1) * A::kStage;
    for (int b = b0 + warp; b <= b1; b += kAttendWarps) {
        copies_wait<A::kRing - 2>();
        __syncwarp();
        fetch(before, true);                                   // the place that the last block has left
        uint32_t km[2][G], vm[2][G];                           // of the keys g and g + 8
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            load_meta<G>(slot + A::kCodes + (g + 8 * r) * 4 * G, km[r]);
            load_meta<G>(slot + 2 * A::kCodes + A::kMeta + (g + 8 * r) * 4 * G, vm[r]);
        }
        const int key = b * 16 + g;
        // some column does not see some of these keys: what is hidden from a column may be anything
        const bool edge = b * 16 + 15 > pos0 || (window > 0 && b * 16 <= last - window);
        bool hidden[4] = {false, false, false, false};
        if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = key + 8 * (e >> 1), mine = pos0 + (GROUPS ? row_of[e & 1] : 0);
                hidden[e] = at > mine || (window > 0 && at <= mine - window);
            }
        }
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint4 w = lds16(slot + i * kBlockBytes + lane * 16);
            uint32_t lo[2][4], hi[2][4];                       // the key g's, and g + 8's
            codes_to_bf16<kExact>(w.x, kZero8, lo[0]);
            codes_to_bf16<kExact>(w.y, kZero8, lo[1]);
            codes_to_bf16<kExact>(w.z, kZero8, hi[0]);
            codes_to_bf16<kExact>(w.w, kZero8, hi[1]);
            const float2 qs = *(const float2*)&q_sum[i][2 * t4];
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            if (!kExact) {
                part[0] = part[2] = -136.f * qs.x;
                part[1] = part[3] = -136.f * qs.y;
            }
#pragma unroll
            for (int term = kTerms - 1; term >= 0; --term) {
                const uint4 qa = q_frag[term][i][0][lane], qb = q_frag[term][i][1][lane];
                const uint32_t qf[8] = {qa.x, qa.y, qa.z, qa.w, qb.x, qb.y, qb.z, qb.w};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const uint32_t a[4] = {lo[st >> 1][2 * (st & 1)], hi[st >> 1][2 * (st & 1)], lo[st >> 1][2 * (st & 1) + 1], hi[st >> 1][2 * (st & 1) + 1]};
                    mma_plain(part, a, qf[2 * st], qf[2 * st + 1]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t sm = km[e >> 1][i];
                s[e] = fmaf(bf16_lo(sm), part[e], fmaf(bf16_hi(sm), (e & 1) ? qs.y : qs.x, s[e]));
            }
        }
        // scores in units of log 2
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (cap > 0.f) {
                if (kExact) s[e] = cap2 * tanhf(s[e] * scale / cap);
                else s[e] = cap2 * (1.f - 2.f * rcp_approx(1.f + ex2_approx(s[e] * in_cap)));
            } else {
                s[e] *= scale2;
            }
            if (hidden[e]) s[e] = -INFINITY;
        }
        float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
        float scale_of[G], most = 0.f;                         // the larger of a lane's two values' scales, where a column sees them
        if (!kExact) {
            const bool seen[2] = {!edge || (key <= last && (window == 0 || key > pos0 - window)), !edge || (key + 8 <= last && (window == 0 || key + 8 > pos0 - window))};
#pragma unroll
            for (int i = 0; i < G; ++i) {
                scale_of[i] = fmaxf(seen[0] ? bf16_lo(vm[0][i]) : 0.f, seen[1] ? bf16_lo(vm[1][i]) : 0.f);
                most = fmaxf(most, scale_of[i] * into[i]);
            }
        }
        if (__any_sync(0xffffffffu, top[0] > best[0] + 8.f || top[1] > best[1] + 8.f || most > kIntoMost)) {
            if (!kExact) {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const float largest = warp_max(scale_of[i]);
                    if (largest * into[i] > kIntoMost && largest < INFINITY) {
                        const float now = into_of(largest), f = now * back_of(into[i]);
                        into[i] = now;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            o[4 * i + j][0] *= f; o[4 * i + j][1] *= f; o[4 * i + j][2] *= f; o[4 * i + j][3] *= f;
                        }
                    }
                }
            }
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
                top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
            }
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float m = fmaxf(best[h], top[h]);
                f[h] = best[h] == m ? 1.f : ex2_approx(best[h] - m);
                best[h] = m;
                sum[h] *= f[h];
#pragma unroll
                for (int i = 0; i < G; ++i) mid[i][h] *= f[h];
            }
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                o[i][0] *= f[0]; o[i][1] *= f[1]; o[i][2] *= f[0]; o[i][3] *= f[1];
            }
        }
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = hidden[e] ? 0.f : ex2_approx(s[e] - best[e & 1]);      // a column may not have seen a key yet
        sum[0] += p[0] + p[2];
        sum[1] += p[1] + p[3];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const float sv[2] = {kExact ? bf16_lo(vm[0][i]) : bf16_lo(vm[0][i]) * into[i], kExact ? bf16_lo(vm[1][i]) : bf16_lo(vm[1][i]) * into[i]};
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = hidden[e] ? 0.f : p[e] * sv[e >> 1];
                mid[i][e & 1] = hidden[e] ? mid[i][e & 1] : fmaf(p[e], bf16_hi(vm[e >> 1][i]), mid[i][e & 1]);
            }
            const uint4 v = lds16(slot + A::kCodes + A::kMeta + i * kBlockBytes + lane * 16);
            const uint32_t words[4] = {v.x, v.y, v.z, v.w};
            if (kExact) {
                uint32_t pb[kTerms][2];
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    const uint32_t a = pack_bf16(w[0], w[1]), b8 = pack_bf16(w[2], w[3]);
                    pb[term][0] = transposed_8x8(a);
                    pb[term][1] = transposed_8x8(b8);
                    w[0] -= bf16_lo(a); w[1] -= bf16_hi(a); w[2] -= bf16_lo(b8); w[3] -= bf16_hi(b8);
                }
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    uint32_t a[4];
                    codes_to_bf16<true>(words[mt], kZero8, a);
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) mma_plain(o[4 * i + mt], a, pb[term][0], pb[term][1]);
                }
            } else {
                const uint32_t p0 = transposed_8x8(pack_half(w[0], w[1])), p8 = transposed_8x8(pack_half(w[2], w[3]));
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    uint32_t a[4];
                    codes_to_half(words[mt], a);
                    mma_half(o[4 * i + mt], a, p0, p8);
                }
            }
        }
        before = slot;
        slot = slot == ring + (A::kRing - 1) * A::kStage ? ring : slot + A::kStage;
    }
    copies_wait<0>();
    // a lane's sums over its keys, added up over the lanes of its heads
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], off);
#pragma unroll
            for (int i = 0; i < G; ++i) mid[i][h] += __shfl_xor_sync(0xffffffffu, mid[i][h], off);
        }
    }
    if (g == 0) {
        warp_ml[warp][2 * t4] = make_float2(best[0], sum[0]);
        warp_ml[warp][2 * t4 + 1] = make_float2(best[1], sum[1]);
    }
    __syncthreads();                                           // the rings are done with: the sums go where they were
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (2 * t4 + h < columns) {
            float* to = sums + (warp * 8 + 2 * t4 + h) * A::kPitch;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                const float back = kExact ? 1.f : back_of(into[i / 4]);       // a power of two
                to[i * 16 + g] = fmaf(o[i][h], back, mid[i / 4][h]);
                to[i * 16 + g + 8] = fmaf(o[i][2 + h], back, mid[i / 4][h]);
            }
        }
    }
    if (threadIdx.x < 8) {
        float m = -INFINITY, l = 0.f;
        for (int w = 0; w < kAttendWarps; ++w) m = fmaxf(m, warp_ml[w][threadIdx.x].x);
        for (int w = 0; w < kAttendWarps; ++w) {
            const float2 ml = warp_ml[w][threadIdx.x];
            const float f = ml.x == m ? 1.f : ex2_approx(ml.x - m);       // a warp without keys: 2^(-inf)
            warp_f[w][threadIdx.x] = f;
            l += f * ml.y;
        }
        cta_ml[threadIdx.x] = make_float2(m, l);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns * DIM; i += blockDim.x) {
        const int h = i / DIM, d = i % DIM;
        const size_t row = n + row_at(h), head = h0 + head_at(h);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kAttendWarps; ++w) v = fmaf(warp_f[w][h], sums[(w * 8 + h) * A::kPitch + d], v);
        if (splits == 1) {
            out[row * out_stride + head * DIM + d] = from_float<T>(v / cta_ml[h].y);
        } else if (clustered) {
            sums[h * A::kPitch + d] = v;                       // nobody else reads the first warp's
        } else {
            const size_t at = (row * n_heads + head) * splits + split;
            part_o[at * DIM + d] = v;
            if (d == 0) part_ml[at] = cta_ml[h];
        }
    }
    }
    if (!clustered) return;
    cluster_meet();
    for (int i = split * blockDim.x + threadIdx.x; i < columns * DIM; i += splits * blockDim.x) {
        const int h = i / DIM, d = i % DIM;
        const uint32_t ml_at = smem_u32(&cta_ml[h]), v_at = smem_u32(&sums[h * A::kPitch + d]);
        float m = -INFINITY, l = 0.f, v = 0.f;
        for (int s = 0; s < splits; ++s) m = fmaxf(m, peer_float(peer_at(ml_at, s)));
        for (int s = 0; s < splits; ++s) {
            const float pm = peer_float(peer_at(ml_at, s)), pl = peer_float(peer_at(ml_at + 4, s));
            if (pl == 0.f) continue;                           // a share without keys: its sums are not there
            const float f = pm == m ? 1.f : ex2_approx(pm - m);
            l = fmaf(f, pl, l);
            v = fmaf(f, peer_float(peer_at(v_at, s)), v);
        }
        out[(size_t)(n + row_at(h)) * out_stride + (size_t)(h0 + head_at(h)) * DIM + d] = from_float<T>(seq < 0 ? 0.f : v / l);
    }
    cluster_meet();                                            // nobody leaves while its sums are read
}

// The shares of a (row, head) added up: one thread a number, or, of 8 and more shares, four threads that each take every fourth
// share.  The loads' latency bounds it: attention and merge of 1 row of 8 heads of 256 over 8,192 keys in 32 shares 20.8 us with one
// thread a number, 14.0 with four; 8 shares 22.8 and 21.4; 3 rows of 32 heads of 128 over 20,000 keys in 12 shares 32.4 and 28.9.
// Few shares of many rows want the threads for other rows: 739 rows in 4 shares 312 us with one, 336 with four.
constexpr int kMergeWays = 4, kWaysFrom = 8;
inline unsigned merge_threads(int dim, int splits) { return dim * (splits >= kWaysFrom ? kMergeWays : 1); }
template <typename T, int DIM>
__global__ void __launch_bounds__(DIM * kMergeWays)
attend4_merge_kernel(T* __restrict__ out, long long out_stride, int n_heads, int splits, const float* __restrict__ part_o, const float2* __restrict__ part_ml) {
    __shared__ float factor[kMaxShares];
    __shared__ float total, sums[kMergeWays - 1][DIM];
    pdl_enter();
    const int n = blockIdx.x / n_heads, h = blockIdx.x % n_heads, d = threadIdx.x % DIM, way = threadIdx.x / DIM, ways = blockDim.x / DIM;
    const size_t at = (size_t)blockIdx.x * splits;
    if (threadIdx.x < 32) {                                    // one warp: every share's weight, 0 for one without keys
        float m = -INFINITY, l = 0.f;
        for (int s = threadIdx.x; s < splits; s += 32) m = fmaxf(m, part_ml[at + s].x);
        m = warp_max(m);
        for (int s = threadIdx.x; s < splits; s += 32) {
            const float2 ml = part_ml[at + s];
            const float f = ml.y == 0.f ? 0.f : (ml.x == m ? 1.f : ex2_approx(ml.x - m));
            factor[s] = f;
            l = fmaf(f, ml.y, l);
        }
        l = warp_sum(l);
        if (threadIdx.x == 0) total = l;
    }
    __syncthreads();
    float v = 0.f;
#pragma unroll 8
    for (int s = way; s < splits; s += ways) {
        const float f = factor[s], o = part_o[(at + s) * DIM + d];     // of a share without keys whatever lies there: asked for all the
        if (f != 0.f) v = fmaf(f, o, v);                               // same, so that eight are under way together
    }
    if (way > 0) sums[way - 1][d] = v;
    if (ways > 1) __syncthreads();
    if (way > 0) return;
    for (int w = 1; w < ways; ++w) v += sums[w - 1][d];
    out[(size_t)n * out_stride + (size_t)h * DIM + d] = from_float<T>(total == 0.f ? 0.f : v / total);      // a padding row has no share with keys
}

template <typename T, int DIM, bool GROUPS>
int launch_attend4(const void* q, long long q_stride, void* out, long long out_stride, const int* token_pos, const int* token_seq, const int* seq_slot,
                   const int* token_slot, const int* cu_seqlens, int row_base, int n_seqs, const Paged4& c, int n_tokens, int n_heads, float scale,
                   float cap, int window, int share, int splits, float* part_o, float2* part_ml, cudaStream_t stream) {
    constexpr int smem = Attend4<DIM>::kShared;
    auto kernel = attend4_kernel<T, DIM, GROUPS>;
    static bool set = false;                                   // once per kernel: the attribute stays
    if (!set) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return check_launch("attend4");
        set = true;
    }
    const int per = n_heads / c.n_kv_heads, chunks = (per + 7) / 8;
    const long long n_groups = GROUPS ? (n_tokens + 8 / per - 1) / (8 / per) + n_seqs : n_tokens;      // a sequence's last may not be full
    const bool clustered = splits > 1 && part_o == nullptr;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_groups * splits), (unsigned)(c.n_kv_heads * chunks));
    cfg.blockDim = dim3(kAttendWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)splits, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = clustered ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, (const T*)q, q_stride, (T*)out, out_stride, token_pos, token_seq, seq_slot, token_slot, cu_seqlens, row_base,
                       n_seqs, n_tokens, c, n_heads, scale, cap, window, share, splits, part_o, part_ml);
    if (splits > 1 && !clustered)
        launch_pdl(attend4_merge_kernel<T, DIM>, dim3((unsigned)((long long)n_tokens * n_heads)), dim3(merge_threads(DIM, splits)), 0, stream, (T*)out, out_stride, n_heads,
                   splits, (const float*)part_o, (const float2*)part_ml);
    return check_launch("attend4");
}

}  // namespace hos

using namespace hos;

// Rows and `held` (or null) have their numbers side by side; sequences' rows are cu_seqlens[s] - row_base .. in order (their entries of
// seq_slot and seq_len_after begin at seq_base), then padding rows.  single: the sequences bring a row each.
extern "C" int hos_store4(const void* rows, int dtype, long long stride, void* held, long long held_stride, const int* token_pos, const int* token_seq,
                          const int* seq_slot, const int* seq_len_after, const int* cu_seqlens, int row_base, int n_seqs, int seq_base, int single,
                          const void* cache, int n_tokens, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    HOS_CHECK_PAGED4("store4");
    const int per_row = 2 * n_kv_heads * (head_dim / 64), piece = dtype == kF32 ? 4 : 8;
    const int vec = (stride % piece == 0 && (uintptr_t)rows % 16 == 0 ? 1 : 0) | (held_stride % piece == 0 && (uintptr_t)held % 16 == 0 ? 2 : 0);
    const long long items = (long long)n_tokens * per_row;
    // Pieces of 64 numbers from which blocks of 16 positions written whole pay (us, a piece's lanes for themselves / blocks of positions;
    // 4 kv heads of 256: 128 rows, 4,096 pieces, 3.3 / 5.0, 512 rows, 16,384, 4.5 / 5.2; 16 of 128: 512 rows, 32,768, 6.6 / 5.9).
    const bool many = items >= 24576 && !single;
    // every sequence may begin and end inside a block
    const dim3 few_grid((unsigned)((items + 31) / 32)), many_grid((unsigned)((n_tokens + 15) / 16 + 2 * n_seqs), (unsigned)((per_row + 7) / 8));
    if (many && many_grid.y > 65535) HOS_REFUSE("store4: %d kv heads", n_kv_heads);
#define HOS_S4(T)                                                                                                                                       \
    do {                                                                                                                                                \
        if (many)                                                                                                                                       \
            launch_pdl(store4_many_kernel<T>, many_grid, dim3(256), 0, stream, (const T*)rows, stride, (T*)held, held_stride, token_pos, cu_seqlens,        \
                       row_base, n_seqs, seq_slot, seq_len_after, seq_base, c, n_tokens, vec);                                                          \
        else                                                                                                                                            \
            launch_pdl(store4_few_kernel<T>, few_grid, dim3(128), 0, stream, (const T*)rows, stride, (T*)held, held_stride, token_pos, token_seq,           \
                       seq_slot, seq_len_after, c, n_tokens, vec);                                                                                      \
    } while (0)
    if (dtype == kF32) HOS_S4(float);
    else HOS_S4(bf16);
    return check_launch("store4");
}

// token_slot: seq_slot[token_seq] of every row, or null.  cu_seqlens: the sequences' rows (less row_base), n_seqs + 1 of them, padding rows
// behind: neighbouring rows of a sequence share a walk if the kv heads have few heads; null: every row alone.  A walk is cut into shares
// of `share` pages, a CTA each: `splits` of them cover the longest row's.  2 to 8 without `parts` are a cluster; else more than one need
// `parts`, n_tokens * n_heads * splits * (head_dim + 2) 32-bit numbers.
extern "C" int hos_attend4(const void* q, int dtype, long long q_stride, void* out, long long out_stride, const int* token_pos, const int* token_seq,
                           const int* seq_slot, const int* token_slot, const int* cu_seqlens, int row_base, int n_seqs, const void* cache, int n_tokens,
                           int n_heads, float scale, float cap, int window, int share, int splits, float* parts, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    HOS_CHECK_PAGED4("attend4");
    if (n_heads <= 0 || n_heads % n_kv_heads) HOS_REFUSE("attend4: %d query heads over %d kv heads", n_heads, n_kv_heads);
    if (share < 1 || splits < 1 || splits > kMaxShares) HOS_REFUSE("attend4: %d shares of %d pages (1..%d shares)", splits, share, kMaxShares);
    if (splits > kClusterShares && parts == nullptr) HOS_REFUSE("attend4: %d shares need a workspace", splits);
    if ((long long)n_tokens * splits > 0x7fffffffll || (long long)n_tokens * n_heads > 0x7fffffffll) HOS_REFUSE("attend4: %d rows in %d shares", n_tokens, splits);
    const size_t n_parts = (size_t)n_tokens * n_heads * splits;
    float2* part_ml = (float2*)parts;                          // pairs first: they want 8 bytes' alignment
    float* part_o = parts == nullptr ? nullptr : parts + 2 * n_parts;
    const bool groups = cu_seqlens != nullptr && 2 * (n_heads / n_kv_heads) <= 8;
#define HOS_A4(T, D)                                                                                                                             \
    return (groups ? launch_attend4<T, D, true> : launch_attend4<T, D, false>)(q, q_stride, out, out_stride, token_pos, token_seq, seq_slot,       \
                                                                               token_slot, cu_seqlens, row_base, n_seqs, c, n_tokens, n_heads,     \
                                                                               scale, cap, window, share, splits, part_o, part_ml, stream)
#define HOS_A4_D(T) do { if (head_dim == 64) HOS_A4(T, 64); else if (head_dim == 128) HOS_A4(T, 128); else if (head_dim == 192) HOS_A4(T, 192); else HOS_A4(T, 256); } while (0)
    if (dtype == kF32) HOS_A4_D(float);
    else HOS_A4_D(bf16);
}

// The shares' sums in `parts` (hos_attend4, hos_attend4_tiles) added up into out.
extern "C" int hos_attend4_merge(void* out, int dtype, long long out_stride, int head_dim, int n_tokens, int n_heads, int splits, float* parts, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (parts == nullptr || splits < 1 || splits > kMaxShares || n_heads <= 0 || (long long)n_tokens * n_heads > 0x7fffffffll)
        HOS_REFUSE("attend4_merge: %d rows of %d heads in %d shares", n_tokens, n_heads, splits);
    const float2* part_ml = (const float2*)parts;
    const float* part_o = parts + 2 * (size_t)n_tokens * n_heads * splits;
#define HOS_AM(T, D)                                                                                                                             \
    launch_pdl(attend4_merge_kernel<T, D>, dim3((unsigned)((long long)n_tokens * n_heads)), dim3(merge_threads(D, splits)), 0, stream, (T*)out,    \
               out_stride, n_heads, splits, part_o, part_ml)
#define HOS_AM_D(T)                                                                                                                              \
    do {                                                                                                                                         \
        if (head_dim == 64) HOS_AM(T, 64);                                                                                                       \
        else if (head_dim == 128) HOS_AM(T, 128);                                                                                                \
        else if (head_dim == 192) HOS_AM(T, 192);                                                                                                \
        else if (head_dim == 256) HOS_AM(T, 256);                                                                                                \
        else HOS_REFUSE("attend4_merge: head size %d", head_dim);                                                                                \
    } while (0)
    if (dtype == kF32) HOS_AM_D(float);
    else HOS_AM_D(bf16);
    return check_launch("attend4_merge");
}
