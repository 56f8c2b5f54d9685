// Attention of pieces over 4-bit pages: sequences that bring many bfloat16 rows.
//
// 128 (row, head) pairs of a kv head to a CTA, 16 to a warp; a page's keys and values are formed once for all of them, as bare codes -8..7,
// exact in bfloat16, in shared memory.  Scales and middles stay out of the operands, as in attention4.cu: a group's part of a score is
// s (q . c) + m sum q in 32 bits; a weight times its value's scale is rounded to half precision (attention4.cuh), for each group of 64
// numbers anew, and the middles' sum goes beside.  The next page is asked for while one is multiplied and formed behind it.  Shares of the
// pages, if rows are few, merge in attention4.cu.
// Measured (B200): a turn of 739 tokens on 7,453, 8 heads over 4 of 256, 312 us, 152 TFLOP/s of the 526 that mma.sync gives at most; the
// kernel of few rows 412.  Bound by latency: the sums of 128 pairs leave registers for 8 warps an SM, which issue in 36% of the clocks; the
// tensor pipe is busy in 33%, shared memory in 19%.  (16 warps, heads of 128, with sums in local memory: 3% faster at most.)
#include "attention4.cuh"

namespace hos {

constexpr int kTileRows = 128;

template <int DIM> struct Tiles4 {
    static constexpr int kGroups = DIM / 64, kRowBytes = DIM * 2;
    static constexpr int kQ = 0, kK = kTileRows * kRowBytes, kV = kK + 2 * 64 * kRowBytes;          // bytes: two pages each
    static constexpr int kMeta = kV + 2 * 64 * kRowBytes, kQSum = kMeta + 2 * 2 * kGroups * 64 * 4, kRaw = kQSum + kTileRows * kGroups * 4;
    static constexpr int kMost = kRaw + 2 * 36 * DIM, kShared = kMost + 3 * 4 * 4;                                             // and a page's codes as they came
    static constexpr int kItems = 128 * kGroups;                                                    // 16-byte pieces of a page's codes
    static constexpr int kEach = (kItems + 255) / 256;
};

template <int DIM>
__global__ void __launch_bounds__(256, DIM == 64 ? 2 : 1)
attend4_tiles_kernel(const bf16* __restrict__ q, long long q_stride, bf16* __restrict__ out, long long out_stride, const int* __restrict__ token_pos,
                     const int* __restrict__ seq_slot, int seq_base, const int* __restrict__ cu_seqlens, int row_base, int n_seqs, int n_tokens, Paged4 c,
                     int n_heads, float scale, float cap, int window, int share, int splits, float* __restrict__ part_o, float2* __restrict__ part_ml) {
    using A = Tiles4<DIM>;
    constexpr int G = A::kGroups;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int per = n_heads / c.n_kv_heads, kvh = blockIdx.y, split = blockIdx.x % splits;
    const RowBlock rows = find_rows(cu_seqlens, row_base, n_seqs, token_pos, n_tokens, blockIdx.x / splits, kTileRows / per, 0);
    if (rows.count <= 0) return;
    const int pairs = rows.count * per;                        // pair j: head kvh * per + j % per of row row0 + j / per
    auto out_at = [&](int j) { return out + (size_t)(rows.row0 + j / per) * out_stride + (size_t)(kvh * per + j % per) * DIM; };
    auto part_at = [&](int j) { return ((size_t)(rows.row0 + j / per) * n_heads + kvh * per + j % per) * splits + split; };
    const int last = rows.pos0 + rows.count - 1, first = window > 0 ? max(0, rows.pos0 - window + 1) : 0;
    const int page0 = first / kPageTokens, page1 = last / kPageTokens + 1, pages = max(share, (page1 - page0 + splits - 1) / splits);
    const int p0 = page0 + split * pages, p1 = rows.seq < 0 ? p0 : min(page1, p0 + pages);
    if (p0 >= p1) {                                            // a share without keys says so; padding rows become zeros
        for (int i = threadIdx.x; i < (splits > 1 ? pairs : pairs * DIM); i += blockDim.x) {
            if (splits > 1) part_ml[part_at(i)] = make_float2(-INFINITY, 0.f);
            else out_at(i / DIM)[i % DIM] = __float2bfloat16_rn(0.f);
        }
        return;
    }
    const int* table = c.page_table + (size_t)seq_slot[seq_base + rows.seq] * c.table_stride;
    auto tile_of = [&](int p) { return ((size_t)table[c.ring_pages > 0 ? p % c.ring_pages : p] * c.n_kv_heads + kvh) * tile4_bytes(DIM); };

    // A page's tiles as they are, on their way: a thread forms what it copied itself.
    const uint32_t raw = smem_u32(smem + A::kRaw);
    auto ask = [&](int p) {
        const size_t tile = tile_of(p);
#pragma unroll
        for (int i = 0; i < A::kEach; ++i) {
            const int item = i * 256 + threadIdx.x;
            if (item < A::kItems) {
                copy16_async(raw + item * 16, c.k_pages + tile + item * 16);
                copy16_async(raw + 36 * DIM + item * 16, c.v_pages + tile + item * 16);
            }
        }
        if (threadIdx.x < 32 * G) {                            // scales and middles: 16 G pieces of each tile
            const int v = threadIdx.x / (16 * G), at = tile4_codes(DIM) + threadIdx.x % (16 * G) * 16;
            copy16_async(raw + v * 36 * DIM + at, (v ? c.v_pages : c.k_pages) + tile + at);
        }
        copies_commit();
    };
    int* most = (int*)(smem + A::kMost);                       // [3][4]: a group's largest scale of the values of page p, at p % 3
    auto form = [&](int p, int buffer) {
        copies_wait<0>();
#pragma unroll
        for (int i = 0; i < A::kEach; ++i) {
            const int item = i * 256 + threadIdx.x;
            if (item >= A::kItems) break;
            const uint4 kv = lds16(raw + item * 16), vv = lds16(raw + 36 * DIM + item * 16);
            const int l = item & 31, block = item >> 5, grp = block % G, row16 = block / G * 16, lg = l >> 2, lt = l & 3;
            const uint32_t kw[4] = {kv.x, kv.y, kv.z, kv.w}, vw[4] = {vv.x, vv.y, vv.z, vv.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {                      // keys [position][number]: eight neighbouring numbers to a word
                uint32_t r[4];
                codes_to_bf16<true>(kw[w], kZero8, r);
                const int key = row16 + lg + 8 * (w >> 1), chunk = 8 * grp + 2 * lt + (w & 1);
                *(uint4*)(smem + A::kK + buffer * 64 * A::kRowBytes + key * A::kRowBytes + ((chunk ^ (key & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {                      // values [number][position]: two neighbouring positions to a register
                uint32_t r[4];
                codes_to_half(vw[w], r);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = grp * 64 + w * 16 + lg + 8 * (e & 1), chunk = (row16 >> 3) + (e >> 1);
                    *(uint32_t*)(smem + A::kV + buffer * 64 * A::kRowBytes + d * 128 + ((chunk ^ (d & 7)) << 4) + lt * 4) = r[e];
                }
            }
        }
        if (threadIdx.x < 32 * G) {
            uint32_t* meta = (uint32_t*)(smem + A::kMeta) + buffer * 2 * G * 64;      // [keys, values][G][64]
            const int v = threadIdx.x / (16 * G), piece = threadIdx.x % (16 * G);
            const uint4 m = lds16(raw + v * 36 * DIM + tile4_codes(DIM) + piece * 16);
            const uint32_t w[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int grp = (4 * piece + e) % G, row = (4 * piece + e) / G, key = p * kPageTokens + row;
                // a key that no row here sees may be anything: it becomes zeros
                const uint32_t m = key <= last && (window == 0 || key > rows.pos0 - window) ? w[e] : 0u;
                meta[(v * G + grp) * 64 + row] = m;
                if (v == 1 && bf16_lo(m) < INFINITY) atomicMax(&most[p % 3 * 4 + grp], __float_as_int(bf16_lo(m)));      // scales are not negative
            }
        }
    };
    if (threadIdx.x < 12) most[threadIdx.x] = 0;
    __syncthreads();
    ask(p0);
    // the pairs' numbers, and their sums over 64
    for (int i = threadIdx.x; i < kTileRows * DIM / 8; i += 256) {
        const int j = i / (DIM / 8), chunk = i % (DIM / 8);
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (j < pairs) v = *(const uint4*)(q + (size_t)(rows.row0 + j / per) * q_stride + (size_t)(kvh * per + j % per) * DIM + chunk * 8);
        *(uint4*)(smem + A::kQ + j * A::kRowBytes + ((chunk ^ (j & 7)) << 4)) = v;
        float s = 0.f;
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) s += bf16_lo(u[e]) + bf16_hi(u[e]);
        s += __shfl_xor_sync(0xffffffffu, s, 1);               // eight neighbouring threads hold 64 numbers
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        if ((i & 7) == 0) ((float*)(smem + A::kQSum))[j * G + chunk / 8] = s;
    }
    form(p0, 0);
    __syncthreads();

    const int row_a = warp * 16 + g, row_b = row_a + 8;        // a lane's two pairs
    const int pos[2] = {rows.pos0 + min(row_a, pairs - 1) / per, rows.pos0 + min(row_b, pairs - 1) / per};
    const int warp_first = rows.pos0 + min(warp * 16, pairs - 1) / per, warp_last = rows.pos0 + min(warp * 16 + 15, pairs - 1) / per;
    const bool busy = warp * 16 < pairs;
    float o[DIM / 8][4], mid[G][2], best[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, into[G];
#pragma unroll
    for (int i = 0; i < G; ++i) into[i] = kIntoFirst;
#pragma unroll
    for (int i = 0; i < DIM / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        mid[i][0] = mid[i][1] = 0.f;
    }
    const float scale2 = scale * 1.44269504f, cap2 = cap * 1.44269504f, in_cap = cap > 0.f ? 2.f * scale2 / cap : 0.f;
    // where a lane's row of an ldmatrix of four begins in a group's 128 bytes, swapped as the rows are
    uint32_t q_at[4], k_at[2];
#pragma unroll
    for (int st = 0; st < 4; ++st)
        q_at[st] = smem_u32(smem + A::kQ) + (warp * 16 + (lane & 15)) * A::kRowBytes + (((2 * st + (lane >> 4)) ^ (lane & 7)) << 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) k_at[h] = ((4 * h + (lane >> 3)) ^ (lane & 7)) << 4;
    const uint32_t k_rows = smem_u32(smem + A::kK) + (lane & 7) * A::kRowBytes, v_rows = smem_u32(smem + A::kV) + (lane & 7) * 128;

    for (int p = p0; p < p1; ++p) {
        const int buffer = (p - p0) & 1;
        if (p + 1 < p1) ask(p + 1);
        if (threadIdx.x < G) most[(p + 2) % 3 * 4 + threadIdx.x] = 0;          // read before the last barrier, raised behind the next
        // what lies wholly behind a warp's rows, or before their windows, is not walked over
        if (busy && p * kPageTokens <= warp_last && !(window > 0 && p * kPageTokens + 63 <= warp_first - window)) {
            const uint32_t page_at = buffer * 64 * A::kRowBytes, k0 = k_rows + page_at + k_at[0], k1 = k_rows + page_at + k_at[1];
            const uint32_t v0 = v_rows + page_at + k_at[0], v1 = v_rows + page_at + k_at[1];
            const uint32_t* km = (const uint32_t*)(smem + A::kMeta) + buffer * 2 * G * 64;
            const uint32_t* vm = km + G * 64;
            float s[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                uint32_t a[4][4];
                const float q_sum[2] = {((const float*)(smem + A::kQSum))[row_a * G + grp], ((const float*)(smem + A::kQSum))[row_b * G + grp]};
#pragma unroll
                for (int st = 0; st < 4; ++st) ldmatrix_x4(a[st], q_at[st] + grp * 128);
#pragma unroll
                for (int n0 = 0; n0 < 8; n0 += 4) {            // four products side by side: one alone would wait for its own sums
                    float part[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t b[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) ldmatrix_x4(b[i], (h ? k1 : k0) + (n0 + i) * 8 * A::kRowBytes + grp * 128);
#pragma unroll
                        for (int st = 0; st < 2; ++st)
#pragma unroll
                            for (int i = 0; i < 4; ++i) mma_bf16(part[i], a[2 * h + st], b[i][2 * st], b[i][2 * st + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 sm = *(const uint2*)&km[grp * 64 + (n0 + i) * 8 + 2 * t4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t w = (e & 1) ? sm.y : sm.x;
                            s[n0 + i][e] = fmaf(bf16_lo(w), part[i][e], fmaf(bf16_hi(w), q_sum[e >> 1], s[n0 + i][e]));
                        }
                    }
                }
            }
            // scores in units of log 2; what some pair does not see may be anything
            const int base = p * kPageTokens;
            const bool edge = base + 63 > rows.pos0 || (window > 0 && base <= last - window);
            uint32_t hidden = 0u;
            float top[2] = {-INFINITY, -INFINITY};
            if (cap > 0.f) {
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = fmaf(-2.f * cap2, rcp_approx(1.f + ex2_approx(s[n][e] * in_cap)), cap2);
            } else {
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] *= scale2;
            }
            if (edge) {
#pragma unroll
                for (int n = 0; n < 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = base + n * 8 + 2 * t4 + (e & 1), mine = pos[e >> 1];
                        if (key > mine || (window > 0 && key <= mine - window)) {
                            s[n][e] = -INFINITY;
                            hidden |= 1u << (n * 4 + e);
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
            if (__any_sync(0xffffffffu, top[0] > best[0] + 8.f || top[1] > best[1] + 8.f)) {
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                    top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                    const float m = fmaxf(best[h], top[h]);
                    f[h] = best[h] == m ? 1.f : ex2_approx(best[h] - m);
                    best[h] = m;
                    sum[h] *= f[h];
#pragma unroll
                    for (int i = 0; i < G; ++i) mid[i][h] *= f[h];
                }
#pragma unroll
                for (int i = 0; i < DIM / 8; ++i) {
                    o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1];
                }
            }
            const float from[2] = {best[0] == -INFINITY ? 0.f : best[0], best[1] == -INFINITY ? 0.f : best[1]};      // no key seen yet: all weights 0
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = ex2_approx(s[n][e] - from[e >> 1]);
                    sum[e >> 1] += s[n][e];
                }
#pragma unroll
            for (int grp = 0; grp < G; ++grp) {
                const float largest = __int_as_float(most[p % 3 * 4 + grp]);
                if (largest * into[grp] > kIntoMost) {
                    const float now = into_of(largest), f = now * back_of(into[grp]);
                    into[grp] = now;
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        o[grp * 8 + d][0] *= f; o[grp * 8 + d][1] *= f; o[grp * 8 + d][2] *= f; o[grp * 8 + d][3] *= f;
                    }
                }
                uint32_t a[4][4];
                if (!edge) {
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint2 sm = *(const uint2*)&vm[grp * 64 + n * 8 + 2 * t4];
                        const float sv[2] = {bf16_lo(sm.x) * into[grp], bf16_lo(sm.y) * into[grp]}, mv[2] = {bf16_hi(sm.x), bf16_hi(sm.y)};
                        a[n >> 1][2 * (n & 1)] = pack_half(s[n][0] * sv[0], s[n][1] * sv[1]);
                        a[n >> 1][2 * (n & 1) + 1] = pack_half(s[n][2] * sv[0], s[n][3] * sv[1]);
                        mid[grp][0] = fmaf(s[n][1], mv[1], fmaf(s[n][0], mv[0], mid[grp][0]));
                        mid[grp][1] = fmaf(s[n][3], mv[1], fmaf(s[n][2], mv[0], mid[grp][1]));
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const uint2 sm = *(const uint2*)&vm[grp * 64 + n * 8 + 2 * t4];
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t m = (e & 1) ? sm.y : sm.x;
                            const bool seen = !((hidden >> (n * 4 + e)) & 1u);
                            w[e] = seen ? s[n][e] * (bf16_lo(m) * into[grp]) : 0.f;
                            if (seen) mid[grp][e >> 1] = fmaf(s[n][e], bf16_hi(m), mid[grp][e >> 1]);
                        }
                        a[n >> 1][2 * (n & 1)] = pack_half(w[0], w[1]);
                        a[n >> 1][2 * (n & 1) + 1] = pack_half(w[2], w[3]);
                    }
                }
#pragma unroll
                for (int d0 = 0; d0 < 8; d0 += 4)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t b[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) ldmatrix_x4(b[i], (h ? v1 : v0) + (grp * 64 + (d0 + i) * 8) * 128);
#pragma unroll
                        for (int st = 0; st < 2; ++st)
#pragma unroll
                            for (int i = 0; i < 4; ++i) mma_half(o[grp * 8 + d0 + i], a[2 * h + st], b[i][2 * st], b[i][2 * st + 1]);
                    }
            }
        }
        if (p + 1 < p1) {
            form(p + 1, buffer ^ 1);                            // nobody reads that one: the walk over it ended before the last barrier
            __syncthreads();
        }
    }
#pragma unroll
    for (int i = 0; i < DIM / 8; ++i) {
        const float back = back_of(into[i / 8]);                  // a power of two
        o[i][0] *= back; o[i][1] *= back; o[i][2] *= back; o[i][3] *= back;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], off);
#pragma unroll
            for (int i = 0; i < G; ++i) mid[i][h] += __shfl_xor_sync(0xffffffffu, mid[i][h], off);
        }
        const int j = h == 0 ? row_a : row_b;
        if (j >= pairs) continue;
        if (splits > 1) {
            const size_t at = part_at(j);
            if (t4 == 0) part_ml[at] = make_float2(best[h], sum[h]);
            float* to = part_o + at * DIM + 2 * t4;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) *(float2*)(to + i * 8) = make_float2(o[i][2 * h] + mid[i / 8][h], o[i][2 * h + 1] + mid[i / 8][h]);
        } else {
            const float f = 1.f / sum[h];
            bf16* to = out_at(j) + 2 * t4;
#pragma unroll
            for (int i = 0; i < DIM / 8; ++i) *(uint32_t*)(to + i * 8) = pack_bf16((o[i][2 * h] + mid[i / 8][h]) * f, (o[i][2 * h + 1] + mid[i / 8][h]) * f);
        }
    }
}

template <int DIM>
int launch_attend4_tiles(const void* q, long long q_stride, void* out, long long out_stride, const int* token_pos, const int* seq_slot, int seq_base,
                         const int* cu_seqlens, int row_base, int n_seqs, const Paged4& c, int n_tokens, int n_heads, float scale, float cap, int window, int share,
                         int splits, float* part_o, float2* part_ml, cudaStream_t stream) {
    auto kernel = attend4_tiles_kernel<DIM>;
    static bool set = false;                                   // once per kernel: the attribute stays
    if (!set) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Tiles4<DIM>::kShared) != cudaSuccess) return check_launch("attend4_tiles");
        set = true;
    }
    const int size = kTileRows / (n_heads / c.n_kv_heads);
    const long long blocks = (n_tokens + size - 1) / size + n_seqs;      // a sequence's last may not be full
    launch_pdl(kernel, dim3((unsigned)(blocks * splits), (unsigned)c.n_kv_heads), dim3(256), Tiles4<DIM>::kShared, stream, (const bf16*)q, q_stride, (bf16*)out,
               out_stride, token_pos, seq_slot, seq_base, cu_seqlens, row_base, n_seqs, n_tokens, c, n_heads, scale, cap, window, share, splits, part_o, part_ml);
    return check_launch("attend4_tiles");
}

}  // namespace hos

using namespace hos;

// As hos_attend4 for bfloat16 rows that come by the sequence (cu_seqlens less row_base, their entries of seq_slot from seq_base on), rows of q
// and out on 16 bytes, heads of 64, 128, 192 or 256.  `parts` as there; the merge is a call of its own.
extern "C" int hos_attend4_tiles(const void* q, long long q_stride, void* out, long long out_stride, const int* token_pos, const int* seq_slot, int seq_base,
                                 const int* cu_seqlens, int row_base, int n_seqs, const void* cache, int n_tokens, int n_heads, float scale, float cap, int window,
                                 int share, int splits, float* parts, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    HOS_CHECK_PAGED4("attend4_tiles");
    if (n_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > kTileRows)
        HOS_REFUSE("attend4_tiles: %d query heads over %d kv heads", n_heads, n_kv_heads);
    if (q_stride % 8 || out_stride % 8 || (uintptr_t)q % 16 || (uintptr_t)out % 16) HOS_REFUSE("attend4_tiles: rows must begin on 16 bytes");
    if (share < 1 || splits < 1 || splits > kMaxShares || (splits > 1 && parts == nullptr)) HOS_REFUSE("attend4_tiles: %d shares of %d pages", splits, share);
    if (n_kv_heads > 65535 || ((long long)n_tokens + n_seqs) * splits > 0x7fffffffll) HOS_REFUSE("attend4_tiles: %d rows, %d kv heads", n_tokens, n_kv_heads);
    const size_t n_parts = (size_t)n_tokens * n_heads * splits;
    float2* part_ml = (float2*)parts;
    float* part_o = parts == nullptr ? nullptr : parts + 2 * n_parts;
#define HOS_AT(D)                                                                                                                                \
    return launch_attend4_tiles<D>(q, q_stride, out, out_stride, token_pos, seq_slot, seq_base, cu_seqlens, row_base, n_seqs, c, n_tokens, n_heads, \
                                   scale, cap, window, share, splits, part_o, part_ml, stream)
    if (head_dim == 64) HOS_AT(64);
    if (head_dim == 128) HOS_AT(128);
    if (head_dim == 192) HOS_AT(192);
    HOS_AT(256);
}
