// Attention of sequences that share pages (forks of a prompt): a shared page is read once for all of them.
//
// The work is a list of items made on the host (parts/shared_attention.py).  An item is a block of rows of the step, a row of the page
// table through which all of them read, and a range of that table's logical pages: the pages that the block's sequences share, or
// the pages that a sequence has for itself (its range without the shared part).  A block's (row, query head) pairs of one kv head, up
// to 16, are the columns of the products S^T = K Q^T and O^T = V^T P^T (m16n8k16, bfloat16, sums in 32 bits), so a page's keys and
// values are read from shared memory once for all pairs.  Masks are a pair's own: keys up to its row's position, the last `window` of
// them; pages outside what any of the rows sees are left out, by the positions on the device, so a list stays right while rows move on.
// Every item leaves unnormalised sums with their maximum and sum of weights, a part of each of its rows; attn_shared_merge_kernel joins a
// row's parts:  m = max m_i,  out = sum e^(m_i - m) o_i / sum e^(m_i - m) l_i.
//
// The walk is persistent, a CTA an SM: a producer warp brings pages by bulk copies through a ring, over the borders of items, four
// consumer warps take 16 keys of a page each.  Weights are rounded to bfloat16 for the product with the values (2^-8 of each at most), their sum
// is of the weights before that rounding.
//
// Compiled per head size: -DHOS_HEAD_DIM=N, a multiple of 16 up to 256.
#include "common.cuh"
#include "kv_layout.cuh"
#include "mma_utils.cuh"
#include "tcgen05_one.cuh"

#ifndef HOS_HEAD_DIM
#define HOS_HEAD_DIM 64
#endif

namespace hos {

constexpr int HD = HOS_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head_dim must be a multiple of 16, at most 256");
constexpr int kGiveUpAttnShared = 7;
constexpr int kPairs = 16;                                   // pairs of an item
constexpr int kTileBytes = kPageTokens * HD * 2;             // a page's keys of a kv head, or its values
constexpr int kConsumers = 128;
constexpr int kThreads = kConsumers + 32;
constexpr long long kWaitCycles = 1ll << 31;                 // about a second
constexpr int kSumsBytes = 4 * kPairs * (HD + 4) * 4;       // the four warps' sums (rows of HD + 4 numbers: no conflicts)
constexpr int kStagesFit = (225 * 1024 - kPairs * HD * 2 - kSumsBytes) / (2 * kTileBytes);
constexpr int kStages = kStagesFit < 6 ? kStagesFit : 6;

struct SharedItem {                                          // as parts/shared_attention.py writes it
    int row0, n_rows;          // places in the list of rows
    int slot;                  // row of the page table
    int lp0, lp1;              // logical pages, lp1 exclusive ...
    int skip0, skip1;          // ... without these
    int share, n_shares;       // which of so many shares of what is left of them
    int part;                  // which part of its rows the item leaves
    int pad0, pad1;
};

struct SharedArgs {
    const bf16* q;
    int q_stride;
    const int* token_pos;
    const SharedItem* items;
    const int* n_items;        // on the device
    const int* rows;
    PagedKV cache;
    int n_heads, parts;        // parts: places of a (row, head) in the workspace
    float* part_o;             // [rows][heads][parts][HD]
    float2* part_ml;           // [rows][heads][parts] (maximum, sum of weights)
    float scale, cap;
    int window;
};

__device__ int* g_shared_error_host = nullptr;

__device__ __forceinline__ void record_give_up() {
    int* w = g_shared_error_host;
    if (w != nullptr) {
        atomicExch_system(w, kGiveUpAttnShared);
        __threadfence_system();
    }
}

// The pages of an item, by the positions of its rows: every warp for itself.
struct Walk {
    int first, count1, second, n;          // logical pages first .. first + count1 - 1, then second ..
    int begin, end;                        // the share's part of them
    int all_from, all_to;                  // the keys that every row sees
};
__device__ __forceinline__ Walk walk_of(const SharedArgs& a, const SharedItem& it, int lane) {
    int low = 0x7fffffff, high = -1;       // the lowest and the highest position of a row
    for (int r = lane; r < it.n_rows; r += 32) {
        const int pos = a.token_pos[a.rows[it.row0 + r]];
        low = min(low, pos);
        high = max(high, pos);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    const int from = max(it.lp0, a.window > 0 ? max(0, low + 1 - a.window) / kPageTokens : 0), to = min(it.lp1, high / kPageTokens + 1);
    Walk w;
    w.all_from = a.window > 0 ? max(0, high + 1 - a.window) : 0;
    w.all_to = low;
    w.first = from;
    w.count1 = max(0, min(to, it.skip0) - from);
    w.second = max(from, it.skip1);
    w.n = w.count1 + max(0, to - w.second);
    const int per = (w.n + it.n_shares - 1) / it.n_shares;
    w.begin = min(w.n, it.share * per);
    w.end = min(w.n, w.begin + per);
    return w;
}
__device__ __forceinline__ int walk_page(const Walk& w, int i) { return i < w.count1 ? w.first + i : w.second + (i - w.count1); }

struct SharedSmem {
    static constexpr int kRing = kStages * 2 * kTileBytes;
    static constexpr int kQ = kPairs * HD * 2;
    static constexpr int kTotal = kRing + kQ + kSumsBytes + 4 * kPairs * 8 + kPairs * 16 + 4 * kStages * 8;
};

__global__ void __launch_bounds__(kThreads, 1) attn_shared_kernel(SharedArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* ring = smem;                                                 // stage: keys, values
    bf16* q_s = reinterpret_cast<bf16*>(smem + SharedSmem::kRing);              // [16][HD], permuted like the pages
    float* sums = reinterpret_cast<float*>(smem + SharedSmem::kRing + SharedSmem::kQ);        // [4][16][HD + 4]
    float2* ml = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(sums) + kSumsBytes);      // [4][16]
    int4* pair_of = reinterpret_cast<int4*>(ml + 4 * kPairs);                   // [16]: row, head, lowest key, position
    uint64_t* k_full = reinterpret_cast<uint64_t*>(pair_of + kPairs);
    uint64_t* v_full = k_full + kStages;
    uint64_t* k_empty = v_full + kStages;
    uint64_t* v_empty = k_empty + kStages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int group = a.n_heads / a.cache.n_kv_heads;
    const int chunks = (group + kPairs - 1) / kPairs;        // sixteens of query heads that share a kv head
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&k_full[s], 1); mbar_init(&v_full[s], 1);
            mbar_init(&k_empty[s], 4); mbar_init(&v_empty[s], 4);
        }
        mbar_fence_init();
    }
    __syncthreads();
    pdl_enter();
    const int per_item = a.cache.n_kv_heads * chunks;
    const int n_work = *a.n_items * per_item;

    if (warp == 4) {
        // ---------------- producer ----------------
        const bf16* k_pages = reinterpret_cast<const bf16*>(a.cache.k_pages);
        const bf16* v_pages = reinterpret_cast<const bf16*>(a.cache.v_pages);
        int t = 0;
        bool ok = true;
        for (int work = blockIdx.x; work < n_work && ok; work += gridDim.x) {
            const SharedItem it = a.items[work / per_item];
            const int kvh = work % per_item / chunks;
            const Walk w = walk_of(a, it, lane);
            const int* table = a.cache.page_table + (size_t)it.slot * a.cache.table_stride;
            for (int i0 = w.begin; i0 < w.end && ok; i0 += 32) {             // 32 pages looked up at a time
                const int page_l = i0 + lane < w.end ? table[kv_table_entry(a.cache, walk_page(w, i0 + lane))] : 0;
                const int n = min(32, w.end - i0);
                for (int i = 0; i < n; ++i, ++t) {
                    const int page = __shfl_sync(0xffffffffu, page_l, i);
                    if (lane == 0) {
                        const int s = t % kStages;
                        const size_t off = kv_tile_offset(a.cache, page, kvh);
                        unsigned char* dst = ring + (size_t)s * 2 * kTileBytes;
                        if (t >= kStages) ok = mbar_wait_cycles(&k_empty[s], ((t / kStages) - 1) & 1, kWaitCycles);
                        if (ok) {
                            mbar_expect_tx(&k_full[s], kTileBytes);
                            bulk_g2s(dst, k_pages + off, kTileBytes, &k_full[s]);
                            if (t >= kStages) ok = mbar_wait_cycles(&v_empty[s], ((t / kStages) - 1) & 1, kWaitCycles);
                        }
                        if (ok) {
                            mbar_expect_tx(&v_full[s], kTileBytes);
                            bulk_g2s(dst + kTileBytes, v_pages + off, kTileBytes, &v_full[s]);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
                    if (!ok) break;
                }
            }
        }
        if (!ok) {
            if (lane == 0) record_give_up();
            let_work_under_way_end();
        }
        return;
    }

    // ---------------- consumers ----------------
    const int g = lane >> 2, t4 = lane & 3;
    const float inv_cap = a.cap > 0.f ? 1.f / a.cap : 0.f;
    const uint32_t q_base = smem_u32(q_s);
    const int upper = (lane >> 3) & 1, right = lane >> 4;
    const int k_row = warp * 16 + (lane & 7) + upper * 8, v_row = warp * 16 + (lane & 7) + right * 8;
    const int q_row = (lane & 7) + right * 8;
    int t = 0;
    bool ok = true;
    auto meet = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    for (int work = blockIdx.x; work < n_work; work += gridDim.x) {
        const SharedItem it = a.items[work / per_item];
        const int kvh = work % per_item / chunks, chunk = work % per_item % chunks;
        const int heads = min(kPairs, group - chunk * kPairs);           // of a row
        const int pairs = min(kPairs, it.n_rows * heads);
        const Walk w = walk_of(a, it, lane);
        meet();                                              // the last item's readers are done
        if (tid < kPairs) {
            const int row = a.rows[it.row0 + min(tid / heads, it.n_rows - 1)];
            const int pos = tid < pairs ? a.token_pos[row] : -1;
            pair_of[tid] = make_int4(row, kvh * group + chunk * kPairs + tid % heads, a.window > 0 ? max(0, pos + 1 - a.window) : 0, pos);
        }
        meet();
        for (int i = tid; i < kPairs * (HD / 8); i += kConsumers) {
            const int p = i / (HD / 8), c = i % (HD / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (p < pairs) v = *reinterpret_cast<const uint4*>(a.q + (size_t)pair_of[p].x * a.q_stride + (size_t)pair_of[p].y * HD + c * 8);
            *reinterpret_cast<uint4*>(q_s + tile_chunk_offset<HD>(p, c)) = v;
        }
        meet();
        const bool two = pairs > 8;                          // columns 8 to 15 are in use
        int lo[2][2], hi[2][2];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int4 p = pair_of[8 * x + 2 * t4 + r];
                lo[x][r] = p.z;
                hi[x][r] = p.w;
            }
        float m_run[2][2] = {{-INFINITY, -INFINITY}, {-INFINITY, -INFINITY}}, l_run[2][2] = {};
        float o[HD / 16][2][4] = {};

        for (int i = w.begin; i < w.end; ++i, ++t) {
            const int s = t % kStages;
            const uint32_t parity = (t / kStages) & 1;
            const uint32_t k_base = smem_u32(ring + (size_t)s * 2 * kTileBytes), v_base = k_base + kTileBytes;
            if (ok) ok = mbar_wait_cycles(&k_full[s], parity, kWaitCycles);
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (!ok) continue;
            float sc[2][4] = {}, sd[2][4] = {};              // two sums of every score, so that a chain is half as long
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
                uint32_t kb[4], qb[4];
                ldmatrix_x4(kb, k_base + 2 * tile_chunk_offset<HD>(k_row, kk * 2 + right));
                ldmatrix_x4(qb, q_base + 2 * tile_chunk_offset<HD>(q_row, kk * 2 + upper));
                auto& to = kk & 1 ? sd : sc;
                mma_bf16(to[0], kb, qb[0], qb[1]);
                if (two) mma_bf16(to[1], kb, qb[2], qb[3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_empty[s]);
            const int key0 = walk_page(w, i) * kPageTokens + warp * 16;
            uint32_t pb[2][2];
            float corr[2][2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (x == 1 && !two) break;
                float m_new[2] = {m_run[x][0], m_run[x][1]};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + g + 8 * (j >> 1), r = j & 1;
                    float v = softcap_fast((sc[x][j] + sd[x][j]) * a.scale, a.cap, inv_cap);
                    v = key >= lo[x][r] && key <= hi[x][r] ? v : -INFINITY;
                    sc[x][j] = v;
                    m_new[r] = fmaxf(m_new[r], v);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int y = 4; y < 32; y <<= 1) m_new[r] = fmaxf(m_new[r], __shfl_xor_sync(0xffffffffu, m_new[r], y));
                    const float use = m_new[r] == -INFINITY ? 0.f : m_new[r];
                    corr[x][r] = __expf(m_run[x][r] - use);
                    m_run[x][r] = m_new[r];
                    l_run[x][r] *= corr[x][r];
#pragma unroll
                    for (int j = r; j < 4; j += 2) {
                        sc[x][j] = __expf(sc[x][j] - use);
                        l_run[x][r] += sc[x][j];
                    }
                }
                pb[x][0] = transposed_8x8(pack_bf16(sc[x][0], sc[x][1]));
                pb[x][1] = transposed_8x8(pack_bf16(sc[x][2], sc[x][3]));
            }
            if (ok) ok = mbar_wait_cycles(&v_full[s], parity, kWaitCycles);
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (!ok) continue;
#pragma unroll
            for (int dd = 0; dd < HD / 16; ++dd) {
                uint32_t va[4];
                ldmatrix_x4_trans(va, v_base + 2 * tile_chunk_offset<HD>(v_row, dd * 2 + upper));
#pragma unroll
                for (int j = 0; j < 4; ++j) o[dd][0][j] *= corr[0][j & 1];
                mma_bf16(o[dd][0], va, pb[0][0], pb[0][1]);
                if (two) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[dd][1][j] *= corr[1][j & 1];
                    mma_bf16(o[dd][1], va, pb[1][0], pb[1][1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_empty[s]);
        }

        // ---- the four warps' sums, each of other keys, are added and leave ----
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int y = 4; y < 32; y <<= 1) l_run[x][r] += __shfl_xor_sync(0xffffffffu, l_run[x][r], y);
                const int p = 8 * x + 2 * t4 + r;
                if (p < pairs) {
                    float* b = sums + (size_t)(warp * kPairs + p) * (HD + 4);
#pragma unroll
                    for (int dd = 0; dd < HD / 16; ++dd) {
                        b[dd * 16 + g] = o[dd][x][r];
                        b[dd * 16 + g + 8] = o[dd][x][2 + r];
                    }
                    if (g == 0) ml[warp * kPairs + p] = make_float2(m_run[x][r], l_run[x][r]);
                }
            }
        meet();
        for (int i = tid; i < pairs * (HD / 4); i += kConsumers) {
            const int p = i / (HD / 4), d = i % (HD / 4) * 4;
            float m = -INFINITY;
#pragma unroll
            for (int y = 0; y < 4; ++y) m = fmaxf(m, ml[y * kPairs + p].x);
            float l = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float2 v = ml[y * kPairs + p];
                const float f = v.x == -INFINITY ? 0.f : __expf(v.x - m);
                const float4 b = *reinterpret_cast<const float4*>(sums + (size_t)(y * kPairs + p) * (HD + 4) + d);
                l += v.y * f;
                acc.x += b.x * f; acc.y += b.y * f; acc.z += b.z * f; acc.w += b.w * f;
            }
            const size_t at = ((size_t)pair_of[p].x * a.n_heads + pair_of[p].y) * a.parts + it.part;
            *reinterpret_cast<float4*>(a.part_o + at * HD + d) = acc;
            if (d == 0) a.part_ml[at] = make_float2(m, l);
        }
    }
    if (!ok && lane == 0) record_give_up();
}

#if (HOS_HEAD_DIM == 64) || (HOS_HEAD_DIM == 128) || (HOS_HEAD_DIM == 256)
// ---- blocks of up to 128 pairs, on tcgen05 -------------------------------------------------------------
// With more than 16 pairs the products above cost more than a page's bytes.  Here the pairs are the 128 rows of the tensor core's
// operand: S = Q K^T (M 128, N 64, two buffers in tensor memory), the softmax by two threads a row, O += P V with O in tensor memory.  A
// page's 16-byte pieces lie in the cache where the 128-byte swizzle wants them, so TMA boxes of [64 rows x 64 columns] are operands
// as they land.  A CTA takes one item and kv head.  Warps: 0 pages, 1 products, 2 to 9 queries, softmax and sums.  The maximum is raised only
// when a tile's exceeds it by 8 (weights up to e^8 do no harm in 32-bit sums and bfloat16 weights).
constexpr int kBlock = 128;
constexpr int kColumns = HD / 64;                            // blocks of 64 numbers of a head
constexpr int kQBlockBytes = kBlock * 128, kTileBlockBytes = kPageTokens * 128, kPBytes = kBlock * 128;
constexpr int kTcStagesFit = (227 * 1024 - kColumns * kQBlockBytes - 2 * kPBytes - 2 * kBlock * 4 - 1024 - 256) / (2 * kTileBytes);
constexpr int kTcStages = kTcStagesFit < 6 ? kTcStagesFit : 6;
constexpr int kTcBarriers = 1 + 4 * kTcStages + 8;
constexpr int kTcShared = kColumns * kQBlockBytes + kTcStages * 2 * kTileBytes + 2 * kPBytes + 2 * kBlock * 4 + kTcBarriers * 8 + 16 + 1008;
static_assert(kTcStages >= 2 && kTcShared <= 227 * 1024, "shared memory of the kernel on tcgen05");
constexpr int kTcThreads = 320;
constexpr int kColS = 0, kColO = 128, kTmemCols = 128 + HD <= 256 ? 256 : 512;
constexpr float kRescaleSlack = 8.f;

// tanh: for |x| <= 0.55 x + x^3 (a + x^2 (b + x^2 c)), relative error 1.3e-6; if any of a warp's scores is larger, 1 - 2 / (1 + e^2x)
// for all of them, absolute error 2e-7.
__device__ __forceinline__ void tanh_scores(float (&t)[32], float pre) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        t[i] *= pre;
        big = fmaxf(big, fabsf(t[i]));
    }
    if (__any_sync(0xffffffffu, !(big <= 0.55f))) {
#pragma unroll
        for (int i = 0; i < 32; ++i) t[i] = fmaf(-2.f, rcp_approx(1.f + ex2_approx(2.88539008f * t[i])), 1.f);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float x = t[i], x2 = x * x;
            t[i] = fmaf(fmaf(fmaf(-0.043099623f, x2, 0.13152355f), x2, -0.33324513f) * x2, x, x);
        }
    }
}
// 2^x = 2^n p(f), n = round(x), f = x - n, p of degree 3, relative error 7.5e-5 (the weights are rounded to 2^-8): on the multiply-add
// pipe, for a quarter of the scores, as the special-function unit takes 16 a clock and an SM
__device__ __forceinline__ float exp2_poly(float x) {
    x = fmaxf(x, -125.f);
    const float xr = x + 12582912.f;
    const float f = x - (xr - 12582912.f);
    float p = fmaf(0.055171646f, f, 0.24261113f);
    p = fmaf(p, f, 0.69326097f);
    p = fmaf(p, f, 0.99992806f);
    return __int_as_float(__float_as_int(p) + (__float_as_int(xr) << 23));
}

__global__ void __launch_bounds__(kTcThreads, 1)
attn_shared_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, SharedArgs a) {
    extern __shared__ unsigned char smem_unaligned[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = smem;
    unsigned char* ring = q_s + kColumns * kQBlockBytes;         // stage: keys, values
    unsigned char* p_s = ring + kTcStages * 2 * kTileBytes;
    float* xchg = reinterpret_cast<float*>(p_s + 2 * kPBytes);   // [2 halves][128 rows]
    uint64_t* bars = reinterpret_cast<uint64_t*>(xchg + 2 * kBlock);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;
    uint64_t* k_empty = k_full + kTcStages;
    uint64_t* v_full = k_empty + kTcStages;
    uint64_t* v_empty = v_full + kTcStages;
    uint64_t* s_full = v_empty + kTcStages;                      // [2]
    uint64_t* s_empty = s_full + 2;
    uint64_t* p_full = s_full + 4;
    uint64_t* pv_done = s_full + 6;
    uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(s_full + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_heads = a.cache.n_kv_heads, kvh = blockIdx.x % kv_heads;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
        mbar_init(q_full, 8);
        for (int s = 0; s < kTcStages; ++s) {
            mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1); mbar_init(&s_empty[s], 8);
            mbar_init(&p_full[s], 8); mbar_init(&pv_done[s], 1);
        }
        mbar_fence_init();
    }
    pdl_enter();
    if (blockIdx.x / kv_heads >= *a.n_items) return;             // (the whole block)
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_smem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const SharedItem it = a.items[blockIdx.x / kv_heads];
    const Walk w = walk_of(a, it, lane);
    const int n_tiles = w.end - w.begin;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_base_smem;
    bool ok = true;                        // false: a wait of this thread (in the softmax warps: of its warp) ran out
    auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_cycles(bar, parity, kWaitCycles); };

    if (warp == 0) {
        // ---------------- pages ----------------
        const int* table = a.cache.page_table + (size_t)it.slot * a.cache.table_stride;
        for (int i0 = 0; i0 < n_tiles && ok; i0 += 32) {         // 32 pages looked up at a time
            const int page_l = i0 + lane < n_tiles ? table[kv_table_entry(a.cache, walk_page(w, w.begin + i0 + lane))] : 0;
            const int n = min(32, n_tiles - i0);
            for (int i = 0; i < n && ok; ++i) {
                const int page = __shfl_sync(0xffffffffu, page_l, i);
                if (lane == 0) {
                    const int j = i0 + i, s = j % kTcStages, row = (page * kv_heads + kvh) * kPageTokens;
                    const uint32_t parity = ((j / kTcStages) - 1) & 1;
                    unsigned char* kd = ring + (size_t)s * 2 * kTileBytes;
                    if (j >= kTcStages) ok = wait(&k_empty[s], parity);
                    if (ok) {
                        mbar_expect_tx(&k_full[s], kTileBytes);
#pragma unroll
                        for (int c = 0; c < kColumns; ++c) tc_tma_2d(kd + c * kTileBlockBytes, &map_k, 64 * c, row, &k_full[s]);
                        if (j >= kTcStages) ok = wait(&v_empty[s], parity);
                    }
                    if (ok) {
                        mbar_expect_tx(&v_full[s], kTileBytes);
#pragma unroll
                        for (int c = 0; c < kColumns; ++c) tc_tma_2d(kd + kTileBytes + c * kTileBlockBytes, &map_v, 64 * c, row, &v_full[s]);
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            }
        }
        if (!ok && lane == 0) record_give_up();
    } else if (warp == 1) {
        // ---------------- products ----------------
        if (lane == 0 && n_tiles > 0) {
            constexpr uint32_t idesc_s = tc_idesc(kBlock, kPageTokens, 0), idesc_o = tc_idesc(kBlock, HD, 1);      // the values lie MN-major
            ok = wait(q_full, 0);
            tc_fence_after_sync();
            auto issue_s = [&](int j) -> bool {
                const int s = j % kTcStages, sb = j & 1;
                if (!wait(&k_full[s], (j / kTcStages) & 1)) return false;
                if (j >= 2 && !wait(&s_empty[sb], ((j >> 1) - 1) & 1)) return false;
                tc_fence_after_sync();
                const uint32_t k_addr = smem_u32(ring + (size_t)s * 2 * kTileBytes);
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    tc_mma(tmem_base + kColS + sb * kPageTokens, desc_kmajor(smem_u32(q_s) + (kk / 4) * kQBlockBytes) + 2 * (kk % 4),
                           desc_kmajor(k_addr + (kk / 4) * kTileBlockBytes) + 2 * (kk % 4), idesc_s, kk > 0 ? 1u : 0u);
                tc_commit(&s_full[sb]);
                tc_commit(&k_empty[s]);
                return true;
            };
            if (ok) ok = issue_s(0);
            for (int j = 0; j < n_tiles && ok; ++j) {
                if (j + 1 < n_tiles && !issue_s(j + 1)) { ok = false; break; }       // the next S runs under this tile's softmax
                const int pb = j & 1, s = j % kTcStages;
                if (!wait(&p_full[pb], (j >> 1) & 1) || !wait(&v_full[s], (j / kTcStages) & 1)) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t v_addr = smem_u32(ring + (size_t)s * 2 * kTileBytes + kTileBytes);
#pragma unroll
                for (int ks = 0; ks < kPageTokens / 16; ++ks)
                    tc_mma(tmem_base + kColO, desc_kmajor(smem_u32(p_s) + pb * kPBytes) + 2 * ks,
                           desc_mnmajor(v_addr + ks * 16 * 128, kTileBlockBytes), idesc_o, (j > 0 || ks > 0) ? 1u : 0u);
                tc_commit(&v_empty[s]);
                tc_commit(&pv_done[pb]);
            }
            if (!ok) record_give_up();
        }
        __syncwarp();
    } else {
        // ---------------- queries, softmax, sums: two threads a row, each 32 of a tile's keys ----------------
        const int quarter = warp & 3, half = (warp - 2) >> 2, tid = threadIdx.x - 64;
        const int r = quarter * 32 + lane;                       // row of the tile = lane of tensor memory
        const int group = a.n_heads / kv_heads, pairs = it.n_rows * group;
        for (int i = tid; i < kBlock * (HD / 8); i += 256) {
            const int p = i / (HD / 8), c = i % (HD / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (p < pairs)
                v = *reinterpret_cast<const uint4*>(a.q + (size_t)a.rows[it.row0 + p / group] * a.q_stride + (size_t)(kvh * group + p % group) * HD + c * 8);
            *reinterpret_cast<uint4*>(q_s + (c / 8) * kQBlockBytes + p * 128 + (((c % 8) ^ (p & 7)) << 4)) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // generic writes -> visible to the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const int row = a.rows[it.row0 + min(r / group, it.n_rows - 1)];
        const int pos = a.token_pos[row], lowest = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
        const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
        // t = tanh(s scale / cap), or s: the score is c_logit t, and a weight 2^(t c2 - m c2)
        const bool capped = a.cap > 0.f;
        const float pre = capped ? a.scale / a.cap : 1.f, c_logit = capped ? a.cap : a.scale;
        const float c2 = c_logit * 1.44269504f, slack = kRescaleSlack / c_logit;
        float m_ref = -INFINITY, l_run = 0.f;                    // l_run: of this thread's keys
        auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
        for (int j = 0; j < n_tiles; ++j) {
            const int sb = j & 1, key0 = walk_page(w, w.begin + j) * kPageTokens;
            float m_half = -INFINITY;
            float sc[32];
            if (ok) ok = warp_wait(&s_full[sb], (j >> 1) & 1);
            if (ok) {
                tc_fence_after_sync();
                {
                    uint32_t v[32];
                    tc_ld32(t_lane + kColS + sb * kPageTokens + 32 * half, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 32; ++i) sc[i] = __uint_as_float(v[i]);
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[sb]);
                if (capped) tanh_scores(sc, pre);
                if (key0 < w.all_from || key0 + kPageTokens - 1 > w.all_to) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int key = key0 + 32 * half + i;
                        sc[i] = key >= lowest && key <= pos ? sc[i] : -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) m_half = fmaxf(m_half, sc[i]);
            }
            // the row's maximum over both halves; two places, so that one barrier is enough
            xchg[half * kBlock + r] = m_half;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float m_tile = fmaxf(m_half, xchg[(half ^ 1) * kBlock + r]);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!ok) continue;
            float factor = 1.f;
            if (m_tile > m_ref + slack || (m_ref == -INFINITY && m_tile > -INFINITY)) {
                factor = m_ref == -INFINITY ? 0.f : __expf((m_ref - m_tile) * c_logit);
                m_ref = m_tile;
            }
            const float m2 = (m_ref == -INFINITY ? 0.f : m_ref) * c2;
            float sum = 0.f;
            uint32_t packed[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                const float e0 = fmaf(sc[i], c2, -m2), e1 = fmaf(sc[i + 1], c2, -m2);
                const bool poly = ((i >> 1) & 3) == 0;
                const float p0 = poly ? exp2_poly(e0) : ex2_approx(e0), p1 = poly ? exp2_poly(e1) : ex2_approx(e1);
                sum += p0 + p1;
                packed[i / 2] = pack_bf16(p0, p1);
            }
            l_run = l_run * factor + sum;
            if (j >= 2) ok = warp_wait(&pv_done[sb], ((j >> 1) - 1) & 1);      // this buffer of weights has been read
            if (!ok) continue;
            if (j > 0 && __any_sync(0xffffffffu, factor != 1.f)) {
                ok = warp_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);      // O is touched only between products
                if (!ok) continue;
                tc_fence_after_sync();
#pragma unroll 1
                for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                    uint32_t o[32];
                    tc_ld32(t_lane + kColO + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                    tc_st32(t_lane + kColO + c, o);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            unsigned char* prow = p_s + (size_t)sb * kPBytes + (size_t)r * 128;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint4*>(prow + (((4 * half + c) ^ (r & 7)) << 4)) =
                    make_uint4(packed[4 * c], packed[4 * c + 1], packed[4 * c + 2], packed[4 * c + 3]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[sb]);
        }
        // ---- the sums leave, not divided ----
        if (ok && n_tiles > 0) ok = warp_wait(&pv_done[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1);
        tc_fence_after_sync();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        xchg[half * kBlock + r] = l_run;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok) {
            const size_t at = ((size_t)row * a.n_heads + kvh * group + r % group) * a.parts + it.part;
            if (half == 0 && r < pairs) a.part_ml[at] = make_float2(m_ref * c_logit, l_run + xchg[kBlock + r]);
            if (n_tiles > 0) {
#pragma unroll 1
                for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                    uint32_t o[32];
                    tc_ld32(t_lane + kColO + c, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (r < pairs) {
                        uint4* dst = reinterpret_cast<uint4*>(a.part_o + at * HD + c);
#pragma unroll
                        for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
        if (!ok && lane == 0) record_give_up();
    }
    tc_fence_before_sync();
    if (__syncthreads_or(!ok)) let_work_under_way_end();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
}
#endif

// A row's parts joined; a row without parts (padding) becomes zeros, and so does one that sees no key.  A block takes a (row, head): HD / 4
// threads a part, as many parts at a time as 256 threads are.
__global__ void __launch_bounds__(256) attn_shared_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                                                                const int* __restrict__ n_parts, int parts, int n_heads, bf16* out, int out_stride) {
    constexpr int ACROSS = HD / 4, DEEP = 256 / ACROSS;
    __shared__ float4 sums[DEEP * ACROSS];
    pdl_enter();
    const int n = blockIdx.x / n_heads, head = blockIdx.x % n_heads;
    const int have = n_parts[n];
    const size_t at = ((size_t)n * n_heads + head) * parts;
    const int across = threadIdx.x % ACROSS, deep = threadIdx.x / ACROSS;
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < have; ++p) m = fmaxf(m, part_ml[at + p].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = deep; p < have; p += DEEP) {
        const float2 v = part_ml[at + p];
        if (deep >= DEEP || v.x == -INFINITY) continue;      // (a part without a key left no sums)
        const float f = __expf(v.x - m);
        const float4 b = *reinterpret_cast<const float4*>(part_o + (at + p) * HD + across * 4);
        acc.x += b.x * f; acc.y += b.y * f; acc.z += b.z * f; acc.w += b.w * f;
    }
    if (deep < DEEP) sums[deep * ACROSS + across] = acc;
    for (int p = 0; p < have; ++p) {
        const float2 v = part_ml[at + p];
        if (v.x != -INFINITY) l += v.y * __expf(v.x - m);
    }
    __syncthreads();
    if (deep == 0) {
#pragma unroll 4
        for (int d = 1; d < DEEP; ++d) {
            const float4 b = sums[d * ACROSS + across];
            acc.x += b.x; acc.y += b.y; acc.z += b.z; acc.w += b.w;
        }
        const float r = l > 0.f ? 1.f / l : 0.f;
        *reinterpret_cast<uint2*>(out + (size_t)n * out_stride + (size_t)head * HD + across * 4) =
            make_uint2(pack_bf16(acc.x * r, acc.y * r), pack_bf16(acc.z * r, acc.w * r));
    }
}

}  // namespace hos

using namespace hos;

extern "C" const char* hos_last_error() { return error_buffer(); }

extern "C" int hos_attn_shared_set_error_word(int* word) {
    if (cudaMemcpyToSymbol(g_shared_error_host, &word, sizeof(word)) != cudaSuccess)
        HOS_REFUSE("attn_shared: cannot set the error word: %s", cudaGetErrorString(cudaGetLastError()));
    return 0;
}

// What a list of work is (parts/shared_attention.py makes one a step and kind of layer): on the device, but for the numbers.
struct SharedWork {
    const int* counts;         // [0] items of up to 16 pairs, [1] of up to 128
    const int* n_parts;        // [rows]
    const int* items;          // of up to 16 pairs, then
    const int* big_items;      // of up to 128
    const int* rows;
    const int* page_table;
    int most, big_most;        // how many items there may be (what the grids are made for)
    int parts;                 // places of a (row, head) in the workspace
    int table_stride, ring_pages, n_heads, n_kv_heads, window;
};

// 1: blocks of up to 128 pairs have a kernel for this head size.
extern "C" int hos_attn_shared_big() { return HD == 64 || HD == 128 || HD == 256; }

// out[n_rows, n_heads * head_dim] = softmax(c tanh(scale q . k / c)) v by the items of the work; see the head of this file.  workspace:
// n_rows * n_heads * parts * (head_dim + 2) floats.
extern "C" int hos_attn_shared(const void* q, int q_stride, void* out, int out_stride, int n_rows, const int* token_pos, const void* k_pages,
                               const void* v_pages, long long n_pages, const SharedWork* work, float scale, float cap, float* workspace,
                               cudaStream_t stream) {
    const SharedWork& k = *work;
    if (n_rows <= 0) return 0;
    if (k.n_kv_heads <= 0 || k.n_heads % k.n_kv_heads) HOS_REFUSE("attn_shared: %d query heads over %d kv heads", k.n_heads, k.n_kv_heads);
    if ((q_stride % 8) || ((uintptr_t)q % 16)) HOS_REFUSE("attn_shared: rows of queries must lie on 16 bytes");
    if ((out_stride % 4) || ((uintptr_t)out % 8)) HOS_REFUSE("attn_shared: rows of the output must lie on 8 bytes");
    if (((uintptr_t)k_pages % 16) || ((uintptr_t)v_pages % 16) || ((uintptr_t)workspace % 16)) HOS_REFUSE("attn_shared: pages and workspace must lie on 16 bytes");
    if ((long long)n_rows * k.n_heads > (1ll << 31) - 1) HOS_REFUSE("attn_shared: %d rows of %d heads", n_rows, k.n_heads);
    const int group = k.n_heads / k.n_kv_heads;
    float* part_ml = workspace + (size_t)n_rows * k.n_heads * k.parts * HD;
    SharedArgs a{(const bf16*)q, q_stride, token_pos, reinterpret_cast<const SharedItem*>(k.items), k.counts, k.rows,
                 PagedKV{const_cast<void*>(k_pages), const_cast<void*>(v_pages), k.page_table, k.table_stride, k.ring_pages, k.n_kv_heads, HD},
                 k.n_heads, k.parts, workspace, reinterpret_cast<float2*>(part_ml), scale, cap, k.window};
    int rc;
    if (k.big_most > 0) {
#if (HOS_HEAD_DIM == 64) || (HOS_HEAD_DIM == 128) || (HOS_HEAD_DIM == 256)
        if (group > kBlock) HOS_REFUSE("attn_shared: %d query heads to a kv head in blocks of %d", group, kBlock);
        CUtensorMap mk, mv;
        const long long page_rows = n_pages * k.n_kv_heads * kPageTokens;
        if (page_rows > (1ll << 31) - 1) HOS_REFUSE("attn_shared: %lld pages of %d kv heads", n_pages, k.n_kv_heads);
        if ((rc = tc_make_map(&mk, k_pages, page_rows, HD, HD, kPageTokens, false))) return rc;
        if ((rc = tc_make_map(&mv, v_pages, page_rows, HD, HD, kPageTokens, false))) return rc;
        static bool set = false;
        if (!set) {
            if (cudaFuncSetAttribute(attn_shared_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcShared) != cudaSuccess)
                HOS_REFUSE("attn_shared: cannot get %d bytes of shared memory", kTcShared);
            set = true;
        }
        SharedArgs b = a;
        b.items = reinterpret_cast<const SharedItem*>(k.big_items);
        b.n_items = k.counts + 1;
        launch_pdl(attn_shared_tc_kernel, dim3((unsigned)(k.big_most * k.n_kv_heads)), dim3(kTcThreads), kTcShared, stream, mk, mv, b);
        if ((rc = check_launch("attn_shared (blocks)"))) return rc;
#else
        HOS_REFUSE("attn_shared: no blocks of %d pairs for heads of %d numbers", 128, HD);
#endif
    }
    if (k.most > 0) {
        static bool set = false;
        if (!set) {
            if (cudaFuncSetAttribute(attn_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SharedSmem::kTotal) != cudaSuccess)
                HOS_REFUSE("attn_shared: cannot get %d bytes of shared memory", SharedSmem::kTotal);
            set = true;
        }
        const long long items = (long long)k.most * k.n_kv_heads * ((group + kPairs - 1) / kPairs);
        const int grid = (int)(items < sm_count_cached() ? items : sm_count_cached());
        launch_pdl(attn_shared_kernel, dim3(grid), dim3(kThreads), SharedSmem::kTotal, stream, a);
        if ((rc = check_launch("attn_shared"))) return rc;
    }
    launch_pdl(attn_shared_merge_kernel, dim3(n_rows * k.n_heads), dim3(256), 0, stream, workspace, reinterpret_cast<const float2*>(part_ml), k.n_parts,
               k.parts, k.n_heads, (bf16*)out, out_stride);
    return check_launch("attn_shared (merge)");
}
