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
// consumer warps take 16 keys of a page each.  Weights are rounded to bfloat16 for the product with the values (2^-9 of each), their sum
// is of the weights before that rounding.
//
// Compiled per head size: -DHOS_HEAD_DIM=N, a multiple of 16 up to 256.
#include "common.cuh"
#include "kv_layout.cuh"
#include "mma_utils.cuh"

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
};
__device__ __forceinline__ Walk walk_of(const SharedArgs& a, const SharedItem& it, int lane) {
    int lo = 0x7fffffff, hi = -1;
    for (int r = lane; r < it.n_rows; r += 32) {
        const int pos = a.token_pos[a.rows[it.row0 + r]];
        lo = min(lo, a.window > 0 ? max(0, pos + 1 - a.window) / kPageTokens : 0);
        hi = max(hi, pos / kPageTokens);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const int from = max(it.lp0, lo), to = min(it.lp1, hi + 1);
    Walk w;
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

// The items' parts of softmax(c tanh(scale q . k / c)) v into the workspace; see the head of this file.  items: on the device,
// *n_items of them, and `most` of them at most (what the grid is made for).
extern "C" int hos_attn_shared(const void* q, int q_stride, const int* token_pos, const int* items, const int* n_items, int most,
                               const int* rows, const void* k_pages, const void* v_pages, const int* page_table, int table_stride,
                               int ring_pages, int n_heads, int n_kv_heads, int head_dim, float scale, float cap, int window, int parts,
                               float* part_o, float* part_ml, cudaStream_t stream) {
    if (most <= 0) return 0;
    if (head_dim != HD) HOS_REFUSE("attn_shared: heads of %d numbers in the library for %d", head_dim, HD);
    if (n_kv_heads <= 0 || n_heads % n_kv_heads) HOS_REFUSE("attn_shared: %d query heads over %d kv heads", n_heads, n_kv_heads);
    if ((q_stride % 8) || ((uintptr_t)q % 16)) HOS_REFUSE("attn_shared: rows of queries must lie on 16 bytes");
    SharedArgs a{(const bf16*)q, q_stride, token_pos, reinterpret_cast<const SharedItem*>(items), n_items, rows,
                 PagedKV{const_cast<void*>(k_pages), const_cast<void*>(v_pages), page_table, table_stride, ring_pages, n_kv_heads, HD},
                 n_heads, parts, part_o, reinterpret_cast<float2*>(part_ml), scale, cap, window};
    static bool set = false;
    if (!set) {
        if (cudaFuncSetAttribute(attn_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SharedSmem::kTotal) != cudaSuccess)
            HOS_REFUSE("attn_shared: cannot get %d bytes of shared memory", SharedSmem::kTotal);
        set = true;
    }
    const long long work = (long long)most * n_kv_heads * ((n_heads / n_kv_heads + kPairs - 1) / kPairs);
    const int grid = (int)(work < sm_count_cached() ? work : sm_count_cached());
    launch_pdl(attn_shared_kernel, dim3(grid), dim3(kThreads), SharedSmem::kTotal, stream, a);
    return check_launch("attn_shared");
}

extern "C" int hos_attn_shared_merge(const float* part_o, const float* part_ml, const int* n_parts, int parts, int n_rows, int n_heads,
                                     void* out, int out_stride, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if ((out_stride % 4) || ((uintptr_t)out % 8)) HOS_REFUSE("attn_shared: rows of the output must lie on 8 bytes");
    if ((long long)n_rows * n_heads > (1ll << 31) - 1) HOS_REFUSE("attn_shared: %d rows of %d heads", n_rows, n_heads);
    launch_pdl(attn_shared_merge_kernel, dim3(n_rows * n_heads), dim3(256), 0, stream, part_o, reinterpret_cast<const float2*>(part_ml), n_parts,
               parts, n_heads, (bf16*)out, out_stride);
    return check_launch("attn_shared_merge");
}
