// What the kernels over 4-bit pages share: the pages as they are handed over, the blocks of a step's rows, the product.
#pragma once
#include "common.cuh"
#include "fourbit.cuh"
#include "kv_layout.cuh"
#include "mma_utils.cuh"

namespace hos {

constexpr int kMaxShares = 1024;        // of a walk over the keys

// One call's view of the pages, as the host hands it over (ops.Paged4).
struct Paged4 {
    uint8_t* k_pages;
    uint8_t* v_pages;
    const int* page_table;
    int table_stride, ring_pages, n_kv_heads, head_dim;
};

__device__ __forceinline__ int page4_of(const Paged4& c, int slot, int pos) {
    const int lp = pos / kPageTokens;
    return c.page_table[(size_t)slot * c.table_stride + (c.ring_pages > 0 ? lp % c.ring_pages : lp)];
}

// Block `left` of the step's rows, cut into blocks of up to `size` rows of one sequence (begun anew where a position is a multiple of
// size if `align` is size - 1, else, 0, at a sequence's first row), in order; after them come the padding rows, `size` at a time (seq
// -1).  Every lane of a warp looks at a sequence, their numbers of blocks are added up.  count <= 0: there is no such block.
struct RowBlock { int seq, row0, pos0, count; };
__device__ __forceinline__ RowBlock find_rows(const int* __restrict__ cu_seqlens, int row_base, int n_seqs, const int* __restrict__ token_pos, int n_tokens,
                                              int left, int size, int align) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
        const int s = s0 + lane;
        int first = 0, n = 0, pos = 0, nb = 0;
        if (s < n_seqs) {
            first = cu_seqlens[s] - row_base;
            n = cu_seqlens[s + 1] - row_base - first;
            pos = n > 0 ? token_pos[first] : 0;
            nb = n > 0 ? ((pos & align) + n + size - 1) / size : 0;
        }
        int upto = nb;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, left < upto);
        if (found != 0) {
            const int who = __ffs(found) - 1, in = left - (__shfl_sync(0xffffffffu, upto, who) - __shfl_sync(0xffffffffu, nb, who));
            first = __shfl_sync(0xffffffffu, first, who);
            n = __shfl_sync(0xffffffffu, n, who);
            pos = __shfl_sync(0xffffffffu, pos, who);
            const int skip = in == 0 ? 0 : size * in - (pos & align);  // rows of the sequence before the block
            return RowBlock{s0 + who, first + skip, pos + skip, min(size - ((pos + skip) & align), n - skip)};
        }
        left -= __shfl_sync(0xffffffffu, upto, 31);
    }
    const int row0 = cu_seqlens[n_seqs] - row_base + size * left;
    return RowBlock{-1, row0, 0, min(size, n_tokens - row0)};
}

// d += a . b, free to be woven into its neighbours.
__device__ __forceinline__ void mma_plain(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace hos

#define HOS_CHECK_PAGED4(what)                                                                                            \
    const Paged4 c = *(const Paged4*)cache;                                                                                \
    const int head_dim = c.head_dim, n_kv_heads = c.n_kv_heads;                                                            \
    if (head_dim % 64 || head_dim < 64 || head_dim > 256) HOS_REFUSE(what ": head size %d (64, 128, 192 or 256)", head_dim);     \
    if (n_kv_heads <= 0) HOS_REFUSE(what ": %d kv heads", n_kv_heads)

