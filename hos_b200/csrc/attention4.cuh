// What the kernels over 4-bit pages share: the pages as they are handed over, the blocks of a step's rows, the product.
#pragma once
#include "common.cuh"
#include "fourbit.cuh"
#include "kv_layout.cuh"
#include "mma_utils.cuh"
#include <cuda_fp16.h>

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

// The same of half precision, and what the products of weights and values take: codes -8..7 (a register's bits lie where 1024 + c or 1024 + 16 c
// is made of them at once) and weights, which are at most 2^8, times the values' scales, brought below 2^7 by a power of two of a
// group's and walk's own (`into`, raised when a scale passes it): rounded to 2^-11 of themselves down to 2^-20 of the largest.
__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t (&r)[4]) {
    const uint32_t up = w >> 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(i < 2 ? w : up), "r"((i & 1) ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        const __half2 c = *reinterpret_cast<const __half2*>(&v);
        const __half2 d = (i & 1) ? __hfma2(c, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hsub2(c, __float2half2_rn(1032.f));
        r[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}
constexpr float kIntoFirst = 8.5070592e37f, kIntoMost = 128.f;        // 2^126: before the first scale
// 1 / into
__device__ __forceinline__ float back_of(float into) { return __uint_as_float((254u << 23) - __float_as_uint(into)); }
__device__ __forceinline__ float into_of(float scale) {                // 2^6 <= scale * into < 2^7
    const int e = (int)((__float_as_uint(scale) >> 23) & 255u) - 127;
    return __uint_as_float((uint32_t)(127 + max(-126, min(126, 6 - e))) << 23);
}

}  // namespace hos

#define HOS_CHECK_PAGED4(what)                                                                                            \
    const Paged4 c = *(const Paged4*)cache;                                                                                \
    const int head_dim = c.head_dim, n_kv_heads = c.n_kv_heads;                                                            \
    if (head_dim % 64 || head_dim < 64 || head_dim > 256) HOS_REFUSE(what ": head size %d (64, 128, 192 or 256)", head_dim);     \
    if (n_kv_heads <= 0) HOS_REFUSE(what ": %d kv heads", n_kv_heads)

