// Keys and values in 4 bits: rows put into the pages, and attention over them.
//
// For every 64 neighbouring numbers of a head a scale s and a middle m in bfloat16 and 64 codes c of 4 bits, -8..7:
//   s = bf16((max - min) / 15), m = bf16(min + 8 s), c = clamp(rint((x - m) / s), -8, 7); what is held is c s + m.
// All numbers alike (s 0 or below the smallest normal number): codes 0, the value m.  A NaN, an infinity or a range that
// overflows makes the 64 numbers NaN.  Divisions and roundings are IEEE's, so that a value is a function of its row alone.
// A page's tile of a kv head is laid out in fourbit.cuh: keys "by row", values "by column".
#include "common.cuh"
#include "fourbit.cuh"
#include "kv_layout.cuh"

namespace hos {

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

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[i];
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(p[i]);
}

// Eight lanes hold 64 numbers, eight each: scale, middle and codes.
__device__ __forceinline__ void quantise64(const float (&x)[8], float& s, float& m, int (&c)[8]) {
    float lo = x[0], hi = x[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        fine = fine && isfinite(x[i]);
    }
    float odd = fine ? 0.f : 1.f;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        odd = fmaxf(odd, __shfl_xor_sync(0xffffffffu, odd, o));
    }
    s = to_float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
    if (!(s >= 1.17549435e-38f)) s = 0.f;            // subnormal or 0 (a NaN is caught below)
    m = to_float(__float2bfloat16_rn(__fadd_rn(lo, 8.f * s)));
    if (odd != 0.f || !isfinite(s) || !isfinite(m)) s = m = __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = (s > 0.f) ? rintf(__fdiv_rn(__fsub_rn(x[i], m), s)) : 0.f;      // NaN: not above 0
        c[i] = (int)fminf(fmaxf(q, -8.f), 7.f);
    }
}

// Eight lanes per 64 numbers; a lane's word of keys, or with its neighbour's codes eight bytes of values.  A row is n_kv_heads * head_dim
// numbers of keys, then as many of values.
template <typename T>
__global__ void __launch_bounds__(256)
store4_kernel(const T* rows, long long stride, T* held, long long held_stride, const int* __restrict__ token_pos, const int* __restrict__ token_seq,
              const int* __restrict__ seq_slot, const int* __restrict__ seq_len_after, Paged4 c, int n_tokens) {
    pdl_enter();
    const int dim = c.head_dim, groups = dim / 64, per_row = 2 * c.n_kv_heads * groups;
    const long long item = (long long)blockIdx.x * 32 + (threadIdx.x >> 3);
    const bool live = item < (long long)n_tokens * per_row;
    const int n = live ? (int)(item / per_row) : 0, r = live ? (int)(item % per_row) : 0, l = threadIdx.x & 7;
    const bool value = r >= c.n_kv_heads * groups;
    const int col = r * 64 + l * 8;                       // column of the row
    float x[8], s, m;
    int q[8];
    load8(rows + (size_t)n * stride + col, x);
    quantise64(x, s, m, q);
    if (live && held != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) held[(size_t)n * held_stride + col + i] = from_float<T>(fmaf((float)q[i], s, m));
    }
    uint32_t w = 0, other;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (uint32_t)(q[i] + 8) << code_shift(i);
    other = __shfl_xor_sync(0xffffffffu, w, 1);
    if (!live) return;
    const int seq = token_seq[n], pos = token_pos[n];
    if (seq < 0) return;
    if (c.ring_pages > 0 && pos + c.ring_pages * kPageTokens < seq_len_after[seq]) return;     // the same step writes over it
    const int head = (r - (value ? c.n_kv_heads * groups : 0)) / groups, g = r % groups, row = pos % kPageTokens;
    const int page = page4_of(c, seq_slot[seq], pos);
    uint8_t* tile = (value ? c.v_pages : c.k_pages) + ((size_t)page * c.n_kv_heads + head) * tile4_bytes(dim);
    uint8_t* block = tile + ((row >> 4) * groups + g) * kBlockBytes;
    if (!value) {
        *(uint32_t*)(block + by_row_word(row & 15, l * 8)) = w;
    } else if ((l & 1) == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            block[by_column_byte(row & 15, l * 8 + i)] = (uint8_t)(((w >> code_shift(i)) & 15u) | (((other >> code_shift(i)) & 15u) << 4));
    }
    if (l == 0) {
        const __nv_bfloat162 sm = __floats2bfloat162_rn(s, m);
        *(__nv_bfloat162*)(tile + tile4_codes(dim) + (row * groups + g) * 4) = sm;
    }
}

// One warp per (row, query head); a lane takes the words lane, lane + 32 of a key.
template <typename T, int DIM>
__global__ void __launch_bounds__(128)
attend4_plain_kernel(const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const int* __restrict__ token_pos,
                     const int* __restrict__ token_seq, const int* __restrict__ seq_slot, Paged4 c, int n_tokens, int n_heads, float scale, float cap,
                     int window) {
    pdl_enter();
    constexpr int kWords = DIM / 8, kPer = (kWords + 31) / 32;
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)n_tokens * n_heads) return;
    const int n = (int)(item / n_heads), h = (int)(item % n_heads), kvh = h / (n_heads / c.n_kv_heads);
    const int seq = token_seq[n], pos = token_pos[n];
    float qv[kPer][8], acc[kPer][8] = {}, best = -INFINITY, sum = 0.f;
    for (int i = 0; i < kPer; ++i)
        for (int j = 0; j < 8; ++j) qv[i][j] = (lane + 32 * i < kWords) ? to_float(q[(size_t)n * q_stride + h * DIM + (lane + 32 * i) * 8 + j]) : 0.f;
    const int first = (seq < 0) ? pos + 1 : (window > 0 ? max(0, pos - window + 1) : 0);
    for (int p = first; p <= pos; ++p) {
        const int page = page4_of(c, seq_slot[seq], p), row = p % kPageTokens;
        const size_t at = ((size_t)page * c.n_kv_heads + kvh) * tile4_bytes(DIM);
        const uint8_t *kt = c.k_pages + at, *vt = c.v_pages + at;
        float dot = 0.f;
        for (int i = 0; i < kPer; ++i) {
            const int d = (lane + 32 * i) * 8, g = d / 64;
            if (d >= DIM) break;
            const uint32_t w = *(const uint32_t*)(kt + ((row >> 4) * (DIM / 64) + g) * kBlockBytes + by_row_word(row & 15, d & 63));
            const uint32_t sm = *(const uint32_t*)(kt + tile4_codes(DIM) + (row * (DIM / 64) + g) * 4);
            for (int j = 0; j < 8; ++j) dot = fmaf(qv[i][j], fmaf((float)((w >> code_shift(j)) & 15u) - 8.f, bf16_lo(sm), bf16_hi(sm)), dot);
        }
        const float score = softcap_precise(warp_sum(dot) * scale, cap), top = fmaxf(best, score);
        const float old = expf(best - top), e = expf(score - top);
        best = top;
        sum = sum * old + e;
        for (int i = 0; i < kPer; ++i) {
            const int d = (lane + 32 * i) * 8, g = d / 64;
            if (d >= DIM) break;
            const uint32_t sm = *(const uint32_t*)(vt + tile4_codes(DIM) + (row * (DIM / 64) + g) * 4);
            for (int j = 0; j < 8; ++j) {
                const int dd = (d & 63) + j;
                const uint8_t b = vt[((row >> 4) * (DIM / 64) + g) * kBlockBytes + by_column_byte(row & 15, dd & ~8)];
                acc[i][j] = acc[i][j] * old + e * fmaf((float)((b >> ((dd & 8) ? 4 : 0)) & 15) - 8.f, bf16_lo(sm), bf16_hi(sm));
            }
        }
    }
    for (int i = 0; i < kPer; ++i)
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * i < kWords) out[(size_t)n * out_stride + h * DIM + (lane + 32 * i) * 8 + j] = from_float<T>(sum > 0.f ? acc[i][j] / sum : 0.f);
}

}  // namespace hos

using namespace hos;

#define HOS_CHECK_PAGED4(what)                                                                                            \
    if (head_dim % 64 || head_dim < 64 || head_dim > 256) HOS_REFUSE(what ": head size %d (64, 128, 192 or 256)", head_dim);     \
    if (n_kv_heads <= 0) HOS_REFUSE(what ": %d kv heads", n_kv_heads);                                                         \
    const Paged4 c{(uint8_t*)k_pages, (uint8_t*)v_pages, page_table, table_stride, ring_pages, n_kv_heads, head_dim}

extern "C" int hos_store4(const void* rows, int dtype, long long stride, void* held, long long held_stride, const int* token_pos, const int* token_seq,
                          const int* seq_slot, const int* seq_len_after, void* k_pages, void* v_pages, const int* page_table, int table_stride, int ring_pages,
                          int n_kv_heads, int head_dim, int n_tokens, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    HOS_CHECK_PAGED4("store4");
    const long long items = (long long)n_tokens * 2 * n_kv_heads * (head_dim / 64);
    const dim3 grid((unsigned)((items + 31) / 32));
    if (dtype == kF32)
        launch_pdl(store4_kernel<float>, grid, dim3(256), 0, stream, (const float*)rows, stride, (float*)held, held_stride, token_pos, token_seq, seq_slot, seq_len_after, c, n_tokens);
    else
        launch_pdl(store4_kernel<bf16>, grid, dim3(256), 0, stream, (const bf16*)rows, stride, (bf16*)held, held_stride, token_pos, token_seq, seq_slot, seq_len_after, c, n_tokens);
    return check_launch("store4");
}

extern "C" int hos_attend4(const void* q, int dtype, long long q_stride, void* out, long long out_stride, const int* token_pos, const int* token_seq,
                           const int* seq_slot, void* k_pages, void* v_pages, const int* page_table, int table_stride, int ring_pages, int n_kv_heads,
                           int head_dim, int n_tokens, int n_heads, float scale, float cap, int window, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    HOS_CHECK_PAGED4("attend4");
    if (n_heads <= 0 || n_heads % n_kv_heads) HOS_REFUSE("attend4: %d query heads over %d kv heads", n_heads, n_kv_heads);
    const dim3 grid((unsigned)(((long long)n_tokens * n_heads + 3) / 4));
#define HOS_A4(T, D) launch_pdl(attend4_plain_kernel<T, D>, grid, dim3(128), 0, stream, (const T*)q, q_stride, (T*)out, out_stride, token_pos, token_seq, seq_slot, c, n_tokens, n_heads, scale, cap, window)
#define HOS_A4_D(T) do { if (head_dim == 64) HOS_A4(T, 64); else if (head_dim == 128) HOS_A4(T, 128); else if (head_dim == 192) HOS_A4(T, 192); else HOS_A4(T, 256); } while (0)
    if (dtype == kF32) HOS_A4_D(float);
    else HOS_A4_D(bf16);
    return check_launch("attend4");
}
