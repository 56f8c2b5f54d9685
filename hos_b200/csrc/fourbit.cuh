// Numbers held in 4 bits, as the operands of mma.sync m16n8k16 want them.
//
// A block is 16 rows x 64 numbers in 512 bytes, 16 to a lane of the warp that multiplies it: with g = lane / 4 and
// t = lane % 4 the MMA wants of its 16 x 16 operand the rows g and g + 8 and four columns a lane, and since a dot product does not
// care in which order its terms come, the four MMA steps of a block take a lane's 16 numbers of a row four by four
// (the other operand is read in the same order).  A 32-bit word holds eight codes; shifted right by 4 r its low nibbles of the two
// halves are the two codes of the operand's register r, so that a register costs a shift and one logical instruction, which also
// sets the bits that make 128 + c of a code c in bfloat16, and one subtraction, exact, that takes the 128 and the zero code away.
//
// Keys (positions x numbers of a head), "by row": word ((row / 8) % 2) * 2 + (d / 8) % 2 of lane (row % 8) * 4 + d / 16, code d % 8
// of the word.  A token's eight neighbouring numbers are one word of its own.
// Weights (features x k) the same with d / 32 in the place of (d / 8) % 2 and (d / 8) % 4 in that of d / 16: a word's step lies in
// one group of 32.
// Values, which the MMA takes transposed (numbers of a head x positions), "by column": word d / 16 of lane (d % 8) * 4 +
// (row % 8) / 2, byte (row % 2) * 2 + row / 8, the low nibble where (d / 8) % 2 is 0.  A byte belongs to one token.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace hos {

constexpr int kBlockRows = 16, kBlockCols = 64, kBlockBytes = 512;

// Bit position of code j (0..7) in its word.
__host__ __device__ __forceinline__ int code_shift(int j) { return 4 * ((j >> 1) + 4 * (j & 1)); }
// Byte of a block at which the word of (row, d..d+7) lies, d a multiple of 8.
__host__ __device__ __forceinline__ int by_row_word(int row, int d) {
    return ((row & 7) * 4 + (d >> 4)) * 16 + (((row >> 3) & 1) * 2 + ((d >> 3) & 1)) * 4;
}
// Byte of a block that holds (row, d) in its low and (row, d + 8) in its high nibble, (d / 8) % 2 == 0.
__host__ __device__ __forceinline__ int by_column_byte(int row, int d) {
    return ((d & 7) * 4 + ((row & 7) >> 1)) * 16 + (d >> 4) * 4 + (row & 1) * 2 + (row >> 3);
}

// A page's tile of one kv head: 64 positions of DIM numbers as blocks [position / 16][d / 64], then for every position and 64
// numbers the scale (low half) and the middle (high half) in bfloat16.
__host__ __device__ __forceinline__ int tile4_codes(int dim) { return 32 * dim; }
__host__ __device__ __forceinline__ int tile4_bytes(int dim) { return 36 * dim; }

// The four operand registers of a word: 128 + code, or (SUBTRACT) the codes minus `zero` ((128 + zero) twice in bfloat16), exact.
template <bool SUBTRACT = true>
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t zero, uint32_t (&r)[4]) {
    const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&zero);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t v;                                            // (w >> 4 i) & mask | bits in one instruction
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(0x43004300u));
        if (!SUBTRACT) {
            r[i] = v;
            continue;
        }
        const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), z);
        r[i] = *reinterpret_cast<const uint32_t*>(&c);
    }
}
constexpr uint32_t kZero8 = 0x43084308u;       // 128 + 8 twice

// bfloat16 pairs
__device__ __forceinline__ float bf16_lo(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// A matrix as the host hands it over (ops.Matrix4): N features (gated: of gate, and as many of up, gate's 16-row tiles first).
struct Matrix4 {
    const uint8_t *codes, *records, *records16;
    const float* powers;                 // records16 and powers: for the products of many rows (weights4_tc.cu)
    int n, k, group, zeros, gated;
};

// 16 bytes from global to shared memory without registers, `bytes` of them read and the rest zeros; groups of a thread's copies
// end in order, and a warp that waits for its own and meets at __syncwarp() sees all of its lanes' copies.
__device__ __forceinline__ void copy16_async(uint32_t smem, const void* gmem, int bytes = 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

}  // namespace hos
