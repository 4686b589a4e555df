// What the kernels over a cache of keys and values in 4 bits share.
//
// A token's key (or value) row of a head, dh numbers, is cut into groups of G (64 where 64 divides dh, else 32, else 16).  A group
// is held as
//     zero = the least of its numbers, rounded to bfloat16
//     step = (the largest − zero) / 15, rounded once to bfloat16 (0 where zero was rounded above the largest)
//     code = (number − zero) / step, rounded once to a whole number (ties to even) and held to 0 … 15; 0 where step = 0
// and a number read back is zero + step · code.  A group that holds a number that is not finite, or whose range is not, gets NaN for
// step and zero, so that it reads back as NaN throughout.
//     codes  uint8    [block][kv_head][BT][dh / 2]      entry 2c in the low half of byte c, 2c + 1 in the high half
//     pairs  bfloat16 [block][kv_head][BT][dh / G][2]   (step, zero)
#pragma once
#include "common.cuh"

namespace {
__host__ __device__ constexpr int packed_group(int dh) {
    return dh <= 0 || dh % 16 != 0 || dh > 256 ? 0 : dh % 64 == 0 ? 64 : dh % 32 == 0 ? 32 : 16;
}
// (step, zero) from the 32-bit word that holds them
__device__ __forceinline__ float pair_step(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float pair_zero(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Eight codes of a 32-bit word in the tensor cores' own way: a bfloat16 whose upper eight bits are zero is its lower eight as a
// whole number, times 2^-133 (numbers below 2^-126 and those of the first binade above have the same spacing), and `mma.sync`
// takes such numbers exactly (checked on the device for all of 0 … 255).  So a code needs no conversion, only a mask: bits 0-3 of
// a half word are its code, bits 4-7 sixteen times its code; the factor 16 is taken out of the other operand or of the result,
// and 2^-133 of the whole product.
constexpr uint32_t PK_LOW = 0x000f000fu, PK_HIGH = 0x00f000f0u;

// the block that holds a token, or −1
__device__ __forceinline__ int packed_block(const int* __restrict__ table, int max_blocks, int n_blocks, int index) {
    const int blk = index >= 0 && index < max_blocks ? table[index] : -1;
    return blk < n_blocks ? blk : -1;
}
}  // namespace
