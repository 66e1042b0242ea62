// The format of a cache whose keys and values are held in 4 bits (cache_4bit.cu writes and reads it back, attention_4bit.cu attends over it).
//
// The numbers.  A head of D numbers is cut into G = D / 32 groups of 32 neighbouring ones.  A group of a token is held as 32
// codes n of 4 bits, a scale s and a least value m, both bfloat16, and stands for m + s n:
//   m = the least of the 32, rounded down to bfloat16;  s = (greatest - m) / 15, rounded up to bfloat16;
//   n = the nearest whole number to (x - m) / s, 0..15.
// Down and up, so that no number of the group lies outside what the codes reach and every one is met within s / 2.  A group that
// holds something not finite, or whose m or s would not be, has s = NaN, m = 0, n = 0: whoever sees it gets NaN, and a key that is
// masked adds 0 * m = 0.  A scale below 2^-126 (the inverse would overflow) is zero: the numbers then differ by less than 2^-122.
//
// Groups of 32 rather than whole heads: a key's few large channels cost precision only among their 31 neighbours.  5 bits a number
// against 16 of the bfloat16 cache.
//
// The bytes of one block (64 tokens) of one head, 20 * 64 * G each for keys and for values:
//   keys:   codes, 32-bit words [64 tokens][4][G]; then [64 tokens][G] pairs (s in the low half, m in the high half)
//           word [t][c][g]: numbers 32 g + 8 c + 2 i + h of token t at bits 4 i + 16 h (i = 0..3, h = 0, 1)
//   values: codes, 32-bit words [4][G][8][4][2]; then s [64 tokens][G]; then m [G][64 tokens]
//           word [a][g][r][c][j]: number 32 g + 16 j + 8 e + r of token 16 a + 4 c + 2 p + h at bits 4 (2 p + e) + 16 h
// Both are the order in which a lane of a tensor-core fragment (m16n8k16) wants them: w & 0x000f000f is a register of two float16
// numbers n 2^-24, w & 0x00f000f0 one of two numbers 16 n 2^-24, and (w >> 8) has the other four codes.  A value word holds four
// neighbouring tokens; whoever appends owns the word of its first token in it and keeps what earlier steps left in the others.
#pragma once
#include "common.cuh"

namespace cache4 {

constexpr int block_bytes(int d) { return 40 * d; }                 // of one head's keys, or values
constexpr int code_bytes(int d) { return 32 * d; }                  // the codes among them

// Numbers of at most this size are held in float16 times 2^-e: the largest then lies in 2^7 .. 2^15, so that what is 2^-21 of it still has float16's 11
// bits.  e is a multiple of 8, so that most blocks of a cache have the same one; a scale and its inverse are normal float32 numbers.
__device__ __forceinline__ int half_exponent(float largest) {
    const int exponent = (int)(__float_as_uint(largest) >> 23) - 127;
    return max(-112, ((exponent - 7) >> 3) * 8);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Float16 blocks (cache_4bit.cu makes them, attention_tcgen05.cu reads them) have a power of two a block and head, for keys and for values.  Where a
// token's largest number is of another step of 2^8 and not of the next one, the block's tokens have powers of their own: 2^-8 of the block's for each of
// the token's steps, so that a large token takes no bits from its neighbours.  A mark a token says how many:
//   keys' scale positive: the low four bits are the groups of 32 values that are not numbers (held as zeros), the high four the values' steps; looked at
//     where the values' scale is negative;
//   keys' scale negative: the low four bits are the keys' steps, the high four the values', up to 14; 15 there: the token has no steps, and the low bits are its
//     groups that are not numbers, all four if it had steps (whoever sees such a token gets NaN in its whole head).
__device__ __forceinline__ int key_steps(uint8_t mark, bool unlike_keys) { return unlike_keys && mark < 0xf0 ? mark & 15 : 0; }
__device__ __forceinline__ int value_steps(uint8_t mark, bool unlike_keys) { return unlike_keys && mark >= 0xf0 ? 0 : mark >> 4; }
__device__ __forceinline__ unsigned marked_groups(uint8_t mark, bool unlike_keys) { return unlike_keys && mark < 0xf0 ? 0u : mark & 15u; }

inline bool takes(int heads, int kv_heads, int head_dim) {
    return kv_heads > 0 && kv_heads <= 65535 && heads % kv_heads == 0 && heads / kv_heads >= 1 && heads / kv_heads <= 16 &&
           (head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128);
}

}  // namespace cache4
