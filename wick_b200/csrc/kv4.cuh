// A paged cache whose keys and values are held in 4 bits: its form, and the value a code stands for.
//
// A page holds 64 positions.  Per page and key head, one behind the other (80 d bytes; d a multiple of 64):
//   keys' codes    [64, d / 2]        eight channels a 32-bit word: channel 8 w + i in bits 4 i .. 4 i + 3 of word w, the word then turned left by 3
//   values' codes  [64, d / 2]        two channels a byte, the even one in the low bits, the byte then turned left by 3; the pieces of 32 bytes of row t
//                                     change places with t (value_turn)
//   keys' scales   [64, d / 32]       a pair of bfloat16 numbers a (low half), b per group of 32 neighbouring channels
//   values' scales [64, d / 32]
// The value of code c is  bf16(b + a (1 + c / 16)),  one rounding.  A group's numbers x are stored with
//   a = bf16(16 (max - min) / 15),  b = bf16(min - a),  c = the whole number nearest to 16 (x - b) / a - 16, within 0 .. 15 (0 where a is 0);
// a group with a number that is none or is beyond 2^127, or whose a or b is beyond bfloat16's range, is stored as a = 0, b = NaN, so that it shows.
//
// Why this form.  1 + c / 16 is the bfloat16 number with the bits of 1 and c in the upper four bits of its mantissa (3 .. 6): two codes that lie
// there, one in either half of a register, are an AND-OR away from two numbers, and one fused multiply-add from two values.  Turned left by 3, a
// word of keys' codes has them there after shifts by 0, 4, 8 and 12.  A byte of values' codes, twice in each half of a register (one
// half a position), has its even channel there at once and the odd one after a shift by 4.  The value is a bfloat16 number by definition, so that every reader
// sees the same ones: those that compute from the codes, and those that open pages first.
#pragma once

#include "common.cuh"

namespace wick {
namespace kv4 {

constexpr int GROUP = 32;                                        // channels that share a scale

__host__ __device__ constexpr int head_bytes(int d) { return 80 * d; }
__host__ __device__ constexpr int value_codes(int d) { return 32 * d; }
__host__ __device__ constexpr int key_scales(int d) { return 64 * d; }
__host__ __device__ constexpr int value_scales(int d) { return 72 * d; }

// Which piece of 32 bytes of row t stands at place p: p ^ value_turn(t).  The kernels read a row's values eight lanes side by side, four rows at
// once (0, 3, 4 and 7, see attn_kv4.cu): with the turn those lie in 32 different banks of shared memory.
template <int D> __host__ __device__ __forceinline__ int value_turn(int t) {
    return D == 256 ? ((t & 1) | ((t >> 1) & 2)) : (D == 128 ? (t >> 2) & 1 : 0);
}
// Byte of row t of the values' codes that holds the channels of byte o of the row in order.
template <int D> __host__ __device__ __forceinline__ int value_byte(int t, int o) { return ((o >> 5) ^ value_turn<D>(t)) * 32 + (o & 31); }

constexpr uint32_t CODE_MASK = 0x00780078u, CODE_ONE = 0x3F803F80u;

// Two codes in bits 3 .. 6 of either half -> two values.  a2, b2: the scales of both.
__device__ __forceinline__ uint32_t two_values(uint32_t x, uint32_t a2, uint32_t b2) {
    uint32_t one, v;
    // (as one instruction: the compiler makes an AND and an OR of it, a third of all instructions of a page)
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(one) : "r"(x), "r"(CODE_MASK), "r"(CODE_ONE));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v) : "r"(one), "r"(a2), "r"(b2));
    return v;
}
__device__ __forceinline__ uint32_t low_halves(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x7632); }
// Whether a pair of scales stands for values that are no numbers.
__device__ __forceinline__ bool no_number(uint32_t scale) { return (scale & 0x7F80u) == 0x7F80u || (scale & 0x7F800000u) == 0x7F800000u; }

// A word of keys' codes: v[i] has channels i and i + 4.
__device__ __forceinline__ void key_word(uint32_t w, uint32_t a2, uint32_t b2, uint32_t (&v)[4]) {
    v[0] = two_values(w, a2, b2);
    v[1] = two_values(w >> 4, a2, b2);
    v[2] = two_values(w >> 8, a2, b2);
    v[3] = two_values(__funnelshift_r(w, w, 12), a2, b2);        // (code 7 goes around the word's end)
}
// Byte k of two positions' words of values' codes (low half: of w0): even and odd channel of both.
template <int k>
__device__ __forceinline__ void value_pair(uint32_t w0, uint32_t w1, uint32_t a2, uint32_t b2, uint32_t& even, uint32_t& odd) {
    const uint32_t x = __byte_perm(w0, w1, k | k << 4 | (k + 4) << 8 | (k + 4) << 12);
    even = two_values(x, a2, b2);
    odd = two_values(x >> 4, a2, b2);
}

}  // namespace kv4
}  // namespace wick
