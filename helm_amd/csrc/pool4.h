// The 4-bit KV pool's pages and their elements (pool4.hip, pool4_attn.hip).
//
// A value is an E2M1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives) times
// its group's power of two; a group is 32 dims of one token and KV head, its
// exponent one byte, e + 127.  e is the smallest with |largest| <= 7 * 2^e,
// -125 <= e <= 125; values are rounded to the nearest code (ties to the even
// one) and those above 6 are 6.  No value is further from its code than half
// the step it would have (6 to 7 lie within 1 of 6, the step there being 2).
// On N(0, 1) rows that keeps an rms error of 0.1119 of the values' rms, against
// 0.1149 where the group's exponent is the largest value's (which cuts 6 to 8
// down to 6) and 0.1155 where no value is cut.  A group that holds an infinity
// or NaN has the exponent byte 255 and stands for NaN; bytes that no write leaves
// (below 2, 253, 254) are hidden tokens' only, and attention takes 253 and 254 for 255.
//
// The limits of e keep every code times 2^e a normal bf16 and fp32 number, so
// that the matrix cores' bf16 operands hold K and V exactly (f16 would not: its
// largest group reaches 2^16).
//
// A page is a row of tiles of 16 tokens per KV head, 17 D bytes each:
//   [K codes 8D][V codes 8D][K exponents D/2][V exponents D/2]
// laid out so that one lane's operands of the 16 x 16 matrix instructions are
// one wide load each, and a wave's load covers a tile's part without gaps:
//   K codes      token-major, dim 2j in the low half of byte j of the row;
//   V codes      chunks of D / 16 dims, chunk-major, then token: a lane reads
//                its chunk of four consecutive tokens at once;
//   K exponents  token-major, one byte a group;
//   V exponents  group-major, one byte a token: four tokens are one word.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace helm {

constexpr int kP4Tok = 16;     // tokens per tile
constexpr int kP4Group = 32;   // dims per exponent

template <int D> struct P4 {
  static constexpr int kVc = 8 * D;            // V codes
  static constexpr int kKe = 16 * D;           // K exponents
  static constexpr int kVe = 16 * D + D / 2;   // V exponents
  static constexpr int kBytes = 17 * D;
  static constexpr int kGroups = D / kP4Group;
  static constexpr int kChunk = D / 32;        // bytes of a V chunk (D / 16 dims)
};

// The group exponent byte of a largest magnitude, from its fp32 bits: 7 is
// 1.75 * 4, so the byte is the magnitude's exponent - 2, one more above 1.75.
__device__ __forceinline__ uint32_t p4_exponent(uint32_t abs_bits) {
  if (abs_bits >= 0x7f800000u) return 255u;
  const int e = (int)((abs_bits + 0x1fffffu) >> 23) - 2;
  return (uint32_t)min(252, max(2, e));
}
__device__ __forceinline__ float p4_scale(uint32_t e) { return __uint_as_float(e << 23); }

}  // namespace helm
