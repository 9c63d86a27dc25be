// Layout of the paged KV cache held in 4 bits, shared by the kernels that write it and the attention that reads it.
//
// Groups of 16 neighbouring dims of a head have a scale; codes are e2m1. A scale byte is the upper half of an f16 behind its sign: 5 exponent and 3
// mantissa bits. An e4m3 scale, with its 4 exponent bits, would lose keys or values whose largest magnitude is below 0.1, or need another factor
// a layer.
// A layer's cache is [num_blocks][Hkv][block_size / 16] cells. A cell is 16 neighbouring tokens of a kv head, 18 D bytes:
//   key codes    [16 tokens][D / 2]    e2m1 pairs, even dim in the low nibble
//   value codes  [16 tokens][D / 2]    the same, but 16-byte piece n (of the cell's D / 2) lies at n ^ 2 (token / 4)
//   key scales   [16 tokens][D / 16]
//   value scales [D / 16][16 tokens]
// What a warp's matrix instruction takes from a cell is then one vector load a lane for each part: a lane that holds four keys 4t..4t+3 finds
// their value scales in one word, and the four rows that a half-warp reads at a time lie in different banks of shared memory. The page's cells of
// a head are one piece of memory, so one bulk copy fetches what a page has for a head. Code times scale has at most 6 significant bits and
// scales end at 10240: exact in f16 and bf16.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace b200 {

constexpr int kCellTokens = 16;
constexpr float kMostFp4Scale = 10240.f;             // (byte 0xe2)
template <int D>
struct Fp4Cell {
  static constexpr int kRow = D / 2;                 // bytes of a token's codes
  static constexpr int kScales = D / 16;             // scales of a token
  static constexpr int kValues = kCellTokens * kRow; // where the value codes begin
  static constexpr int kKeyScales = 2 * kValues;
  static constexpr int kValueScales = kKeyScales + kCellTokens * kScales;
  static constexpr int kBytes = kValueScales + kCellTokens * kScales;
  // Byte `at` of a token's value codes.
  static __host__ __device__ constexpr int value_at(int token, int at) {
    return kValues + ((token * kRow + at) ^ (32 * (token >> 2)));
  }
};

#ifdef __CUDACC__
__device__ __forceinline__ float fp4_scale_value(uint8_t b) { return __half2float(__ushort_as_half((unsigned short)(b << 7))); }
// The nearest scale to v >= 0, ties to even; saturates, NaN stays NaN.
__device__ __forceinline__ uint8_t fp4_scale_byte(float v) {
  const uint32_t u = __float_as_uint(v);
  if (u > 0x7f800000u) return 0xff;
  if (v >= kMostFp4Scale) return 0xe2;
  if (v < 6.103515625e-5f) return (uint8_t)__float2int_rn(v * 131072.f);       // below 2^-14: multiples of 2^-17
  return (uint8_t)(((u + 0x7ffffu + (u >> 20 & 1)) >> 20) - ((127 - 15) << 3));
}
#endif

}  // namespace b200
