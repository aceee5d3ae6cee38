// Layout of the 4-bit KV cache and the device-side pieces that its kernels share.
//
// The cache is [pages][kv heads][block]: a page holds T tokens (a power of two, 16 to
// 256), a block the K and V rows of one kv head for a page's tokens,
// T * D + 4 * T * NG bytes (NG = D / groupsize scale groups a row):
//   * K codes  [T][4 g][D/32 w][8 i] nibbles: dim 32 w + 8 g + i of a token.  Lane group
//              g of a 16x16x32 MFMA reads its D/32 words at once, and k-step w then
//              covers dims [32 w, 32 w + 32), so that scale groups of 32 end with a k-step.
//   * V codes  [T/4][D/8 b][4 t][8 i] nibbles: dim 8 b + i of token 4 q + t.  One 16-byte
//              load gives a lane four tokens of its 8 dims: the tokens are the reduction
//              index of the second product, which an MFMA operand holds along a register.
//   * K scales, V scales: fp16 [T/4][NG][4 t].
// A code c stands for (c - 8) * s, as in the packed weights.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sm24_device.h"

namespace kv4 {

using sm24::float4_t;
using sm24::half2_t;
using sm24::half4_t;
using sm24::half8_t;
using sm24::u32x2;
using sm24::u32x4;

enum : int { F16 = 0, BF16 = 1 };

constexpr float kScaleMax = 65504.0f;  // largest finite fp16: scales saturate there

// Element `h` (raw 16 bits) of a row of fp16 or bf16.
template <int TYPE>
__device__ __forceinline__ float to_float(uint16_t h) {
  if constexpr (TYPE == F16) return (float)__builtin_bit_cast(_Float16, h);
  else return __builtin_bit_cast(float, (uint32_t)h << 16);
}
// Rounded to nearest, ties to even; NaN stays NaN.
template <int TYPE>
__device__ __forceinline__ uint16_t from_float(float x) {
  if constexpr (TYPE == F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else return __builtin_bit_cast(uint16_t, (__bf16)x);
}

template <int TYPE>
__device__ __forceinline__ void unpack8(const u32x4& w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = to_float<TYPE>((uint16_t)(w[i] & 0xFFFFu));
    x[2 * i + 1] = to_float<TYPE>((uint16_t)(w[i] >> 16));
  }
}
template <int TYPE>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; i++)
    w[i] = (uint32_t)from_float<TYPE>(x[2 * i]) | (uint32_t)from_float<TYPE>(x[2 * i + 1]) << 16;
  return w;
}

// Byte offsets inside a block (o: token within the page).
template <int D>
__device__ __forceinline__ int k_word(int o, int b) {  // word of dims [8 b, 8 b + 8)
  return o * (D / 2) + 4 * ((b & 3) * (D / 32) + (b >> 2));
}
template <int D>
__device__ __forceinline__ int v_word(int T, int o, int b) {
  return T * (D / 2) + (o >> 2) * (2 * D) + b * 16 + (o & 3) * 4;
}
template <int D, int NG>
__device__ __forceinline__ int k_scale(int T, int o, int n) {
  return T * D + ((o >> 2) * NG + n) * 8 + (o & 3) * 2;
}
template <int D, int NG>
__device__ __forceinline__ int v_scale(int T, int o, int n) {
  return k_scale<D, NG>(T, o, n) + 2 * T * NG;
}
template <int D, int NG>
__device__ __forceinline__ int block_bytes(int T) {
  return T * (D + 4 * NG);
}

}  // namespace kv4
