// Quantizing writes into the 4-bit KV cache: what the kernels that append rows share.
#pragma once
#include <type_traits>

#include "kv4_device.h"

namespace kv4 {

constexpr int kRowThreads = 256;

struct RowArgs {
  void* k;
  void* v;
  uint8_t* cache;
  const int32_t* slots;
  long long kt, kh, vt, vh;  // strides in elements
  int tokens, heads, log_page, num_pages;
};

// (In fp32 with a flag for NaN, over the lanes by shuffles, and codes inserted one by one, the
// append took 24.5 us where it now takes 20.0: it was bound by its operations.)
// Bits of the largest |x| over the 8 dims and the G/8 lanes of a scale group: of fp16 and of
// bf16 the bits without the sign order as the values do, and a NaN's are above infinity's.
template <int G>
__device__ __forceinline__ uint32_t group_max(const u32x4& raw) {
  typedef uint16_t pair __attribute__((ext_vector_type(2)));
  auto magnitude = [](uint32_t w) { return __builtin_bit_cast(pair, w & 0x7FFF7FFFu); };
  const pair p = __builtin_elementwise_max(__builtin_elementwise_max(magnitude(raw.x), magnitude(raw.y)),
                                           __builtin_elementwise_max(magnitude(raw.z), magnitude(raw.w)));
  uint32_t m = max((uint32_t)p.x, (uint32_t)p.y);
  auto over = [&](auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, c, 0xF, 0xF, true));
  };
  over(std::integral_constant<int, 0xB1>());                            // lanes 1 0 3 2 of four
  over(std::integral_constant<int, 0x4E>());                            // 2 3 0 1
  if constexpr (G >= 64) over(std::integral_constant<int, 0x141>());    // 7 ... 0 of eight
  if constexpr (G >= 128) over(std::integral_constant<int, 0x140>());   // 15 ... 0 of sixteen
  return m;
}

// Eight dims [8 b, 8 b + 8) of a row (raw, as in memory) into a slot that exists; the D/8 lanes of the
// row call it together.
template <int D, int NG, int TYPE>
__device__ __forceinline__ void write_row(const RowArgs& a, int slot, int head, int b, bool is_v, const u32x4& raw) {
  constexpr int G = D / NG;
  float x[8];
  unpack8<TYPE>(raw, x);
  const uint32_t bits = group_max<G>(raw);
  const float amax = TYPE == F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __builtin_bit_cast(float, bits << 16);
  // the weights' quantizer: fp16(max * 2/15), saturating (fminf would drop a NaN)
  float scaled = amax * (2.0f / 15.0f);
  if (scaled > kScaleMax) {  // the quotients stay finite
    scaled = kScaleMax;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __builtin_amdgcn_fmed3f(x[i], -8.f * kScaleMax, 8.f * kScaleMax);
  }
  const _Float16 s16 = (_Float16)scaled;
  const float s = (float)s16;
  // x / s correctly rounded where that decides a code: one Newton step on x * (1 / s), within
  // +-8 (ties such as 2.5 are exact and must stay so).  Four codes are summed in fp32, where
  // 16 bits are exact: 8 + 8 16 + 8 16^2 + 8 16^3 is their offset.
  const float inv = __builtin_amdgcn_rcpf(s);
  float half[2] = {34952.f, 34952.f};
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float q0 = x[i] * inv;
    const float q = __builtin_fmaf(__builtin_fmaf(-q0, s, x[i]), inv, q0);
    const float c = __builtin_amdgcn_fmed3f(__builtin_rintf(q), -8.f, 7.f);
    half[i / 4] = __builtin_fmaf(c, (float)(1 << (4 * (i % 4))), half[i / 4]);
  }
  uint32_t word = (uint32_t)half[0] | (uint32_t)half[1] << 16;
  if (!(s > 0.f)) word = 0x88888888u;
  const int T = 1 << a.log_page, o = slot & (T - 1);
  uint8_t* block = a.cache + ((size_t)(slot >> a.log_page) * a.heads + head) * block_bytes<D, NG>(T);
  *reinterpret_cast<uint32_t*>(block + (is_v ? v_word<D>(T, o, b) : k_word<D>(o, b))) = word;
  if (b % (G / 8) == 0) {
    const int n = b / (G / 8);
    *reinterpret_cast<_Float16*>(block + (is_v ? v_scale<D, NG>(T, o, n) : k_scale<D, NG>(T, o, n))) = s16;
  }
}

}  // namespace kv4
