// Rotary positions: the table of a step's angles, and rows turned by it.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kv4_host.h"
#include "rotary_device.h"

namespace rotary {

// A frequency is a fixed-point number of turns a position, 2^-64 of a turn each: its product
// with the position, modulo 2^64, is the exact place on the circle, at any distance and below
// zero too.  sincospi then needs no reduction.  One thread a pair; bound by its latency (1.4 us
// for a token) or by the write of 16 bytes a pair (2.6 us for 2047 tokens of 40 pairs).
__global__ __launch_bounds__(kThreads) void rotary_angles_kernel(const int32_t* positions, const uint64_t* freqs,
                                                                 double2_t* out, unsigned pairs, long long total,
                                                                 double factor) {
  const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (i >= total) return;
  const unsigned token = (unsigned)(i / pairs), pair = (unsigned)(i - (long long)token * pairs);
  const uint64_t place = (uint64_t)(int64_t)positions[token] * freqs[pair];
  double s, c;
  sincospi((double)(int64_t)place * 0x1p-63, &s, &c);
  out[i] = (double2_t){c * factor, s * factor};
}

template <int TYPE, bool INTERLEAVED, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Rows a, Shape s, int heads_per) {
  const int head0 = (int)blockIdx.y * heads_per;
  turn_rows<TYPE, INTERLEAVED, ALIGNED>(a, s, (int)blockIdx.x * s.tokens, head0, min(head0 + heads_per, a.heads));
}

}  // namespace rotary

extern "C" {

int marlin_hip_rotary_angles(const void* positions, const void* freqs, void* angles, int tokens, int pairs,
                             double factor, int dev, hipStream_t stream) {
  if (tokens < 0 || pairs < 0) return kv4::refuse("rotary_angles takes no negative sizes");
  const long long total = (long long)tokens * pairs;
  if (total > 0xFFFFFF00ll) return kv4::refuse("rotary_angles: too many angles for one launch");
  if (total == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const dim3 grid((unsigned)((total + rotary::kThreads - 1) / rotary::kThreads)), block(rotary::kThreads);
  hipLaunchKernelGGL(rotary::rotary_angles_kernel, grid, block, 0, stream, static_cast<const int32_t*>(positions),
                     static_cast<const uint64_t*>(freqs), static_cast<rotary::double2_t*>(angles), (unsigned)pairs, total,
                     factor);
  return sm24::launch_error(hipGetLastError());
}

int marlin_hip_rotary(const void* x, const void* angles, void* out, int tokens, int heads, int head_dim, int rotary_dim,
                      long long x_token_stride, long long x_head_stride, long long out_token_stride,
                      long long out_head_stride, int interleaved, int dtype, int dev, hipStream_t stream) {
  if (tokens < 0 || heads < 0) return kv4::refuse("rotary takes no negative sizes");
  if (head_dim < 8 || head_dim > 1024 || head_dim % 8 != 0 || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return kv4::refuse("rotary takes heads of a multiple of 8 dims, 1024 at most, of which an even number turns");
  if ((x_token_stride | x_head_stride | out_token_stride | out_head_stride) & 7)
    return kv4::refuse("rotary needs strides that are multiples of 8 elements");
  if (dtype != 0 && dtype != 1) {
    sm24::set_error("marlin_hip: rotary has kernels for fp16 and bf16 rows");
    return MARLIN_HIP_ERR_KERN_SHAPE;
  }
  if (tokens == 0 || heads == 0) return MARLIN_HIP_OK;
  const int pairs = rotary_dim / 2;
  const rotary::Shape s = rotary::shape_of(head_dim, pairs, interleaved != 0, heads);
  const unsigned tiles = ((unsigned)tokens + s.tokens - 1) / s.tokens;
  if (tiles > 0xFFFFFF) return kv4::refuse("rotary: more tokens than one launch takes");
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const rotary::Rows a{static_cast<const uint16_t*>(x), static_cast<uint16_t*>(out),
                       static_cast<const rotary::double2_t*>(angles), x_token_stride, x_head_stride, out_token_stride,
                       out_head_stride, tokens, heads, head_dim, pairs};
  // Few tokens: a workgroup for each round of heads; many: a thread keeps its angles for all of them.
  const int rounds = (heads + s.heads - 1) / s.heads;
  int per = tiles < 512 ? 1 : rounds;
  if ((rounds + per - 1) / per > 65535) per = (rounds + 65534) / 65535;
  const dim3 grid(tiles, (unsigned)((rounds + per - 1) / per)), block(rotary::kThreads);
  rotary::dispatch(pairs, interleaved != 0, [&](auto i, auto al) {
    constexpr bool I = decltype(i)::value, AL = decltype(al)::value;
    if (dtype == kv4::F16) hipLaunchKernelGGL((rotary::rotary_kernel<kv4::F16, I, AL>), grid, block, 0, stream, a, s, per * s.heads);
    else hipLaunchKernelGGL((rotary::rotary_kernel<kv4::BF16, I, AL>), grid, block, 0, stream, a, s, per * s.heads);
  });
  return sm24::launch_error(hipGetLastError());
}

}  // extern "C"
