// Rows of a step turned by their positions on the way into the 4-bit KV cache: q is turned and
// written out, k turned, rounded to its type and quantized, v quantized, in one launch.
//
// K thereby is not written and read once more between the two.  Bound by memory: of 4096 tokens
// of 32 heads and 32 kv heads q, k and v are read, q and the cache's rows written: 163 MB in 32 us, 5.1 TB/s,
// what a large copy reaches.  24 tokens 4 us, latency.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4_host.h"
#include "kv4_rows.h"
#include "rotary_device.h"

namespace kv4 {

struct AppendRotaryArgs {
  RowArgs rows;
  rotary::Rows q;
  rotary::Shape shape;            // of q's workgroups
  int q_parts, q_heads_per;       // workgroups of a token tile, heads of each
  int q_blocks, kv_blocks;        // workgroups of q, then of K, then of V
  int parts, heads_per;           // of K's and V's token tiles
};

// The first workgroups turn q (rotary_device.h); the others write K and V as the plain append
// does, consecutive tokens of a head, and keep a token's angles for several heads.
template <int D, int NG, int TYPE, bool INTERLEAVED, bool ALIGNED>
__global__ __launch_bounds__(kRowThreads) void kv4_append_rotary_kernel(AppendRotaryArgs a) {
  static_assert(kRowThreads == rotary::kThreads, "");
  const int block = (int)blockIdx.x;
  if (block < a.q_blocks) {
    const int tile = block / a.q_parts, head0 = (block - tile * a.q_parts) * a.q_heads_per;
    rotary::turn_rows<TYPE, INTERLEAVED, ALIGNED>(a.q, a.shape, tile * a.shape.tokens, head0,
                                                  min(head0 + a.q_heads_per, a.q.heads));
    return;
  }
  constexpr int B = D / 8;
  const bool is_v = block - a.q_blocks >= a.kv_blocks;
  const int i = block - a.q_blocks - (is_v ? a.kv_blocks : 0);
  const int tile = i / a.parts, head0 = (i - tile * a.parts) * a.heads_per;
  const int head1 = min(head0 + a.heads_per, a.rows.heads);
  const int token = tile * (kRowThreads / B) + (int)threadIdx.x / B, b = threadIdx.x % B;
  if (token >= a.rows.tokens) return;
  const int slot = a.rows.slots[token];
  if (slot < 0 || (slot >> a.rows.log_page) >= a.rows.num_pages) return;  // (all lanes of the row)
  const long long stride = is_v ? a.rows.vh : a.rows.kh;
  const uint16_t* row = static_cast<const uint16_t*>(is_v ? a.rows.v : a.rows.k);
  row += token * (is_v ? a.rows.vt : a.rows.kt) + head0 * stride;
  if (is_v) {
    for (int h = head0; h < head1; h++, row += stride)
      write_row<D, NG, TYPE>(a.rows, slot, h, b, true, *reinterpret_cast<const u32x4*>(row + 8 * b));
    return;
  }
  const rotary::double2_t* at = a.q.angles + (size_t)token * a.q.pairs;
  const rotary::Turn<TYPE, INTERLEAVED, ALIGNED> turn(at, a.q.pairs, b);
  for (int h = head0; h < head1; h++, row += stride) {
    const u32x4 raw = turn(*reinterpret_cast<const u32x4*>(row + 8 * b), row, at, a.q.pairs, b);
    write_row<D, NG, TYPE>(a.rows, slot, h, b, false, raw);
  }
}

}  // namespace kv4

extern "C" int marlin_hip_kv4_append_rotary(
    const void* q, const void* k, const void* v, const void* angles, void* q_out, void* cache, const void* slots,
    int tokens, int q_heads, int kv_heads, int head_dim, int rotary_dim, long long q_token_stride,
    long long q_head_stride, long long k_token_stride, long long k_head_stride, long long v_token_stride,
    long long v_head_stride, long long out_token_stride, long long out_head_stride, int page_size, int num_pages,
    int groupsize, int interleaved, int dtype, int dev, hipStream_t stream) {
  using namespace kv4;
  const int err = check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if (tokens < 0 || q_heads < 0) return refuse("kv4_append_rotary takes no negative sizes");
  if (tokens > (1 << 30)) return refuse("more rows than one launch of the KV cache takes");
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return refuse("kv4_append_rotary turns an even number of dims, 2 at least and head_dim at most");
  if ((q_token_stride | q_head_stride | k_token_stride | k_head_stride | v_token_stride | v_head_stride |
       out_token_stride | out_head_stride) & 7)
    return refuse("kv4_append_rotary needs strides that are multiples of 8 elements");
  if (tokens == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const int pairs = rotary_dim / 2;
  AppendRotaryArgs a{};
  a.rows = RowArgs{const_cast<void*>(k), const_cast<void*>(v), static_cast<uint8_t*>(cache),
                   static_cast<const int32_t*>(slots), k_token_stride, k_head_stride, v_token_stride, v_head_stride,
                   tokens, kv_heads, 31 - __builtin_clz((unsigned)page_size), num_pages};
  a.q = rotary::Rows{static_cast<const uint16_t*>(q), static_cast<uint16_t*>(q_out),
                     static_cast<const rotary::double2_t*>(angles), q_token_stride, q_head_stride, out_token_stride,
                     out_head_stride, tokens, q_heads, head_dim, pairs};
  long long q_blocks = 0;
  if (q_heads > 0) {
    a.shape = rotary::shape_of(head_dim, pairs, interleaved != 0, q_heads);
    const int tiles = (tokens + a.shape.tokens - 1) / a.shape.tokens;
    const int rounds = (q_heads + a.shape.heads - 1) / a.shape.heads, per = tiles < 512 ? 1 : rounds;
    a.q_heads_per = per * a.shape.heads;
    a.q_parts = (rounds + per - 1) / per;
    q_blocks = (long long)tiles * a.q_parts;
  }
  const int per_block = kRowThreads / (head_dim / 8), tiles = (tokens + per_block - 1) / per_block;
  // Heads of a workgroup, which share the tokens' angles: one where there are few workgroups.
  a.heads_per = (long long)tiles * kv_heads >= 2048 ? 4 : 1;
  a.parts = (kv_heads + a.heads_per - 1) / a.heads_per;
  const long long kv_blocks = (long long)tiles * a.parts;
  if (q_blocks + 2 * kv_blocks > 0x7FFFFF) return refuse("more rows than one launch of the KV cache takes");
  a.q_blocks = (int)q_blocks;
  a.kv_blocks = (int)kv_blocks;
  const dim3 grid((unsigned)(q_blocks + 2 * kv_blocks)), block(kRowThreads);
  rotary::dispatch(pairs, interleaved != 0, [&](auto i, auto al) {
    constexpr bool I = decltype(i)::value, AL = decltype(al)::value;
    dispatch(head_dim, groups(head_dim, groupsize), [&](auto d, auto g) {
      constexpr int D = decltype(d)::value, NG = decltype(g)::value;
      if (dtype == F16) hipLaunchKernelGGL((kv4_append_rotary_kernel<D, NG, F16, I, AL>), grid, block, 0, stream, a);
      else hipLaunchKernelGGL((kv4_append_rotary_kernel<D, NG, BF16, I, AL>), grid, block, 0, stream, a);
    });
  });
  return sm24::launch_error(hipGetLastError());
}
