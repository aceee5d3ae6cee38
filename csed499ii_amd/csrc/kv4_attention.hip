// Attention over the 4-bit paged KV cache: launch plan and entry points.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv4_host.h"
#include "kv4_split.h"

namespace kv4 {

int compute_units(int dev) {
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
  return n;
}

struct Plan {
  int row_blocks, splits;
  long long tiles;
};

// Splits of the cache's length: enough workgroups for `cus` compute units four times over,
// each wave with a step at least.
Plan plan(int requests, int q_heads, int kv_heads, int max_q, int max_kv, int cus) {
  Plan p;
  p.row_blocks = (int)(((long long)max_q * (q_heads / kv_heads) + 15) / 16);
  p.tiles = (long long)requests * kv_heads * p.row_blocks;
  const long long most = ((long long)max_kv + kStep * kWaves - 1) / (kStep * kWaves);
  long long s = p.tiles > 0 ? (4ll * cus + p.tiles - 1) / p.tiles : 1;
  if (s > most) s = most;
  if (s < 1 || p.tiles * (long long)sizeof(uint32_t) > (long long)sm24::kCounterBytes) s = 1;
  p.splits = (int)s;
  return p;
}

int check(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int page_size, int num_pages,
          int max_pages, int groupsize, int max_q, int max_kv, float scale, int dtype) {
  const int err = check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if (tokens < 0 || requests < 0 || max_pages < 0 || max_q < 0 || max_kv < 0)
    return refuse("kv4_attention takes no negative sizes");
  if (q_heads <= 0 || q_heads % kv_heads != 0) return refuse("kv4_attention needs q_heads to be a multiple of kv_heads");
  if ((long long)max_pages * page_size > (1ll << 30)) return refuse("a block table row covers more than 2^30 tokens");
  if (!(scale > 0.f) || !isfinite(scale)) return refuse("kv4_attention needs a positive, finite scale");
  return MARLIN_HIP_OK;
}

}  // namespace kv4

extern "C" {

int marlin_hip_kv4_plan(int requests, int q_heads, int kv_heads, int head_dim, int groupsize, int max_q, int max_kv,
                        int sms, int* out) {
  const int err = kv4::check(0, requests, q_heads, kv_heads, head_dim, 16, 1, 0, groupsize, max_q, max_kv, 1.f, 0);
  if (err != MARLIN_HIP_OK) return err;
  const kv4::Plan p = kv4::plan(requests, q_heads, kv_heads, max_q, max_kv, sms > 0 ? sms : 256);
  out[0] = 0;
  out[1] = (int)(p.tiles * p.splits);
  out[2] = p.splits;
  return MARLIN_HIP_OK;
}

int marlin_hip_kv4_attention(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                             const void* cu_q, void* out, void* lse, int tokens, int requests, int q_heads,
                             int kv_heads, int head_dim, long long q_token_stride, long long q_head_stride,
                             int page_size, int num_pages, int max_pages, int groupsize, int max_q, int max_kv,
                             float scale, int dtype, int dev, hipStream_t stream) {
  using namespace kv4;
  int err = check(tokens, requests, q_heads, kv_heads, head_dim, page_size, num_pages, max_pages, groupsize, max_q,
                  max_kv, scale, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if ((q_token_stride | q_head_stride) & 7) return refuse("kv4_attention needs strides that are multiples of 8 elements");
  if (num_pages < 1) return refuse("kv4_attention needs a cache of at least one page");
  if (tokens == 0 || requests == 0 || max_q == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  Plan p = plan(requests, q_heads, kv_heads, max_q, max_kv, compute_units(dev));
  AttnArgs a{};
  a.q = q;
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = static_cast<const int32_t*>(block_table);
  a.kv_lens = static_cast<const int32_t*>(kv_lens);
  a.cu_q = static_cast<const int32_t*>(cu_q);
  a.out = out;
  a.lse = static_cast<float*>(lse);
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.tokens = tokens;
  a.requests = requests;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.num_pages = num_pages;
  a.max_pages = max_pages;
  a.log_page = 31 - __builtin_clz((unsigned)page_size);
  a.max_rows = 0x7FFFFFFF;
  a.c1 = scale * 1.4426950408889634f;
  if (p.splits > 1) {
    err = sm24::get_scratch(dev, stream, (size_t)p.tiles * p.splits * 16 * (head_dim + 2) * sizeof(float),
                            &a.counters, &a.partial);
    if (err != MARLIN_HIP_OK) return err;
    if (!a.counters) p.splits = 1;  // capturing, and this stream has no scratch yet
  }
  a.row_blocks = p.row_blocks;
  a.splits = p.splits;
  const long long blocks = p.tiles * p.splits;
  if (blocks > 0xFFFFFFll) return refuse("kv4_attention: more row blocks than one launch takes");
  dispatch(head_dim, groups(head_dim, groupsize), [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    const dim3 grid((unsigned)blocks), block(64 * kWaves);
    if (dtype == F16) hipLaunchKernelGGL((kv4_split_kernel<D, NG, F16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv4_split_kernel<D, NG, BF16>), grid, block, 0, stream, a);
  });
  return sm24::launch_error(hipGetLastError());
}

}  // extern "C"
