// Attention over the 4-bit paged KV cache: launch plan and entry points.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kv4_host.h"
#include "kv4_split.h"

namespace kv4 {

hipError_t launch_prompt(const AttnArgs& a, int workgroups, int head_dim, int ng, int dtype, hipStream_t stream);

// Requests of at most so many rows (new tokens times the query heads of a kv head) go to the
// split kernel, the others to the prompt kernel, each of which passes over the other's.  The
// split kernel's time grows with the rows, the prompt kernel's is the same up to 256: 12
// requests of 4096 tokens on 8 heads of 128 dims, 64, 80, 96 and 128 rows, 53, 55, 70 and 82
// us beside 72 to 73; with groups of 32, 128, 144 and 160 rows, 104, 123 and 133 beside 108,
// 125 and 125.
// Few tiles leave the prompt kernel's large parts waiting: one request of 8192 tokens, 24 us
// beside 34 at 64 rows, 41 beside 57 at 256.
int split_rows(int requests, int kv_heads, int head_dim, int ng, int cus) {
  if ((long long)requests * kv_heads <= cus / 16) return 256;
  return head_dim == 128 && ng == 4 ? 144 : 80;
}

// (the query takes the host 0.2 us of each call, so its answer is kept)
int compute_units(int dev) {
  static std::atomic<int> known[64];
  if (dev >= 0 && dev < 64 && known[dev].load(std::memory_order_relaxed) > 0)
    return known[dev].load(std::memory_order_relaxed);
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
  if (dev >= 0 && dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

struct Plan {
  int workgroups, log_kw, lead, pieces;
  bool split;  // a tile may be divided: the call needs scratch
  bool rest;   // the prompt kernel's last blocks, too, where they are few
};

// Two workgroups of eight waves fill a compute unit.  All eight waves take one block of 16
// rows and meet in LDS: a piece of a block costs its write and read in memory, and so there
// are few (one request of 131072 tokens on 8 heads: 38.4 us with eight, 63 with four, 113 with two; 64 requests of
// 4096: 61, 65, 66).  From two blocks a workgroup on, a workgroup goes through many short
// ones instead, and two waves take a block (64 requests of 4096 tokens on 32 heads: 220 us
// with eight, 215 with four, 210 with two; 200 of 1000: 208, 187, 177).
Plan plan(int requests, int q_heads, int kv_heads, int max_q, int max_kv, int cus) {
  Plan p{};
  const long long row_blocks = ((long long)max_q * (q_heads / kv_heads) + 15) / 16;
  const long long steps = ((long long)max_kv + kStep - 1) / kStep;
  const long long most = 2ll * cus;
  const long long blocks = requests * row_blocks * kv_heads;
  p.log_kw = blocks <= 2 * most ? kLogWaves : 1;
  const int hw = kWaves >> p.log_kw;
  const long long units = steps < 1 ? 1 : (steps + (1 << p.log_kw) - 1) >> p.log_kw;
  const long long w = requests * ((row_blocks * kv_heads + hw - 1) / hw) * units;
  p.lead = w > most ? kLead : 0;
  p.workgroups = (int)(w < most ? w : most);
  p.split = units > 1;
  return p;
}

// The prompt kernel: a workgroup of eight waves fills a compute unit.  Fewer tiles (256 rows
// of a head) than compute units are divided over their tokens on the device, which knows the
// lengths; this is the grid, which bounds the tiles by the tokens.
Plan prompt_plan(int tokens, int requests, int q_heads, int kv_heads, int max_q, int max_kv, int max_rows, int cus) {
  const long long group = q_heads / kv_heads, rows = tokens * group;
  long long kinds = rows / kPromptRows + (requests < rows / (max_rows + 1) ? requests : rows / (max_rows + 1));
  const long long most = requests * ((max_q * group + kPromptRows - 1) / kPromptRows);
  if (kinds > most) kinds = most;
  Plan p{};
  p.pieces = cus / kv_heads;
  p.split = max_kv > kTile && p.pieces > 1;
  // (of one fresh prompt the last blocks see few tokens: 60 us whole, 67 with workgroups for
  // them, 1500 tokens on 64 and 8 heads)
  p.rest = p.split && kinds > p.pieces && (requests > 1 || max_kv >= 2ll * max_q);
  const long long w = (p.rest ? kinds + p.pieces : p.split && kinds < p.pieces ? p.pieces : kinds) * kv_heads;
  p.workgroups = w > 0x7FFFFF ? -1 : (int)w;
  return p;
}

// Which kernels a call launches, and what each is given.
struct Choice {
  bool prompts, split;
  int few_rows, split_q;  // rows of a request that go to the split kernel, new tokens of one
};
Choice choose(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int ng, int max_q, bool cu, int cus) {
  Choice c;
  const int group = q_heads / kv_heads;
  c.few_rows = split_rows(requests, kv_heads, head_dim, ng, cus);
  c.prompts = (long long)max_q * group > c.few_rows;
  c.split_q = c.prompts ? c.few_rows / group : max_q;
  // (where the tokens say that no request can be short, the prompt kernel takes all)
  c.split = !c.prompts || (cu && c.split_q > 0 && tokens <= c.split_q + (long long)(requests - 1) * max_q);
  return c;
}

int check(int tokens, int requests, int q_heads, int kv_heads, int head_dim, int page_size, int num_pages,
          int max_pages, int groupsize, int max_q, int max_kv, float scale, int dtype) {
  const int err = check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if (tokens < 0 || requests < 0 || max_pages < 0 || max_q < 0 || max_kv < 0)
    return refuse("kv4_attention takes no negative sizes");
  if (q_heads <= 0 || q_heads % kv_heads != 0) return refuse("kv4_attention needs q_heads to be a multiple of kv_heads");
  if ((long long)tokens * (q_heads / kv_heads) > (1ll << 30) || (long long)max_q * (q_heads / kv_heads) > (1ll << 30))
    return refuse("kv4_attention takes at most 2^30 rows (tokens times query heads of a kv head)");
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
  out[0] = out[1] = out[2] = 0;
  if (requests == 0 || max_q == 0) return MARLIN_HIP_OK;
  using namespace kv4;
  const int cus = sms > 0 ? sms : 256, ng = groups(head_dim, groupsize), most = (1 << 30) / (q_heads / kv_heads);
  const int tokens = (long long)requests * max_q < most ? requests * max_q : most;
  const Choice c = choose(tokens, requests, q_heads, kv_heads, head_dim, ng, max_q, max_q > 1, cus);
  if (requests > kMaxRequests) requests = kMaxRequests;  // (of the first launch)
  if (c.split_q > 0) {
    const Plan p = plan(requests, q_heads, kv_heads, c.split_q, max_kv, cus);
    out[1] = p.workgroups;
    out[2] = p.split;
  }
  if (c.prompts) {
    const Plan p = prompt_plan(tokens, requests, q_heads, kv_heads, max_q, max_kv, c.split ? c.few_rows : 0, cus);
    if (p.workgroups < 0) return refuse("kv4_attention: too many rows for one launch");
    out[0] = 1;
    out[1] = p.workgroups;
    out[2] |= p.split;  // (shorter requests may go to the other kernel)
  }
  return MARLIN_HIP_OK;
}

int marlin_hip_kv4_attention_ctx(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                                 const void* cu_q, const void* context_lens, void* out, void* lse, int tokens,
                                 int requests, int q_heads, int kv_heads, int head_dim, long long q_token_stride,
                                 long long q_head_stride, int page_size, int num_pages, int max_pages, int groupsize,
                                 int max_q, int max_kv, float scale, int dtype, int dev, hipStream_t stream) {
  using namespace kv4;
  // (a bound that may be far above what there is, e.g. a fixed one of all steps: the choice of
  // kernels and their grids go by rows that exist)
  if (tokens >= 0 && max_q > tokens) max_q = tokens;
  int err = check(tokens, requests, q_heads, kv_heads, head_dim, page_size, num_pages, max_pages, groupsize, max_q,
                  max_kv, scale, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if ((q_token_stride | q_head_stride) & 7) return refuse("kv4_attention needs strides that are multiples of 8 elements");
  if (num_pages < 1) return refuse("kv4_attention needs a cache of at least one page");
  if (tokens == 0 || requests == 0 || max_q == 0) return MARLIN_HIP_OK;
  // (request i is token i: its row of q, and of the output, must be there)
  if (cu_q == nullptr && tokens < requests) return refuse("kv4_attention without cu_q needs a token for every request");
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  AttnArgs a{};
  a.q = q;
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = static_cast<const int32_t*>(block_table);
  a.kv_lens = static_cast<const int32_t*>(kv_lens);
  a.cu_q = static_cast<const int32_t*>(cu_q);
  a.ctx = static_cast<const int32_t*>(context_lens);
  a.out = out;
  a.lse = static_cast<float*>(lse);
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.tokens = tokens;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  const int group = q_heads / kv_heads, ng = groups(head_dim, groupsize);
  const long long page_bytes = (long long)page_size * (head_dim + 4 * ng) * kv_heads;
  if (page_bytes > 0xFFFFFFFFll) return refuse("kv4_attention: a page of 2^32 bytes or more");
  a.page_stride = (uint32_t)page_bytes;
  a.num_pages = num_pages;
  a.max_pages = max_pages;
  a.log_page = 31 - __builtin_clz((unsigned)page_size);
  a.group = group;
  a.max_q = max_q;
  a.c1 = scale * 1.4426950408889634f;
  const int cus = compute_units(dev);
  const Choice c = choose(tokens, requests, q_heads, kv_heads, head_dim, ng, max_q, cu_q != nullptr, cus);
  a.max_rows = c.split ? c.few_rows : 0;
  for (a.first = 0; a.first < requests; a.first += kMaxRequests) {
    a.requests = requests - a.first < kMaxRequests ? requests - a.first : kMaxRequests;
    if (c.prompts) {
      const Plan p = prompt_plan(tokens, a.requests, q_heads, kv_heads, max_q, max_kv, a.max_rows, cus);
      if (p.workgroups < 0) return refuse("kv4_attention: too many rows for one launch");
      a.pieces = p.pieces;
      a.rest = p.rest;
      if (p.split) {
        const size_t rows = (size_t)p.pieces * kv_heads * kPromptRows;
        err = sm24::get_scratch(dev, stream, (rows * head_dim + 2 * rows * 2) * sizeof(float), &a.counters, &a.partial);
        if (err != MARLIN_HIP_OK) return err;
        if (a.partial) a.partial_ml = a.partial + rows * head_dim;  // (null: blocks stay whole)
      }
      err = sm24::launch_error(launch_prompt(a, p.workgroups, head_dim, ng, dtype, stream));
      if (err != MARLIN_HIP_OK) return err;
      a.partial = nullptr;
    }
    if (c.split) {
      const Plan p = plan(a.requests, q_heads, kv_heads, c.split_q, max_kv, cus);
      a.log_kw = p.log_kw;
      a.lead = p.lead;
      a.slots = 2 * cus;
      if (p.split) {
        const size_t rows = (size_t)p.workgroups * 2 * 16 * (kWaves >> p.log_kw);
        err = sm24::get_scratch(dev, stream, rows * (head_dim + 2) * sizeof(float), &a.counters, &a.partial);
        if (err != MARLIN_HIP_OK) return err;
        // (null while the stream is captured and has no scratch yet: tiles stay whole)
        if (a.partial) a.partial_ml = a.partial + rows * head_dim;
      }
      dispatch(head_dim, ng, [&](auto d, auto g) {
        constexpr int D = decltype(d)::value, NG = decltype(g)::value;
        const dim3 grid((unsigned)p.workgroups), block(64 * kWaves);
        if (dtype == F16) hipLaunchKernelGGL((kv4_split_kernel<D, NG, F16>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((kv4_split_kernel<D, NG, BF16>), grid, block, 0, stream, a);
      });
      err = sm24::launch_error(hipGetLastError());
      if (err != MARLIN_HIP_OK) return err;
      a.partial = nullptr;
    }
    a.kv_lens += a.requests;
    a.table += (size_t)a.requests * max_pages;
    if (a.cu_q) a.cu_q += a.requests;
    if (a.ctx) a.ctx += a.requests;
  }
  return MARLIN_HIP_OK;
}

int marlin_hip_kv4_attention(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                             const void* cu_q, void* out, void* lse, int tokens, int requests, int q_heads,
                             int kv_heads, int head_dim, long long q_token_stride, long long q_head_stride,
                             int page_size, int num_pages, int max_pages, int groupsize, int max_q, int max_kv,
                             float scale, int dtype, int dev, hipStream_t stream) {
  return marlin_hip_kv4_attention_ctx(q, cache, block_table, kv_lens, cu_q, nullptr, out, lse, tokens, requests,
                                      q_heads, kv_heads, head_dim, q_token_stride, q_head_stride, page_size, num_pages,
                                      max_pages, groupsize, max_q, max_kv, scale, dtype, dev, stream);
}

}  // extern "C"
