// The 4-bit KV cache's bookkeeping and rows: block tables and slot maps of a step,
// quantizing writes, and the read-back of the values that cached rows stand for.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4_device.h"
#include "kv4_host.h"

namespace kv4 {

// ---------------------------------------------------------------------------
// Tables: request i has ctx_i tokens and gets new_i more.  New tokens are numbered
// through all requests; a page is taken from the free list for each new token that is the
// first of its page, in that order.
//
// Two prefix sums over the requests (tokens, pages) and a write per token.  Every
// workgroup makes the sums for itself, kTabRequests requests at a time, and writes the
// tokens of its range: that reads 8 bytes a request once per workgroup, from L2, and
// needs no second launch and no exchange.  Bound by the latency of its steps: 64 requests
// 3.9 us, 1000 requests with 131 tokens each on average 7.5.
// ---------------------------------------------------------------------------

constexpr int kTabThreads = 512;
constexpr int kTabRequests = 2 * kTabThreads;  // requests per round, two a thread
constexpr int kTabTokens = 2048;               // tokens per workgroup

struct TableArgs {
  const int32_t* ctx;
  const int32_t* fresh;
  const int32_t* free_pages;
  int32_t* table;
  int32_t* slots;
  int32_t* cu;
  int32_t* kv;
  int32_t* used;
  int requests, num_free, max_pages, log_page, tokens;
};

__global__ __launch_bounds__(kTabThreads) void kv4_tables_kernel(TableArgs a) {
  __shared__ uint32_t tok0[kTabRequests + 1];  // first token of each request of the round
  __shared__ uint32_t page0[kTabRequests];     // its first page's place in the free list
  __shared__ int32_t have[kTabRequests];       // its context, in tokens
  __shared__ uint32_t wave_sum[2][kTabThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lp = a.log_page;
  const long long cap = (long long)a.max_pages << lp;
  const uint32_t t_lo = blockIdx.x * (uint32_t)kTabTokens;
  const uint32_t t_hi = min(t_lo + kTabTokens, (uint32_t)a.tokens);
  uint32_t tok_carry = 0, page_carry = 0;

  for (int base = 0; base < a.requests; base += kTabRequests) {
    uint32_t n[2], p[2];
    int32_t c[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int r = base + 2 * tid + u;
      const bool in = r < a.requests;
      c[u] = in ? max(a.ctx[r], 0) : 0;
      n[u] = in ? (uint32_t)max(a.fresh[r], 0) : 0u;
      // lengths past the table's width are cut there: no page is taken for what it cannot name
      const long long before = min((long long)c[u], cap), after = min((long long)c[u] + n[u], cap);
      const long long round = (1ll << lp) - 1;
      p[u] = (uint32_t)(((after + round) >> lp) - ((before + round) >> lp));
      if (in && blockIdx.x == 0) a.kv[r] = (int32_t)after;
    }
    uint32_t ts = n[0] + n[1], ps = p[0] + p[1];  // inclusive sums over the wave's threads
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t x = __shfl_up(ts, d), y = __shfl_up(ps, d);
      if (lane >= d) ts += x, ps += y;
    }
    __syncthreads();  // the previous round's readers are done
    if (lane == 63) wave_sum[0][wave] = ts, wave_sum[1][wave] = ps;
    __syncthreads();
    uint32_t tb = tok_carry, pb = page_carry, tall = tok_carry, pall = page_carry;
#pragma unroll
    for (int w = 0; w < kTabThreads / 64; w++) {
      if (w < wave) tb += wave_sum[0][w], pb += wave_sum[1][w];
      tall += wave_sum[0][w], pall += wave_sum[1][w];
    }
    tb += ts - n[0] - n[1];
    pb += ps - p[0] - p[1];
    tok0[2 * tid] = tb;
    tok0[2 * tid + 1] = tb + n[0];
    page0[2 * tid] = pb;
    page0[2 * tid + 1] = pb + p[0];
    have[2 * tid] = c[0];
    have[2 * tid + 1] = c[1];
    if (tid == 0) tok0[kTabRequests] = tall;
    if (blockIdx.x == 0) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int r = base + 2 * tid + u;
        if (r < a.requests) a.cu[r] = (int32_t)(u ? tb + n[0] : tb);
      }
    }
    __syncthreads();
    const uint32_t first = max(t_lo, tok_carry), last = min(t_hi, tall);
    for (uint32_t t = first + tid; t < last; t += kTabThreads) {
      int lo = 0, hi = kTabRequests;  // the last request of the round whose first token is <= t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tok0[mid] <= t) lo = mid;
        else hi = mid;
      }
      const long long pos = (long long)have[lo] + (t - tok0[lo]);
      int32_t page = -1;
      if (pos < cap) {
        const int j = (int)(pos >> lp);
        const int old = (int)(((long long)have[lo] + ((1ll << lp) - 1)) >> lp);  // pages it has
        int32_t* entry = a.table + (size_t)(base + lo) * a.max_pages + j;
        if (j < old) {
          page = *entry;
        } else {
          const uint32_t rank = page0[lo] + (uint32_t)(j - old);
          page = rank < (uint32_t)a.num_free ? a.free_pages[rank] : -1;
          if ((pos & ((1ll << lp) - 1)) == 0) *entry = page;
        }
      }
      const long long slot = ((long long)page << lp) + (pos & ((1ll << lp) - 1));
      a.slots[t] = page < 0 || slot > 0x7FFFFFFFll ? -1 : (int32_t)slot;
    }
    tok_carry = tall;
    page_carry = pall;
    if (blockIdx.x != 0 && tall >= t_hi) return;  // (the first workgroup writes every request's sums)
  }
  for (uint32_t t = max(t_lo, tok_carry) + tid; t < t_hi; t += kTabThreads) a.slots[t] = -1;
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[a.requests] = (int32_t)tok_carry;
    a.used[0] = (int32_t)page_carry;
  }
}

// ---------------------------------------------------------------------------
// Rows in and out.  D/8 lanes hold a row, 8 dims (16 bytes, one code word) each; a
// workgroup's threads take K rows, then V rows, of consecutive (token, head) pairs.
// Bound by memory: 2 D bytes of fp16 and D/2 + 2 NG of codes and scales a row.
// ---------------------------------------------------------------------------

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
  over(Int<0xB1>());                            // lanes 1 0 3 2 of four
  over(Int<0x4E>());                            // 2 3 0 1
  if constexpr (G >= 64) over(Int<0x141>());    // 7 ... 0 of eight
  if constexpr (G >= 128) over(Int<0x140>());   // 15 ... 0 of sixteen
  return m;
}

// Eight dims a thread: 16 bytes of a row, a word of codes.  A workgroup writes consecutive
// tokens of one head, so that the words of a block's lines, which four tokens share in V,
// meet in one L2 (a workgroup of one token's heads: 27.4 us where this took 24.5; read back
// 21.0 and 17.5).  4096 tokens of 32 heads of 128 dims take 20.0 us, 4.2 TB/s of the 5.1 that
// a large copy reaches, read back 18.0; 24 tokens 3.1, the latency of slot, row and write.
template <int D, int NG, int TYPE>
__global__ __launch_bounds__(kRowThreads) void kv4_append_kernel(RowArgs a) {
  constexpr int B = D / 8, G = D / NG;
  const int token = (int)(blockIdx.x / (unsigned)a.heads * (kRowThreads / B) + threadIdx.x / B);
  const int head = (int)(blockIdx.x % (unsigned)a.heads), b = threadIdx.x % B;
  const bool is_v = blockIdx.y != 0;
  if (token >= a.tokens) return;
  const int slot = a.slots[token];
  const int T = 1 << a.log_page;
  if (slot < 0 || (slot >> a.log_page) >= a.num_pages) return;  // (all lanes of the row)
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.v : a.k);
  src += is_v ? token * a.vt + head * a.vh : token * a.kt + head * a.kh;
  const u32x4 raw = *reinterpret_cast<const u32x4*>(src + 8 * b);
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
  const int o = slot & (T - 1);
  uint8_t* block = a.cache + ((size_t)(slot >> a.log_page) * a.heads + head) * block_bytes<D, NG>(T);
  *reinterpret_cast<uint32_t*>(block + (is_v ? v_word<D>(T, o, b) : k_word<D>(o, b))) = word;
  if (b % (G / 8) == 0) {
    const int n = b / (G / 8);
    *reinterpret_cast<_Float16*>(block + (is_v ? v_scale<D, NG>(T, o, n) : k_scale<D, NG>(T, o, n))) = s16;
  }
}

template <int D, int NG, int TYPE>
__global__ __launch_bounds__(kRowThreads) void kv4_gather_kernel(RowArgs a) {
  constexpr int B = D / 8, G = D / NG;
  const int token = (int)(blockIdx.x / (unsigned)a.heads * (kRowThreads / B) + threadIdx.x / B);
  const int head = (int)(blockIdx.x % (unsigned)a.heads), b = threadIdx.x % B;
  const bool is_v = blockIdx.y != 0;
  if (token >= a.tokens) return;
  const int slot = a.slots[token];
  const int T = 1 << a.log_page;
  float x[8] = {};
  if (slot >= 0 && (slot >> a.log_page) < a.num_pages) {
    const int o = slot & (T - 1);
    const uint8_t* block = a.cache + ((size_t)(slot >> a.log_page) * a.heads + head) * block_bytes<D, NG>(T);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(block + (is_v ? v_word<D>(T, o, b) : k_word<D>(o, b)));
    const int n = b / (G / 8);
    const float s = (float)*reinterpret_cast<const _Float16*>(
        block + (is_v ? v_scale<D, NG>(T, o, n) : k_scale<D, NG>(T, o, n)));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = ((float)((word >> (4 * i)) & 15u) - 8.f) * s;
  }
  uint16_t* dst = static_cast<uint16_t*>(is_v ? a.v : a.k) + ((size_t)token * a.heads + head) * D + 8 * b;
  *reinterpret_cast<u32x4*>(dst) = pack8<TYPE>(x);
}

int log2_of(int x) { return 31 - __builtin_clz((unsigned)x); }

int rows(bool append, const RowArgs& a, int head_dim, int ng, int dtype, hipStream_t stream) {
  const int per = kRowThreads / (head_dim / 8);  // tokens of a workgroup, all of one head
  const long long blocks = ((long long)a.tokens + per - 1) / per * a.heads;
  if (blocks > 0xFFFFFFFFll / kRowThreads) return refuse("more rows than one launch of the KV cache takes");
  const dim3 grid((unsigned)blocks, 2), block(kRowThreads);
  dispatch(head_dim, ng, [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    if (append) {
      if (dtype == F16) hipLaunchKernelGGL((kv4_append_kernel<D, NG, F16>), grid, block, 0, stream, a);
      else hipLaunchKernelGGL((kv4_append_kernel<D, NG, BF16>), grid, block, 0, stream, a);
    } else {
      if (dtype == F16) hipLaunchKernelGGL((kv4_gather_kernel<D, NG, F16>), grid, block, 0, stream, a);
      else hipLaunchKernelGGL((kv4_gather_kernel<D, NG, BF16>), grid, block, 0, stream, a);
    }
  });
  return sm24::launch_error(hipGetLastError());
}

}  // namespace kv4

extern "C" {

int marlin_hip_kv4_tables(const void* context_lens, const void* new_lens, const void* free_pages, void* block_table,
                          void* slots, void* cu_new, void* kv_lens, void* pages_used, int requests, int num_free,
                          int max_pages, int page_size, int tokens, int dev, hipStream_t stream) {
  if (requests < 0 || num_free < 0 || max_pages < 0 || tokens < 0)
    return kv4::refuse("kv4_tables takes no negative sizes");
  if (!kv4::page_ok(page_size)) return kv4::refuse("the KV cache's page_size must be 16, 32, 64, 128 or 256");
  // (lengths are cut there, and are int32)
  if ((long long)max_pages * page_size > (1ll << 30)) return kv4::refuse("a block table row covers more than 2^30 tokens");
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  kv4::TableArgs a{};
  a.ctx = static_cast<const int32_t*>(context_lens);
  a.fresh = static_cast<const int32_t*>(new_lens);
  a.free_pages = static_cast<const int32_t*>(free_pages);
  a.table = static_cast<int32_t*>(block_table);
  a.slots = static_cast<int32_t*>(slots);
  a.cu = static_cast<int32_t*>(cu_new);
  a.kv = static_cast<int32_t*>(kv_lens);
  a.used = static_cast<int32_t*>(pages_used);
  a.requests = requests;
  a.num_free = num_free;
  a.max_pages = max_pages;
  a.log_page = kv4::log2_of(page_size);
  a.tokens = tokens;
  const unsigned blocks = tokens > 0 ? ((unsigned)tokens + kv4::kTabTokens - 1) / kv4::kTabTokens : 1;
  hipLaunchKernelGGL(kv4::kv4_tables_kernel, dim3(blocks), dim3(kv4::kTabThreads), 0, stream, a);
  return sm24::launch_error(hipGetLastError());
}

int marlin_hip_kv4_append(const void* k, const void* v, void* cache, const void* slots, int tokens, int kv_heads,
                          int head_dim, long long k_token_stride, long long k_head_stride, long long v_token_stride,
                          long long v_head_stride, int page_size, int num_pages, int groupsize, int dtype, int dev,
                          hipStream_t stream) {
  const int err = kv4::check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if (tokens < 0 || ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7))
    return kv4::refuse("kv4_append needs strides that are multiples of 8 elements");
  if (tokens == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const kv4::RowArgs a{const_cast<void*>(k), const_cast<void*>(v), static_cast<uint8_t*>(cache),
                       static_cast<const int32_t*>(slots), k_token_stride, k_head_stride, v_token_stride,
                       v_head_stride, tokens, kv_heads, kv4::log2_of(page_size), num_pages};
  return kv4::rows(true, a, head_dim, kv4::groups(head_dim, groupsize), dtype, stream);
}

int marlin_hip_kv4_gather(const void* cache, const void* slots, void* k, void* v, int tokens, int kv_heads,
                          int head_dim, int page_size, int num_pages, int groupsize, int dtype, int dev,
                          hipStream_t stream) {
  const int err = kv4::check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, dtype);
  if (err != MARLIN_HIP_OK) return err;
  if (tokens < 0) return kv4::refuse("kv4_gather takes no negative sizes");
  if (tokens == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const kv4::RowArgs a{k, v, const_cast<uint8_t*>(static_cast<const uint8_t*>(cache)),
                       static_cast<const int32_t*>(slots), 0, 0, 0, 0, tokens, kv_heads, kv4::log2_of(page_size),
                       num_pages};
  return kv4::rows(false, a, head_dim, kv4::groups(head_dim, groupsize), dtype, stream);
}

}  // extern "C"
