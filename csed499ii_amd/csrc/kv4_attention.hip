// Attention over the 4-bit paged KV cache: launch plan and entry points.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kv4_host.h"
#include "kv4_prompt.h"

namespace kv4 {

// Requests of at most so many rows (new tokens times the query heads of a kv head) go to the
// split kernel, the others to the prompt kernel, each of which passes over the other's.  The
// split kernel's time grows with the rows, the prompt kernel's is the same up to 256: 12
// requests of 4096 tokens on 8 heads of 128 dims, 64, 80, 96 and 128 rows, 53, 55, 70 and 82
// us beside 72 to 73; with groups of 32, 128, 144 and 160 rows, 104, 123 and 133 beside 108,
// 125 and 125.
// Few tiles leave the prompt kernel's large parts waiting: one request of 8192 tokens, 24 us
// beside 34 at 64 rows, 41 beside 57 at 256.  (Of a prefix, whose parts need not meet, only tiles that
// kMaxParts leaves compute units without one, `few` = cus / 64: 32 requests on 64 and 8 heads behind 8192 tokens in one
// and two groups 63 and 82 us in the split kernel, 58 and 64 here; 64 on 16 and 4 heads 45 and 49.)
int split_rows(int requests, int kv_heads, int head_dim, int ng, int few) {
  if ((long long)requests * kv_heads <= few) return 256;
  return head_dim == 128 && ng == 4 ? 144 : 80;
}

// Compute units that launches are planned for: the stream's arrival counters, one a workgroup of the split kernel
// (two of which fill a unit) and one a wave of a part of the prompt kernel (one of which does), are enough for so many.
constexpr int kMostUnits = (int)(sm24::kCounterBytes / sizeof(uint32_t)) / kPromptWaves;
static_assert(kPromptWaves >= 2, "");

// (the query takes the host 0.2 us of each call, so its answer is kept)
int compute_units(int dev) {
  static std::atomic<int> known[64];
  if (dev >= 0 && dev < 64 && known[dev].load(std::memory_order_relaxed) > 0)
    return known[dev].load(std::memory_order_relaxed);
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) return 256;
  if (n > kMostUnits) n = kMostUnits;
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
Plan plan(int requests, int q_heads, int kv_heads, int max_q, int max_kv, int cus, bool behind = false) {
  Plan p{};
  const long long row_blocks = ((long long)max_q * (q_heads / kv_heads) + 15) / 16;
  const long long steps = ((long long)max_kv + kStep - 1) / kStep;
  const long long most = 2ll * cus;
  const long long blocks = requests * row_blocks * kv_heads;
  p.log_kw = behind ? (blocks <= most ? 3 : blocks <= 2 * most ? 2 : 1) : blocks <= 2 * most ? kLogWaves : 1;
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
  c.few_rows = split_rows(requests, kv_heads, head_dim, ng, cus / 16);
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

// ---------------------------------------------------------------------------
// The prefix that the requests of a group share: the whole pages, from the first on, that are the
// same in their tables and lie within their contexts.  A workgroup for each group compares every
// request's row with the first one's; one more for the requests of no group.  Once a step, for all
// layers.  64 rows of 512 entries in one group take 10 us, what one compute unit reads at; 4 groups of 8 rows 4.1.
// ---------------------------------------------------------------------------

constexpr int kMaxGroups = 1 << 20;
constexpr int kSharedThreads = 1024, kSharedRound = 1024, kSharedWaves = kSharedThreads / 64, kSharedRows = 4;

struct SharedArgs {
  const int32_t* table;
  const int32_t* ctx;
  const int32_t* cu_q;       // null: a token each
  const int32_t* cu_groups;  // [groups + 1]
  int32_t* lens;             // [groups] tokens of the prefix
  int32_t* leads;            // [groups] a request that holds it
  int32_t* cu_rows;          // [groups + 1] first token of each group
  int32_t* start;            // [requests] tokens of the prefix, 0 for a request that does not share it
  int requests, groups, max_pages, log_page;
};

__global__ __launch_bounds__(kSharedThreads) void kv4_shared_kernel(SharedArgs a) {
  __shared__ int first[kSharedRound];  // column in which a request's row differs
  __shared__ int lead, least, sharers;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = (int)blockIdx.x;
  auto border = [&](int i) { return min(max(a.cu_groups[i], 0), a.requests); };
  auto token = [&](int r) { return a.cu_q == nullptr ? r : max(a.cu_q[r], 0); };
  if (g == a.groups) {
    const int r0 = border(0), r1 = border(a.groups);
    for (int r = tid; r < a.requests; r += kSharedThreads)
      if (r < r0 || r >= r1) a.start[r] = 0;
    if (tid == 0) a.cu_rows[a.groups] = token(r1);
    return;
  }
  const int r0 = border(g), r1 = max(border(g + 1), r0);
  // whole pages that may be shared: none of a request without new tokens
  auto pages = [&](int r) {
    if (a.cu_q != nullptr && a.cu_q[r + 1] <= a.cu_q[r]) return 0;
    return min(max(a.ctx[r], 0) >> a.log_page, a.max_pages);
  };
  if (tid == 0) lead = 0x7FFFFFFF, least = 0x7FFFFFFF, sharers = 0;
  __syncthreads();
  const bool one_round = r1 - r0 <= kSharedRound;  // (what `first` holds then serves below)
  for (int from = r0; from < r1; from += kSharedRound)
    if (from + tid < r1) {
      const int n = first[tid] = pages(from + tid);
      if (n > 0) atomicMin(&lead, from + tid);
    }
  __syncthreads();
  const int leader = lead;
  const bool any = leader < r1;
  const int most = !any ? 0 : one_round ? first[leader - r0] : pages(leader);
  const int32_t* lead_row = a.table + (size_t)(any ? leader : r0) * a.max_pages;
  for (int from = r0; from < r1; from += kSharedRound) {
    const int n = min(r1 - from, kSharedRound);
    __syncthreads();  // the round before is done with LDS
    if (!one_round) {
      if (tid < n) first[tid] = pages(from + tid);
      __syncthreads();
    }
    // A wave takes four rows, 256 columns of each in flight.
    for (int i0 = kSharedRows * wave; i0 < n; i0 += kSharedRows * kSharedWaves) {
      int common[kSharedRows];
#pragma unroll
      for (int k = 0; k < kSharedRows; k++) common[k] = most;
      for (int j0 = 0; j0 < most; j0 += 256) {
        int want[4], page[kSharedRows][4];
#pragma unroll
        for (int u = 0; u < 4; u++) {  // (those past the last repeat it)
          const int j = min(j0 + 64 * u + lane, most - 1);
          want[u] = lead_row[j];
#pragma unroll
          for (int k = 0; k < kSharedRows; k++) page[k][u] = a.table[(size_t)(from + min(i0 + k, n - 1)) * a.max_pages + j];
        }
        bool more = false;
#pragma unroll
        for (int k = 0; k < kSharedRows; k++) {
#pragma unroll
          for (int u = 3; u >= 0; u--) {
            const uint64_t differ = __ballot(page[k][u] != want[u]);
            if (differ != 0) common[k] = min(common[k], j0 + 64 * u + __builtin_ctzll(differ));
          }
          more |= common[k] >= j0 + 256;
        }
        if (!more) break;
      }
#pragma unroll
      for (int k = 0; k < kSharedRows; k++)
        if (lane == 0 && i0 + k < n) first[i0 + k] = min(first[i0 + k], common[k]);
    }
    __syncthreads();
    if (tid < n) {
      const int common = first[tid];
      if (!one_round) a.start[from + tid] = common;
      if (common > 0) {
        atomicMin(&least, common);
        atomicAdd(&sharers, 1);
      }
    }
  }
  __syncthreads();
  const int len = sharers > 1 ? least << a.log_page : 0;
  for (int from = r0; from < r1; from += kSharedRound)
    if (from + tid < r1) a.start[from + tid] = (one_round ? first[tid] : a.start[from + tid]) > 0 ? len : 0;
  if (tid == 0) {
    a.lens[g] = len;
    a.leads[g] = any ? leader : 0;
    a.cu_rows[g] = token(r0);
  }
}

struct Problem {
  int tokens, requests, q_heads, kv_heads, head_dim, ng, max_q, max_kv, dtype, dev, cus;
  hipStream_t stream;
};

// Every launch of a call, or of one pass of it, on the kernels that `c` names.
template <int FORM>
int attend(AttnArgs a, const Problem& p, const Choice& c) {
  int err = MARLIN_HIP_OK;
  a.max_rows = c.split ? c.few_rows : 0;
  for (a.first = 0; a.first < p.requests; a.first += kMaxRequests) {
    a.requests = p.requests - a.first < kMaxRequests ? p.requests - a.first : kMaxRequests;
    if (c.prompts) {
      const Plan plan = prompt_plan(p.tokens, a.requests, p.q_heads, p.kv_heads, p.max_q, p.max_kv, a.max_rows, p.cus);
      if (plan.workgroups < 0) return refuse("kv4_attention: too many rows for one launch");
      a.pieces = plan.pieces;
      a.rest = plan.rest;
      if (plan.split) {
        const size_t rows = (size_t)plan.pieces * p.kv_heads * kPromptRows;
        err = sm24::get_scratch(p.dev, p.stream, (rows * p.head_dim + 2 * rows * 2) * sizeof(float), &a.counters, &a.partial);
        if (err != MARLIN_HIP_OK) return err;
        if (a.partial) a.partial_ml = a.partial + rows * p.head_dim;  // (null: blocks stay whole)
      }
      err = sm24::launch_error(launch_prompt<FORM>(a, plan.workgroups, p.head_dim, p.ng, p.dtype, p.stream));
      if (err != MARLIN_HIP_OK) return err;
      a.partial = nullptr;
    }
    if (c.split) {
      // (through a window a row's tokens are no more than the window's and the sinks')
      const long long reach = FORM == WINDOW ? (long long)a.window + a.sinks + c.split_q + 2 * kStep : p.max_kv;
      const Plan plan = kv4::plan(a.requests, p.q_heads, p.kv_heads, c.split_q, reach < p.max_kv ? (int)reach : p.max_kv, p.cus,
                                  FORM == SHARED && a.start != nullptr);
      a.log_kw = plan.log_kw;
      a.lead = plan.lead;
      a.slots = 2 * p.cus;
      if (plan.split) {
        const size_t rows = (size_t)plan.workgroups * 2 * 16 * (kWaves >> plan.log_kw);
        err = sm24::get_scratch(p.dev, p.stream, rows * (p.head_dim + 2) * sizeof(float), &a.counters, &a.partial);
        if (err != MARLIN_HIP_OK) return err;
        // (null while the stream is captured and has no scratch yet: tiles stay whole)
        if (a.partial) a.partial_ml = a.partial + rows * p.head_dim;
      }
      err = sm24::launch_error(launch_split<FORM>(a, plan.workgroups, p.head_dim, p.ng, p.dtype, p.stream));
      if (err != MARLIN_HIP_OK) return err;
      a.partial = nullptr;
    }
    a.kv_lens += a.requests;
    if (FORM == SHARED && a.leads != nullptr) a.leads += a.requests;
    else a.table += (size_t)a.requests * (size_t)a.max_pages;
    if (FORM == SHARED && a.start != nullptr) a.start += a.requests;
    if (a.cu_q) a.cu_q += a.requests;
    if (a.ctx) a.ctx += a.requests;
  }
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
  const int cus = sms <= 0 ? 256 : sms < kMostUnits ? sms : kMostUnits, ng = groups(head_dim, groupsize), most = (1 << 30) / (q_heads / kv_heads);
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

}  // extern "C"

namespace kv4 {

// The prefix that groups of requests share (marlin_hip_kv4_shared).
struct Prefix {
  const int32_t *lens, *leads, *cu_rows, *start;
  int groups;
  float* workspace;
  long long bytes;
  bool always;
};

// Whether two passes can pay: what falls away, in steps of 16 rows and 32 tokens, if the prefix were all of max_kv
// (where it is far shorter they do not: 16 requests on 64 and 8 heads behind 64 tokens, max_kv 16384, 30 us where 15).
// A block of 256 rows of the prompt kernel counts as eight.  (With the second launch and the sums between
// them the passes cost 15 to 20 us, an undivided pass 0.5 ns a step.  In graphs: 16 requests on 64 and 8 heads behind
// 8192 tokens, 17000 steps fewer, 44.5 us where 42 in one pass; four groups of 8 on 32 heads behind 1500,
// 47000 fewer, 42 where 53; 32 on 32 heads behind 4096, 130000 fewer, 47 where 98.  The worst that was found: 32
// requests of 4 tokens on 64 and 8 heads behind 4096, 43000 fewer, 62 where 56.  A prefix in the prompt kernel from half
// as many more on: 64 on 64 and 8 heads behind 2000 in two groups, 25000 fewer, 46 where 33.  Prompts, which the second
// pass takes through the same kernel, from four times as many on.)
bool shares(int groups, const Problem& p, int group, bool first_prompts, bool prompts) {
  auto blocks = [&](int n, bool big) {
    const long long rows = ((long long)p.tokens + n - 1) / n * group;
    return n * (big ? (rows + kPromptRows - 1) / kPromptRows * 8 : (rows + 15) / 16);
  };
  const long long fewer = blocks(p.requests, prompts) - blocks(groups, first_prompts);
  return fewer * p.kv_heads * (p.max_kv / kStep) >= (prompts ? 81920 : first_prompts ? 32768 : 20480);
}

// How a call with a prefix runs, the same for the call and for the query of its workspace.
struct SharedPlan {
  bool two;                 // passes
  Choice first;             // of the first one
  bool parts;               // its divided blocks leave their parts to the second one
  size_t parts_at, places;  // floats before the parts, rows that they hold
  size_t least, bytes;      // of workspace: what two passes need, and what serves them best
};
SharedPlan plan_shared(const Problem& p, const Choice& c, int groups, bool always) {
  SharedPlan s{};
  const int group = p.q_heads / p.kv_heads, average = (p.tokens + groups - 1) / groups;  // tokens that a group has
  const bool big = (long long)average * group > split_rows(groups, p.kv_heads, p.head_dim, p.ng, p.cus / 64);
  s.two = always || shares(groups, p, group, big, c.prompts);
  if (!s.two) return s;
  // One kernel takes all groups, by the rows that a group has on average.
  s.first.prompts = big;
  s.first.split = !big;
  s.first.few_rows = 0x7FFFFFFF;
  s.first.split_q = average;
  // Blocks of rows that the prompt kernel divides leave their parts where the second pass, if it runs on the
  // split kernel alone, adds them as it writes: they would meet through memory that is not cached.
  // (One launch of the first pass: a second would write over its parts.  And one block a workgroup of the
  // second: 128 requests on 32 heads of 8192 shared tokens, 47 and 106 us so, 52 and 84 joined.)
  const size_t rows = (size_t)p.tokens * p.q_heads;
  s.places = ((size_t)p.cus / p.kv_heads) * p.kv_heads * kPromptRows;
  s.parts_at = (rows * (p.head_dim + 4) + 3) & ~(size_t)3;
  const long long blocks = (long long)p.requests * ((c.split_q * group + 15) / 16) * p.kv_heads;
  s.parts = big && !c.prompts && blocks <= 2 * p.cus && groups <= kMaxRequests && s.places <= 0x7FFFFFFF;
  s.least = rows * (p.head_dim + 2) * sizeof(float);
  s.bytes = s.parts ? (s.parts_at + s.places * (p.head_dim + 2)) * sizeof(float) : s.least;
  return s;
}

int attention(const void* q, const void* cache, const void* block_table, const void* kv_lens, const void* cu_q,
              const void* context_lens, void* out, void* lse, int tokens, int requests, int q_heads, int kv_heads,
              int head_dim, long long q_token_stride, long long q_head_stride, int page_size, int num_pages, int max_pages,
              int groupsize, int max_q, int max_kv, float scale, int dtype, int dev, hipStream_t stream, int window,
              int sinks, const Prefix* prefix) {
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
  a.window = window;
  a.sinks = sinks;
  const Problem p{tokens, requests, q_heads, kv_heads, head_dim, ng, max_q, max_kv, dtype, dev, compute_units(dev), stream};
  const Choice c = choose(tokens, requests, q_heads, kv_heads, head_dim, ng, max_q, cu_q != nullptr, p.cus);
  if (window > 0) return attend<WINDOW>(a, p, c);
  if (prefix == nullptr) return attend<PLAIN>(a, p, c);
  const SharedPlan s = plan_shared(p, c, prefix->groups, prefix->always);
  if (!s.two) return attend<PLAIN>(a, p, c);
  const size_t rows = (size_t)tokens * q_heads;
  if (prefix->bytes < (long long)s.least)
    return refuse("kv4_attention of a shared prefix needs a workspace of head_dim + 2 floats a row");
  a.before = prefix->workspace;
  a.before_ml = a.before + rows * head_dim;
  // First pass: a group is a request whose tokens are the prefix and whose rows, behind it, see all of them.
  AttnArgs b = a;
  b.kv_lens = b.ctx = prefix->lens;
  b.leads = prefix->leads;
  b.cu_q = prefix->cu_rows;
  b.max_q = tokens;
  Problem first = p;
  first.requests = prefix->groups;
  first.max_q = tokens;
  if (s.parts && prefix->bytes >= (long long)s.bytes) {
    a.where = b.where = reinterpret_cast<int2*>(a.before_ml + 2 * rows);
    a.parts = b.parts = prefix->workspace + s.parts_at;
    a.parts_ml = b.parts_ml = a.parts + s.places * head_dim;
    a.places = b.places = (int)s.places;
  }
  err = attend<SHARED>(b, first, s.first);
  if (err != MARLIN_HIP_OK) return err;
  a.start = prefix->start;
  return attend<SHARED>(a, p, c);
}

}  // namespace kv4

extern "C" {

int marlin_hip_kv4_shared_plan(int tokens, int requests, int groups, int q_heads, int kv_heads, int head_dim,
                               int groupsize, int max_q, int max_kv, int cu_q, int always, int dev, long long* out) {
  using namespace kv4;
  if (tokens >= 0 && max_q > tokens) max_q = tokens;
  const int err = check(tokens, requests, q_heads, kv_heads, head_dim, 16, 1, 0, groupsize, max_q, max_kv, 1.f, 0);
  if (err != MARLIN_HIP_OK) return err;
  if (groups < 0 || groups > kMaxGroups) return refuse("kv4_attention takes prefixes of 2^20 groups at most");
  out[0] = out[1] = out[2] = 0;
  if (tokens == 0 || requests == 0 || max_q == 0 || groups == 0) return MARLIN_HIP_OK;
  const Problem p{tokens, requests, q_heads, kv_heads, head_dim, kv4::groups(head_dim, groupsize), max_q, max_kv, 0, dev,
                  dev < 0 ? 256 : compute_units(dev), nullptr};
  const SharedPlan s = plan_shared(p, choose(tokens, requests, q_heads, kv_heads, head_dim, p.ng, max_q, cu_q != 0, p.cus),
                                   groups, always != 0);
  out[0] = (long long)s.bytes;
  out[1] = s.first.prompts;
  out[2] = s.parts;
  return MARLIN_HIP_OK;
}

int marlin_hip_kv4_attention_ctx(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                                 const void* cu_q, const void* context_lens, void* out, void* lse, int tokens,
                                 int requests, int q_heads, int kv_heads, int head_dim, long long q_token_stride,
                                 long long q_head_stride, int page_size, int num_pages, int max_pages, int groupsize,
                                 int max_q, int max_kv, float scale, int dtype, int dev, hipStream_t stream) {
  return kv4::attention(q, cache, block_table, kv_lens, cu_q, context_lens, out, lse, tokens, requests, q_heads, kv_heads,
                        head_dim, q_token_stride, q_head_stride, page_size, num_pages, max_pages, groupsize, max_q, max_kv,
                        scale, dtype, dev, stream, 0, 0, nullptr);
}

int marlin_hip_kv4_attention_window(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                                    const void* cu_q, const void* context_lens, void* out, void* lse, int tokens,
                                    int requests, int q_heads, int kv_heads, int head_dim, long long q_token_stride,
                                    long long q_head_stride, int page_size, int num_pages, int max_pages, int groupsize,
                                    int max_q, int max_kv, float scale, int window, int sinks, int dtype, int dev,
                                    hipStream_t stream) {
  if (window < 1 || sinks < 0) return kv4::refuse("kv4_attention needs a window of a token at least and no negative sinks");
  // (no position passes 2^30: as many see all)
  if (window > 1 << 30) window = 1 << 30;
  if (sinks > 1 << 30) sinks = 1 << 30;
  return kv4::attention(q, cache, block_table, kv_lens, cu_q, context_lens, out, lse, tokens, requests, q_heads, kv_heads,
                        head_dim, q_token_stride, q_head_stride, page_size, num_pages, max_pages, groupsize, max_q, max_kv,
                        scale, dtype, dev, stream, window, sinks, nullptr);
}

int marlin_hip_kv4_attention_shared(const void* q, const void* cache, const void* block_table, const void* kv_lens,
                                    const void* cu_q, const void* context_lens, const void* shared, void* out, void* lse,
                                    void* workspace, int tokens, int requests, int groups, int q_heads, int kv_heads,
                                    int head_dim, long long q_token_stride, long long q_head_stride, int page_size,
                                    int num_pages, int max_pages, int groupsize, int max_q, int max_kv, float scale,
                                    int dtype, long long workspace_bytes, int always, int dev, hipStream_t stream) {
  if (groups < 0 || groups > kv4::kMaxGroups) return kv4::refuse("kv4_attention takes prefixes of 2^20 groups at most");
  const int32_t* at = static_cast<const int32_t*>(shared);
  const kv4::Prefix prefix{at, at + groups, at + 2 * (size_t)groups, at + 3 * (size_t)groups + 1, groups,
                           static_cast<float*>(workspace), workspace_bytes, always != 0};
  return kv4::attention(q, cache, block_table, kv_lens, cu_q, context_lens, out, lse, tokens, requests, q_heads, kv_heads,
                        head_dim, q_token_stride, q_head_stride, page_size, num_pages, max_pages, groupsize, max_q, max_kv,
                        scale, dtype, dev, stream, 0, 0, groups > 0 ? &prefix : nullptr);
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

int marlin_hip_kv4_shared(const void* block_table, const void* context_lens, const void* cu_q, const void* cu_groups,
                          void* shared, int requests, int groups, int max_pages, int page_size, int dev,
                          hipStream_t stream) {
  if (requests < 0 || groups < 0 || max_pages < 0) return kv4::refuse("kv4_shared takes no negative sizes");
  if (requests > (1 << 30)) return kv4::refuse("kv4_shared takes at most 2^30 requests");  // (as of pages)
  if (!kv4::page_ok(page_size)) return kv4::refuse("the KV cache's page_size must be 16, 32, 64, 128 or 256");
  if ((long long)max_pages * page_size > (1ll << 30)) return kv4::refuse("a block table row covers more than 2^30 tokens");
  if (groups > kv4::kMaxGroups) return kv4::refuse("kv4_shared takes at most 2^20 groups");
  if (requests == 0 || groups == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  int32_t* out = static_cast<int32_t*>(shared);
  const kv4::SharedArgs a{static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(context_lens),
                          static_cast<const int32_t*>(cu_q), static_cast<const int32_t*>(cu_groups), out, out + groups,
                          out + 2 * (size_t)groups, out + 3 * (size_t)groups + 1, requests, groups, max_pages,
                          31 - __builtin_clz((unsigned)page_size)};
  hipLaunchKernelGGL(kv4::kv4_shared_kernel, dim3((unsigned)groups + 1), dim3(kv4::kSharedThreads), 0, stream, a);
  return sm24::launch_error(hipGetLastError());
}

}  // extern "C"
