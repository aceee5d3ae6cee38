// Attention of a few query rows over the 4-bit paged cache, split over the cache's length.
//
// For one request and kv head the query rows are its new tokens times the query heads
// that share the kv head (row i: token i / G, head i % G).  With codes c (less 8), scales k
// and v:
//   x_j = k_j (q . c_j)                   (per scale group, summed over the groups)
//   p_j = exp2(x_j c1 - M)                (c1 = scale log2 e; M: the row's reference)
//   O_d = sum_j (p_j v_j) c_jd,   L = sum_j p_j,   out = O / L
// so that the scales leave both products and the matrix cores multiply small integers,
// which fp16 holds exactly.
//
// A tile is HW blocks of 16 rows (an MFMA's columns) over all the tokens that they see: all
// of a head's rows, then the next head's, so that blocks that read the same codes mostly
// share a compute unit's path to memory.  (Several blocks to a wave, which unpacks for all:
// 66.9 us where this takes 65.9, 12 requests of 5 tokens and 8 query heads to a kv head.)
// A workgroup gives each block KW of its eight waves, which take turns at the 32-token
// steps: a unit is a step for each.  The tiles' units, end to end, are divided evenly over the workgroups,
// whatever the requests' lengths: a workgroup takes the end of one tile, whole tiles, the
// beginning of another.  Per step and wave:
//   S^T = K Q^T  16x16x32 MFMAs, A = codes (rows = 16 tokens), B = Q, held in registers;
//                lane (c, g) gets row c's sums of tokens 4 g .. 4 g + 3: what the second
//                product wants as its B operand, if its reduction index counts tokens
//                4 g + i of the step's two halves, so p never leaves its lane;
//   O^T = V^T P^T  A = codes of V, each word's 8 dims spread over the accumulators.
// (The offset 8 is taken off the codes, one packed operation for two.  Left in the products
// and subtracted from the sums it costs less, but the sums then grow to 8 sum p v and lose
// in fp32 what a small output has: 10^-6 of the largest v was seen.)
//
// M is not the running maximum but a reference that is only changed, by a wave-uniform branch,
// when a row's p v, which is rounded to fp16 for the matrix cores, would pass 2^15 (or its sum
// of p 2^100): rare after the first step.  The branch brings the row's largest p v so far to 2^7,
// however large the v of tokens of little weight.  So p v has fp16's 11 bits where it is not
// below 2^-14, and is off by 2^-25 at most there: an output by 2^-11 sum_j w_j |v_j| (w: the
// softmax) and 2^-32 a token of the largest w_j s_j of the row, all its scale groups alike, which
// share M.  With the largest v in M's place, however small its weight, values 2^21 below it lost
// bits, and all of them 2^31 below.  Sums are fp32.
//
// What does not exist must not count: tokens past the row's last one, pages whose table
// entry is not a page, slots never written (their scales may be NaN).  Their p v is set to
// zero after the product, not multiplied by zero.
//
// Bound by HBM where the cache is long and one block of rows reads it: 64 requests of 1024 to
// 16384 tokens on 8 heads of 128 dims, eight query heads each, take 128 us, 4.6 TB/s of the
// 5.1 that a large copy reaches.  From two blocks on, by the unpacking, which every block
// repeats (12 requests of five tokens, 40 rows, 4096 in all: 47 us, 36 at 24 rows).  Short ones
// by latencies one after the other (lengths, table, codes, the meeting): one request of 1000
// tokens on 32 heads, 11.0 us.
//
// The waves meet in LDS; the partial sums of a divided tile go through the uncached
// scratch, and the last of its workgroups to arrive on its counter adds them in order: one
// launch, and the same bits from run to run.
#pragma once
#include "kv4_device.h"

namespace kv4 {

constexpr int kLogWaves = 3, kWaves = 1 << kLogWaves;
constexpr int kLogStep = 5, kStep = 1 << kLogStep;  // tokens per wave and step
// Units that a tile counts more than it has, for what a workgroup's turn to another tile costs,
// where there are more units than workgroups
// (24 requests of 17 to 4096 tokens on 32 heads: 94.3 us with none, 57.8 with 2, 59.6 with 4;
// 64 of 1024 to 16384 on 8: 133.0, 128.2, 129.3; one of 131072: 41.4, 38.4, 37.8).
constexpr int kLead = 2;
// Units that a whole tile may take beyond an even share before tiles are divided: what the
// meeting of the pieces costs.  four requests of 1000 tokens (four units), 40 rows on 20 heads,
// 23.3 us divided, 16.6 whole; 16 of 1000 on 8 heads 14.3 and 14.2; one of 1000 on 32 heads,
// which stays divided, 11.0 and 12.7.
constexpr int kWhole = 3;
constexpr int kTilesAt = 43;       // bit of a sum of units
constexpr int kMaxSplits = 32;     // pieces of one tile: each costs its last workgroup's read of it
constexpr int kTile = 64;          // tokens of a tile of the prompt kernel
constexpr int kPromptWaves = 8, kPromptRows = 32 * kPromptWaves;
constexpr int kMaxRequests = 2 * 64 * kWaves;  // of a launch that divides by the requests' lengths
constexpr float kVTop = 7.f;       // a new reference brings the row's largest p v to 2^7
constexpr float kMostPV = 1 << 15; // ... which later ones may pass by 2^8 (65504 is the largest fp16)
constexpr float kSlack = 8.f;      // of a reference that is rounded, in log2 units
constexpr float kMostL = 0x1p100f; // of a row's sum of p, before it gets a new reference
constexpr float kMostShift = 90.f; // p <= 2^90 at a new reference, however small its v
constexpr float kBig = 1 << 20;    // of a row's largest score, in log2 units
constexpr float kNone = -1.0e30f;  // reference of a row that has seen nothing

struct AttnArgs {
  const void* q;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu_q;  // null: request i is token i
  void* out;
  float* lse;           // null: not wanted
  float* partial;       // [workgroup][first, last][row][D] (prompt kernel: [part][wave][..]); null: no tile is divided
  float* partial_ml;    // as many pairs of a reference and a sum
  uint32_t* counters;   // [workgroup] (prompt kernel: [block of rows][wave]), zero between launches
  long long qt, qh;     // strides of q in elements
  int tokens, requests, q_heads, kv_heads;
  uint32_t page_stride; // bytes of a page, all heads
  int num_pages, max_pages, log_page;
  int first;            // token of request 0 where cu_q is null
  int pieces;           // of the prompt kernel: workgroups a head that fill the machine
  bool rest;            // whether its grid has as many more, to divide the last blocks
  int max_q;            // a request's later tokens are not computed
  int max_rows;         // requests of at most so many rows a head are the split kernel's, others the prompt kernel's
  int log_kw;           // KW waves of a workgroup share a head (KW HW = kWaves)
  int slots;            // workgroups that fill the machine
  int lead;             // units that a tile counts more than it has
  int group;            // query heads of a kv head
  float c1;             // softmax scale * log2 e
  const int32_t* ctx;   // positions of the first new tokens; null: they are the last of kv_lens
};

struct Request {
  int first, n, kv;  // first token, new tokens in q, tokens in all that the table covers
  int past;          // position of the first new token
};
__device__ __forceinline__ Request request_of(const AttnArgs& a, int r) {
  Request q;
  int cap = a.max_pages << a.log_page;  // (at most 2^30)
  asm volatile("" : "+s"(cap));         // (else kept in a vector register all the while)
  const int kv = max(a.kv_lens[r], 0);
  q.kv = min(kv, cap);
  int n = 1;
  if (a.cu_q == nullptr) {
    q.first = a.first + r;
    q.n = 1;
  } else {
    const int begin = max(a.cu_q[r], 0), end = max(a.cu_q[r + 1], 0);
    n = max(end - begin, 0);
    q.first = min(begin, a.tokens);
    q.n = max(min(end, a.tokens) - q.first, 0);
  }
  // positions go by the lengths as they are: what the table or q cuts off moves no token
  q.past = min(kv - n, 1 << 30);
  return q;
}
// With the position that the caller gives.  (Apart, for the loads that a short call waits for:
// loaded with the lengths it costs one of 1000 tokens 0.3 of its 11 us.)
__device__ __forceinline__ void set_past(const AttnArgs& a, int r, Request& q) {
  if (__builtin_expect(a.ctx != nullptr, 0)) q.past = min(max(a.ctx[r], 0), 1 << 30);
}

// Tokens that new token t sees.
__device__ __forceinline__ int seen_by(const Request& q, int t) { return max(min(q.past + t + 1, q.kv), 0); }

// Rows of a head that are computed.
__device__ __forceinline__ int rows_of(const AttnArgs& a, const Request& q) { return min(q.n, a.max_q) * a.group; }

// Codes of one 32-token step as loaded.  BLOCKS: 8-dim words of a scale group, whose 16
// MFMA rows are word row / PARTS, part row % PARTS.
template <int D, int NG>
struct Shape {
  static constexpr int KW = D / 32;             // words of K a lane holds per half = k-steps
  static constexpr int BLOCKS = D / NG / 8;     // 16, 8 or 4
  static constexpr int PARTS = 16 / BLOCKS;     // 1, 2 or 4
  static constexpr int OPS = 8 / PARTS;         // MFMAs per scale group
  static constexpr int STEPS = KW / NG;         // k-steps per scale group
  // A step in LDS: K codes of 32 tokens, V codes, scales [half][K, V][quad][NG][4].
  static constexpr int V_AT = kStep * D / 2, S_AT = kStep * D, STAGE = S_AT + 128 * NG;
  static constexpr int LOADS = D / 32 + (NG == 4 ? 2 : 1);  // DMA instructions of a step
  // 128 registers let two workgroups share a compute unit.  With several groups of 128 dims
  // V's codes and scales do not fit them, and are read from LDS as they are needed (12 requests
  // of five tokens with groups of 32, as first built: 53.5 us; all at once, one workgroup a unit
  // and four steps in flight, 56.6).
  static constexpr bool LATE = NG > 1 && D == 128;
  static constexpr int RING = 2;  // steps of a wave in flight or in use
};

// x and its value in the lane 16 (32) places over, in one order or the other.  (In assembly:
// given one value twice, the compiler takes the builtin's two results for the same.  The
// wait states are those it puts between a VALU write and this read.)
struct Pair {
  float a, b;
};
__device__ __forceinline__ Pair across16(float x) {
  Pair p = {x, x};
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(p.a), "+v"(p.b));
  return p;
}
__device__ __forceinline__ Pair across32(float x) {
  Pair p = {x, x};
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(p.a), "+v"(p.b));
  return p;
}
// Over the four lanes of an MFMA column.
__device__ __forceinline__ float column_max(float x) {
  const Pair p = across16(x), q = across32(fmaxf(p.a, p.b));
  return fmaxf(q.a, q.b);
}
__device__ __forceinline__ float column_sum(float x) {
  const Pair p = across16(x), q = across32(p.a + p.b);
  return q.a + q.b;
}

// Four bytes per lane from the lane's own address into lds + 4 lane.
__device__ __forceinline__ void dma4(uint32_t lds, const void* src) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\t"
      "global_load_lds_dword %1, off" ::"s"(lds),
      "v"(src)
      : "memory", "m0");
}

template <int D, int NG>
struct Codes {
  uint32_t k[2][D / 32];
  u32x4 v[2][NG];       // four tokens each
  half4_t ks[2][NG], vs[2][NG];
};

// Constants of the unpacking, kept in registers the compiler cannot see through: with
// literals it takes v_and_b32 and v_or_b32 where v_and_or_b32 does both.
struct Magic {
  uint32_t even, odd, exponent;
  __device__ __forceinline__ Magic() {
    asm("s_mov_b32 %0, 0x000f000f" : "=s"(even));
    asm("s_mov_b32 %0, 0x00f000f0" : "=s"(odd));
    asm("v_mov_b32 %0, 0x64006400" : "=v"(exponent));
  }
  // Nibbles 0 and 4, then 1 and 5 of a word, less 8 (see sm24::dequant4).
  __device__ __forceinline__ half4_t codes(uint32_t q) const {
    const half2_t l = __builtin_bit_cast(half2_t, (q & even) | exponent) - (half2_t){(_Float16)1032.f, (_Float16)1032.f};
    const half2_t h = __builtin_bit_cast(half2_t, (q & odd) | exponent) * (half2_t){(_Float16)0.0625f, (_Float16)0.0625f} +
                      (half2_t){(_Float16)-72.f, (_Float16)-72.f};
    return (half4_t){l.x, l.y, h.x, h.y};
  }
};

// Codes of a word less 8, in nibble order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half8_t k_operand(const Magic& m, uint32_t w) {
  const half4_t a = m.codes(w), b = m.codes(w >> 8);
  return (half8_t){a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// Of four fp16 numbers, without their signs; of two such, the larger (a NaN is larger still).
__device__ __forceinline__ half4_t magnitude(half4_t v) {
  return __builtin_bit_cast(half4_t, __builtin_bit_cast(u32x2, v) & 0x7FFF7FFFu);
}
__device__ __forceinline__ half4_t larger(half4_t a, half4_t b) {
  typedef uint16_t quad __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(half4_t, __builtin_elementwise_max(__builtin_bit_cast(quad, a), __builtin_bit_cast(quad, b)));
}

// Selectors of v_perm_b32 that pair the parts of two tokens' words (first token low).
template <int PARTS>
__device__ __forceinline__ uint32_t part_selector(int part) {
  if constexpr (PARTS == 2) return part ? 0x07060302u : 0x05040100u;
  else return 0x0C040C00u + 0x00010001u * (uint32_t)part;  // one byte each, zero above
}

// Operands of a scale group from eight tokens' words: operand i holds dim (8 / PARTS) part + i
// of the words.  Where a word is one part, its low and its high half in turn, to spare
// registers.
template <int PARTS>
constexpr int kTurns = PARTS == 1 ? 2 : 1;
template <int PARTS>
constexpr int kTurnOps = 8 / PARTS / kTurns<PARTS>;
template <int PARTS>
__device__ __forceinline__ void v_operands(const Magic& m, const u32x4& a, const u32x4& b, uint32_t sel, int turn,
                                           half8_t (&out)[kTurnOps<PARTS>]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int p = 0; p < 4; p++) {
    // a part of the even token's word in the low half, of the odd one's in the high: their
    // nibbles 0 become one pair, their nibbles 1 the next
    const uint32_t t = __builtin_amdgcn_perm(w[2 * p + 1], w[2 * p],
                                             PARTS > 1 ? sel : turn ? 0x07060302u : 0x05040100u);
#pragma unroll
    for (int i = 0; i < kTurnOps<PARTS>; i += 2) {
      const half4_t h = m.codes(i ? t >> 8 : t);
      out[i][2 * p] = h.x, out[i][2 * p + 1] = h.y;
      out[i + 1][2 * p] = h.z, out[i + 1][2 * p + 1] = h.w;
    }
  }
}

template <int D, int NG, int TYPE>
__global__ __launch_bounds__(64 * kWaves, 4) void kv4_split_kernel(AttnArgs a) {
  using S = Shape<D, NG>;
  // the waves' rings; later 16 rows of D + 4 floats in each
  static_assert(S::RING * S::STAGE >= 16 * (D + 4) * 4 && S::RING * S::STAGE >= 16 * (kMaxSplits + 2) * 4, "");
  __shared__ __align__(16) uint8_t lds[kWaves * S::RING * S::STAGE];
  __shared__ uint32_t begins[kMaxRequests];
  __shared__ int few_first[64], few_n[64], few_kv[64], few_past[64];
  __shared__ long long wave_sum[kWaves];
  __shared__ int wave_max[kWaves];
  __shared__ uint32_t arrived;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.group;
  const int T = 1 << a.log_page;
  const int KW = 1 << a.log_kw, HW = kWaves >> a.log_kw;
  const int kw = wave & (KW - 1), hw = wave >> a.log_kw;

  // ---- the division: every request's tiles are as long as its last one; rows that see
  // nothing take a unit, to write their zeros.  Without scratch, and where the units do
  // not fit 31 bits, tiles count as one and stay whole ----
  auto blocks_of = [&](const Request& q) { return rows_of(a, q) > a.max_rows ? 0 : (rows_of(a, q) + 15) / 16; };
  auto units_of = [&](const Request& q) { return max((q.kv + kStep * KW - 1) >> (kLogStep + a.log_kw), 1) + a.lead; };
  bool divided = a.partial != nullptr;
  uint32_t total, share;
  // Up to 64 requests are one to a lane, in every wave alike, and found by a ballot; more
  // are two to a thread and searched for.
  const bool few = a.requests <= 64;
  Request own{0, 0, 0, 0};
  if (few && lane < a.requests) own = request_of(a, lane);
  while (true) {
    long long mine[2] = {0, 0};
    int longest = 1;
    auto cost = [&](const Request& q) {
      long long n = ((long long)blocks_of(q) * a.kv_heads + HW - 1) >> (kLogWaves - a.log_kw);
      if (divided) {  // units, and above them tiles: as many as the sums have room for
        if (n > 0) longest = max(longest, units_of(q));
        n = min(n * units_of(q), 1ll << 32) + (min(n, 1023ll) << kTilesAt);
      }
      return n;
    };
    if (few) {
      mine[0] = cost(own);
      if (__ballot(mine[0] > 0) == 0) return;  // beside prompts, no request of few rows
    } else {
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (2 * tid + u < a.requests) mine[u] = cost(request_of(a, 2 * tid + u));
    }
    long long sum = mine[0] + mine[1], all, before;
    if (a.requests > 1) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const long long x = __shfl_up(sum, d);
        if (lane >= d) sum += x;
        longest = max(longest, __shfl_xor(longest, d));
      }
    }
    before = sum - mine[0] - mine[1];
    if (few) {
      const int at = a.requests - 1;
      all = (long long)(uint32_t)__builtin_amdgcn_readlane((int)(sum >> 32), at) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((int)sum, at);
      if (wave == 0) {
        begins[lane] = (uint32_t)before;
        few_first[lane] = own.first, few_n[lane] = own.n, few_kv[lane] = own.kv, few_past[lane] = own.past;
      }
      __syncthreads();
    } else {
      if (lane == 63) {
        wave_sum[wave] = sum;
        wave_max[wave] = longest;
      }
      __syncthreads();
      all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        if (w < wave) before += wave_sum[w];
        all += wave_sum[w];
        longest = max(longest, wave_max[w]);
      }
      begins[2 * tid] = (uint32_t)before;
      begins[2 * tid + 1] = (uint32_t)(before + mine[0]);
      __syncthreads();
    }
    if (divided) {
      const long long tiles = all >> kTilesAt, units = all & ((1ll << kTilesAt) - 1);
      // tiles stay whole, one a workgroup, where none takes much more than an even share
      const bool whole = tiles <= gridDim.x &&
                         (longest - a.lead - kWhole) * (long long)a.slots <= units - tiles * a.lead;
      if (__builtin_amdgcn_readfirstlane((int)(whole || units > 0x7FFFFFFFll))) {
        divided = false;
        continue;
      }
      all = units;
    }
    total = __builtin_amdgcn_readfirstlane((uint32_t)all);
    share = (total + gridDim.x - 1) / gridDim.x;
    // pieces of one unit: no more than one a compute unit (one request of 4000 tokens on 32
    // heads 16.3 us with two, 13.3 so)
    if (divided && share == 1 && total > (uint32_t)a.slots / 2) share = 2;
    // a tile lies in kMaxSplits shares at most
    if (divided) share = max(share, (uint32_t)((longest + kMaxSplits - 2) / (kMaxSplits - 1)));
    share = __builtin_amdgcn_readfirstlane(share);
    break;
  }

  // The lane's index anew, as a value of this piece only: neither it nor what is computed from
  // it is kept in registers through the loop.
  auto lane_again = [] {
    uint32_t ones = ~0u;
    asm volatile("" : "+s"(ones));
    return (int)__builtin_amdgcn_mbcnt_hi(ones, __builtin_amdgcn_mbcnt_lo(ones, 0));
  };
  const Magic magic;
  const uint32_t block = block_bytes<D, NG>(T);
  uint8_t* const ring = lds + wave * (S::RING * S::STAGE);
  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(
      (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)ring));

  const uint32_t first_unit = blockIdx.x * share, last_unit = min(first_unit + share, total);
  uint32_t unit = first_unit;
  while (unit < last_unit) {
    // ---- the piece: steps [s0, s1) of a tile ----
    int r = 0;  // the last request that begins at the unit or before
    Request rq;
    uint32_t r_begin;
    if (few) {
      const int i = lane_again();
      r = 63 - __builtin_clzll(__ballot(i < a.requests && begins[i] <= unit));
      rq = Request{few_first[r], few_n[r], few_kv[r], few_past[r]};
    } else {
      for (int hi = a.requests; hi - r > 1;) {
        const int mid = (r + hi) >> 1;
        if (__builtin_amdgcn_readfirstlane(begins[mid]) <= unit) r = mid;
        else hi = mid;
      }
      rq = request_of(a, r);
    }
    r_begin = begins[r];
    r = __builtin_amdgcn_readfirstlane(r);
    rq.first = __builtin_amdgcn_readfirstlane(rq.first);
    rq.n = __builtin_amdgcn_readfirstlane(rq.n);
    rq.kv = __builtin_amdgcn_readfirstlane(rq.kv);
    rq.past = __builtin_amdgcn_readfirstlane(rq.past);
    set_past(a, r, rq);
    r_begin = __builtin_amdgcn_readfirstlane(r_begin);
    const int rows = rows_of(a, rq), row_blocks = blocks_of(rq), len = divided ? units_of(rq) : 1;
    const int tile = (int)((unit - r_begin) / (uint32_t)len);
    const uint32_t tile_unit = r_begin + (uint32_t)tile * len;
    // the wave's blocks of rows of all heads (it may have none)
    const int own_block = tile * HW + hw, own = min(own_block, row_blocks * a.kv_heads - 1);
    const bool exists = own == own_block;
    const int head = row_blocks == 1 ? own : own / row_blocks, row0 = (own - head * row_blocks) * 16;
    const bool one = rq.n == 1;  // (spares the divisions of a row's index)
    const int t_first = one ? 0 : row0 / G, t_last = one ? 0 : min((row0 + 15) / G, rq.n - 1);
    const int end = seen_by(rq, t_last);   // tokens that some row of the tile sees
    const int all = seen_by(rq, t_first);  // ... that every row sees
    const int steps = (end + kStep - 1) / kStep;
    // this wave's steps: s0, s0 + KW, ... (the tile's first units are its lead)
    const uint32_t next_unit = min(tile_unit + len, last_unit), work_unit = tile_unit + (divided ? a.lead : 0);
    if (next_unit <= work_unit) break;
    const int s0 = (divided ? (int)(max(unit, work_unit) - work_unit) * KW : 0) + kw;
    const int s1 = divided ? min(steps, (int)(next_unit - work_unit) * KW) : steps;
    const int count = exists && s1 > s0 ? (s1 - s0 + KW - 1) >> a.log_kw : 0;
    const bool whole = unit <= work_unit && next_unit == tile_unit + len;
    const bool first_piece = unit == first_unit;
    if (!first_piece) __syncthreads();  // the piece before is done with LDS

    // ---- Q: lane (c, g) holds row c's dims [32 w + 8 g, + 8), slots in the order the
    // unpacking gives ----
    const int lane = lane_again(), c = lane & 15, g = lane >> 4;
    const int blk = c / S::PARTS, part = c % S::PARTS;
    const uint32_t sel = S::PARTS == 1 ? 0u : part_selector<S::PARTS == 1 ? 2 : S::PARTS>(part);
    half8_t qf[S::KW];
    float c1 = a.c1;
    const int row = row0 + c, t_row = one ? 0 : row / G, h_row = one ? min(row, G - 1) : row - t_row * G;
    const int seen = row < rows ? seen_by(rq, t_row) : 0;  // tokens the row sees
    float x[S::KW][8];
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(rq.first + min(t_row, rq.n - 1)) * a.qt +
                          (long long)(head * G + h_row) * a.qh + 8 * g;
    float amax = 0.f;
#pragma unroll
    for (int w = 0; w < S::KW; w++) {
      unpack8<TYPE>(*reinterpret_cast<const u32x4*>(src + 32 * w), x[w]);
#pragma unroll
      for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[w][i]));
    }
    if constexpr (TYPE == BF16) {
      // bf16's range does not fit fp16: rows are brought to [2^7, 2^8) by a power of two
      amax = column_max(amax);
      const int e = amax > 0.f && amax < __builtin_inff() ? 8 - __builtin_amdgcn_frexp_expf(amax) : 0;
#pragma unroll
      for (int w = 0; w < S::KW; w++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[w][i] = __builtin_amdgcn_ldexpf(x[w][i], e);
      c1 = __builtin_amdgcn_ldexpf(c1, -e);
    }
    constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
    for (int w = 0; w < S::KW; w++)
#pragma unroll
      for (int i = 0; i < 8; i++) qf[w][i] = (_Float16)x[w][order[i]];

    // ---- the loop ----
    float4_t O[NG][S::OPS];
    bool big = false, some_big = false;  // the row, some row
    bool fresh = true;                   // (wave-uniform) no step yet
    float M = kNone, L = 0.f, shift = 0.f, x_top = 0.f;  // M = x_top c1 - shift, x_top a score
#pragma unroll
    for (int n = 0; n < NG; n++)
#pragma unroll
      for (int i = 0; i < S::OPS; i++) O[n][i] = (float4_t){0.f, 0.f, 0.f, 0.f};
    const int32_t* pages = a.table + (size_t)r * a.max_pages;
    const uint8_t* const cache = a.cache + (size_t)head * block;

    // Places of 32 of the wave's steps from k on: lane i has half i % 2 of step k + i / 2,
    // the byte offset of its K codes (bit 63: no such page).
    auto places = [&](int k) {
      const int tok = (s0 + (k + (lane >> 1)) * KW) * kStep + 16 * (lane & 1);
      const int id = tok < end ? pages[tok >> a.log_page] : -1;
      const bool there = (uint32_t)id < (uint32_t)a.num_pages;
      // a page that is not there is read as the first one and masked
      const uint64_t at = (uint64_t)(there ? (uint32_t)id : 0u) * a.page_stride + (uint32_t)(tok & (T - 1)) * (D / 2);
      return there ? at : at | 1ull << 63;
    };
    uint64_t now = places(0), then = places(32);  // of steps [32 b, 32 b + 32) and the 32 after
    auto place = [&](uint64_t v, int i) {
      return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
             (uint32_t)__builtin_amdgcn_readlane((int)v, i);
    };
    // Sends step k into a stage of the ring.
    auto send = [&](int k, uint64_t p0, uint64_t p1, uint32_t to) {
      const uint8_t* k0 = cache + (p0 & ~(1ull << 63));
      const uint8_t* k1 = cache + (p1 & ~(1ull << 63));
      const uint32_t v_off = (uint32_t)T * (D / 2);
      if constexpr (D == 128) {  // 16 tokens are 64 lanes' 16 bytes
        sm24::dma16x1(to, 16 * lane, k0);
        sm24::dma16x1(to + 1024, 16 * lane, k1);
        sm24::dma16x1(to + S::V_AT, 16 * lane, k0 + v_off);
        sm24::dma16x1(to + S::V_AT + 1024, 16 * lane, k1 + v_off);
      } else {
        const uint8_t* kl = (lane < 32 ? k0 : k1 - 512) + 16 * lane;
        sm24::dma16(to, kl);
        sm24::dma16(to + S::V_AT, kl + v_off);
      }
      // scales: 8 NG lanes for K and for V of a half; they lie T D - o (D/2 - 2 NG) behind the K codes
      constexpr int L8 = 8 * NG;
      const uint32_t tok = (uint32_t)(s0 + k * KW) * kStep;
      const uint32_t o0 = tok & (T - 1), o1 = (tok + 16) & (T - 1);
      const uint8_t* sc0 = k0 + (uint32_t)T * D - o0 * (D / 2 - 2 * NG);
      const uint8_t* sc1 = k1 + (uint32_t)T * D - o1 * (D / 2 - 2 * NG);
      const uint32_t at = (lane % L8) * 4 + (lane / L8 % 2) * (2 * NG * (uint32_t)T);
      if constexpr (NG == 4) {
        dma4(to + S::S_AT, sc0 + at);
        dma4(to + S::S_AT + 256, sc1 + at);
      } else if (lane < 4 * L8) {
        dma4(to + S::S_AT, (lane < 2 * L8 ? sc0 : sc1) + at);
      }
    };
    auto read_v = [&](const uint8_t* from, int u, int n) {
      return *reinterpret_cast<const u32x4*>(from + S::V_AT + u * (8 * D) + g * (2 * D) + (n * S::BLOCKS + blk) * 16);
    };
    auto read_ks = [&](const uint8_t* from, int u, int n) {
      return *reinterpret_cast<const half4_t*>(from + S::S_AT + u * (64 * NG) + (g * NG + n) * 8);
    };
    auto read_vs = [&](const uint8_t* from, int u, int n) {
      return *reinterpret_cast<const half4_t*>(from + S::S_AT + u * (64 * NG) + 32 * NG + (g * NG + n) * 8);
    };
    auto receive = [&](const uint8_t* from, int u, Codes<D, NG>& f) {
      const uint8_t* kp = from + u * (8 * D) + c * (D / 2) + g * (D / 8);
      if constexpr (D == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kp);
        f.k[u][0] = w.x, f.k[u][1] = w.y, f.k[u][2] = w.z, f.k[u][3] = w.w;
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(kp);
        f.k[u][0] = w.x, f.k[u][1] = w.y;
      }
#pragma unroll
      for (int n = 0; n < NG; n++) {
        if (!S::LATE) {
          f.v[u][n] = read_v(from, u, n);
          f.vs[u][n] = read_vs(from, u, n);
        }
        f.ks[u][n] = read_ks(from, u, n);
      }
    };
    auto compute = [&](int s, bool there0, bool there1, Codes<D, NG>& f, const uint8_t* from) {
      float x[2][4];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        if constexpr (S::LATE) receive(from, u, f);
        float4_t sum[NG];
#pragma unroll
        for (int n = 0; n < NG; n++) {
          sum[n] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < S::STEPS; w++) {
            const half8_t k = k_operand(magic, f.k[u][n * S::STEPS + w]);
            sum[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[n * S::STEPS + w], sum[n], 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          x[u][i] = sum[0][i] * (float)f.ks[u][0][i];
#pragma unroll
          for (int n = 1; n < NG; n++) x[u][i] = __builtin_fmaf(sum[n][i], (float)f.ks[u][n][i], x[u][i]);
        }
      }
      half4_t vs[2][NG];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int n = 0; n < NG; n++) vs[u][n] = S::LATE ? read_vs(from, u, n) : f.vs[u][n];
      // (wave-uniform) a step that some row does not see whole
      const bool masked = (s + 1) * kStep > all || !there0 || !there1;
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int tok = s * kStep + 16 * u + 4 * g + i;
            const bool in = tok < seen && (u ? there1 : there0);
            x[u][i] = in ? x[u][i] : -__builtin_inff();
            // (the scale of a token that the row does not see may be anything)
#pragma unroll
            for (int n = 0; n < NG; n++) vs[u][n][i] = in ? vs[u][n][i] : (_Float16)0.f;
          }
      }
      half4_t vt[2];  // of V, a token's largest scale (of the sizes: bits order as they do)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        vt[u] = magnitude(vs[u][0]);
#pragma unroll
        for (int n = 1; n < NG; n++) vt[u] = larger(vt[u], magnitude(vs[u][n]));
      }
      half8_t P[NG];
      float p[8], sum = 0.f, most = 0.f;  // of this step's tokens: their sum, the largest p v
      auto refer = [&] {
        // A new reference (the four lanes of a row agree): the row's largest score m, and the
        // largest p v of this step, e, and of those before, e_old, in log2 of 2^m's units.
        float m = x[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) m = fmaxf(m, x[i / 4][i % 4]);
        m = column_max(m);
        const bool none = M == kNone;
        const float old_max = none ? kNone : M + shift;
        // Past kBig, where M's rounding would show, scores are taken less the largest one, x_top.
        const bool risen = big ? m > x_top : m * c1 > old_max;
        const float new_max = risen ? m * c1 : old_max;
        const float drop = big ? (risen ? x_top - m : 0.f) * c1 : old_max - new_max;  // (<= 0)
        if (risen) {
          big = fabsf(new_max) > kBig;
          x_top = m;
        }
        float e = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float v = x[i / 4][i % 4];
          e = fmaxf(e, (big ? (v - x_top) * c1 : __builtin_fmaf(v, c1, -new_max)) +
                           __builtin_amdgcn_logf((float)vt[i / 4][i % 4]));
        }
        e = column_max(e);
        const float e_old = none ? e : kVTop - shift + drop;
        // (2^24: below the least v; where all v so far are zero the next may be any)
        const float new_shift = fminf(kVTop - fmaxf(e, e_old), none ? kVTop + 24.f : kMostShift);
        const float new_M = new_max <= kNone ? kNone : new_max - new_shift;
        const float f = none ? 0.f : __builtin_amdgcn_exp2f(big ? drop + (new_shift - shift) : M - new_M);
        M = new_M;
        shift = new_shift;
        some_big = __any(big);
        L *= f;
#pragma unroll
        for (int n = 0; n < NG; n++)
#pragma unroll
          for (int i = 0; i < S::OPS; i++) O[n][i] *= f;
      };
      auto weigh = [&] {
        if (some_big) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float v = x[i / 4][i % 4];
            p[i] = big ? __builtin_fmaf(v - x_top, c1, shift) : __builtin_fmaf(v, c1, -M);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) p[i] = __builtin_fmaf(x[i / 4][i % 4], c1, -M);
        }
        sum = 0.f, most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          p[i] = __builtin_amdgcn_exp2f(p[i]);
          sum += p[i];
          if constexpr (NG > 1) {
            most = fmaxf(most, p[i] * (float)vt[i / 4][i % 4]);
          }
          if constexpr (!S::LATE) {
#pragma unroll
            for (int n = 0; n < NG; n++) {
              const float pv = p[i] * (float)vs[i / 4][n][i % 4];
              if constexpr (NG == 1) most = fmaxf(most, fabsf(pv));
              P[n][i] = (_Float16)pv;
            }
          }
        }
      };
      if (!fresh) weigh();
      // (a row without a reference has p = 2^(10^30) of what it sees)
      if (fresh || __any(!(L + sum < kMostL) || most > kMostPV)) {
        refer();
        fresh = false;
        weigh();
      }
      L += sum;
      if (S::LATE && masked) {  // (a sign marks what is not seen)
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = x[i / 4][i % 4] == -__builtin_inff() ? -0.f : p[i];
      }
#pragma unroll
      for (int n = 0; n < NG; n++) {
        u32x4 v0, v1;
        if constexpr (S::LATE) {
          v0 = read_v(from, 0, n), v1 = read_v(from, 1, n);
          const half4_t s[2] = {read_vs(from, 0, n), read_vs(from, 1, n)};
#pragma unroll
          for (int i = 0; i < 8; i++) P[n][i] = (_Float16)(p[i] * (float)s[i / 4][i % 4]);
          if (masked) {  // what is not seen is zero, whatever its scale (a seen NaN shows)
#pragma unroll
            for (int i = 0; i < 8; i++) P[n][i] = __builtin_signbit(p[i]) ? (_Float16)0.f : P[n][i];
          }
        } else {
          v0 = f.v[0][n], v1 = f.v[1][n];
        }
#pragma unroll
        for (int turn = 0; turn < kTurns<S::PARTS>; turn++) {
          constexpr int OT = kTurnOps<S::PARTS>;
          half8_t vo[OT];
          v_operands<S::PARTS>(magic, v0, v1, sel, turn, vo);
#pragma unroll
          for (int i = 0; i < OT; i++)
            O[n][turn * OT + i] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(vo[i], P[n], O[n][turn * OT + i], 0, 0, 0);
        }
        if constexpr (S::LATE) __builtin_amdgcn_sched_barrier(0);  // (registers: a group at a time)
      }
    };

#pragma unroll
    for (int k = 0; k < S::RING; k++)
      if (k < count) send(k, place(now, 2 * k), place(now, 2 * k + 1), ring_at + k * S::STAGE);
    int stage = 0;
#pragma unroll 1
    for (int k = 0; k < count; k++) {
      if (k > 0 && (k & 31) == 0) {
        now = then;
        then = places(k + 32);
      }
      const int i = 2 * (k & 31);
      const bool there0 = __builtin_amdgcn_readlane((int)(now >> 32), i) >= 0;
      const bool there1 = __builtin_amdgcn_readlane((int)(now >> 32), i + 1) >= 0;
      if (k + S::RING <= count) sm24::wait_vm<(S::RING - 1) * S::LOADS>();
      else sm24::wait_vm<0>();
      Codes<D, NG> f;
      if constexpr (!S::LATE) {
        receive(ring + stage * S::STAGE, 0, f);
        receive(ring + stage * S::STAGE, 1, f);
      }
      if (S::LATE) compute(s0 + k * KW, there0, there1, f, ring + stage * S::STAGE);
      // the stage's reads are done before it is filled again
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (k + S::RING < count) {
        const int j = 2 * ((k + S::RING) & 31);
        if ((k & 31) + S::RING < 32) send(k + S::RING, place(now, j), place(now, j + 1), ring_at + stage * S::STAGE);
        else send(k + S::RING, place(then, j), place(then, j + 1), ring_at + stage * S::STAGE);
      }
      stage = stage + 1 == S::RING ? 0 : stage + 1;
      if (!S::LATE) compute(s0 + k * KW, there0, there1, f, nullptr);
    }

    // ---- the waves of a block of rows meet: lane (c, g) holds row c's dims of MFMA
    // rows 4 g + i; then the waves share out the items (row, four dims) ----
    constexpr int RP = D + 4, Q4 = D / 4;  // floats of a row in LDS, items of a row
    const int et = lane_again(), ec = et & 15, eg = et >> 4;
    const int item0 = et + 64 * kw, items = 64 << a.log_kw;
    uint8_t* const group = lds + (hw << a.log_kw) * (S::RING * S::STAGE);  // those waves' rings
    const int live_rows = min(rows - row0, 16);
    // a piece's place in the scratch, and a row of this head in it
    auto slot_row = [&](uint32_t w, int second, int row) {
      return (((size_t)w * 2 + second) * HW + hw) * 16 + row;
    };
    auto write = [&](int row, int d0, float m, float l, const float4_t& o) {
      const int i = row0 + row, t = one ? 0 : i / G;
      const size_t at = (size_t)(rq.first + t) * a.q_heads + head * G + i - t * G;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // no token seen: zeros (a NaN stays one)
      uint16_t* dst = static_cast<uint16_t*>(a.out) + at * D + d0;
      *reinterpret_cast<u32x2*>(dst) =
          (u32x2){(uint32_t)from_float<TYPE>(o.x * inv) | (uint32_t)from_float<TYPE>(o.y * inv) << 16,
                  (uint32_t)from_float<TYPE>(o.z * inv) | (uint32_t)from_float<TYPE>(o.w * inv) << 16};
      if (a.lse != nullptr && d0 == 0)
        a.lse[at] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    };
    __syncthreads();  // the rings are done with
    L = column_sum(L);
    float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int n = 0; n < NG; n++)
#pragma unroll
      for (int i = 0; i < S::OPS; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int m = 4 * eg + k;
          mine[ec * RP + 8 * (n * S::BLOCKS + m / S::PARTS) + (8 / S::PARTS) * (m % S::PARTS) + i] = O[n][i][k];
        }
    if (eg == 0) *reinterpret_cast<float2*>(mine + ec * RP + D) = make_float2(M, L);
    __syncthreads();
#pragma unroll 1
    for (int it = item0; it < 16 * Q4; it += items) {
      const int row = it / Q4, d0 = it % Q4 * 4;
      if (!exists || row >= live_rows) break;  // (rows ascend)
      const float* from = reinterpret_cast<const float*>(group) + row * RP;
      constexpr int NEXT = S::RING * S::STAGE / 4;  // floats from a wave's to the next
      float m = kNone, l = 0.f;
      float4_t o = {0.f, 0.f, 0.f, 0.f};
      float2 ml[kWaves];
      float4_t v[kWaves];
#pragma unroll
      for (int w = 0; w < kWaves; w++) {  // (all reads in flight; those past KW repeat the last and do not count)
        const float* at = from + min(w, KW - 1) * NEXT;
        ml[w] = *reinterpret_cast<const float2*>(at + D);
        v[w] = *reinterpret_cast<const float4_t*>(at + d0);
      }
#pragma unroll
      for (int w = 0; w < kWaves; w++) m = fmaxf(m, ml[w].x);
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float f = w < KW ? __builtin_amdgcn_exp2f(ml[w].x - m) : 0.f;
        l += f * ml[w].y;
        o += v[w] * f;
      }
      if (whole) {
        write(row, d0, m, l, o);
      } else {
        const size_t at = slot_row(blockIdx.x, first_piece ? 0 : 1, row);
        *reinterpret_cast<float4_t*>(a.partial + at * D + d0) = o;
        if (d0 == 0) *reinterpret_cast<float2*>(a.partial_ml + at * 2) = make_float2(m, l);
      }
    }
    if (!whole) {
      // every thread's stores are done before the barrier, the counter (the first
      // workgroup's: only its last piece is a tile's beginning) moves after it
      const uint32_t w0 = work_unit / share, pieces = (tile_unit + len - 1) / share - w0 + 1;
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_waitcnt(0);
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __syncthreads();
      if (wave == 0 && et == 0)
        arrived = __hip_atomic_fetch_add(a.counters + w0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
      __syncthreads();
      if (arrived == pieces) {
        if (wave == 0 && et == 0) __hip_atomic_store(a.counters + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // only the first workgroup's piece may be its second
        const int second0 = w0 * share < tile_unit ? 1 : 0;
        float* weight = reinterpret_cast<float*>(group);  // [row][piece], then [row] {reference, sum}
        float* row_ml = weight + 16 * kMaxSplits;
        const int left = exists ? live_rows : 0;
        // lane s reads a row's reference and sum of piece s; the wave weighs the pieces
        float2 ml[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const int row = kw + (j << a.log_kw);
          ml[j] = make_float2(kNone, 0.f);
          if (row < left && et < (int)pieces)
            ml[j] = *reinterpret_cast<const float2*>(
                a.partial_ml + slot_row(w0 + et, et == 0 ? second0 : 0, row) * 2);
        }
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const int row = kw + (j << a.log_kw);
          if (row < left) {  // (wave-uniform)
            float m = ml[j].x;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
            const float f = et < (int)pieces ? __builtin_amdgcn_exp2f(ml[j].x - m) : 0.f;
            float l = f * ml[j].y;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
            if (et < kMaxSplits) weight[row * kMaxSplits + et] = f;
            if (et == 0) row_ml[2 * row] = m, row_ml[2 * row + 1] = l;
          }
        }
        __syncthreads();
#pragma unroll 1
        for (int it = item0; it < left * Q4; it += items) {
          const int row = it / Q4, d0 = it % Q4 * 4;
          float4_t o = {0.f, 0.f, 0.f, 0.f};
          constexpr int FLIGHT = 8;  // pieces in flight
#pragma unroll 1
          for (uint32_t s = 0; s < pieces; s += FLIGHT) {
            float4_t v[FLIGHT];
#pragma unroll
            for (int k = 0; k < FLIGHT; k++) {
              const uint32_t p = min(s + k, pieces - 1);
              v[k] = *reinterpret_cast<const float4_t*>(
                  a.partial + slot_row(w0 + p, p == 0 ? second0 : 0, row) * D + d0);
            }
#pragma unroll
            for (int k = 0; k < FLIGHT; k++) o += v[k] * weight[row * kMaxSplits + s + k];  // (zero past the last)
          }
          write(row, d0, row_ml[2 * row], row_ml[2 * row + 1], o);
        }
      }
    }
    unit = next_unit;
  }
}

}  // namespace kv4
