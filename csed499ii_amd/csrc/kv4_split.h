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
// A workgroup takes 16 rows (one MFMA's columns) of one head and a range of 32-token
// steps, its waves every fourth step.  Per step and wave:
//   S^T = K Q^T  16x16x32 MFMAs, A = codes (rows = 16 tokens), B = Q, held in registers;
//                lane (c, g) gets row c's sums of tokens 4 g .. 4 g + 3: what the second
//                product wants as its B operand, if its reduction index counts tokens
//                4 g + i of the step's two halves, so p never leaves its lane;
//   O^T = V^T P^T  A = codes of V, each word's 8 dims spread over the accumulators.
// (The offset 8 is taken off the codes, one packed operation for two.  Left in the products
// and subtracted from the sums it costs less, but the sums then grow to 8 sum p v and lose
// in fp32 what a small output has: 10^-6 of the largest v was seen.)
//
// M is not the running maximum but a reference it may exceed by 2^kSlack before
// accumulators are rescaled, which a wave-uniform branch does then: rare after the first
// steps, and the exact maximum is not needed for an exact softmax.  M also carries the
// power of two that keeps p v in fp16's normal range (p v is rounded to fp16 for the
// matrix cores, relative error 2^-12, averaged over the tokens; sums are fp32): M rises
// when a larger v is met, too.
//
// What does not exist must not count: tokens past the row's last one, pages whose table
// entry is not a page, slots never written (their scales may be NaN).  Their p v is set to
// zero after the product, not multiplied by zero.
//
// The waves meet in LDS; with more than one split the partial sums go through the
// uncached scratch, and the last workgroup to arrive on the tile's counter adds them in
// split order: one launch, and the same bits from run to run.
#pragma once
#include "kv4_device.h"

namespace kv4 {

constexpr int kWaves = 4;
constexpr int kStep = 32;          // tokens per wave and step
constexpr float kSlack = 8.f;      // p <= 2^8 of the reference
constexpr float kVTop = 7.f;       // v 2^shift <= 2^7, so p v <= 2^15 < 65504
constexpr float kNone = -1.0e30f;  // reference of a row that has seen nothing

struct AttnArgs {
  const void* q;
  const uint8_t* cache;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu_q;  // null: request i is token i
  void* out;
  float* lse;           // null: not wanted
  float* partial;       // [tile][split][16][D + 2]
  uint32_t* counters;   // [tile], zero between launches
  long long qt, qh;     // strides of q in elements
  int tokens, requests, q_heads, kv_heads;
  int num_pages, max_pages, log_page;
  int row_blocks, splits;
  int max_rows;         // rows of a request above this are another kernel's
  float c1;             // softmax scale * log2 e
};

struct Request {
  int first, n, kv;  // first token, new tokens, tokens in all
};
__device__ __forceinline__ Request request_of(const AttnArgs& a, int r) {
  Request q;
  q.kv = min(max(a.kv_lens[r], 0), a.max_pages << a.log_page);  // (at most 2^30)
  if (a.cu_q == nullptr) {
    q.first = r;
    q.n = 1;
  } else {
    q.first = min(max(a.cu_q[r], 0), a.tokens);
    q.n = max(min(a.cu_q[r + 1], a.tokens) - q.first, 0);
  }
  return q;
}

// Codes of one 32-token step as loaded.  BLOCKS: 8-dim words of a scale group, whose 16
// MFMA rows are word row / PARTS, part row % PARTS.
template <int D, int NG>
struct Shape {
  static constexpr int KW = D / 32;             // words of K a lane holds per half = k-steps
  static constexpr int BLOCKS = D / NG / 8;     // 16, 8 or 4
  static constexpr int PARTS = 16 / BLOCKS;     // 1, 2 or 4
  static constexpr int OPS = 8 / PARTS;         // MFMAs per scale group
  static constexpr int STEPS = KW / NG;         // k-steps per scale group
};

template <int D, int NG>
struct Codes {
  uint32_t k[2][D / 32];
  u32x4 v[2][NG];       // four tokens each
  half4_t ks[2][NG], vs[2][NG];
};

// Codes of a word less 8, in nibble order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half8_t k_operand(uint32_t w) {
  const half4_t a = sm24::dequant4(w), b = sm24::dequant4(w >> 8);
  return (half8_t){a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

// Selectors of v_perm_b32 that pair the parts of two tokens' words (first token low).
template <int PARTS>
__device__ __forceinline__ uint32_t part_selector(int part) {
  if constexpr (PARTS == 2) return part ? 0x07060302u : 0x05040100u;
  else return 0x0C040C00u + 0x00010001u * (uint32_t)part;  // one byte each, zero above
}

// Operands 0 .. OPS - 1 of a scale group from eight tokens' words: operand i holds dim
// (8 / PARTS) part + i of the words.
template <int PARTS>
__device__ __forceinline__ void v_operands(const u32x4& a, const u32x4& b, uint32_t sel, half8_t (&out)[8 / PARTS]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int p = 0; p < 4; p++) {
    const uint32_t x = w[2 * p], y = w[2 * p + 1];
    // t: a part of x's word in the low half, of y's in the high one; dequant4 pairs their
    // nibbles 0, then their nibbles 1
    auto put = [&](int i, uint32_t t) {
      const half4_t h = sm24::dequant4(t);
      out[i][2 * p] = h.x, out[i][2 * p + 1] = h.y;
      out[i + 1][2 * p] = h.z, out[i + 1][2 * p + 1] = h.w;
    };
    if constexpr (PARTS == 1) {
      const uint32_t t0 = __builtin_amdgcn_perm(y, x, 0x05040100u), t1 = __builtin_amdgcn_perm(y, x, 0x07060302u);
      put(0, t0);
      put(2, t0 >> 8);
      put(4, t1);
      put(6, t1 >> 8);
    } else {
      const uint32_t t = __builtin_amdgcn_perm(y, x, sel);
      put(0, t);
      if constexpr (PARTS == 2) put(2, t >> 8);
    }
  }
}

template <int D, int NG, int TYPE>
__global__ __launch_bounds__(64 * kWaves) void kv4_split_kernel(AttnArgs a) {
  using S = Shape<D, NG>;
  constexpr int RP = D + 4;  // floats per row in LDS
  __shared__ __align__(16) float red[kWaves][16][RP];
  __shared__ float red_m[kWaves][16], red_l[kWaves][16];
  __shared__ uint32_t arrived;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % a.splits;
  const int tile = blockIdx.x / a.splits;  // (request, head, row block)
  const int rb = tile % a.row_blocks;
  const int head = tile / a.row_blocks % a.kv_heads;
  const int r = tile / a.row_blocks / a.kv_heads;
  const int G = a.q_heads / a.kv_heads;
  const int T = 1 << a.log_page;

  const Request rq = request_of(a, r);
  const int rows = rq.n * G;
  if (rows > a.max_rows || rb * 16 >= rows) return;
  const int past = rq.kv - rq.n;  // token t sees tokens 0 .. past + t
  const int t_first = rb * 16 / G, t_last = min((rb * 16 + 15) / G, rq.n - 1);
  const int end = max(past + t_last + 1, 0);  // tokens that some row of the block sees
  const int all = min(max(past + t_first + 1, 0), end);  // ... that every row sees

  // this split's steps: at least one a wave, so short requests take fewer splits
  const int steps = (end + kStep - 1) / kStep;
  const int per = max((steps + a.splits - 1) / a.splits, kWaves);
  const int live = max((steps + per - 1) / per, 1);
  if (split >= live) return;
  const int s0 = split * per, s1 = min(s0 + per, steps);

  // ---- Q: lane (c, g) holds row c's dims [32 w + 8 g, + 8), slots in the order the
  // unpacking gives ----
  const int row = rb * 16 + c;
  const int t_row = row / G, h_row = head * G + row % G;
  const int seen = row < rows ? max(past + t_row + 1, 0) : 0;  // tokens the row sees
  half8_t qf[S::KW];
  float c1 = a.c1;
  {
    float x[S::KW][8];
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(rq.first + min(t_row, rq.n - 1)) * a.qt +
                          (long long)h_row * a.qh + 8 * g;
    float amax = 0.f;
#pragma unroll
    for (int w = 0; w < S::KW; w++) {
      unpack8<TYPE>(*reinterpret_cast<const u32x4*>(src + 32 * w), x[w]);
#pragma unroll
      for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[w][i]));
    }
    if constexpr (TYPE == BF16) {
      // bf16's range does not fit fp16: rows are brought to [2^7, 2^8) by a power of two
      amax = fmaxf(amax, __shfl_xor(amax, 16));
      amax = fmaxf(amax, __shfl_xor(amax, 32));
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
  }

  // ---- the loop ----
  float4_t O[NG][S::OPS];
  float M = kNone, L = 0.f;
#pragma unroll
  for (int n = 0; n < NG; n++)
#pragma unroll
    for (int i = 0; i < S::OPS; i++) O[n][i] = (float4_t){0.f, 0.f, 0.f, 0.f};
  float shift = 0.f, v_top = 0.f;  // v 2^shift <= 2^kVTop while v <= v_top
  float x_top = kNone;              // x above which M rises
  const int blk = c / S::PARTS, part = c % S::PARTS;
  const uint32_t sel = S::PARTS == 1 ? 0u : part_selector<S::PARTS == 1 ? 2 : S::PARTS>(part);
  const size_t block = block_bytes<D, NG>(T);
  const int32_t* pages = a.table + (size_t)r * a.max_pages;

  // page ids of the wave's next 32 steps: lane i holds the page of half i % 2 of step i / 2
  auto fetch_ids = [&](int s) {
    const int tok = (s + (lane >> 1) * kWaves) * kStep + 16 * (lane & 1);
    const int id = tok < end ? pages[tok >> a.log_page] : -1;
    return (uint32_t)id < (uint32_t)a.num_pages ? id : -1;
  };
  auto fetch = [&](int s, int id0, int id1, Codes<D, NG>& f) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int id = u ? id1 : id0;
      const int o = (s * kStep + 16 * u) & (T - 1);
      // a page that is not there is read as the first one and masked
      const uint8_t* b = a.cache + ((size_t)max(id, 0) * a.kv_heads + head) * block;
      const uint8_t* kp = b + (o + c) * (D / 2) + g * (D / 8);
      if constexpr (D == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(kp);
        f.k[u][0] = w.x, f.k[u][1] = w.y, f.k[u][2] = w.z, f.k[u][3] = w.w;
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(kp);
        f.k[u][0] = w.x, f.k[u][1] = w.y;
      }
#pragma unroll
      for (int n = 0; n < NG; n++) {
        f.v[u][n] = *reinterpret_cast<const u32x4*>(b + v_word<D>(T, o + 4 * g, n * S::BLOCKS + blk));
        f.ks[u][n] = *reinterpret_cast<const half4_t*>(b + k_scale<D, NG>(T, o + 4 * g, n));
        f.vs[u][n] = *reinterpret_cast<const half4_t*>(b + v_scale<D, NG>(T, o + 4 * g, n));
      }
    }
  };
  auto compute = [&](int s, int id0, int id1, const Codes<D, NG>& f) {
    float x[2][4];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      float4_t sum[NG];
#pragma unroll
      for (int n = 0; n < NG; n++) {
        sum[n] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < S::STEPS; w++)
          sum[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k_operand(f.k[u][n * S::STEPS + w]), qf[n * S::STEPS + w],
                                                          sum[n], 0, 0, 0);
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
      for (int n = 0; n < NG; n++) vs[u][n] = f.vs[u][n];
    // (wave-uniform) a step that some row does not see whole
    const bool masked = (s + 1) * kStep > all || id0 < 0 || id1 < 0;
    if (masked) {
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int tok = s * kStep + 16 * u + 4 * g + i;
          const bool in = tok < seen && (u ? id1 : id0) >= 0;
          x[u][i] = in ? x[u][i] : -__builtin_inff();
#pragma unroll
          for (int n = 0; n < NG; n++) vs[u][n][i] = in ? vs[u][n][i] : (_Float16)0.f;
        }
    }
    float xm = x[0][0], vm = 0.f;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        xm = fmaxf(xm, x[u][i]);
#pragma unroll
        for (int n = 0; n < NG; n++) vm = fmaxf(vm, (float)vs[u][n][i]);
      }
    if (__any(xm > x_top || vm > v_top)) {
      // new reference: the rows' maxima so far and the largest v of all lanes
      xm = fmaxf(xm, __shfl_xor(xm, 16));
      xm = fmaxf(xm, __shfl_xor(xm, 32));
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) vm = fmaxf(vm, __shfl_xor(vm, d));
      float new_shift = shift;
      if (vm > v_top) {
        // vm <= 2^e; 2^24 bounds the shift where every v so far is tiny or zero
        new_shift = fminf(kVTop - (float)__builtin_amdgcn_frexp_expf(vm), 24.f);
        v_top = __builtin_amdgcn_exp2f(kVTop - new_shift);
      }
      // M = max - shift: rows keep the larger of the old maximum and this step's
      const float old_max = M == kNone ? kNone : M + shift;
      const float new_max = fmaxf(old_max, xm * c1);
      const float new_M = new_max <= kNone ? kNone : new_max - new_shift;
      const float f = M == kNone ? 0.f : __builtin_amdgcn_exp2f(M - new_M);
      M = new_M;
      shift = new_shift;
      x_top = M == kNone ? kNone : (new_max + kSlack) / c1;
      L *= f;
#pragma unroll
      for (int n = 0; n < NG; n++)
#pragma unroll
        for (int i = 0; i < S::OPS; i++) O[n][i] *= f;
    }
    half4_t ph[2][NG];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], c1, -M));
        L += p;
#pragma unroll
        for (int n = 0; n < NG; n++) ph[u][n][i] = (_Float16)(p * (float)vs[u][n][i]);
      }
#pragma unroll
    for (int n = 0; n < NG; n++) {
      const half8_t P = {ph[0][n][0], ph[0][n][1], ph[0][n][2], ph[0][n][3],
                         ph[1][n][0], ph[1][n][1], ph[1][n][2], ph[1][n][3]};
      half8_t vo[S::OPS];
      v_operands<S::PARTS>(f.v[0][n], f.v[1][n], sel, vo);
#pragma unroll
      for (int i = 0; i < S::OPS; i++) O[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vo[i], P, O[n][i], 0, 0, 0);
    }
  };

  for (int base = s0 + wave; base < s1; base += 32 * kWaves) {
    const int ids = fetch_ids(base);
    const int count = min((s1 - base + kWaves - 1) / kWaves, 32);
    auto id = [&](int i) { return __builtin_amdgcn_readlane(ids, i); };
    Codes<D, NG> f[2];
    fetch(base, id(0), id(1), f[0]);
    for (int k = 0; k < count; k += 2) {
      if (k + 1 < count) fetch(base + (k + 1) * kWaves, id(2 * k + 2), id(2 * k + 3), f[1]);
      compute(base + k * kWaves, id(2 * k), id(2 * k + 1), f[0]);
      if (k + 1 < count) {
        if (k + 2 < count) fetch(base + (k + 2) * kWaves, id(2 * k + 4), id(2 * k + 5), f[0]);
        compute(base + (k + 1) * kWaves, id(2 * k + 2), id(2 * k + 3), f[1]);
      }
    }
  }

  // ---- the waves meet: lane (c, g) holds row c's dims of MFMA rows 4 g + i ----
  L += __shfl_xor(L, 16);
  L += __shfl_xor(L, 32);
#pragma unroll
  for (int n = 0; n < NG; n++)
#pragma unroll
    for (int i = 0; i < S::OPS; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int m = 4 * g + k;
        const int d = 8 * (n * S::BLOCKS + m / S::PARTS) + (8 / S::PARTS) * (m % S::PARTS) + i;
        red[wave][c][d] = O[n][i][k];
      }
  if (g == 0) {
    red_m[wave][c] = M;
    red_l[wave][c] = L;
  }
  __syncthreads();
  // thread: row tid / 16, dims [D/16 * (tid % 16), + D/16)
  constexpr int E = D / 16;
  const int rr = tid >> 4, d0 = E * (tid & 15);
  const bool exists = rb * 16 + rr < rows;
  float m = red_m[0][rr];
#pragma unroll
  for (int w = 1; w < kWaves; w++) m = fmaxf(m, red_m[w][rr]);
  float l = 0.f, o[E] = {};
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const float f = __builtin_amdgcn_exp2f(red_m[w][rr] - m);
    l += f * red_l[w][rr];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] += f * red[w][rr][d0 + e];
  }
  if (live > 1) {
    constexpr int W = D + 2;
    float* part = a.partial + ((size_t)tile * a.splits + split) * 16 * W + (size_t)rr * W;
    if (exists) {
#pragma unroll
      for (int e = 0; e < E; e += 2) *reinterpret_cast<float2*>(part + d0 + e) = make_float2(o[e], o[e + 1]);
      if ((tid & 15) == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
    }
    // every thread's stores are done before the barrier, the counter moves after it
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (tid == 0)
      arrived = __hip_atomic_fetch_add(a.counters + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    __syncthreads();
    if (arrived != (uint32_t)live) return;
    if (tid == 0) __hip_atomic_store(a.counters + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!exists) return;
    const float* all_parts = a.partial + (size_t)tile * a.splits * 16 * W + (size_t)rr * W;
    m = kNone;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.f;
    for (int s = 0; s < live; s++) {
      const float* p = all_parts + (size_t)s * 16 * W;
      const float2 ml = *reinterpret_cast<const float2*>(p + D);
      const float nm = fmaxf(m, ml.x);
      const float f0 = __builtin_amdgcn_exp2f(m - nm), f1 = __builtin_amdgcn_exp2f(ml.x - nm);
      m = nm;
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 v = *reinterpret_cast<const float2*>(p + d0 + e);
        o[e] = o[e] * f0 + v.x * f1;
        o[e + 1] = o[e + 1] * f0 + v.y * f1;
      }
    }
  }
  if (!exists) return;
  const int t_out = (rb * 16 + rr) / G, h_out = head * G + (rb * 16 + rr) % G;
  const size_t at = (size_t)(rq.first + t_out) * a.q_heads + h_out;
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no token seen: zeros (a NaN stays one)
  uint16_t* dst = static_cast<uint16_t*>(a.out) + at * D + d0;
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(dst + e) =
        (uint32_t)from_float<TYPE>(o[e] * inv) | (uint32_t)from_float<TYPE>(o[e + 1] * inv) << 16;
  if (a.lse != nullptr && (tid & 15) == 0)
    a.lse[at] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

}  // namespace kv4
