// Attention of many query rows (prompts, chunks of prompts) over the 4-bit paged cache.
//
// The sums of kv4_split.h, on 32x32x16 MFMAs: a wave keeps 32 rows, a workgroup of eight
// goes through the tokens that its rows see, 64 at a time.  Its waves turn the tile's codes
// into fp16 (less 8, exact) once for all eight, straight into the MFMAs' operand order in
// LDS, one tile ahead of the products; the codes come from memory two tiles ahead.
//   S^T = K Q^T    A = K from LDS, B = Q in registers; lane (c, h) gets row c's sums of tokens
//                  8 b + 4 h + i of a half tile (32 tokens)
//   O^T = V^T P^T  A = V from LDS, B = p v, whose reduction index counts those tokens: p
//                  stays in its lane
// Sixteen tokens lie in one page, and are what a wave loads at once: the page is the wave's,
// so that a tile costs it a few scalar operations and one load.
//
// Bound by issue: a wave issues an operation of any kind every 4.1 to 4.8 cycles, two waves of
// a SIMD in parallel, and an MFMA takes its 32 cycles and hides nearly no other operation of
// either wave (32 + 2.1 n cycles for one beside n of the vector ALU, with two waves).  So what
// counts is operations per score, of any kind, and neither LDS (254 of 256 bytes a clock with
// eight waves) nor the order of products and softmax.  A tile of 128 dims takes 4400 cycles:
// 2048 of MFMAs, some 1600 of vector operations at their rates, the rest waits.  4096 tokens
// on 32 heads of 128 dims: 161 us, 854 TFLOP/s, where a large library product reaches 1161;
// MFMAs are 36 % of all its cycles, beginnings, ends and the division included.
// Tried: four waves and 128 rows (198), 32-token tiles and three workgroups a compute unit
// (232), scales as fp16 in mixed FMAs (168 where this took 164), products and softmax of two tiles interleaved
// (186 to 191); 64 dims in 128 registers, for two workgroups a compute unit, spill.
//
// Fewer blocks of rows than compute units are divided over their tokens, one part a
// workgroup; the waves of the same rows meet in the uncached scratch, and the last to arrive
// adds the parts in order.  A 512-token chunk on 64 and 8 heads with 4096 in all: 134 us
// whole, 87 in two parts, whose write and read take 6.
//
// SHARED, first pass: 64 requests on 64 and 8 heads that share 8192 tokens are 512 rows a head, 16
// blocks in 16 parts of 8 tiles: 37 us, 460 TFLOP/s, of which beginnings, the write of the parts (34 MB)
// and 8 tiles' worth of filling take half.  WINDOW: 8000 tokens on 32 heads through 1024 and a few first
// ones, 231 us where 126 GFLOP are seen: of a block's 21 tiles twelve are whole.
#pragma once
#include "kv4_split.h"

namespace kv4 {

constexpr int kMaxKinds = 256;     // row blocks of a launch whose tokens are divided
constexpr int kMaxParts = kMaxPartsLeft;  // of a row block's tokens
constexpr float kMinShare = 4.f;   // tiles: a part costs its write and its read

typedef float float16_t __attribute__((ext_vector_type(16)));

// Place of dim 8 blk + i of V among the MFMA rows: the rows of a scale group fill
// whole MFMAs, and consecutive words go to consecutive rows.
template <int D, int NG>
__device__ __forceinline__ constexpr int v_row(int blk, int i) {
  constexpr int BL = D / 8 / NG;
  return blk / BL * (8 * BL) + i * BL + blk % BL;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, (half2_t){(_Float16)lo, (_Float16)hi});
}

template <int D, int NG, int TYPE, int FORM = PLAIN>
__global__ __launch_bounds__(64 * kPromptWaves, 2) void kv4_prompt_kernel(AttnArgs a) {
  constexpr int W = kPromptWaves;
  constexpr int KU = D / 16;          // k-steps of the first product
  constexpr int GU = KU / NG;         // ... per scale group
  constexpr int DT = D / 32;          // MFMAs of 32 dims of the second
  constexpr int BL = D / 8 / NG;      // words of a scale group
  constexpr int K_BYTES = kTile * D * 2, V_BYTES = K_BYTES, S_BYTES = 2 * NG * kTile * 4;
  constexpr int BUF = K_BYTES + V_BYTES + S_BYTES;  // operands and scales of a tile
  constexpr int PIECES = kTile * D / 2 / 16;  // 16-byte pieces of K codes, and of V codes
  constexpr int GROUPS = kTile / 16;          // of tokens in one page
  // Halves of a tile whose scores are held at once: both, for products and softmax side by
  // side, where the products are long enough for it (2048 tokens of 4096 on 64 and 8 heads of 128
  // dims, groups of 32: 339 us with both, 353 one by one, of 64 272 and 274; 4000 on 16 and 4
  // heads of 64 dims 109 and 100).
  constexpr int HALVES = D == 128 ? 2 : 1;
  __shared__ __align__(16) uint8_t lds[2 * BUF];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const int G = a.group, T = 1 << a.log_page;

  // ---- the piece: which request's, which block of rows, which part of its tokens ----
  // Heads fastest, so that a head stays on one XCD; a request's last block, the longest, first.
  __shared__ __align__(16) int kinds[kMaxKinds], kind_tiles[kMaxKinds];
  const int head = blockIdx.x % a.kv_heads, index = blockIdx.x / a.kv_heads;
  auto blocks_of = [&](const Request& q) { return rows_of(a, q) > a.max_rows ? (rows_of(a, q) + kPromptRows - 1) / kPromptRows : 0; };
  // tokens that some row of a block sees
  auto end_of = [&](const Request& q, int block) {
    return seen_by(q, min((block * kPromptRows + kPromptRows - 1) / G, q.n - 1));
  };
  // (WINDOW) the tiles of tokens that some row of a block sees
  auto reach_of = [&](const Request& q, int block) {
    const int t0 = block * kPromptRows / G, t1 = min((block * kPromptRows + kPromptRows - 1) / G, q.n - 1);
    return Reach(a, q, t0, t1, seen_by(q, t1), kLogTile);
  };
  auto tiles_in = [&](const Request& q, int block) {
    if constexpr (FORM == WINDOW) return reach_of(q, block).steps;
    return (end_of(q, block) + kTile - 1) / kTile;
  };
  const int per = (a.requests + 63) / 64, r_lane = lane * per;  // a lane's requests
  int own = 0;
  for (int r = r_lane; r < min(r_lane + per, a.requests); r++) own += blocks_of(request_of<FORM>(a, r));
  auto scan = [&](int x) {  // what the lanes before have
    int sum = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(sum, d);
      if (lane >= d) sum += y;
    }
    return sum - x;
  };
  const int before = scan(own), all = __builtin_amdgcn_readlane(before + own, 63);
  if (all == 0) return;
  int r, block, part = 0, parts = 1, most = 0;
  uint32_t slot = blockIdx.x;  // a divided block's workgroup's place in the scratch
  if (a.partial == nullptr || all > min(a.pieces, kMaxKinds)) {
    // Workgroups for all compute units: whole, but for the last ones, where they would keep
    // less than half of the units busy (nine requests of 256 new tokens, 2048 in all, on 32
    // heads, 288 blocks: 155 us whole, 116 with the last 32 divided).
    const int rest = a.partial != nullptr && a.rest ? all % a.pieces : 0;
    const int ways = 2 * rest <= a.pieces && rest > 0 ? min(a.pieces / rest, kMaxParts) : 1;
    const int whole = ways > 1 ? all - rest : all;
    int kind = index;
    if (index >= whole) {
      kind = whole + (index - whole) / ways;
      if (ways == 1 || kind >= all) return;
      part = (index - whole) % ways;
      most = ways;
      slot = (uint32_t)((index - whole) * a.kv_heads + head);
    }
    const int at = __builtin_ctzll(__ballot(before + own > kind));
    int i = kind - __builtin_amdgcn_readlane(before, at);
    r = at * per;
    int n = blocks_of(request_of<FORM>(a, r));
    while (i >= n) {
      i -= n;
      n = blocks_of(request_of<FORM>(a, ++r));
    }
    block = n - 1 - i;
  } else {
    // Divided: parts of (nearly) one length, the shortest of 64 that give no more parts than
    // there are workgroups for this head.
    if (wave == 0) {
      // a request after the other, its blocks over the lanes
      for (uint64_t with = __ballot(own > 0); with != 0; with &= with - 1) {
        const int at = __builtin_ctzll(with);
        int i = __builtin_amdgcn_readlane(before, at);
        for (int r = at * per; r < min(at * per + per, a.requests); r++) {
          Request q = request_of<FORM>(a, r);
          set_past(a, r, q);
          const int n = blocks_of(q);
          for (int b = lane; b < n; b += 64) {
            kinds[i + b] = r * kMaxKinds + n - 1 - b;
            kind_tiles[i + b] = max(tiles_in(q, n - 1 - b), 1);
          }
          i += n;
        }
      }
    }
    __syncthreads();
    int tiles_of[4];  // of the kinds 4 lane + (0 .. 3)
    float sum = 0.f, longest = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      tiles_of[k] = 4 * lane + k < all ? kind_tiles[4 * lane + k] : 0;
      sum += (float)tiles_of[k];
      longest = fmaxf(longest, (float)tiles_of[k]);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      sum += __shfl_xor(sum, d);
      longest = fmaxf(longest, __shfl_xor(longest, d));
    }
    const float lo = fmaxf(fmaxf(sum / (float)a.pieces, kMinShare), longest / (float)kMaxParts), hi = fmaxf(lo, longest);
    // (in the other forms from the shortest itself on, in equal ratios: of 128 tiles in two blocks and 32 workgroups
    // 16 parts of 8 where steps of hi / 64 make 13 of 10)
    const float per_tile = FORM == PLAIN
        ? 1.f / (lo + (hi - lo) * ((float)(lane + 1) / 64.f))
        : __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(hi / lo) * ((float)lane / -63.f)) / lo;
    auto parts_of = [&](int tiles, float f) { return max((int)ceilf((float)tiles * f - 0.001f), 1); };
    int n = 0;
    for (int i = 0; i < all; i += 4) {
      const int4 t = *reinterpret_cast<const int4*>(kind_tiles + i);
      n += parts_of(t.x, per_tile) + (i + 1 < all ? parts_of(t.y, per_tile) : 0) +
           (i + 2 < all ? parts_of(t.z, per_tile) : 0) + (i + 3 < all ? parts_of(t.w, per_tile) : 0);
    }
    const float f = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, per_tile), __builtin_ctzll(__ballot(n <= a.pieces || lane == 63))));
    int parts_to[5] = {0};  // of this lane's kinds, up to each
#pragma unroll
    for (int k = 0; k < 4; k++) parts_to[k + 1] = parts_to[k] + (tiles_of[k] > 0 ? parts_of(tiles_of[k], f) : 0);
    const int ahead = scan(parts_to[4]);
    const uint64_t past_it = __ballot(ahead + parts_to[4] > index);
    if (past_it == 0) return;
    const int at = __builtin_ctzll(past_it), left = index - __builtin_amdgcn_readlane(ahead, at);
    int i = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int from = __builtin_amdgcn_readlane(parts_to[k], at), to = __builtin_amdgcn_readlane(parts_to[k + 1], at);
      if (left >= from && left < to) i = 4 * at + k, part = left - from, parts = to - from;
    }
    const int kind = __builtin_amdgcn_readfirstlane(kinds[i]);
    r = kind / kMaxKinds, block = kind % kMaxKinds;
  }
  Request rq = request_of<FORM>(a, r);
  set_past(a, r, rq);
  const int rows = rows_of(a, rq), row0 = block * kPromptRows;
  const int w_row0 = row0 + 32 * wave;
  // tokens that some row of the workgroup, some row of the wave and every row of it sees
  const int end = end_of(rq, block);
  Reach reach;
  if constexpr (FORM == WINDOW) reach = reach_of(rq, block);
  auto token_of = [&](int tile) { return FORM == WINDOW ? reach.at(tile, kLogTile) : tile * kTile; };
  const int tiles = FORM == WINDOW ? reach.steps : (end + kTile - 1) / kTile;
  if (most > 0) {
    if constexpr (FORM == WINDOW) parts = max(min(most, tiles / (int)kMinShare), 1);
    else parts = max(min(most, (end + kTile - 1) / (kTile * (int)kMinShare)), 1);
    if (part >= parts) return;
  }
  const int w_end = w_row0 < rows ? seen_by(rq, min((w_row0 + 31) / G, rq.n - 1)) : 0;
  const int w_all = min(seen_by(rq, w_row0 / G), w_end);
  // (WINDOW) where the wave's first window begins, and its last
  const int w_low = FORM == WINDOW ? window_of(a, rq, w_row0 / G) : 0;
  const int w_high = FORM == WINDOW ? window_of(a, rq, min((w_row0 + 31) / G, rq.n - 1)) : 0;

  typedef __attribute__((address_space(3))) uint8_t lds_u8;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_u8*)lds;

  // Where 64 groups of 16 tokens (16 tiles) from 64 b on begin, one a lane: the table's entries
  // as they come (a look at once would wait for them and for every load before them), then the
  // byte offset of the K codes (bit 63: no such page, which is read as the first one and masked).
  const int t0 = tiles * part / parts, t1 = tiles * (part + 1) / parts;
  const int32_t* pages = pages_of<FORM>(a, r, rq);
  // (first token of a lane's group of the block)
  auto group_at = [&](int b) {
    if constexpr (FORM == WINDOW) return token_of(16 * b + (lane >> 2)) + 16 * (lane & 3);
    return (64 * b + lane) * 16;
  };
  auto entries = [&](int b) { return pages[min(group_at(b), end - 1) >> a.log_page]; };
  int entry0 = 0, entry1 = 0, entry = 0;  // (here, so that they and Q come together)
  if (t0 < t1) {
    entry0 = entries(t0 >> 4);
    entry1 = entries((t0 >> 4) + 1);
    entry = entries((t0 >> 4) + 2);
  }

  // ---- Q ----
  const int seen = w_row0 + c < rows ? seen_by(rq, min((w_row0 + c) / G, rq.n - 1)) : 0;
  const int hidden = FORM == WINDOW ? window_of(a, rq, min((w_row0 + c) / G, rq.n - 1)) : 0;  // tokens before it: sinks only
  half8_t qf[KU];
  float down = 1.f, up = 1.f;  // scores per product of the row's operands (a power of two), and back
  {
    const int row = w_row0 + c, t_row = min(row / G, rq.n - 1), h_row = head * G + row % G;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(rq.first + t_row) * a.qt +
                          (long long)h_row * a.qh + 8 * h;
    u32x4 raw[KU];
#pragma unroll
    for (int u = 0; u < KU; u++) raw[u] = *reinterpret_cast<const u32x4*>(src + 16 * u);
    if constexpr (TYPE == BF16) {
      float amax = 0.f;
#pragma unroll
      for (int u = 0; u < KU; u++) {
        float x[8];
        unpack8<TYPE>(raw[u], x);
#pragma unroll
        for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));
      }
      const Pair p = across32(amax);
      amax = fmaxf(p.a, p.b);
      // (2^100 where all is so small that its scores are zero anyway)
      const int e = amax > 0.f && amax < __builtin_inff() ? min(8 - __builtin_amdgcn_frexp_expf(amax), 100) : 0;
#pragma unroll
      for (int u = 0; u < KU; u++) {
        float x[8];
        unpack8<TYPE>(raw[u], x);
        constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for (int i = 0; i < 8; i++) qf[u][i] = (_Float16)__builtin_amdgcn_ldexpf(x[order[i]], e);
      }
      down = __builtin_amdgcn_ldexpf(1.f, -e);
      up = __builtin_amdgcn_ldexpf(1.f, e);
    } else {
#pragma unroll
      for (int u = 0; u < KU; u++) {
        const half8_t q = __builtin_bit_cast(half8_t, raw[u]);
        qf[u] = (half8_t){q[0], q[4], q[1], q[5], q[2], q[6], q[3], q[7]};
      }
    }
  }

  // ---- the codes of a tile: a wave's pieces are all of K or all of V ----
  const Magic magic;
  const uint8_t* const cache = a.cache + (size_t)head * block_bytes<D, NG>(T);
  // a wave's pieces: of K (the first waves) or of V, of one group (D = 128) or of two
  constexpr int KWAVES = PIECES / 64;
  static_assert(2 * KWAVES <= W && (KWAVES == GROUPS || 2 * KWAVES == GROUPS), "");
  const bool is_k = wave < KWAVES, is_v = !is_k && wave < 2 * KWAVES;

  auto places = [&](int b, int entry) {
    const int tok = group_at(b);
    const bool there = (uint32_t)entry < (uint32_t)a.num_pages;
    const uint64_t at = (uint64_t)(there ? (uint32_t)entry : 0u) * a.page_stride + (uint32_t)(tok & (T - 1)) * (D / 2);
    return there || tok >= end ? at : at | 1ull << 63;
  };
  uint64_t now = 0, then = 0;  // of the block of the tile in use, and of the one after
  auto place = [&](int tile, int g, int block_now) {
    const int i = (tile & 15) * GROUPS + g;
    const uint64_t v = tile >> 4 == block_now ? now : then;
    return cache + ((uint64_t)(uint32_t)(__builtin_amdgcn_readlane((int)(v >> 32), i) & 0x7FFFFFFF) << 32 |
                    (uint32_t)__builtin_amdgcn_readlane((int)v, i));
  };
  u32x4 raw;
  uint32_t raw_scales;
  auto fetch = [&](int tile, int block_now) {
    if (!is_k && !is_v) return;
    const uint32_t v_off = is_k ? 0u : (uint32_t)T * (D / 2);
    if constexpr (KWAVES == GROUPS) {
      raw = *reinterpret_cast<const u32x4*>(place(tile, wave % GROUPS, block_now) + v_off + (uint32_t)(16 * lane));
    } else {
      const int g = wave % KWAVES * 2;
      const uint8_t *p0 = place(tile, g, block_now) + v_off, *p1 = place(tile, g + 1, block_now) + v_off;
      raw = *reinterpret_cast<const u32x4*>((lane < 32 ? p0 : p1) + (uint32_t)(16 * (lane & 31)));
    }
  };
  // Scales of a group: 8 NG lanes of K, as many of V.  (The waves without V's longer unpacking.)
  const int s_group = KWAVES == GROUPS ? wave : wave - 2 * KWAVES;
  const bool s_mine = s_group >= 0 && s_group < GROUPS;
  const uint32_t s_lane = (lane % (8 * NG)) * 4 + (lane / (8 * NG)) * (2 * NG * (uint32_t)T) + (uint32_t)T * D;
  auto fetch_scales = [&](int tile, int block_now) {
    raw_scales = 0;
    if (s_mine) {
      const uint32_t o = (uint32_t)(token_of(tile) + 16 * s_group) & (T - 1);
      const uint8_t* b = place(tile, s_group, block_now) - o * (D / 2 - 2 * NG);
      if (lane < 16 * NG) raw_scales = *reinterpret_cast<const uint32_t*>(b + s_lane);
    }
  };
  // Slot of token t among a tile's of a K operand: turned by the reader's lane group, so that
  // the writing lanes (four words of a row side by side) hit different banks.
  auto k_slot = [](int t, int g) { return (t + 4 * g) & (kTile - 1); };
  // Where a thread writes V's operands in a tile: quad q gives reduction steps of 16 tokens,
  // lanes' halves, first or second four.  (One register: the compiler would keep its terms.)
  const int v_piece = tid - PIECES, v_quad = v_piece / (D / 8), v_blk = v_piece % (D / 8);
  uint32_t v_to = K_BYTES + ((v_quad >> 2) * 2 + (v_quad & 1)) * (D * 16) + (v_quad >> 1 & 1) * 8 + v_row<D, NG>(v_blk, 0) * 16;
  asm volatile("" : "+v"(v_to));
  auto unpack = [&](int tile) {
    uint8_t* const to = lds + (tile & 1) * BUF;
    if (s_mine && lane < 16 * NG) {
      // fp32, K's with the softmax's factor: a score is one FMA.  (Kept as fp16 for mixed FMAs,
      // which issue at half the rate, and the factor apart: 168 us where this takes 164, 4096
      // tokens on 32 heads; with groups of 32 465 and 448, 2048 on 64 and 8 heads of 4096.)
      const half2_t v = __builtin_bit_cast(half2_t, raw_scales);
      const float f = lane < 8 * NG ? a.c1 : 1.f;
      *reinterpret_cast<float2*>(to + K_BYTES + V_BYTES + s_group * (128 * NG) + lane * 8) =
          make_float2((float)v.x * f, (float)v.y * f);
    }
    if (is_k) {
      constexpr int PT = D / 32;  // pieces of a token
      const int t = tid / PT;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int word = tid % PT * 4 + j, g = word / (D / 32), b = 4 * (word % (D / 32)) + g;
        *reinterpret_cast<half8_t*>(to + (b * kTile + k_slot(t, g)) * 16) = k_operand(magic, raw[j]);
      }
    } else if (is_v) {
      uint8_t* const v = to + v_to;
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const uint32_t s = half ? 0x07060302u : 0x05040100u;
        const uint32_t x = __builtin_amdgcn_perm(raw.y, raw.x, s), y = __builtin_amdgcn_perm(raw.w, raw.z, s);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const half4_t lo = magic.codes(k ? x >> 8 : x), hi = magic.codes(k ? y >> 8 : y);
          const int i = 4 * half + 2 * k;
          *reinterpret_cast<half4_t*>(v + i * BL * 16) = (half4_t){lo.x, lo.y, hi.x, hi.y};
          *reinterpret_cast<half4_t*>(v + (i + 1) * BL * 16) = (half4_t){lo.z, lo.w, hi.z, hi.w};
        }
      }
    }
  };

  float16_t O[DT];
  // M as in kv4_split.h; the scores, in units of `down`, are taken less `base`, which is M, or
  // 0 before there is one
  float M = kNone, base = 0.f, L = 0.f;
  bool some_none = true;  // some row of the wave that has tokens here has no M
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) O[t][i] = 0.f;

  // LDS addresses of this lane's operands in the tile in use: everything else of an address
  // is an instruction's constant.
  auto read16 = [](uint32_t at, int more) {
    return *(const __attribute__((address_space(3))) half8_t*)(uintptr_t)(at + more);
  };
  // Scales [group of 16][K, V][quad][NG][4] of tokens 8 b + 4 h + (0 .. 3) of half j.
  auto scale_of = [&](uint32_t scales_lane, int kv, int n, int j, int b) {
    const int more = (2 * j + b / 2) * (128 * NG) + kv * (64 * NG) + (2 * (b & 1) * NG + n) * 16;
    return *(const __attribute__((address_space(3))) float4_t*)(uintptr_t)(scales_lane + more);
  };
  auto compute = [&](int tile, uint32_t hole) {
    const uint32_t buf = lds_at + (tile & 1) * BUF;
    uint32_t scales_lane = buf + K_BYTES + V_BYTES + 16 * NG * h;
    uint32_t even[2] = {buf + (h * kTile + k_slot(c, h)) * 16, buf + (h * kTile + k_slot(32 + c, h)) * 16};
    uint32_t odd[2] = {buf + (h * kTile + k_slot(c, 2 + h)) * 16, buf + (h * kTile + k_slot(32 + c, 2 + h)) * 16};
    const int tok0 = token_of(tile);
    const bool masked = tok0 + kTile > w_all || hole != 0 || (FORM == WINDOW && tok0 < w_high && tok0 + kTile > a.sinks);
    // Scores of half j, less base.
    auto scores_of = [&](int j, float (&x)[16]) {
#pragma unroll
      for (int n = 0; n < NG; n++) {
        float16_t S;
#pragma unroll
        for (int i = 0; i < 16; i++) S[i] = 0.f;
#pragma unroll
        for (int u = n * GU; u < (n + 1) * GU; u++)
          S = __builtin_amdgcn_mfma_f32_32x32x16_f16(read16((u & 1 ? odd : even)[j], u * (2 * kTile * 16)), qf[u], S, 0, 0, 0);
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float4_t s = scale_of(scales_lane, 0, n, j, b);
#pragma unroll
          for (int i = 0; i < 4; i++)
            x[4 * b + i] = __builtin_fmaf(S[4 * b + i], s[i], n == 0 ? -base : x[4 * b + i]);
        }
      }
    };
    // -infinity for what a row does not see, `least` at least for what it does (NaN stays): once
    // there is a reference so much that p is not zero, which what is not seen is told by.
    auto mask = [&](int j, float (&x)[16], float least) {
      int left = seen - tok0 - 4 * h;
      asm volatile("" : "+v"(left));  // (else done for every tile)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int t = 32 * j + 8 * (i / 4) + i % 4;
        const bool in = t < left && !(hole >> (2 * j + i / 8) & 1);
        x[i] = in ? x[i] < least ? least : x[i] : -__builtin_inff();
      }
    };
    // The same through a window, by a bit for each token of a half tile, from 4 h on, that the lane's row sees:
    // two operations a score and two a pair of p v, where comparisons take twelve.  (Through a window of 1024 nine
    // tiles of a block of rows are masked in some wave: 8000 tokens on 32 heads, 291 us so and 260 by bits.)
    uint32_t bits[2] = {0, 0};
    if (FORM == WINDOW && masked) {
      int mine = tok0 + 4 * h;
      asm volatile("" : "+v"(mine));
#pragma unroll
      for (int j = 0; j < 2; j++) {
        auto below = [&](int t) { return t - mine - 32 * j >= 32 ? ~0u : (1u << max(t - mine - 32 * j, 0)) - 1u; };
        bits[j] = below(seen);
        if constexpr (FORM == WINDOW) bits[j] &= ~below(hidden) | below(a.sinks);
        if (hole >> (2 * j) & 1) bits[j] &= 0xFFFF0000u;
        if (hole >> (2 * j + 1) & 1) bits[j] &= 0x0000FFFFu;
      }
    }
    auto sees = [&](int j, int i) { return (uint32_t)__builtin_amdgcn_sbfe((int)bits[j], 8 * (i / 4) + i % 4, 1); };  // all ones or none
    auto hide = [&](int j, float (&x)[16]) {
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const uint32_t s = sees(j, i);
        x[i] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x[i]) & s) | (0xFF800000u & ~s));
      }
    };
    // p and p v (fp16 pairs) of half j; sum of p, the largest p v.
    auto weigh = [&](int j, float (&x)[16], u32x4 (&P)[NG][2], float& sum, float& most) {
      sum = 0.f, most = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) {
        x[i] = __builtin_amdgcn_exp2f(x[i] * down);
        sum += x[i];
      }
#pragma unroll
      for (int n = 0; n < NG; n++) {
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float4_t s = scale_of(scales_lane, 1, n, j, b);
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float lo = x[4 * b + i] * s[i], hi = x[4 * b + i + 1] * s[i + 1];
            most = fmaxf(fmaxf(most, fabsf(lo)), fabsf(hi));
            P[n][b >> 1][2 * (b & 1) + i / 2] = pack2(lo, hi);
          }
        }
        asm volatile("" : "+v"(sum), "+v"(most));  // (now, not when all of p v is in registers)
      }
      if (masked) {  // what a row does not see is zero, whatever its scale
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          uint32_t keep;
          if constexpr (FORM != WINDOW) keep = (x[i] == 0.f ? 0u : 0xFFFFu) | (x[i + 1] == 0.f ? 0u : 0xFFFF0000u);
          else keep = (sees(j, i) & 0xFFFFu) | (sees(j, i + 1) & 0xFFFF0000u);
#pragma unroll
          for (int n = 0; n < NG; n++) P[n][i / 8][i % 8 / 2] &= keep;
        }
      }
    };
    // A new reference from the scores x of half j, which come to lie less it; what it is higher by.
    // In log2 units: the largest score xm and the largest p v, which lies e over it, are brought
    // to 2^-rel and to 2^kVTop at most.
    auto refer = [&](int j, float (&x)[16]) {
      float xm = -__builtin_inff(), e = xm;
#pragma unroll
      for (int i = 0; i < 16; i++) xm = fmaxf(xm, x[i]);
      const Pair px = across32(xm);
      xm = fmaxf(px.a, px.b);
#pragma unroll
      for (int b = 0; b < 4; b++) {
        float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NG; n++) {
          const float4_t s = scale_of(scales_lane, 1, n, j, b);
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = fmaxf(v[i], fabsf(s[i]));
        }
#pragma unroll
        for (int i = 0; i < 4; i++)  // (what is not seen makes -inf or NaN, which count for nothing)
          e = fmaxf(e, __builtin_fmaf(x[4 * b + i] - xm, down, __builtin_amdgcn_logf(v[i])));
      }
      const Pair pe = across32(e);
      e = fmaxf(pe.a, pe.b);
      const bool none = M == kNone, any = xm > -__builtin_inff();
      const float rel = fmaxf(e - kVTop, none && !(e > -__builtin_inff()) ? -kNoV : -kMostShift);
      const bool rises = any && (none || __builtin_fmaf(xm, down, rel) > 0.f);
      const float new_base = rises ? base + __builtin_fmaf(rel, up, xm) : base;
      float less = new_base - base;
      // (scores so large that base's rounding moves it by more than the slack: p = 1 for the largest)
      const bool coarse = rises && !(fabsf(__builtin_fmaf(xm - less, down, rel)) <= kSlack);
      if (coarse) less = xm;
      base = coarse ? base + xm : new_base;
      const float f = none ? 0.f : __builtin_amdgcn_exp2f(-less * down);
      M = none && !any ? kNone : base * down;
      some_none = __any(M == kNone && seen > token_of(t0));
      L *= f;
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] -= less;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) O[t][i] *= f;
      return less;
    };
    const float least = -126.f * up;
    const uint32_t v_at = buf + K_BYTES + (h * D + c) * 16;
#pragma unroll
    for (int j0 = 0; j0 < 2; j0 += HALVES) {
      float x[HALVES][16];
#pragma unroll
      for (int jj = 0; jj < HALVES; jj++) scores_of(j0 + jj, x[jj]);
      if (masked) {
#pragma unroll
        for (int jj = 0; jj < HALVES; jj++) {
          if constexpr (FORM != WINDOW) mask(j0 + jj, x[jj], some_none ? -__builtin_inff() : least);
          else hide(j0 + jj, x[jj]);
        }
      }
#pragma unroll
      for (int jj = 0; jj < HALVES; jj++) {
        const int j = j0 + jj;
        u32x4 P[NG][2];
        float sum = 0.f, most = 0.f;
        auto refer_to = [&] {
          const float less = refer(j, x[jj]);
          if (jj + 1 < HALVES) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[HALVES - 1][i] -= less;
          }
          if (FORM != WINDOW && masked) {
#pragma unroll
            for (int k = jj; k < HALVES; k++) mask(j0 + k, x[k], least);
          }
          asm volatile("" ::: "memory");  // (else V's scales are kept in registers)
        };
        const bool first = some_none;
        if (!first) weigh(j, x[jj], P, sum, most);
        if (first || __any(!(L + sum < kMostL) || most > kMostPV)) {
          // Rare; from the scores on once more, which are not kept, for their registers.  (Else
          // what is read both times is, and addresses by the dozen.)
          if (!first) {
            asm volatile("" : "+v"(even[j]), "+v"(odd[j]), "+v"(scales_lane)::"memory");
            scores_of(j, x[jj]);
            if (masked) {
              if constexpr (FORM != WINDOW) mask(j, x[jj], -__builtin_inff());
              else hide(j, x[jj]);
            }
          }
          refer_to();
          weigh(j, x[jj], P, sum, most);
        }
        L += sum;
#pragma unroll
        for (int n = 0; n < NG; n++)
#pragma unroll
          for (int s = 0; s < 2; s++)
#pragma unroll
            for (int t = n * (DT / NG); t < (n + 1) * (DT / NG); t++)
              O[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read16(v_at, ((2 * j + s) * 2 * D + 32 * t) * 16),
                                                            __builtin_bit_cast(half8_t, P[n][s]), O[t], 0, 0, 0);
      }
    }
  };

  if (t0 < t1) {
    const int b0 = t0 >> 4;
    now = places(b0, entry0);
    then = places(b0 + 1, entry1);
    uint64_t missing = __ballot((int64_t)now < 0);  // groups of the block whose page is not there
    fetch(t0, b0);
    fetch_scales(t0, b0);
    unpack(t0);
    fetch_scales(t0 + 1, b0);
    fetch(t0 + 1, b0);
    __syncthreads();
#pragma unroll 1
    for (int tile = t0; tile < t1; tile++) {
      const int b = tile >> 4;
      if (tile > t0 && (tile & 15) == 0) {
        now = then;
        then = places(b + 1, entry);
        entry = entries(b + 2);
        missing = __ballot((int64_t)now < 0);
      }
      if (FORM == WINDOW ? token_of(tile) < w_end && (token_of(tile) + kTile > w_low || token_of(tile) < a.sinks)
                         : tile * kTile < w_end)
        compute(tile, (uint32_t)(missing >> ((tile & 15) * GROUPS)) & ((1u << GROUPS) - 1));
      if (tile + 1 < t1) {
        unpack(tile + 1);
        fetch_scales(tile + 2, b);
        fetch(tile + 2, b);
      }
      __syncthreads();
    }
  }

  // (the thread's index anew: what is made from it is not kept in registers through the loop)
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));
  const int out_lane = thread & 63, out_c = out_lane & 31, out_h = out_lane >> 5;
  const int row = w_row0 + out_c, t_row = row / G, h_row = head * G + row - t_row * G;
  // ---- out: lane (c, h) holds row c's dims of MFMA rows 8 (k / 4) + 4 h + k % 4 ----
  const Pair pl = across32(L);
  float l = pl.a + pl.b;
  if (parts > 1) {
    // The waves of the same rows meet in memory; the last to arrive (its own stores and
    // those it reads are ordered by its wait and by the counter) adds the parts in order.
    if (w_row0 >= rows) return;
    constexpr int kPart = DT * 16 * 64;  // floats of a wave's part
    const uint32_t stride = (uint32_t)a.kv_heads * W;  // from a part's waves to the next one's
    const uint32_t first = (slot - (uint32_t)(part * a.kv_heads)) * W + wave, mine = first + part * stride;
    if (FORM == SHARED && a.parts != nullptr) {
      // left for the second pass (below)
    } else if constexpr (FORM != PLAIN) {
      // By pairs: of two neighbouring sums the first to arrive leaves its own and ends, the other adds
      // it, the earlier part's first, and goes on with the pair's.  (One wave for all parts reads them one
      // after the other: 13 parts of 512 rows on 8 heads, 8192 tokens, 58 us where this takes 55.)
      uint32_t low = part;  // of the parts that O sums
      for (uint32_t width = 1; width < (uint32_t)parts; width *= 2) {
        const uint32_t other = low ^ width;
        if (other >= (uint32_t)parts) continue;
        uint32_t* const met = a.counters + first + max(low, other) * stride;
        uint32_t there = 0;
        if (out_lane == 0) there = __hip_atomic_load(met, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__builtin_amdgcn_readfirstlane(there) == 0) {
          float* const o_low = a.partial + (size_t)(first + low * stride) * kPart + 4 * out_lane;
#pragma unroll
          for (int t = 0; t < DT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              *reinterpret_cast<float4_t*>(o_low + (4 * t + i) * 256) =
                  (float4_t){O[t][4 * i], O[t][4 * i + 1], O[t][4 * i + 2], O[t][4 * i + 3]};
          *reinterpret_cast<float2*>(a.partial_ml + (size_t)(first + low * stride) * 128 + 2 * out_lane) = make_float2(M, l);
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
          __builtin_amdgcn_s_waitcnt(0);
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
          if (out_lane == 0) there = __hip_atomic_fetch_add(met, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (__builtin_amdgcn_readfirstlane(there) == 0) return;
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        if (out_lane == 0) __hip_atomic_store(met, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const float2 x = *reinterpret_cast<const float2*>(a.partial_ml + (size_t)(first + other * stride) * 128 + 2 * out_lane);
        const float* const o = a.partial + (size_t)(first + other * stride) * kPart + 4 * out_lane;
        float4_t v[DT * 4];
#pragma unroll
        for (int i = 0; i < DT * 4; i++) v[i] = *reinterpret_cast<const float4_t*>(o + i * 256);
        const float most = fmaxf(M, x.x), f = __builtin_amdgcn_exp2f(M - most), g = __builtin_amdgcn_exp2f(x.x - most);
        const bool after = other < low;
        l = after ? __builtin_fmaf(x.y, g, l * f) : __builtin_fmaf(l, f, x.y * g);
        M = most;
#pragma unroll
        for (int i = 0; i < DT * 16; i++) {
          const float mine_i = O[i / 16][i % 16], v_i = v[i / 4][i % 4];
          O[i / 16][i % 16] = after ? __builtin_fmaf(v_i, g, mine_i * f) : __builtin_fmaf(mine_i, f, v_i * g);
        }
        low = min(low, other);
      }
    } else {
    float* const o_mine = a.partial + (size_t)mine * kPart + 4 * out_lane;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        *reinterpret_cast<float4_t*>(o_mine + (4 * t + i) * 256) =
            (float4_t){O[t][4 * i], O[t][4 * i + 1], O[t][4 * i + 2], O[t][4 * i + 3]};
    float* const ml = a.partial_ml + 2 * out_lane;
    *reinterpret_cast<float2*>(ml + (size_t)mine * 128) = make_float2(M, l);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    uint32_t arrived = 0;
    if (out_lane == 0) arrived = __hip_atomic_fetch_add(a.counters + first, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    if ((int)__builtin_amdgcn_readfirstlane(arrived) != parts) return;
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (out_lane == 0) __hip_atomic_store(a.counters + first, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float most = M;
    for (int p = 0; p < parts; p += 8) {
      float m[8];  // (those past the last repeat it)
#pragma unroll
      for (int i = 0; i < 8; i++) m[i] = ml[(size_t)(first + min(p + i, parts - 1) * stride) * 128];
#pragma unroll
      for (int i = 0; i < 8; i++) most = fmaxf(most, m[i]);
    }
    float16_t sum[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int i = 0; i < 16; i++) sum[t][i] = 0.f;
    l = 0.f;
#pragma unroll 1
    for (int p = 0; p < parts; p++) {
      const uint32_t at = first + p * stride;
      const float2 x = *reinterpret_cast<const float2*>(ml + (size_t)at * 128);
      const float* o = a.partial + (size_t)at * kPart + 4 * out_lane;
      float4_t v[DT * 4];
#pragma unroll
      for (int i = 0; i < DT * 4; i++) v[i] = *reinterpret_cast<const float4_t*>(o + i * 256);
      const float f = __builtin_amdgcn_exp2f(x.x - most);
      l += f * x.y;
#pragma unroll
      for (int i = 0; i < DT * 16; i++) sum[i / 16][i % 16] = __builtin_fmaf(v[i / 4][i % 4], f, sum[i / 16][i % 16]);
    }
    M = most;
#pragma unroll
    for (int t = 0; t < DT; t++) O[t] = sum[t];
    }
  }
  // (the passes' addresses from the kernel's arguments anew: not kept in registers through the loop either)
  typedef const __attribute__((address_space(4))) AttnArgs* Late;
  Late late = (Late)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(late));
  const size_t at = (size_t)(rq.first + t_row) * a.q_heads + h_row;
  uint16_t* const dst = static_cast<uint16_t*>(a.out) + at * D;
  float own_f = 1.f, before_f = 0.f;  // (SHARED, second pass) factors of these sums and of the first pass's
  size_t left_at = at;  // where a first pass leaves its sums
  float* left = nullptr;
  if constexpr (FORM == SHARED) {
    left = late->before;
    if (late->parts != nullptr && late->start == nullptr) {
      if (parts > 1) {
        // (a slot's rows are the block's; the parts of a block are kv_heads slots apart)
        left = late->parts;
        left_at = (size_t)slot * kPromptRows + 32 * wave + out_c;
      }
      if (part == 0 && out_h == 0 && row < rows) late->where[at] = make_int2((int)left_at, parts > 1 ? parts : 0);
    }
    if (late->start != nullptr && rq.start > 0 && row < rows) {
      const float2 ml = *reinterpret_cast<const float2*>(late->before_ml + 2 * at);
      const float most = fmaxf(M, ml.x);
      own_f = __builtin_amdgcn_exp2f(M - most), before_f = __builtin_amdgcn_exp2f(ml.x - most);
      M = most, l = own_f * l + before_f * ml.y;
    }
  }
  // (SHARED) the first pass leaves its sums; the second adds them
  const bool leaves = FORM == SHARED && late->start == nullptr;
  const float norm = l == 0.f ? 0.f : 1.f / l;  // no token seen: zeros (a NaN stays one)
  const float inv = leaves ? 1.f : FORM == SHARED ? own_f * norm : norm;
  if constexpr (FORM == SHARED) before_f *= norm;
  auto finish = [&](float (&x)[8], int d) {
    if (row >= rows) return;
    if constexpr (FORM == SHARED) {
      if (rq.start > 0) {
        const float4_t* const b = reinterpret_cast<const float4_t*>(late->before + at * D + d);
        const float4_t v[2] = {b[0], b[1]};
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __builtin_fmaf(v[i / 4][i % 4], before_f, x[i]);
      }
    }
    *reinterpret_cast<u32x4*>(dst + d) = pack8<TYPE>(x);
  };
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) O[t][i] *= inv;
  // f(eight dims, the first one's place) of the lane's row
  auto words = [&](auto f) {
  if constexpr (BL >= 8) {
    // all eight dims of a word: row v_row(blk, i) of the group
#pragma unroll
    for (int n = 0; n < NG; n++)
#pragma unroll
      for (int k = 0; k < BL / 2; k++) {  // words 4 out_h + k % 4 + 8 (k / 4) of the group
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const int m = i * BL + 8 * (k / 4);  // MFMA row less 4 out_h + k % 4
          x[i] = O[n * (BL / 4) + m / 32][m % 32 / 8 * 4 + k % 4];
        }
        f(x, 8 * (n * BL + 8 * (k / 4) + 4 * out_h + k % 4));
      }
  } else {
    // a lane has every other dim (2 e + out_h) of each of the group's four words: the lanes of a
    // row exchange, and write two words each
#pragma unroll
    for (int n = 0; n < NG; n++)
#pragma unroll
      for (int k = 0; k < 2; k++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float low = O[n][4 * e + k], high = O[n][4 * e + k + 2];  // (by value: a choice of elements becomes an index)
          const float keep = out_h ? high : low, give = out_h ? low : high;
          const float got = __shfl_xor(give, 32);
          x[2 * e] = out_h ? got : keep;
          x[2 * e + 1] = out_h ? keep : got;
        }
        f(x, 8 * (n * 4 + k + 2 * out_h));
      }
  }
  };
  if constexpr (FORM == SHARED) {
    if (leaves) {
      // Through LDS, which the tiles no longer need: a wave's rows, 16 at a time, come out side by side.  (Each
      // lane's eight dims straight to memory: 42.9 us where this takes 38.5, 64 requests on 64 and 8 heads that
      // share 8192 tokens.)
      constexpr int RP = 16 * (D + 4) * 4 * W <= 2 * BUF ? D + 4 : D;
      static_assert(16 * RP * 4 * W <= 2 * BUF, "");
      float* const mine = reinterpret_cast<float*>(lds) + wave * (16 * RP);
#pragma unroll 1
      for (int half = 0; half < 2; half++) {
        words([&](float (&x)[8], int d) {
          if (out_c >> 4 != half) return;
          float4_t* const to = reinterpret_cast<float4_t*>(mine + (out_c & 15) * RP + d);
          to[0] = (float4_t){x[0], x[1], x[2], x[3]};
          to[1] = (float4_t){x[4], x[5], x[6], x[7]};
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        constexpr int ITEMS = 16 * D / 4 / 64;  // of four dims
        float4_t v[ITEMS];
        uint32_t lo[ITEMS], hi[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
          const int item = out_lane + 64 * i, r = item / (D / 4), d = item % (D / 4) * 4;
          v[i] = *reinterpret_cast<const float4_t*>(mine + r * RP + d);
          lo[i] = __shfl((int)(uint32_t)left_at, 16 * half + r), hi[i] = __shfl((int)(uint32_t)(left_at >> 32), 16 * half + r);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
          const int item = out_lane + 64 * i, r = item / (D / 4), d = item % (D / 4) * 4;
          if (w_row0 + 16 * half + r < rows)
            *reinterpret_cast<float4_t*>(left + ((size_t)hi[i] << 32 | lo[i]) * D + d) = v[i];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    } else {
      words(finish);
    }
  } else {
    words(finish);
  }
  if constexpr (FORM == SHARED) {
    if (leaves) {
      float* const ml = left == late->before ? late->before_ml : late->parts_ml;
      if (out_h == 0 && row < rows) *reinterpret_cast<float2*>(ml + 2 * left_at) = make_float2(M, l);
      return;
    }
  }
  if (a.lse != nullptr && out_h == 0 && row < rows)
    a.lse[at] = l == 0.f ? -__builtin_inff() : (M + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// Launch of the kernel in one form (kv4_prompt*.hip).
template <int FORM>
hipError_t launch_prompt(const AttnArgs& a, int workgroups, int head_dim, int ng, int dtype, hipStream_t stream);

}  // namespace kv4
