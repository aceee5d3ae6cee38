// Pages of the 4-bit KV cache: which are free, copies of them in the caches of all layers, requests
// made from others, and the held pages moved together.
//
// The block table with the lengths is the only state: a page is held if an entry of a written
// token names it, however many do.  What these kernels decide they decide anew from the table.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv4_device.h"
#include "kv4_host.h"

namespace kv4 {

constexpr int kMaxLayers = 128;  // of one launch: their addresses are kernel arguments
struct Layers {
  uint8_t* at[kMaxLayers];
  int count;
};

struct Tables {
  const int32_t* table;  // [requests][max_pages]
  const int32_t* lens;
  int requests, max_pages, log_page, num_pages;
};
// Entries of a request that tokens have been written behind.
__device__ __forceinline__ int entries_of(const Tables& t, int len) {
  const long long n = ((long long)max(len, 0) + (1ll << t.log_page) - 1) >> t.log_page;
  return (int)min(n, (long long)t.max_pages);
}

// ---------------------------------------------------------------------------
// Marks: a byte for each page, 1 where it is held.  Setting a byte needs no atomic.
//
// Few pages and a small table: one workgroup, the bytes in LDS.  Else a launch that clears them in
// memory, one that sets them from all compute units, and one that reads them: a single workgroup
// takes a table at the 64 bytes a clock of its compute unit.  16384 pages, 256 requests: 1.9, 3.1 and 7.3 us; the
// last is every workgroup's count of all the bytes.  7.0 us in one where both are small.
// ---------------------------------------------------------------------------

constexpr int kMarkThreads = 1024, kMarkWaves = kMarkThreads / 64;
constexpr int kSmallPages = 32768;    // marks that one workgroup keeps in LDS ...
constexpr int kSmallEntries = 32768;  // ... and table entries that it looks at

__global__ __launch_bounds__(256) void kv4_clear_marks_kernel(u32x4* marks, int pieces) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i < pieces) marks[i] = (u32x4){0, 0, 0, 0};
}

__global__ __launch_bounds__(256) void kv4_mark_kernel(Tables t, uint8_t* marks) {
  for (int r = (int)blockIdx.x; r < t.requests; r += (int)gridDim.x) {
    const int n = entries_of(t, t.lens[r]);
    const int32_t* row = t.table + (size_t)r * t.max_pages;
    for (long long j = (long long)blockIdx.y * 256 + threadIdx.x; j < n; j += (long long)gridDim.y * 256) {
      const int page = row[j];
      if ((uint32_t)page < (uint32_t)t.num_pages) marks[page] = 1;
    }
  }
}

constexpr int kStrip = 256;  // pages that a wave looks at together

// Held pages before each chunk of `step` pages (kMarkThreads chunks), in LDS, and in all.
struct Census {
  int step, held;
};
__device__ __forceinline__ Census census(const uint8_t* marks, int num_pages, int (&before)[kMarkThreads + 1], int (&wave_sum)[kMarkWaves]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Census c;
  c.step = ((num_pages + kMarkThreads - 1) / kMarkThreads + kStrip - 1) & ~(kStrip - 1);
  // 16 bytes a lane, side by side: sixteen lanes have a strip, all strips of a chunk add up
  before[tid] = 0;
  __syncthreads();
  constexpr int FLIGHT = 4;
  const int pieces = (num_pages + 15) / 16, per_chunk = c.step / 16;  // (the marks end on 16 bytes; past the last page they are 0)
  for (int p0 = tid; p0 < ((pieces + 63) & ~63); p0 += FLIGHT * kMarkThreads) {
    u32x4 w[FLIGHT];
#pragma unroll
    for (int k = 0; k < FLIGHT; k++) {
      const int p = p0 + k * kMarkThreads;
      w[k] = reinterpret_cast<const u32x4*>(marks)[min(p, pieces - 1)];
    }
#pragma unroll
    for (int k = 0; k < FLIGHT; k++) {
      int n = __popc(w[k].x) + __popc(w[k].y) + __popc(w[k].z) + __popc(w[k].w);
      if (p0 + k * kMarkThreads >= pieces) n = 0;
      n += __builtin_amdgcn_update_dpp(0, n, 0x128, 0xF, 0xF, true);  // the lane 8, 4, 2, 1 places on of sixteen
      n += __builtin_amdgcn_update_dpp(0, n, 0x124, 0xF, 0xF, true);
      n += __builtin_amdgcn_update_dpp(0, n, 0x122, 0xF, 0xF, true);
      n += __builtin_amdgcn_update_dpp(0, n, 0x121, 0xF, 0xF, true);
      if ((lane & 15) == 0 && n > 0) atomicAdd(&before[(p0 + k * kMarkThreads) / per_chunk], n);
    }
  }
  __syncthreads();
  const int n = before[tid];
  int sum = n;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(sum, d);
    if (lane >= d) sum += x;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int base = 0;
  c.held = 0;
#pragma unroll
  for (int w = 0; w < kMarkWaves; w++) {
    if (w < wave) base += wave_sum[w];
    c.held += wave_sum[w];
  }
  before[tid] = base + sum - n;
  if (tid == 0) before[kMarkThreads] = c.held;
  __syncthreads();
  return c;
}

// f(page, held, held pages before it) for every page, over all waves of `workgroups` workgroups.
template <class F>
__device__ __forceinline__ void each_page(const uint8_t* marks, int num_pages, const Census& c, const int (&before)[kMarkThreads + 1],
                                          int workgroup, int workgroups, F&& f) {
  const int lane = threadIdx.x & 63;
  const int chunks = (num_pages + c.step - 1) / c.step;
  for (int chunk = workgroup * kMarkWaves + (int)(threadIdx.x >> 6); chunk < chunks; chunk += workgroups * kMarkWaves) {
    const long long first = (long long)chunk * c.step, last = min(first + c.step, (long long)num_pages);
    int seen = before[chunk];
    for (long long p = first; p < last; p += kStrip) {
      // a lane's four pages; held ones before them, of all lanes
      const long long page = p + 4 * lane;
      const uint32_t word = page < last ? *reinterpret_cast<const uint32_t*>(&marks[page]) : 0u;
      int before_lane = 0, all = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint64_t m = __ballot((word >> (8 * k) & 1u) != 0);
        before_lane += __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        all += (int)__popcll(m);
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const bool held = (word >> (8 * k) & 1u) != 0;
        if (page + k < last) f((int)page + k, held, seen + before_lane);
        before_lane += held;
      }
      seen += all;
    }
  }
}

// The free pages in ascending order, then -1.
struct FreeArgs {
  int32_t* free_pages;
  int32_t* count;
  int num_pages;
};
__device__ __forceinline__ void plan_of(const FreeArgs& a, const uint8_t* marks, int (&before)[kMarkThreads + 1],
                                           int (&wave_sum)[kMarkWaves], int workgroup, int workgroups) {
  const Census c = census(marks, a.num_pages, before, wave_sum);
  const int count = a.num_pages - c.held;
  each_page(marks, a.num_pages, c, before, workgroup, workgroups, [&](int page, bool held, int held_before) {
    if (!held) a.free_pages[page - held_before] = page;
  });
  for (long long i = (long long)count + workgroup * kMarkThreads + (int)threadIdx.x; i < a.num_pages;
       i += (long long)workgroups * kMarkThreads)
    a.free_pages[i] = -1;
  if (workgroup == 0 && threadIdx.x == 0) a.count[0] = count;
}

// Held pages above the number of held pages, in ascending order, go to the free ones below it.
struct MovePlan {
  int32_t* counts;  // held pages, pages that move
  int32_t* from;    // [move]
  int32_t* to;      // [move]
  int32_t* rank;    // [page]: its move
  int num_pages;
};
__device__ __forceinline__ void plan_of(const MovePlan& a, const uint8_t* marks, int (&before)[kMarkThreads + 1],
                                            int (&wave_sum)[kMarkWaves], int workgroup, int workgroups) {
  const Census c = census(marks, a.num_pages, before, wave_sum);
  // held pages below the border
  int below = 0;
  if (c.held < a.num_pages) {
    const int chunk = c.held / c.step;
    below = before[chunk];
    for (int p = chunk * c.step; p < c.held; p += 64) {
      const int page = p + (int)(threadIdx.x & 63);
      below += (int)__popcll(__ballot(page < c.held && marks[page] != 0));
    }
  } else {
    below = c.held;
  }
  each_page(marks, a.num_pages, c, before, workgroup, workgroups, [&](int page, bool held, int held_before) {
    if (held && page >= c.held) {
      a.from[held_before - below] = page;
      a.rank[page] = held_before - below;
    } else if (!held && page < c.held) {
      a.to[page - held_before] = page;
    }
  });
  if (workgroup == 0 && threadIdx.x == 0) a.counts[0] = c.held, a.counts[1] = c.held - below;
}

template <class Args>
__global__ __launch_bounds__(kMarkThreads) void kv4_page_plan_kernel(Args a, const uint8_t* marks) {
  __shared__ int before[kMarkThreads + 1], wave_sum[kMarkWaves];
  plan_of(a, marks, before, wave_sum, (int)blockIdx.x, (int)gridDim.x);
}

// The same with the marks in LDS.
template <class Args>
__global__ __launch_bounds__(kMarkThreads) void kv4_small_page_plan_kernel(Args a, Tables t) {
  __shared__ __align__(16) uint8_t marks[kSmallPages];
  __shared__ int before[kMarkThreads + 1], wave_sum[kMarkWaves];
  const int tid = threadIdx.x;
  for (int i = tid; i < (t.num_pages + 15) / 16; i += kMarkThreads) reinterpret_cast<u32x4*>(marks)[i] = (u32x4){0, 0, 0, 0};
  __syncthreads();
  // every entry, several of a thread in flight; its row and column go on without a division
  constexpr int FLIGHT = 8;
  const int all = t.requests * t.max_pages;  // (at most kSmallEntries)
  if (all > 0) {
    const int rows = kMarkThreads / t.max_pages, columns = kMarkThreads - rows * t.max_pages;
    int row = tid / t.max_pages, column = tid - row * t.max_pages;
    for (int e = tid; e < all; e += FLIGHT * kMarkThreads) {
      int page[FLIGHT], len[FLIGHT], at[FLIGHT];
#pragma unroll
      for (int k = 0; k < FLIGHT; k++) {
        page[k] = t.table[min(e + k * kMarkThreads, all - 1)];
        len[k] = t.lens[min(row, t.requests - 1)];
        at[k] = row < t.requests ? column : t.max_pages;
        row += rows, column += columns;
        if (column >= t.max_pages) row++, column -= t.max_pages;
      }
#pragma unroll
      for (int k = 0; k < FLIGHT; k++)
        if (at[k] < entries_of(t, len[k]) && (uint32_t)page[k] < (uint32_t)t.num_pages) marks[page[k]] = 1;
    }
  }
  __syncthreads();
  plan_of(a, marks, before, wave_sum, 0, 1);
}

template <class Args>
void plan_pages(const Args& a, const Tables& t, void* workspace, hipStream_t stream) {
  if (t.num_pages <= kSmallPages && (long long)t.requests * t.max_pages <= kSmallEntries) {
    hipLaunchKernelGGL((kv4_small_page_plan_kernel<Args>), dim3(1), dim3(kMarkThreads), 0, stream, a, t);
    return;
  }
  uint8_t* marks = static_cast<uint8_t*>(workspace);
  const int pieces = (t.num_pages + 15) / 16;
  hipLaunchKernelGGL(kv4_clear_marks_kernel, dim3((pieces + 255) / 256), dim3(256), 0, stream,
                     reinterpret_cast<u32x4*>(marks), pieces);
  if (t.requests > 0 && t.max_pages > 0) {
    const unsigned rows = t.requests < 4096 ? t.requests : 4096;
    unsigned across = (4096 + rows - 1) / rows, most = (t.max_pages + 255) / 256;
    if (across > most) across = most;
    hipLaunchKernelGGL(kv4_mark_kernel, dim3(rows, across), dim3(256), 0, stream, t, marks);
  }
  hipLaunchKernelGGL((kv4_page_plan_kernel<Args>), dim3(64), dim3(kMarkThreads), 0, stream, a, (const uint8_t*)marks);
}

// ---------------------------------------------------------------------------
// Whole pages.  A wave copies kPiece bytes, four 16-byte loads a lane in flight: 163 MB of moves (read and
// written) in 28 us where part of it lies in the last cache, some 36 (4.5 TB/s) where none does.
// ---------------------------------------------------------------------------

constexpr int kCopyThreads = 256, kCopyWaves = kCopyThreads / 64;
constexpr uint32_t kPiece = 4096;

// Pages from[i] to to[i] of every layer, over the waves of the grid.
__device__ __forceinline__ void copy_pages(const Layers& layers, const int32_t* from, const int32_t* to, int pairs,
                                           uint32_t page_bytes, int num_pages) {
  const uint32_t pieces = (page_bytes + kPiece - 1) / kPiece;
  const long long total = (long long)pairs * layers.count * pieces;
  const int lane = threadIdx.x & 63;
  for (long long i = (long long)blockIdx.x * kCopyWaves + (threadIdx.x >> 6); i < total; i += (long long)gridDim.x * kCopyWaves) {
    const long long page = i / pieces;
    const uint32_t piece = (uint32_t)(i - page * pieces);
    const int layer = (int)(page % layers.count), pair = (int)(page / layers.count);
    const int a = from[pair], b = to[pair];
    if ((uint32_t)a >= (uint32_t)num_pages || (uint32_t)b >= (uint32_t)num_pages || a == b) continue;
    uint8_t* base = layers.at[layer] + (size_t)piece * kPiece + 16 * lane;
    const uint8_t* src = base + (size_t)a * page_bytes;
    uint8_t* dst = base + (size_t)b * page_bytes;
    const uint32_t left = page_bytes - piece * kPiece, at = 16 * lane;  // (a multiple of 16)
    u32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (at + 1024 * k < left) v[k] = *reinterpret_cast<const u32x4*>(src + 1024 * k);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (at + 1024 * k < left) *reinterpret_cast<u32x4*>(dst + 1024 * k) = v[k];
  }
}

__global__ __launch_bounds__(kCopyThreads) void kv4_copy_pages_kernel(Layers layers, const int32_t* from, const int32_t* to,
                                                                      int pairs, uint32_t page_bytes, int num_pages) {
  copy_pages(layers, from, to, pairs, page_bytes, num_pages);
}

__global__ __launch_bounds__(kCopyThreads) void kv4_move_kernel(Layers layers, Tables t, MovePlan plan, int32_t* new_table,
                                                                uint32_t page_bytes) {
  const int held = plan.counts[0];
  for (int r = (int)blockIdx.x; r < t.requests; r += (int)gridDim.x) {
    const int n = entries_of(t, t.lens[r]);
    const size_t row = (size_t)r * t.max_pages;
    for (int j = (int)threadIdx.x; j < t.max_pages; j += kCopyThreads) {
      const int page = j < n ? t.table[row + j] : -1;
      const bool there = (uint32_t)page < (uint32_t)t.num_pages;
      new_table[row + j] = !there ? -1 : page < held ? page : plan.to[plan.rank[page]];
    }
  }
  copy_pages(layers, plan.from, plan.to, plan.counts[1], page_bytes, t.num_pages);
}

// ---------------------------------------------------------------------------
// Forks.  New request i is old request parents[i]: its entries are the parent's.  Pages that are
// full are shared.  One that is not may be written by one request only: the first that holds
// it, unless another holds it as a full page; the others get a copy of its written tokens (in fours, as
// V lies) on a fresh page.  Requests share a page at one place of their tables only, so a request
// looks at that column of the others.  64 samples of one prompt, 32 layers of 32 heads: 3.3 us for the
// tables and 19.5 for the copies, of 69 MB, nearly all written (3.5 TB/s).
// ---------------------------------------------------------------------------

struct ForkArgs {
  Tables old;
  const int32_t* parents;
  const int32_t* free_pages;
  int32_t* table;
  int32_t* lens;
  int32_t* used;
  int32_t* copies;  // [new request]: the page that it gets a copy of, or -1
  int rows, num_free;
};

__device__ __forceinline__ int fork_len(const ForkArgs& a, int i) {
  const int p = a.parents[i];
  if ((uint32_t)p >= (uint32_t)a.old.requests) return 0;
  return (int)min((long long)max(a.old.lens[p], 0), (long long)a.old.max_pages << a.old.log_page);
}

__global__ __launch_bounds__(256) void kv4_fork_table_kernel(ForkArgs a) {
  __shared__ int shared;
  const int i = (int)blockIdx.x, tid = threadIdx.x, lp = a.old.log_page;
  const int len = fork_len(a, i), n = entries_of(a.old, len);
  const int32_t* from = a.old.table + (size_t)max(a.parents[i], 0) * a.old.max_pages;  // (not read where len is 0)
  int32_t* to = a.table + (size_t)i * a.old.max_pages;
  for (int j = tid; j < a.old.max_pages; j += 256) {
    const int page = j < n ? from[j] : -1;
    to[j] = (uint32_t)page < (uint32_t)a.old.num_pages ? page : -1;
  }
  const int last = len >> lp;
  const bool part = (len & ((1 << lp) - 1)) != 0;
  const int page = part ? from[last] : -1;
  if (tid == 0) shared = 0;
  __syncthreads();
  if ((uint32_t)page < (uint32_t)a.old.num_pages) {
    for (int k = tid; k < a.rows; k += 256) {
      const int other = fork_len(a, k);
      const bool full = other >> lp > last;
      if (k == i || !(full || (k < i && other > last << lp))) continue;
      if (a.old.table[(size_t)a.parents[k] * a.old.max_pages + last] == page) shared = 1;
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.lens[i] = len;
    a.copies[i] = shared ? page : -1;
  }
}

constexpr int kForkRound = 1024;

__global__ __launch_bounds__(kCopyThreads) void kv4_fork_copy_kernel(Layers layers, ForkArgs a, int heads, int head_dim, int ng) {
  __shared__ int sources[kForkRound], targets[kForkRound], fours_of[kForkRound];
  __shared__ int wave_sum[kCopyWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lp = a.old.log_page, T = 1 << lp;
  const uint32_t blocks = (uint32_t)layers.count * heads;  // (below 2^22: the heads are checked on the host)
  const uint32_t block = (uint32_t)(T * (head_dim + 4 * ng)), page_bytes = block * heads;
  constexpr int FLIGHT = 4;
  const uint32_t half_lane = lane & 31;
  const uint32_t per_four = head_dim / 8, codes_of_page = (T / 4) * per_four;  // 16-byte runs of K's codes, or of V's
  const uint32_t code_at = lane < 32 ? 0 : (uint32_t)(T * head_dim / 2);
  const uint32_t scale_at = (uint32_t)(T * head_dim) + (lane < 32 ? 0 : 2 * T * ng);
  int taken = 0;  // pages that the rounds before took
  for (int r0 = 0; r0 < a.rows; r0 += kForkRound) {
    // the round's requests that get a copy, in order
    constexpr int PER = kForkRound / kCopyThreads;
    int own[PER], len[PER], n = 0;
#pragma unroll
    for (int u = 0; u < PER; u++) {
      const int r = r0 + PER * tid + u;
      own[u] = r < a.rows ? a.copies[r] : -1;
      len[u] = r < a.rows ? a.lens[r] : 0;
      n += own[u] >= 0;
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(sum, d);
      if (lane >= d) sum += x;
    }
    __syncthreads();  // the round before is done with LDS
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int at = sum - n, all = 0;
#pragma unroll
    for (int w = 0; w < kCopyWaves; w++) {
      if (w < wave) at += wave_sum[w];
      all += wave_sum[w];
    }
#pragma unroll
    for (int u = 0; u < PER; u++) {
      if (own[u] >= 0) {
        const int r = r0 + PER * tid + u, rank = taken + at;
        const int fresh = rank < a.num_free ? a.free_pages[rank] : -1;
        const bool there = (uint32_t)fresh < (uint32_t)a.old.num_pages;
        if (blockIdx.x == 0) a.table[(size_t)r * a.old.max_pages + (len[u] >> lp)] = there ? fresh : -1;
        sources[at] = own[u];
        targets[at] = fresh;
        fours_of[at] = there ? ((len[u] & (T - 1)) + 3) >> 2 : 0;  // (no page: nothing to copy)
        at++;
      }
    }
    __syncthreads();
    // A wave takes one head of one layer and a run of the copies, and keeps what it has read for those
    // of the same page (samples of one prompt).  Lanes 0 to 31 have K's codes and scales, the others V's.
    if (all > 0) {
      const uint32_t waves = gridDim.x * kCopyWaves, id = blockIdx.x * kCopyWaves + wave;
      const uint32_t runs = min(max(waves / blocks, 1u), (uint32_t)all);
      const uint32_t most = ((uint32_t)all + runs - 1) / runs;
      for (uint32_t item = id; item < blocks * runs; item += waves) {
        const uint32_t b = item / runs, k0 = (item - b * runs) * most, k1 = min(k0 + most, (uint32_t)all);
        const uint32_t layer = b / (uint32_t)heads, head = b - layer * (uint32_t)heads;
        uint8_t* const base = layers.at[layer] + (size_t)head * block;
        for (uint32_t c0 = 0; c0 < codes_of_page; c0 += 32 * FLIGHT) {
          u32x4 v[FLIGHT];
          u32x2 s[FLIGHT];
          int held = -1, held_fours = 0;  // what v and s hold
          bool more = false;              // some copy goes on past this part
          for (uint32_t k = k0; k < k1; k++) {
            const int source = __builtin_amdgcn_readfirstlane(sources[k]), target = __builtin_amdgcn_readfirstlane(targets[k]);
            const int fours = __builtin_amdgcn_readfirstlane(fours_of[k]);
            const uint32_t codes = (uint32_t)fours * per_four, scales = (uint32_t)fours * ng;
            if (codes <= c0) continue;
            more |= codes > c0 + 32 * FLIGHT;
            if (source != held || fours > held_fours) {
              const uint8_t* src = base + (size_t)(uint32_t)source * page_bytes;
#pragma unroll
              for (int u = 0; u < FLIGHT; u++) {
                const uint32_t c = c0 + 32 * u + half_lane;
                if (c < codes) v[u] = *reinterpret_cast<const u32x4*>(src + code_at + 16 * c);
                if (c < scales) s[u] = *reinterpret_cast<const u32x2*>(src + scale_at + 8 * c);
              }
              held = source, held_fours = fours;
            }
            uint8_t* dst = base + (size_t)(uint32_t)target * page_bytes;
#pragma unroll
            for (int u = 0; u < FLIGHT; u++) {
              const uint32_t c = c0 + 32 * u + half_lane;
              if (c < codes) *reinterpret_cast<u32x4*>(dst + code_at + 16 * c) = v[u];
              if (c < scales) *reinterpret_cast<u32x2*>(dst + scale_at + 8 * c) = s[u];
            }
          }
          if (!more) break;
        }
      }
    }
    taken += all;
  }
  if (blockIdx.x == 0 && tid == 0) a.used[0] = taken;
}

// Launches f(layers) for every kMaxLayers of the caches.
template <class F>
void each_layers(const void* const* caches, int count, F&& f) {
  for (int first = 0; first == 0 || first < count; first += kMaxLayers) {
    Layers l{};
    l.count = count - first < kMaxLayers ? count - first : kMaxLayers;
    for (int i = 0; i < l.count; i++) l.at[i] = const_cast<uint8_t*>(static_cast<const uint8_t*>(caches[first + i]));
    f(l);
  }
}

int check_tables(int requests, int max_pages, int page_size, int num_pages) {
  if (requests < 0 || max_pages < 0) return refuse("the KV cache's pages take no negative sizes");
  // (the kernels go through them in steps that must not pass 31 bits)
  if (requests > (1 << 30)) return refuse("the KV cache's pages take tables of at most 2^30 requests");
  if (!page_ok(page_size)) return refuse("the KV cache's page_size must be 16, 32, 64, 128 or 256");
  if (num_pages < 1 || (long long)num_pages * page_size > 0x7FFFFFFFll)
    return refuse("the KV cache holds a page at least and 2^31 - 1 tokens at most");
  if ((long long)max_pages * page_size > (1ll << 30)) return refuse("a block table row covers more than 2^30 tokens");
  return MARLIN_HIP_OK;
}

int check_pool(int layers, int kv_heads, int head_dim, int page_size, int num_pages, int groupsize, uint32_t* page_bytes) {
  const int err = check_geometry(kv_heads, head_dim, groupsize, page_size, num_pages, 0);
  if (err != MARLIN_HIP_OK) return err;
  if (layers < 0) return refuse("the KV cache's pages take no negative sizes");
  const long long bytes = (long long)page_size * (head_dim + 4 * groups(head_dim, groupsize)) * kv_heads;
  if (bytes > 0x7FFFFFFFll) return refuse("a page of 2^31 bytes or more");
  *page_bytes = (uint32_t)bytes;
  return MARLIN_HIP_OK;
}

int log2_page(int x) { return 31 - __builtin_clz((unsigned)x); }

// Workgroups that copy: enough to fill the machine, no more than there are pieces (0: not known).
unsigned copy_grid(long long waves) {
  const long long w = (waves + kCopyWaves - 1) / kCopyWaves;
  return (unsigned)(w < 1 ? 1 : w < 2048 ? w : 2048);
}

}  // namespace kv4

extern "C" {

int marlin_hip_kv4_free_pages(const void* block_table, const void* kv_lens, void* free_pages, void* count,
                              void* workspace, int requests, int max_pages, int page_size, int num_pages, int dev,
                              hipStream_t stream) {
  using namespace kv4;
  const int err = check_tables(requests, max_pages, page_size, num_pages);
  if (err != MARLIN_HIP_OK) return err;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const Tables t{static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(kv_lens), requests, max_pages,
                 log2_page(page_size), num_pages};
  plan_pages(FreeArgs{static_cast<int32_t*>(free_pages), static_cast<int32_t*>(count), num_pages}, t, workspace, stream);
  return sm24::launch_error(hipGetLastError());
}

int marlin_hip_kv4_copy_pages(const void* const* caches, int layers, const void* from, const void* to, int pairs,
                              int kv_heads, int head_dim, int page_size, int num_pages, int groupsize, int dev,
                              hipStream_t stream) {
  using namespace kv4;
  uint32_t page_bytes = 0;
  const int err = check_pool(layers, kv_heads, head_dim, page_size, num_pages, groupsize, &page_bytes);
  if (err != MARLIN_HIP_OK) return err;
  if (pairs < 0) return refuse("kv4_copy_pages takes no negative sizes");
  if (pairs == 0 || layers == 0) return MARLIN_HIP_OK;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  each_layers(caches, layers, [&](const Layers& l) {
    const long long waves = (long long)pairs * l.count * ((page_bytes + kPiece - 1) / kPiece);
    hipLaunchKernelGGL(kv4_copy_pages_kernel, dim3(copy_grid(waves)), dim3(kCopyThreads), 0, stream, l,
                       static_cast<const int32_t*>(from), static_cast<const int32_t*>(to), pairs, page_bytes, num_pages);
  });
  return sm24::launch_error(hipGetLastError());
}

int marlin_hip_kv4_compact(const void* const* caches, int layers, const void* block_table, const void* kv_lens,
                           void* new_table, void* counts, void* workspace, int requests, int max_pages, int kv_heads,
                           int head_dim, int page_size, int num_pages, int groupsize, int dev, hipStream_t stream) {
  using namespace kv4;
  uint32_t page_bytes = 0;
  int err = check_pool(layers, kv_heads, head_dim, page_size, num_pages, groupsize, &page_bytes);
  if (err == MARLIN_HIP_OK) err = check_tables(requests, max_pages, page_size, num_pages);
  if (err != MARLIN_HIP_OK) return err;
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const Tables t{static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(kv_lens), requests, max_pages,
                 log2_page(page_size), num_pages};
  int32_t* lists = static_cast<int32_t*>(workspace);
  const size_t n = ((size_t)num_pages + 15) & ~(size_t)15;
  const MovePlan plan{static_cast<int32_t*>(counts), lists, lists + n, lists + 2 * n, num_pages};
  plan_pages(plan, t, lists + 3 * n, stream);
  err = sm24::launch_error(hipGetLastError());
  if (err != MARLIN_HIP_OK) return err;
  each_layers(caches, layers, [&](const Layers& l) {
    hipLaunchKernelGGL(kv4_move_kernel, dim3(2048), dim3(kCopyThreads), 0, stream, l, t, plan,
                       static_cast<int32_t*>(new_table), page_bytes);
  });
  return sm24::launch_error(hipGetLastError());
}

int marlin_hip_kv4_fork(const void* const* caches, int layers, const void* block_table, const void* kv_lens,
                        const void* parents, const void* free_pages, void* new_table, void* new_lens, void* pages_used,
                        void* workspace, int requests, int new_requests, int num_free, int max_pages, int kv_heads,
                        int head_dim, int page_size, int num_pages, int groupsize, int dev, hipStream_t stream) {
  using namespace kv4;
  uint32_t page_bytes = 0;
  int err = check_pool(layers, kv_heads, head_dim, page_size, num_pages, groupsize, &page_bytes);
  if (err == MARLIN_HIP_OK) err = check_tables(requests, max_pages, page_size, num_pages);
  if (err != MARLIN_HIP_OK) return err;
  if (new_requests < 0 || num_free < 0) return refuse("kv4_fork takes no negative sizes");
  if (kv_heads > 32767) return refuse("kv4_fork takes at most 32767 heads");
  // (each looks at the others' entries of one column)
  if (new_requests > 65536) return refuse("kv4_fork makes at most 65536 requests");
  sm24::DeviceScope scope(dev);
  if (!scope.ok) return MARLIN_HIP_ERR_LAUNCH;
  const Tables t{static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(kv_lens), requests, max_pages,
                 log2_page(page_size), num_pages};
  const ForkArgs a{t, static_cast<const int32_t*>(parents), static_cast<const int32_t*>(free_pages),
                   static_cast<int32_t*>(new_table), static_cast<int32_t*>(new_lens), static_cast<int32_t*>(pages_used),
                   static_cast<int32_t*>(workspace), new_requests, num_free};
  if (new_requests > 0) {
    hipLaunchKernelGGL(kv4_fork_table_kernel, dim3((unsigned)new_requests), dim3(256), 0, stream, a);
    err = sm24::launch_error(hipGetLastError());
    if (err != MARLIN_HIP_OK) return err;
  }
  each_layers(caches, layers, [&](const Layers& l) {
    const long long waves = (long long)new_requests * l.count * kv_heads;
    hipLaunchKernelGGL(kv4_fork_copy_kernel, dim3(copy_grid(waves)), dim3(kCopyThreads), 0, stream, l, a, kv_heads, head_dim,
                       groups(head_dim, groupsize));
  });
  return sm24::launch_error(hipGetLastError());
}

}  // extern "C"
