// Host-side checks shared by the entry points of the 4-bit KV cache.
#pragma once
#include <string>
#include <type_traits>

#include "../../include/marlin_hip.h"
#include "sm24_host.h"

namespace kv4 {

// Scale groups of a row (1, 2 or 4), 0 for a geometry without kernels.
inline int groups(int head_dim, int groupsize) {
  if (head_dim != 64 && head_dim != 128) return 0;
  const int g = groupsize == -1 ? head_dim : groupsize;
  if (g != 32 && g != 64 && g != 128) return 0;
  return head_dim % g == 0 ? head_dim / g : 0;
}

inline bool page_ok(int page_size) {
  return page_size >= 16 && page_size <= 256 && (page_size & (page_size - 1)) == 0;
}

inline int refuse(const std::string& why) {
  sm24::set_error("marlin_hip: " + why);
  return MARLIN_HIP_ERR_PROB_SHAPE;
}

inline int check_geometry(int kv_heads, int head_dim, int groupsize, int page_size, int num_pages, int dtype) {
  if (kv_heads <= 0 || num_pages < 0) return refuse("the KV cache needs at least one head and no negative page count");
  if (!page_ok(page_size)) return refuse("the KV cache's page_size must be 16, 32, 64, 128 or 256");
  // a slot is an int32, and a call's heads are one grid dimension
  if ((long long)num_pages * page_size > 0x7FFFFFFFll) return refuse("the KV cache holds more than 2^31 - 1 tokens");
  if (groups(head_dim, groupsize) == 0 || (dtype != 0 && dtype != 1)) {
    sm24::set_error("marlin_hip: the KV cache has kernels for head_dim 64 and 128, groupsize 32, 64, 128 or -1 "
                    "that divides it, fp16 and bf16 rows");
    return MARLIN_HIP_ERR_KERN_SHAPE;
  }
  return MARLIN_HIP_OK;
}

template <int N>
using Int = std::integral_constant<int, N>;

// f(Int<D>, Int<NG>) of a checked geometry.
template <class F>
auto dispatch(int head_dim, int ng, F&& f) {
  if (head_dim == 64) return ng == 1 ? f(Int<64>{}, Int<1>{}) : f(Int<64>{}, Int<2>{});
  return ng == 1 ? f(Int<128>{}, Int<1>{}) : ng == 2 ? f(Int<128>{}, Int<2>{}) : f(Int<128>{}, Int<4>{});
}

}  // namespace kv4
