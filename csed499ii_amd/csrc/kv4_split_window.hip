// Launcher of the split kernel of the 4-bit KV cache (kv4_split.h): a sliding window and sinks.
#include "kv4_host.h"
#include "kv4_split.h"

namespace kv4 {

template <>
hipError_t launch_split<WINDOW>(const AttnArgs& a, int workgroups, int head_dim, int ng, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)workgroups), block(64 * kWaves);
  dispatch(head_dim, ng, [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    if (dtype == F16) hipLaunchKernelGGL((kv4_split_kernel<D, NG, F16, WINDOW>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv4_split_kernel<D, NG, BF16, WINDOW>), grid, block, 0, stream, a);
  });
  return hipGetLastError();
}

}  // namespace kv4
