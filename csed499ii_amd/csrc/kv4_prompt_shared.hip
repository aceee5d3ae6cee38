// Launcher of the prompt kernel of the 4-bit KV cache (kv4_prompt.h): a prefix that requests share.
#include "kv4_host.h"
#include "kv4_prompt.h"

namespace kv4 {

template <>
hipError_t launch_prompt<SHARED>(const AttnArgs& a, int workgroups, int head_dim, int ng, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)workgroups), block(64 * kPromptWaves);
  dispatch(head_dim, ng, [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, NG = decltype(g)::value;
    if (dtype == F16) hipLaunchKernelGGL((kv4_prompt_kernel<D, NG, F16, SHARED>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((kv4_prompt_kernel<D, NG, BF16, SHARED>), grid, block, 0, stream, a);
  });
  return hipGetLastError();
}

}  // namespace kv4
