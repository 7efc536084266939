// Launches of the attention over a shared prefix and of the received weights for one configuration.  The build compiles
// this unit once per padded width P (32, 64, 96, 128; keys and values both) and element type IN (0 fp32, 1 bf16, 2 fp16),
// given as -DSTA_PREFIX_P= and -DSTA_PREFIX_IN=.
#include "api_common.hpp"
#include "prefix_attn.hip"

#if !defined(STA_PREFIX_P) || !defined(STA_PREFIX_IN)
#error "launch_prefix.hip is compiled with -DSTA_PREFIX_P= -DSTA_PREFIX_IN="
#endif

namespace sta_api {

// The rows of one walk: finished, or their partials.  values 0: statistics alone.
template <int P, int IN>
int launch_prefix(const sta::PrefixArgs& a, const sta::PrefixWalk& w, int share, int values, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(a.kv) * (a.batch / w.span) * w.tiles * w.nsplit;
  if (grid <= 0 || grid > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  auto launch = [&](auto kernel, int lds) {
    if (lds > 64 * 1024 - 16) {  // with the kernels' own few bytes past 64 KB
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return hip_status(e);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), lds, s, a, w);
    return check_launch();
  };
  constexpr int wide = sta::win_lds_bytes<P, IN, false>(), shared = sta::win_lds_bytes<P, IN, true>();
  if (values) {
    return share ? launch(sta::prefix_attention_kernel<P, IN, true, true>, shared)
                 : launch(sta::prefix_attention_kernel<P, IN, false, true>, wide);
  }
  return share ? launch(sta::prefix_attention_kernel<P, IN, true, false>, shared)
               : launch(sta::prefix_attention_kernel<P, IN, false, false>, wide);
}

template <int P, int IN>
int launch_received(const sta::ReceivedArgs& w, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(w.a.kv) * w.a.batch * w.tiles * w.nsplit;
  if (grid <= 0 || grid > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  hipLaunchKernelGGL((sta::received_kernel<P, IN>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, w);
  return check_launch();
}

template int launch_prefix<STA_PREFIX_P, STA_PREFIX_IN>(const sta::PrefixArgs&, const sta::PrefixWalk&, int, int, hipStream_t);
template int launch_received<STA_PREFIX_P, STA_PREFIX_IN>(const sta::ReceivedArgs&, hipStream_t);

}  // namespace sta_api
