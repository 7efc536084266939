// Launches of the attention over a shared prefix and of the received weights for one configuration.  The build compiles
// this unit once per padded width P (32, 64, 96, 128; keys and values both) and element type IN (0 fp32, 1 bf16, 2 fp16),
// given as -DSTA_PREFIX_P= and -DSTA_PREFIX_IN=.
#include "prefix_plan.hpp"

#if !defined(STA_PREFIX_P) || !defined(STA_PREFIX_IN)
#error "launch_prefix.hip is compiled with -DSTA_PREFIX_P= -DSTA_PREFIX_IN="
#endif

namespace sta_api {

// The walks of a plan; values 0: statistics alone (one walk).
template <int P, int IN>
int launch_prefix(const sta::PrefixArgs& a, const PrefixPlan& p, int values, hipStream_t s) {
  int64_t grid[2] = {0, 0};
  for (int i = 0; i < p.walks; ++i)
    grid[i] = static_cast<int64_t>(a.kv) * (a.batch / p.walk[i].span) * p.walk[i].tiles * p.walk[i].nsplit;
  if (grid[0] <= 0 || grid[0] + grid[1] > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(grid[0] + grid[1]));
  auto launch = [&](auto kernel, int lds, auto... args) {
    if (lds > 64 * 1024 - 16) {  // with the kernels' own few bytes past 64 KB
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return hip_status(e);
    }
    hipLaunchKernelGGL(kernel, g, dim3(256), lds, s, a, args...);
    return check_launch();
  };
  constexpr int shared = sta::win_lds_bytes<P, IN, true>(), rows = 4 * sta::win_join_floats<P>();
  const int by_rows = a.parts && values ? rows : 0;
  auto least = [&](int bytes) { return bytes > by_rows ? bytes : by_rows; };
  const int wide = least(sta::win_lds_bytes<P, IN, false>());
  const int ga = static_cast<int>(grid[0]), gb = static_cast<int>(grid[1]);
  if constexpr (IN != sta::F32) {
    if (p.stream && !p.share[0] && a.d % 8 == 0 && (!values || a.dv % 8 == 0)) {
      const int lds = values ? least(sta::prefix_stream_bytes<P, true>()) : sta::prefix_stream_bytes<P, false>();
      if (p.walks == 2)
        return launch(sta::prefix_walks_kernel<P, IN, false, true, true>, lds > shared ? lds : shared, p.walk[0], p.walk[1], ga,
                      gb);
      return values ? launch(sta::prefix_attention_kernel<P, IN, false, true, true>, lds, p.walk[0])
                    : launch(sta::prefix_attention_kernel<P, IN, false, false, true>, lds, p.walk[0]);
    }
  }
  if (p.walks == 2) {
    if (p.share[0] && p.share[1])
      return launch(sta::prefix_walks_kernel<P, IN, true, true, false>, shared, p.walk[0], p.walk[1], ga, gb);
    if constexpr (IN == sta::F32) {  // 16-bit rows that are walked apart are few
      if (!p.share[1])
        return launch(sta::prefix_walks_kernel<P, IN, false, false, false>, wide, p.walk[0], p.walk[1], ga, gb);
    }
    return launch(sta::prefix_walks_kernel<P, IN, false, true, false>, wide > shared ? wide : shared, p.walk[0], p.walk[1], ga,
                  gb);
  }
  if (values) {
    return p.share[0] ? launch(sta::prefix_attention_kernel<P, IN, true, true, false>, shared, p.walk[0])
                      : launch(sta::prefix_attention_kernel<P, IN, false, true, false>, wide, p.walk[0]);
  }
  return p.share[0] ? launch(sta::prefix_attention_kernel<P, IN, true, false, false>, shared, p.walk[0])
                    : launch(sta::prefix_attention_kernel<P, IN, false, false, false>, wide, p.walk[0]);
}

template <int P, int IN>
int launch_received(const sta::ReceivedArgs& w, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(w.a.kv) * w.a.batch * w.tiles * w.nsplit;
  if (grid <= 0 || grid > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(grid));
  if (w.few) {
    const int lds = sta::received_few_bytes<P, IN>((w.a.n * w.a.group + 31) / 32 * 32);
    if (lds > 64 * 1024) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(sta::received_few_kernel<P, IN>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return hip_status(e);
    }
    hipLaunchKernelGGL((sta::received_few_kernel<P, IN>), g, dim3(256), lds, s, w);
    return check_launch();
  }
  if constexpr (IN != sta::F32) {
    if (w.stream && w.a.d % 8 == 0) {
      hipLaunchKernelGGL((sta::received_kernel<P, IN, true>), g, dim3(256), 0, s, w);
      return check_launch();
    }
  }
  hipLaunchKernelGGL((sta::received_kernel<P, IN, false>), g, dim3(256), 0, s, w);
  return check_launch();
}

template int launch_prefix<STA_PREFIX_P, STA_PREFIX_IN>(const sta::PrefixArgs&, const PrefixPlan&, int, hipStream_t);
template int launch_received<STA_PREFIX_P, STA_PREFIX_IN>(const sta::ReceivedArgs&, hipStream_t);

}  // namespace sta_api
