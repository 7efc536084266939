// Launches of a step over the cache that keeps the most attended tokens for one configuration.  The build compiles this
// unit once per element type (0 fp32, 1 bf16, 2 fp16) and count of 32-column key blocks, given as -DSTA_HEAVY_ST= and
// -DSTA_HEAVY_NBK=; each holds the four counts of value blocks.
#include "api_common.hpp"
#include "heavy_cache.hip"

#if !defined(STA_HEAVY_ST) || !defined(STA_HEAVY_NBK)
#error "launch_heavy.hip is compiled with -DSTA_HEAVY_ST= -DSTA_HEAVY_NBK="
#endif

namespace sta_api {

template <int ST, int NBK>
int launch_heavy(const sta::HeavyArgs& h, hipStream_t s) {
  const sta::RingArgs& a = h.r;
  const int64_t grid = static_cast<int64_t>(a.streams) * a.kv * a.chunks * a.nsplit;
  const int64_t outputs = static_cast<int64_t>(a.streams) * a.heads;
  const int64_t ranges = (h.pitch + sta::HEAVY_SLOTS - 1) / sta::HEAVY_SLOTS;
  const int64_t join = outputs + static_cast<int64_t>(a.streams) * a.kv * ranges;
  if (grid <= 0 || grid > sta::MAX_GROUPS || (!h.alone && join > sta::MAX_GROUPS / 2)) return STA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(grid));
  const int lds = static_cast<int>(sta::heavy_lds_bytes(a.group, a.nbv, h.pitch, h.local));
  auto launch = [&](auto kernel) {
    if (lds > 64 * 1024 - 1024) {  // with the kernel's own arrays past 64 KB
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return hip_status(e);
    }
    hipLaunchKernelGGL(kernel, g, dim3(256), lds, s, h);
    return check_launch();
  };
  const int st = a.nbv == 1   ? launch(sta::heavy_attention_kernel<NBK, 1, ST>)
                 : a.nbv == 2 ? launch(sta::heavy_attention_kernel<NBK, 2, ST>)
                 : a.nbv == 3 ? launch(sta::heavy_attention_kernel<NBK, 3, ST>)
                              : launch(sta::heavy_attention_kernel<NBK, 4, ST>);
  if (st != STA_OK) return st;
  if (!h.alone)
    hipLaunchKernelGGL((sta::heavy_join_kernel<ST>), dim3(static_cast<unsigned>(join)), dim3(512), 0, s, h,
                       static_cast<int>(outputs), static_cast<int>(ranges));
  return check_launch();
}

template int launch_heavy<STA_HEAVY_ST, STA_HEAVY_NBK>(const sta::HeavyArgs&, hipStream_t);

}  // namespace sta_api
