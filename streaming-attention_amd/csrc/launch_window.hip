// Launches of the windowed attention kernels for one configuration.  The build compiles this unit once per padded
// width P (32, 64, 96, 128; keys and values both) and element type IN (0 fp32, 1 bf16, 2 fp16), given as
// -DSTA_WIN_P= and -DSTA_WIN_IN=.
#include "api_common.hpp"
#include "window_attn.hip"

#if !defined(STA_WIN_P) || !defined(STA_WIN_IN)
#error "launch_window.hip is compiled with -DSTA_WIN_P= -DSTA_WIN_IN="
#endif

namespace sta_api {

template <int P, int IN>
int launch_window_forward(const sta::WinArgs& a, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(a.batch) * a.heads * a.tiles;
  if (grid <= 0 || grid > 0x7fffffff) return STA_ERR_SHAPE;
  hipLaunchKernelGGL((sta::window_forward_kernel<P, IN>), dim3(static_cast<unsigned>(grid)), dim3(256), 0, s, a);
  return check_launch();
}

// D and dq, then dk and dv, then the sums of the sinks
template <int P, int IN>
int launch_window_backward(const sta::WinArgs& a, hipStream_t s) {
  const int64_t bkv = static_cast<int64_t>(a.batch) * (a.heads / a.group);
  const int64_t grid_q = static_cast<int64_t>(a.batch) * a.heads * a.tiles;
  const int64_t grid_k = bkv * (a.tiles + static_cast<int64_t>(a.sink_tiles) * a.far_chunks);
  const int64_t grid_s = (bkv * a.sink_rows * (a.d + a.dv) + 255) / 256;
  if (grid_q <= 0 || grid_q > 0x7fffffff || grid_k > 0x7fffffff || grid_s > 0x7fffffff) return STA_ERR_SHAPE;
  hipLaunchKernelGGL((sta::window_dq_kernel<P, IN>), dim3(static_cast<unsigned>(grid_q)), dim3(256), 0, s, a);
  constexpr int lds = sta::win_dkv_lds<P, IN>();
  if constexpr (lds > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&sta::window_dkv_kernel<P, IN>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return hip_status(e);
  }
  hipLaunchKernelGGL((sta::window_dkv_kernel<P, IN>), dim3(static_cast<unsigned>(grid_k)), dim3(256), lds, s, a);
  if (a.far_chunks > 0)
    hipLaunchKernelGGL((sta::window_sink_kernel<IN>), dim3(static_cast<unsigned>(grid_s)), dim3(256), 0, s, a);
  return check_launch();
}

template int launch_window_forward<STA_WIN_P, STA_WIN_IN>(const sta::WinArgs&, hipStream_t);
template int launch_window_backward<STA_WIN_P, STA_WIN_IN>(const sta::WinArgs&, hipStream_t);

}  // namespace sta_api
