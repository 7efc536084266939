// Launches of the windowed attention kernels for one configuration.  The build compiles this unit once per padded
// width P (32, 64, 96, 128; keys and values both) and element type IN (0 fp32, 1 bf16, 2 fp16), given as
// -DSTA_WIN_P= and -DSTA_WIN_IN=.
#include "api_common.hpp"
#include "window_attn.hip"

#if !defined(STA_WIN_P) || !defined(STA_WIN_IN)
#error "launch_window.hip is compiled with -DSTA_WIN_P= -DSTA_WIN_IN="
#endif

namespace sta_api {

template <typename Kernel>
static int launch(Kernel kernel, int64_t grid, int lds, const sta::WinArgs& a, hipStream_t s) {
  if (grid <= 0 || grid > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  if (lds > 64 * 1024 - 16) {  // with the kernels' own few bytes past 64 KB
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return hip_status(e);
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), lds, s, a);
  return check_launch();
}

template <int P, int IN>
int launch_window_forward(const sta::WinArgs& a, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(a.batch) * a.heads * a.tiles;
  if (a.share) return launch(sta::window_forward_kernel<P, IN, true>, grid, sta::win_lds_bytes<P, IN, true>(), a, s);
  return launch(sta::window_forward_kernel<P, IN, false>, grid, sta::win_lds_bytes<P, IN, false>(), a, s);
}

// D and dq, then dk and dv, then the sums of the sinks.  The rows behind the window of up to 32 sinks go to workgroups whose
// waves share 32 of them, in a launch of their own: in tiles of 128 keys they take as many steps for 4 keys as for 128
// (backward, 8 x 16 heads of 4096 rows, 64 wide, window 256: 4 sinks 484 -> 442 us, 32 425 -> 412, 64 419 -> 420; 2 x 16 heads,
// 128 wide, 64 sinks 255 -> 268).  Below a sixteenth of the steps that launch costs what it saves (32 heads of 16384 rows, 128
// wide, window 4096 3744 -> 3788 us).
template <int P, int IN>
int launch_window_backward(const sta::WinArgs& a, hipStream_t s) {
  const int64_t bkv = static_cast<int64_t>(a.batch) * (a.heads / a.group);
  const int64_t grid_q = static_cast<int64_t>(a.batch) * a.heads * a.tiles;
  const int64_t behind = a.n - a.window, steps = static_cast<int64_t>(a.key_tiles) * (a.window + sta::WIN_ROWS);
  const bool apart = !a.key_share && a.far_chunks > 0 && a.sinks <= 32 && 16 * behind > steps;
  sta::WinArgs keys = a, far = a;
  if (apart) {
    keys.sink_tiles = 0;
    far.key_tiles = 0;
    far.sink_tiles = (a.sinks + 31) / 32;
  }
  const int64_t grid_k = bkv * (a.key_tiles + static_cast<int64_t>(keys.sink_tiles) * a.far_chunks);
  const int64_t grid_s = (bkv * a.sink_rows * (a.d + a.dv) + 255) / 256;
  if (grid_q > sta::MAX_GROUPS || grid_k > sta::MAX_GROUPS || grid_s > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  int st = a.share ? launch(sta::window_dq_kernel<P, IN, true>, grid_q, sta::win_lds_bytes<P, IN, true>(), a, s)
                   : launch(sta::window_dq_kernel<P, IN, false>, grid_q, sta::win_lds_bytes<P, IN, false>(), a, s);
  if (st != STA_OK) return st;
  constexpr bool FULL = sta::win_pipe<P, IN, false>();
  if (a.key_share)
    st = launch(sta::window_dkv_kernel<P, IN, true, false>, grid_k, sta::win_dkv_lds<P, IN, true>(), keys, s);
  else if (FULL && a.d == P && a.dv == P)
    st = launch(sta::window_dkv_kernel<P, IN, false, FULL>, grid_k, sta::win_dkv_lds<P, IN, false>(), keys, s);
  else
    st = launch(sta::window_dkv_kernel<P, IN, false, false>, grid_k, sta::win_dkv_lds<P, IN, false>(), keys, s);
  if (st == STA_OK && apart)
    st = launch(sta::window_dkv_kernel<P, IN, true, false>, bkv * far.sink_tiles * a.far_chunks,
                sta::win_dkv_lds<P, IN, true>(), far, s);
  if (st != STA_OK || a.far_chunks == 0) return st;
  return launch(sta::window_sink_kernel<IN>, grid_s, 0, a, s);
}

template int launch_window_forward<STA_WIN_P, STA_WIN_IN>(const sta::WinArgs&, hipStream_t);
template int launch_window_backward<STA_WIN_P, STA_WIN_IN>(const sta::WinArgs&, hipStream_t);

}  // namespace sta_api
