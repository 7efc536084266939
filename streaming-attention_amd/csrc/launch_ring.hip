// Launches of the single-token attention over a cache for one configuration.  The build compiles this unit once per
// storage (0 fp32, 1 bf16, 2 fp16, 3 four bits), element type of the queries and count of 32-column key blocks, given as
// -DSTA_RING_ST=, -DSTA_RING_Q= and -DSTA_RING_NBK=; each holds the four counts of value blocks.
#include "api_common.hpp"
#include "ring_cache.hip"

#if !defined(STA_RING_ST) || !defined(STA_RING_Q) || !defined(STA_RING_NBK)
#error "launch_ring.hip is compiled with -DSTA_RING_ST= -DSTA_RING_Q= -DSTA_RING_NBK="
#endif

namespace sta_api {

template <int ST, int Q, int NBK>
int launch_ring(const sta::RingArgs& a, hipStream_t s) {
  const int64_t grid = static_cast<int64_t>(a.streams) * a.kv * a.chunks * a.nsplit;
  const int64_t heads = static_cast<int64_t>(a.streams) * a.heads;
  const bool join = a.nsplit > 1 || (a.append && a.chunks > 1);  // 512 threads a head
  if (grid <= 0 || grid > sta::MAX_GROUPS || (join && heads > sta::MAX_GROUPS / 2)) return STA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(grid));
  switch (a.nbv) {
    case 1: hipLaunchKernelGGL((sta::ring_attention_kernel<NBK, 1, ST, Q>), g, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL((sta::ring_attention_kernel<NBK, 2, ST, Q>), g, dim3(256), 0, s, a); break;
    case 3: hipLaunchKernelGGL((sta::ring_attention_kernel<NBK, 3, ST, Q>), g, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((sta::ring_attention_kernel<NBK, 4, ST, Q>), g, dim3(256), 0, s, a);
  }
  if (join)
    hipLaunchKernelGGL((sta::ring_join_kernel<Q>), dim3(static_cast<unsigned>(heads)), dim3(512), 0, s, a);
  return check_launch();
}

template int launch_ring<STA_RING_ST, STA_RING_Q, STA_RING_NBK>(const sta::RingArgs&, hipStream_t);

}  // namespace sta_api
