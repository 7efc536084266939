// The compiled configuration of an attention over a shared prefix, for the entry points that launch it.
#pragma once

#include "prefix_plan.hpp"

namespace sta_api {

// launch_prefix.hip, one object per (P, IN)
template <int P, int IN>
int launch_prefix(const sta::PrefixArgs& a, const PrefixPlan& p, int values, hipStream_t s);
template <int P, int IN>
int launch_received(const sta::ReceivedArgs& w, hipStream_t s);

template <typename Call>
int prefix_by_type(int dtype, int width, Call call) {
#define STA_PREFIX_CASE(P)                                                                                 \
  if (width <= P) {                                                                                        \
    if (dtype == STA_F32) return call(std::integral_constant<int, P>{}, std::integral_constant<int, sta::F32>{});   \
    if (dtype == STA_BF16) return call(std::integral_constant<int, P>{}, std::integral_constant<int, sta::BF16>{}); \
    return call(std::integral_constant<int, P>{}, std::integral_constant<int, sta::F16>{});                \
  }
  STA_PREFIX_CASE(32)
  STA_PREFIX_CASE(64)
  STA_PREFIX_CASE(96)
  STA_PREFIX_CASE(128)
#undef STA_PREFIX_CASE
  return STA_ERR_UNSUPPORTED;
}

// rows on 16 bytes (of 2-byte elements)
inline bool on_units(const sta::Rows& t) {
  return ((reinterpret_cast<uintptr_t>(t.p) | 2 * t.sb | 2 * t.sh | 2 * t.sn) & 15) == 0;
}

// the walks of a plan
inline int run_prefix(const sta::PrefixArgs& a, PrefixPlan p, int dtype, int values, hipStream_t s) {
  const bool prefix = p.walk[0].prefix, own = p.walks == 1 && p.walk[0].own;  // of the first walk
  p.stream = (!own || on_units(a.k)) && (!prefix || on_units(a.pk)) &&
             (!values || ((!own || on_units(a.v)) && (!prefix || on_units(a.pv))));
  return prefix_by_type(dtype, values && a.dv > a.d ? a.dv : a.d, [&](auto width, auto in) {
    return launch_prefix<decltype(width)::value, decltype(in)::value>(a, p, values, s);
  });
}

}  // namespace sta_api
