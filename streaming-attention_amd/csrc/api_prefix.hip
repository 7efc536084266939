// Entry points of the attention over a shared prefix and of the received weights (see include/streamattn.h): argument
// checks, plans, launches.
#include "prefix_dispatch.hpp"

#include <utility>

using namespace sta_api;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int IN>
void join(const sta::PrefixArgs& a, bool few, dim3 grid, hipStream_t s) {
  if (few) hipLaunchKernelGGL((sta::prefix_join_few_kernel<IN>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((sta::prefix_join_kernel<IN>), grid, dim3(128), 0, s, a);
}

// The partials of every row, in rows of 2^20 workgroups.
int join_rows(const sta::PrefixArgs& a, int dtype, hipStream_t s) {
  const bool few = a.parts <= sta::PREFIX_FEW_PARTS;
  const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * a.n;
  const int64_t groups = few ? ceil_div(rows, a.out ? 256 / (a.pitch / 4) : 256) : rows;
  const int64_t x = groups < 1 << 20 ? groups : 1 << 20, y = ceil_div(groups, x);
  if (y > 65535) return STA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(x), static_cast<unsigned>(y));
  if (dtype == STA_F32) join<sta::F32>(a, few, g, s);
  else if (dtype == STA_BF16) join<sta::BF16>(a, few, g, s);
  else join<sta::F16>(a, few, g, s);
  return check_launch();
}

// How the received weights are dealt out.  Few rows: as many workgroups as the card holds at a time (two a compute unit, four
// of up to 64 columns of 16 bits), whose waves have four blocks of keys at least (16 x 8 key heads of 8192 rows, 128 wide, 128
// rows: 64 us, 77 with 2048; 16 x 16 of 64: 47 with 1024, 54 with 512, 49 with 2048; fp32 175, 180 with 2048).  Many: a
// workgroup a tile of keys, and where that leaves fewer than 4096 several that share its rows, of which the first tiles have
// most, 8 row tiles of 64 at least (4 x 8 x 4 heads of 1024 rows of 128: 41 us, 45 with 16, 45 with 4), 2 of up to 512
// workgroups and 1 of up to 256 (8 x 4 heads of 256 rows 9.5 us, 11 with 2, 36 with 16; of 512 rows 15, of 1024 21, and 35).
void plan_received(sta::ReceivedArgs& w, int dtype) {
  const sta::PrefixArgs& a = w.a;
  const int64_t units = static_cast<int64_t>(a.batch) * a.kv, rows = static_cast<int64_t>(a.n) * a.group;
  w.few = rows <= sta::RECEIVED_FEW;
  w.nsplit = 1;
  if (w.few) {
    const int64_t want = ceil_div(dtype != STA_F32 && a.d <= 64 ? 1024 : 512, units), most = ceil_div(a.m, 4 * 4 * 32);
    w.tiles = static_cast<int>(want < most ? want : most);
    return;
  }
  w.tiles = static_cast<int>(ceil_div(a.m, dtype == STA_F32 ? 128 : 256));
  const int64_t row_tiles = a.group * ceil_div(a.n, 64);
  for (const auto& [groups, least] : {std::pair<int64_t, int64_t>{256, 1}, {512, 2}, {4096, 8}}) {
    const int64_t want = groups / (units * w.tiles), most = ceil_div(row_tiles, least), split = want < most ? want : most;
    if (split > w.nsplit) w.nsplit = static_cast<int>(split);
  }
}

int64_t received_sum_bytes(const sta::ReceivedArgs& w) {
  return w.nsplit == 1 ? 0 : 4 * ceil_div(static_cast<int64_t>(w.nsplit) * w.a.batch * w.a.kv * w.a.m, 4) * 4;
}
int64_t received_lse_bytes(const sta::PrefixArgs& a) {
  return 4 * ceil_div(static_cast<int64_t>(a.batch) * a.heads * a.n, 4) * 4;
}

}  // namespace

extern "C" {

int64_t sta_prefix_attention_bytes(int dtype, int64_t batch, int heads, int kv_heads, int64_t sets, int64_t n, int64_t m,
                                   int64_t p, int d, int dv) {
  sta::PrefixArgs a;
  if (prefix_shape(a, dtype, batch, heads, kv_heads, sets, n, m, p, d, dv, 1.f) != STA_OK || m < 1 || dv < 1) return -1;
  return prefix_part_bytes(a, plan_prefix(a, dtype, true).parts);
}

int sta_prefix_attention(const void* q, const void* k, const void* v, const void* prefix_k, const void* prefix_v, int dtype,
                         int64_t batch, int heads, int kv_heads, int64_t sets, int64_t n, int64_t m, int64_t p, int d,
                         int dv, const int64_t* strides, float scale, const int32_t* lengths, const int32_t* counts,
                         const int32_t* prefix_lengths, void* out, float* lse, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  if (!q || !k || !v || !out || !strides || (p > 0 && (!prefix_k || !prefix_v))) return STA_ERR_ARG;
  sta::PrefixArgs a;
  if (const int st = prefix_shape(a, dtype, batch, heads, kv_heads, sets, n, m, p, d, dv, scale)) return st;
  if (m < 1 || dv < 1) return STA_ERR_SHAPE;
  if (!aligned16(out)) return STA_ERR_ARG;
  if (!prefix_strides_ok(strides, p > 0 ? 5 : 3, dtype)) return STA_ERR_UNSUPPORTED;
  const PrefixPlan plan = plan_prefix(a, dtype, true);
  const int64_t need = prefix_part_bytes(a, plan.parts);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return STA_ERR_SCRATCH;
  a.q = prefix_rows_of(q, strides);
  a.k = prefix_rows_of(k, strides + 3);
  a.v = prefix_rows_of(v, strides + 6);
  if (p > 0) {
    a.pk = prefix_rows_of(prefix_k, strides + 9);
    a.pv = prefix_rows_of(prefix_v, strides + 12);
  }
  a.lengths = lengths;
  a.counts = counts;
  a.prefix_lengths = prefix_lengths;
  a.out = out;
  a.lse = lse;
  set_parts(a, workspace, plan.parts);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int st = run_prefix(a, plan, dtype, 1, s);
  return st == STA_OK && plan.parts ? join_rows(a, dtype, s) : st;
}

int64_t sta_received_attention_bytes(int dtype, int64_t batch, int heads, int kv_heads, int64_t n, int64_t m, int d,
                                     int with_lse) {
  sta::ReceivedArgs w{};
  if (prefix_shape(w.a, dtype, batch, heads, kv_heads, batch, n, m, 0, d, 0, 1.f) != STA_OK || m < 1) return -1;
  plan_received(w, dtype);
  int64_t bytes = received_sum_bytes(w);
  if (!with_lse) bytes += received_lse_bytes(w.a) + prefix_part_bytes(w.a, plan_prefix(w.a, dtype, true).parts);
  return bytes;
}

int sta_received_attention(const void* q, const void* k, int dtype, int64_t batch, int heads, int kv_heads, int64_t n,
                           int64_t m, int d, const int64_t* strides, float scale, const int32_t* lengths,
                           const int32_t* counts, const float* lse, float* weights, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  if (!q || !k || !weights || !strides) return STA_ERR_ARG;
  sta::ReceivedArgs w{};
  sta::PrefixArgs& a = w.a;
  if (const int st = prefix_shape(a, dtype, batch, heads, kv_heads, batch, n, m, 0, d, 0, scale)) return st;
  if (m < 1) return STA_ERR_SHAPE;
  if (!prefix_strides_ok(strides, 2, dtype)) return STA_ERR_UNSUPPORTED;
  const int64_t need = sta_received_attention_bytes(dtype, batch, heads, kv_heads, n, m, d, lse != nullptr);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return STA_ERR_SCRATCH;
  a.q = prefix_rows_of(q, strides);
  a.k = prefix_rows_of(k, strides + 3);
  a.lengths = lengths;
  a.counts = counts;
  plan_received(w, dtype);
  w.stream = on_units(a.q);
  char* room = static_cast<char*>(workspace);
  w.sums = reinterpret_cast<float*>(room);
  room += received_sum_bytes(w);
  w.weights = weights;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (lse) {
    a.lse = const_cast<float*>(lse);
  } else {
    a.lse = reinterpret_cast<float*>(room);
    room += received_lse_bytes(a);
    const PrefixPlan plan = plan_prefix(a, dtype, true);
    set_parts(a, room, plan.parts);
    int st = run_prefix(a, plan, dtype, 0, s);
    if (st == STA_OK && plan.parts) st = join_rows(a, dtype, s);
    if (st != STA_OK) return st;
  }
  const int st = prefix_by_type(dtype, d, [&](auto width, auto in) {
    return launch_received<decltype(width)::value, decltype(in)::value>(w, s);
  });
  if (st != STA_OK || w.nsplit == 1) return st;
  const int64_t groups = ceil_div(static_cast<int64_t>(a.batch) * a.kv * a.m, 256);
  if (groups > sta::MAX_GROUPS) return STA_ERR_SHAPE;
  hipLaunchKernelGGL(sta::received_join_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, s, w);
  return check_launch();
}

}  // extern "C"
