// Entry points of the windowed attention (see include/streamattn.h): argument checks, the gradient's plan and the
// choice of the compiled configuration.
#include <cmath>

#include "api_common.hpp"
#include "window_attn.hip"

using namespace sta_api;

namespace sta_api {
template <int P, int IN>
int launch_window_forward(const sta::WinArgs& a, hipStream_t s);
template <int P, int IN>
int launch_window_backward(const sta::WinArgs& a, hipStream_t s);
}  // namespace sta_api

namespace {

constexpr int kMaxWindowD = 128;
constexpr int64_t kMaxWindowRows = int64_t(1) << 30;  // rows and their sums with a window stay in 32 bits

int element_size(int dtype) { return dtype == STA_F32 ? 4 : 2; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

sta::Rows rows_of(const void* p, const int64_t* strides) { return sta::Rows{p, strides[0], strides[1], strides[2], 0}; }

// a tile's rows are reached by 32-bit offsets from its first
bool strides_ok(const int64_t* strides, int tensors, int dtype) {
  for (int i = 0; i < tensors; ++i) {
    const int64_t sn = strides[3 * i + 2];
    if (sn < 0 || sn > (int64_t(1) << 24) / element_size(dtype)) return false;
  }
  return true;
}

// The number of 128-row tiles (128-key tiles for dk and dv) below which the waves of a workgroup share 32 rows instead (the
// card has 256 compute units).  Long windows gain more, short ones pay for staging a tile four times; shared tiles of 128
// columns leave one wave a SIMD, as those of dk and dv do above 64; fp32 products take 16 times as long, so balance counts for
// more.  Wide / shared in us, 2048 rows a head (tiles: 16 a head):
//   16 bits, window 1024: out d = 64, 256 tiles 26 / 21, 384 33 / 29, 512 34 / 38; dq 256 31 / 29, 384 41 / 40;
//     d = 96, out 256 33 / 32, 384 42 / 43; dq 384 56 / 52; d = 128, out + dq 128 86 / 66, 160 87 / 92, 192 88 / 105
//   window 256: out + dq d = 64, 128 33 / 23, 160 33 / 31, 192 32 / 31, 256 32 / 35; d = 128, 128 45 / 39, 160 46 / 59
//   dk, dv: d = 64, window 1024, 256 47 / 40, 384 56 / 56, window 256, 256 29 / 29, 384 43 / 39; d = 128, window 1024, 128
//     55 / 51, 160 56 / 71, window 256, 64 31 / 31, 128 31 / 41
//   fp32, d = 64, all of them: window 256, 256 tiles 218 / 216, 512 370 / 403; window 2048, 256 696 / 447, 768 1600 / 1320
int64_t share_below(int es, int width, int64_t window, bool keys) {
  if (es == 4) return window >= 1024 ? 1024 : 448;
  if (keys) return width <= 64 ? 448 : (window >= 1024 ? 144 : 96);
  return window >= 1024 && width <= 96 ? 448 : 160;
}

// The shape part of the arguments; STA_OK or what is wrong with it.
int window_shape(sta::WinArgs& a, int dtype, int64_t batch, int heads, int kv_heads, int64_t n, int d, int dv,
                 float scale, int64_t window, int64_t sinks) {
  if (!dtype_ok(dtype)) return STA_ERR_DTYPE;
  const int es = element_size(dtype);
  if (batch < 1 || heads < 1 || kv_heads < 1 || n < 1 || d < 1 || dv < 1 || heads % kv_heads != 0)
    return STA_ERR_SHAPE;
  if (window < 1 || sinks < 0 || !std::isfinite(scale)) return STA_ERR_ARG;
  if (d > kMaxWindowD || dv > kMaxWindowD || d * es < 16 || dv * es < 16 || n > kMaxWindowRows || batch > 0x7fffffff) return STA_ERR_UNSUPPORTED;
  a = sta::WinArgs{};
  a.batch = static_cast<int>(batch);
  a.heads = heads;
  a.group = heads / kv_heads;
  a.n = static_cast<int>(n);
  a.d = d;
  a.dv = dv;
  a.window = static_cast<int>(window < n ? window : n);
  a.sinks = static_cast<int>(sinks < n ? sinks : n);
  a.scale = scale;
  // above 0: a hidden pair's logit, -inf, stays one times c
  a.c = std::fmax(std::fabs(scale) * 1.44269504088896340736f, 1e-37f);
  const int64_t wide = (n + sta::WIN_ROWS - 1) / sta::WIN_ROWS;
  const int width = d > dv ? d : dv;
  a.share = batch * heads * wide < share_below(es, width, a.window, false);
  a.key_share = batch * kv_heads * wide < share_below(es, width, a.window, true);
  a.tiles = static_cast<int>(a.share ? (n + 31) / 32 : wide);
  a.key_tiles = static_cast<int>(a.key_share ? (n + 31) / 32 : wide);
  a.lift = a.drop = 1.f;
  return STA_OK;
}

// How the rows behind the window of the sinks are dealt out: as many workgroups as the card holds at a time (256 compute
// units, two each of 16-bit rows up to 64 columns), chunks of at least 256 rows.  Backward, window 256, 4 sinks: 8 x 16 heads of
// 4096 x 64, 256 workgroups 450 us, 512 442, 1024 456, 2048 464; 2 x 16 heads of 4096 x 128, 256 227, 512 238; chunks of at
// least 64 rows, 4 query heads of one key head of 32768 x 64, window 512, 186 us, of 256 158.
void plan_sinks(sta::WinArgs& a, int es) {
  const int64_t behind = a.n - a.window;
  if (a.sinks == 0 || behind <= 0) return;
  const int64_t bkv = static_cast<int64_t>(a.batch) * (a.heads / a.group);
  a.sink_rows = a.sinks;
  const int rows = a.key_share ? 32 : sta::WIN_ROWS;
  a.sink_tiles = (a.sinks + rows - 1) / rows;
  const int64_t room = es == 2 && a.d <= 64 && a.dv <= 64 ? 512 : 256;
  int64_t chunks = room / (bkv * a.sink_tiles);
  if (chunks > (behind + 255) / 256) chunks = (behind + 255) / 256;
  if (chunks < 1) chunks = 1;
  const int64_t chunk = ((behind + chunks - 1) / chunks + 31) / 32 * 32;
  a.far_rows = static_cast<int>(chunk);
  a.far_chunks = static_cast<int>((behind + chunk - 1) / chunk);
}

int64_t delta_floats(const sta::WinArgs& a) {
  return (static_cast<int64_t>(a.batch) * a.heads * a.n + 63) / 64 * 64;
}

int64_t part_floats(const sta::WinArgs& a) {
  if (a.far_chunks == 0) return 0;
  return static_cast<int64_t>(a.batch) * (a.heads / a.group) * (a.far_chunks + 1) * a.sink_rows * (a.d + a.dv);
}

template <int P>
int by_type(bool backward, const sta::WinArgs& a, int dtype, hipStream_t s) {
  if (dtype == STA_F32)
    return backward ? launch_window_backward<P, sta::F32>(a, s) : launch_window_forward<P, sta::F32>(a, s);
  if (dtype == STA_BF16)
    return backward ? launch_window_backward<P, sta::BF16>(a, s) : launch_window_forward<P, sta::BF16>(a, s);
  return backward ? launch_window_backward<P, sta::F16>(a, s) : launch_window_forward<P, sta::F16>(a, s);
}

int dispatch(bool backward, const sta::WinArgs& a, int dtype, void* stream) {
  const int width = a.d > a.dv ? a.d : a.dv;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (width <= 32) return by_type<32>(backward, a, dtype, s);
  if (width <= 64) return by_type<64>(backward, a, dtype, s);
  if (width <= 96) return by_type<96>(backward, a, dtype, s);
  return by_type<128>(backward, a, dtype, s);
}

}  // namespace

extern "C" {

int sta_window_attention(const void* q, const void* k, const void* v, int dtype, int64_t batch, int heads,
                         int kv_heads, int64_t n, int d, int dv, const int64_t* strides, float scale, int64_t window,
                         int64_t sinks, const int32_t* lengths, void* out, void* rest, float* lse, void* stream) {
  if (!q || !k || !v || !out || !strides || !aligned16(out) || !aligned16(rest)) return STA_ERR_ARG;
  sta::WinArgs a;
  if (const int st = window_shape(a, dtype, batch, heads, kv_heads, n, d, dv, scale, window, sinks)) return st;
  if (!strides_ok(strides, 3, dtype)) return STA_ERR_UNSUPPORTED;
  a.q = rows_of(q, strides);
  a.k = rows_of(k, strides + 3);
  a.v = rows_of(v, strides + 6);
  a.lengths = lengths;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  return dispatch(false, a, dtype, stream);
}

int64_t sta_window_backward_bytes(int dtype, int64_t batch, int heads, int kv_heads, int64_t n, int d, int dv,
                                  int64_t window, int64_t sinks) {
  sta::WinArgs a;
  if (window_shape(a, dtype, batch, heads, kv_heads, n, d, dv, 1.f, window, sinks) != STA_OK) return -1;
  plan_sinks(a, element_size(dtype));
  return 4 * (delta_floats(a) + part_floats(a));
}

int sta_window_attention_backward(const void* grad, const void* q, const void* k, const void* v, const void* out,
                                  const void* rest, const float* lse, int dtype, int64_t batch, int heads, int kv_heads, int64_t n,
                                  int d, int dv, const int64_t* strides, float scale, int64_t window, int64_t sinks,
                                  const int32_t* lengths, void* dq, void* dk, void* dv_out, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (!grad || !q || !k || !v || !out || !lse || !strides || !dq || !dk || !dv_out || !workspace) return STA_ERR_ARG;
  if (!aligned16(out) || !aligned16(rest) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv_out) || !aligned16(workspace))
    return STA_ERR_ARG;
  sta::WinArgs a;
  if (const int st = window_shape(a, dtype, batch, heads, kv_heads, n, d, dv, scale, window, sinks)) return st;
  plan_sinks(a, element_size(dtype));
  if (workspace_bytes < 4 * (delta_floats(a) + part_floats(a))) return STA_ERR_SCRATCH;
  if (!strides_ok(strides, 4, dtype)) return STA_ERR_UNSUPPORTED;
  a.q = rows_of(q, strides);
  a.k = rows_of(k, strides + 3);
  a.v = rows_of(v, strides + 6);
  a.go = rows_of(grad, strides + 9);
  a.lengths = lengths;
  a.out = const_cast<void*>(out);
  a.rest = const_cast<void*>(rest);
  a.lse = const_cast<float*>(lse);
  a.delta = static_cast<float*>(workspace);
  a.part = a.delta + delta_floats(a);
  a.dq = dq;
  a.dk = dk;
  a.dv_out = dv_out;
  if (dtype == STA_F16) {
    // fp16 weights of long rows are subnormal (1 / 4096 has 10 bits left): they and their gradients are carried times
    // a power of two near the number of keys, at most 2^10; the gradients of rows and keys for which that is too much
    // are lowered from there (win_lower)
    const int64_t keys = static_cast<int64_t>(a.window) + a.sinks < a.n ? a.window + a.sinks : a.n;
    int e = 0;
    while (e < 10 && (int64_t(2) << e) <= keys) ++e;
    a.lift = std::ldexp(1.f, e);
    a.drop = std::ldexp(1.f, -e);
  }
  return dispatch(true, a, dtype, stream);
}

}  // extern "C"
