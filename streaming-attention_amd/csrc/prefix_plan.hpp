// How the rows and keys of an attention over a shared prefix are dealt out, for the entry points that launch it.
#pragma once

#include "api_common.hpp"
#include "prefix_attn.hip"

namespace sta_api {

constexpr int kMaxPrefixD = 128;
constexpr int64_t kMaxPrefixRows = int64_t(1) << 30;
constexpr int kMaxPrefixParts = 256;  // prefix_join_kernel's weights

// The walks of a call: one over prefix and own tokens together, or two, whose partials are joined.
struct PrefixPlan {
  int walks;
  sta::PrefixWalk walk[2];
  int share[2];     // tiles of 32 rows whose waves share the keys, see deal_out; of two walks of 16-bit rows the second's always
  int parts;        // 0: one workgroup finishes a row
  int stream;       // the first walk's keys and values lie on 16 bytes: prefix_stream_pass where the widths allow it
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One walk over `keys` keys of units of `rows` rows: the tile and the number of workgroups that share a tile's keys.
// Up to 64 rows: tiles of 32 whose waves share the keys (8 key heads of 16384 x 128 and 64 rows: 27 us, 32 with a tile of
// 128; 96 rows 33 and 33, 128 rows 38 and 34).  A share has at least `least` keys; room: workgroups that the walk is to fill
// the card with, which holds 512 at a time (256 compute units, two each of 128 columns).
inline void deal_out(sta::PrefixWalk& w, int& share, int64_t units, int64_t rows, int64_t keys, int64_t room, int64_t least) {
  share = rows <= 64;
  w.tiles = static_cast<int>(ceil_div(rows, share ? 32 : sta::WIN_ROWS));
  int64_t want = room / (units * w.tiles);
  const int64_t most = ceil_div(keys, least);
  if (want > most) want = most;
  if (want > kMaxPrefixParts / 2) want = kMaxPrefixParts / 2;
  w.nsplit = static_cast<int>(want < 1 ? 1 : want);
}

// A share of 256 keys is two tiles of 32 a wave (fp32, whose products take 16 times as long: 128; four rows
// over 8 x 2048 keys 14 -> 11 us).
// own: the sequences' own tokens take part.  The sequences of a set lie in one tile for the prefix (two walks, whose partials
// are joined) where each has few rows and there are keys enough:
// * up to 512 keys a workgroup goes over both for itself, without partials (4 x 8 heads of 64 over 256 and 64 keys 10.3 -> 9.1
//   us, 64 x 4 of 64 rows 19.7 -> 11.2; over 576 keys 8 x 8 x 4 rows take 10.6 and 10.1, 32 x 32 of one row 18.5 and 20.4);
//   fp32 up to 128 (64 x 8 x 4 rows of 128 over 128 keys 46 -> 41 us, of 64 23 -> 16, 2 x 2 of 128 19 -> 21; over 256 keys 49
//   and 56);
// * above 64 rows its tile of 128 is full enough (64 x 4 of 96 rows of 64 over 16384: 272 -> 176 us, 16 x 8 142 -> 97, 4 x
//   8 38.6 -> 37.1); not in fp32 (4 x 8 of 96 rows of 128 over 4096: 95 and 109 us).
// One workgroup of the prefix's walk a compute unit leaves room for one of the other's, and has half the partials of two (64
// x 32 heads of 128 over 16384 shared and 1024 own rows: 79 us, 92 with two; 64 rows over 8 x 16384 alone 27 and 32); with
// many tiles and more than 1024 keys a share, two (64 x 4 of 48 rows of 64 over 16384: 134 -> 82 us, 32 rows 73 -> 57, 16
// x 8 of 32 rows 43 -> 38; of 1024 keys 28 and 27, 30 and 30, of 512 23 and 26).  Many are 32, or 16 up to 64 columns (64 x
// 32 heads over 32768 shared and 1024 own rows, 64 wide 57 -> 50 us, 128 wide 108 and 110).
inline PrefixPlan plan_prefix(const sta::PrefixArgs& a, int dtype, bool own) {
  const int64_t least = dtype == STA_F32 ? 128 : 256, keys = static_cast<int64_t>(a.p) + a.m;
  const bool one = keys <= (dtype == STA_F32 ? 128 : 512);
  PrefixPlan p{};
  const int64_t rows = static_cast<int64_t>(a.n) * a.group, units = static_cast<int64_t>(a.batch) * a.kv;
  const bool packed =
      a.p > 0 && (!own || (!one && a.per_set > 1 && rows < (dtype == STA_F32 ? sta::WIN_ROWS : sta::WIN_ROWS / 2 + 1)));
  if (packed) {
    const int64_t sets = static_cast<int64_t>(a.sets) * a.kv, together = rows * a.per_set;
    const int64_t tiles = sets * ceil_div(together, sta::WIN_ROWS);
    p.walks = own ? 2 : 1;
    p.walk[0].span = a.per_set;
    p.walk[0].prefix = 1;
    const bool two = a.p * tiles > 256 * 1024 && tiles >= (a.d <= 64 && a.dv <= 64 ? 16 : 32);
    deal_out(p.walk[0], p.share[0], sets, together, a.p, two ? 512 : 256, least);
    p.parts = p.walk[0].nsplit;
    if (own) {
      p.walk[1].span = 1;
      p.walk[1].own = 1;
      p.walk[1].first = p.parts;
      deal_out(p.walk[1], p.share[1], units, rows, a.m, 512, least);
      p.parts += p.walk[1].nsplit;
    }
    return p;
  }
  p.walks = 1;
  p.walk[0].span = 1;
  p.walk[0].prefix = a.p > 0;
  p.walk[0].own = 1;
  deal_out(p.walk[0], p.share[0], units, rows, keys, one ? 1 : 512, least);
  p.parts = p.walk[0].nsplit > 1 ? p.walk[0].nsplit : 0;
  return p;
}

// the partials: sums, then statistics
inline int64_t prefix_sum_bytes(const sta::PrefixArgs& a, int parts) {
  return 4 * static_cast<int64_t>(a.batch) * a.heads * a.n * parts * a.pitch;
}
inline int64_t prefix_part_bytes(const sta::PrefixArgs& a, int parts) {
  return prefix_sum_bytes(a, parts) + ceil_div(8 * static_cast<int64_t>(a.batch) * a.heads * a.n * parts, 16) * 16;
}
inline void set_parts(sta::PrefixArgs& a, void* room, int parts) {
  a.part = static_cast<float*>(room);
  a.stat = reinterpret_cast<float*>(static_cast<char*>(room) + prefix_sum_bytes(a, parts));
  a.parts = parts;
}

// The shape part of the arguments; d and dv padded are the caller's.
inline int prefix_shape(sta::PrefixArgs& a, int dtype, int64_t batch, int heads, int kv_heads, int64_t sets, int64_t n,
                        int64_t m, int64_t p, int d, int dv, float scale) {
  if (!dtype_ok(dtype)) return STA_ERR_DTYPE;
  const int es = dtype == STA_F32 ? 4 : 2;
  if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || sets < 1 || batch % sets || n < 1 || m < 0 || p < 0 ||
      d < 1 || dv < 0)
    return STA_ERR_SHAPE;
  if (!(scale == scale && scale - scale == 0.f)) return STA_ERR_ARG;  // finite
  if (d > kMaxPrefixD || dv > kMaxPrefixD || d * es < 16 || (dv && dv * es < 16) || n > kMaxPrefixRows ||
      m > kMaxPrefixRows || p > kMaxPrefixRows || batch > 0x7fffffff / heads ||
      static_cast<int64_t>(batch / sets) * n > kMaxPrefixRows / (heads / kv_heads))
    return STA_ERR_UNSUPPORTED;
  a = sta::PrefixArgs{};
  a.batch = static_cast<int>(batch);
  a.heads = heads;
  a.kv = kv_heads;
  a.group = heads / kv_heads;
  a.sets = static_cast<int>(sets);
  a.per_set = static_cast<int>(batch / sets);
  a.n = static_cast<int>(n);
  a.m = static_cast<int>(m);
  a.p = static_cast<int>(p);
  a.d = d;
  a.dv = dv;
  a.pitch = (dv + 3) / 4 * 4;
  a.scale = scale;
  const float c = (scale < 0.f ? -scale : scale) * 1.44269504088896340736f;
  a.c = c > 1e-37f ? c : 1e-37f;  // above 0: a hidden pair's logit, -inf, stays one times c
  return STA_OK;
}

// a tile's rows are reached by 32-bit offsets from its first
inline bool prefix_strides_ok(const int64_t* strides, int tensors, int dtype) {
  for (int i = 0; i < tensors; ++i) {
    const int64_t sn = strides[3 * i + 2];
    if (sn < 0 || sn > (int64_t(1) << 24) / (dtype == STA_F32 ? 4 : 2)) return false;
  }
  return true;
}

inline sta::Rows prefix_rows_of(const void* p, const int64_t* strides) {
  return sta::Rows{p, strides[0], strides[1], strides[2], 0};
}

}  // namespace sta_api
