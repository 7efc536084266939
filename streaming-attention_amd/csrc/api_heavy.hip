// Entry points of the cache that keeps the most attended tokens (see include/streamattn.h): argument checks, the split of
// a step, launches.
#include <cmath>

#include "heavy_cache.hip"
#include "prefix_dispatch.hpp"

using namespace sta_api;

namespace sta_api {
template <int ST, int NBK>
int launch_heavy(const sta::HeavyArgs& h, hipStream_t s);
}  // namespace sta_api

namespace {

constexpr int kMaxHeavyD = 128;
constexpr int64_t kMaxHeavySlots = int64_t(1) << 30;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

sta::Rows rows_of(const void* p, int64_t sb, int64_t sh, int64_t sn) { return sta::Rows{p, sb, sh, sn, 0}; }

int heavy_shape(sta::HeavyArgs& h, int dtype, int64_t streams, int heads, int kv_heads, int d, int dv, int64_t recent,
                int64_t kept) {
  h = sta::HeavyArgs{};
  if (!dtype_ok(dtype)) return STA_ERR_DTYPE;
  if (streams < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || d < 1 || dv < 1) return STA_ERR_SHAPE;
  if (recent < 1 || kept < 1) return STA_ERR_ARG;
  if (d > kMaxHeavyD || dv > kMaxHeavyD || recent > kMaxHeavySlots || kept > kMaxHeavySlots - recent ||
      streams > 0x7fffffff / kv_heads || streams > 0x7fffffff / heads || heads / kv_heads > sta::HEAVY_HEADS)
    return STA_ERR_UNSUPPORTED;
  sta::RingArgs& a = h.r;
  a.streams = static_cast<int>(streams);
  a.heads = heads;
  a.kv = kv_heads;
  a.group = heads / kv_heads;
  a.chunks = (a.group + 15) / 16;
  a.d = d;
  a.dv = dv;
  a.nbk = (d + 31) / 32;
  a.nbv = (dv + 31) / 32;
  h.recent = static_cast<int>(recent);
  h.kept = static_cast<int>(kept);
  h.ring = h.recent + 1;
  a.slots = h.ring + h.kept;
  a.tiles = (a.slots + 31) / 32;
  a.nsplit = 1;
  h.pitch = 32 * a.tiles;
  h.part_pitch = (dv + 3) / 4 * 4;
  return STA_OK;
}

// Workgroups that share a key head's slots: one a compute unit of the whole launch, whose waves have a tile at least (32 x 8
// key heads of 2048 slots of 128: 49 us, 62 with two a compute unit, 8 of 16000 20 and 20, fp32 39 and 49; 8 of 1024 slots in
// shares of four tiles 12 us, of eight 13, fp32 15 and 21).  Short caches have one, which finishes their key heads in one
// launch (64 wide, 800 slots 9.1 us, 9.4 shared, 1050 slots 10.3 and 9.4; 128 wide, 430 slots 9.0 and 9.7, 560 slots 12.4 and
// 11.8 with four query heads; fp32 128 wide, 170 slots 12.4 and 12.6, 300 slots 15 and 12).  Above 128 key heads two shares
// would leave a second turn half empty, and one is best (17 x 8 key heads of 16000 slots of 128: 193 us, two 253, three 198;
// 25 x 8: 255, 296 and 307; 31 x 8: 328, 358 and 358).  fp32 has a workgroup a compute unit at a time: three shares of up to
// 170 key heads take two turns of a third each (17 x 8 of 4096 slots of 128: 178 -> 142 us, 20 x 8 183 -> 150; of 2048 95 ->
// 83, 64 wide 47 -> 44; of 1024 54 and 53, 64 wide 27 and 29).
int splits_of(const sta::RingArgs& a, int dtype) {
  const int64_t work = static_cast<int64_t>(a.streams) * a.kv * a.chunks, blocks = static_cast<int64_t>(a.tiles) * (a.nbk + a.nbv);
  if (blocks <= (dtype == STA_F32 ? 40 : 104)) return 1;
  const bool thirds = dtype == STA_F32 && work > 128 && 3 * work <= 512 && blocks >= 256;
  const int64_t want = thirds ? 3 : 256 / work, most = (a.tiles + 3) / 4, split = want < most ? want : most;
  return static_cast<int>(split < 1 ? 1 : split);
}

// A shared prefix in front of the cache: one row a head, that of the one own token, which the walk leaves to the cache.
int prefix_of(sta::PrefixArgs& p, const sta::RingArgs& a, int dtype, int64_t sets, int64_t rows, float scale) {
  return prefix_shape(p, dtype, a.streams, a.heads, a.kv, sets, 1, 1, rows, a.d, a.dv, scale);
}

int64_t round16(int64_t x) { return (x + 15) / 16 * 16; }

// The workspace: logits, then of steps that several workgroups share what they do to the slots, their partials and the
// prefix's.
struct Workspace {
  int64_t logits, moves, part, prefix;
  int64_t total() const { return logits + moves + part + prefix; }
};
Workspace workspace_of(const sta::HeavyArgs& h, const sta::PrefixArgs* p, int prefix_parts) {
  const sta::RingArgs& a = h.r;
  const int64_t heads = static_cast<int64_t>(a.streams) * a.heads;
  Workspace w{};
  w.logits = h.local ? 0 : 4 * heads * h.pitch;
  if (h.alone) return w;
  w.moves = static_cast<int64_t>(sizeof(sta::HeavyMove)) * a.streams * a.kv;
  w.part = round16(4 * heads * a.nsplit * h.part_pitch) + round16(8 * heads * a.nsplit);
  if (p) w.prefix = prefix_part_bytes(*p, prefix_parts);
  return w;
}
void plan_heavy(sta::HeavyArgs& h, int dtype, int prefix_parts) {
  h.r.nsplit = splits_of(h.r, dtype);
  h.prefix_parts = prefix_parts;
  h.alone = h.r.nsplit == 1 && h.r.chunks == 1 && prefix_parts == 0;
  // two workgroups a compute unit with the logits in LDS, and the kernel's own kilobyte
  h.local = h.alone && sta::heavy_lds_bytes(h.r.group, h.r.nbv, h.pitch, true) <= 79 * 1024;
}

template <int ST>
int by_keys(const sta::HeavyArgs& h, hipStream_t s) {
  switch (h.r.nbk) {
    case 1: return launch_heavy<ST, 1>(h, s);
    case 2: return launch_heavy<ST, 2>(h, s);
    case 3: return launch_heavy<ST, 3>(h, s);
    default: return launch_heavy<ST, 4>(h, s);
  }
}

template <typename Call>
void by_type(int dtype, Call call) {
  if (dtype == STA_F32) call(std::integral_constant<int, sta::F32>{});
  else if (dtype == STA_BF16) call(std::integral_constant<int, sta::BF16>{});
  else call(std::integral_constant<int, sta::F16>{});
}

int state_of(sta::HeavyArgs& h, void* keys, void* values, int64_t* counts, float* weights, int64_t* positions,
             uint64_t* lowest) {
  if (!keys || !values || !counts || !weights || !positions || !lowest || !aligned16(keys) || !aligned16(values) ||
      !aligned16(weights) || !aligned16(positions))
    return STA_ERR_ARG;
  h.r.keys = static_cast<uint8_t*>(keys);
  h.r.values = static_cast<uint8_t*>(values);
  h.counts = counts;
  h.weights = weights;
  h.positions = positions;
  h.lowest = reinterpret_cast<unsigned long long*>(lowest);
  return STA_OK;
}

// a workgroup a tile of the cache, in rows of 2^20
bool tile_grid(const sta::RingArgs& a, dim3& g) {
  const int64_t tiles = static_cast<int64_t>(a.streams) * a.kv * a.tiles, x = tiles < 1 << 20 ? tiles : 1 << 20;
  const int64_t y = (tiles + x - 1) / x;
  g = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
  return y <= 65535;
}
// and one a key head
bool head_grid(const sta::RingArgs& a, int threads, dim3& g) {
  const int64_t heads = static_cast<int64_t>(a.streams) * a.kv;
  g = dim3(static_cast<unsigned>(heads));
  return heads <= (int64_t(1) << 32) / threads - 1;
}

}  // namespace

extern "C" {

int sta_heavy_layout(int dtype, int64_t streams, int kv_heads, int d, int dv, int64_t recent, int64_t kept,
                     int64_t* sizes) {
  if (!sizes) return STA_ERR_ARG;
  sta::HeavyArgs h;
  if (const int st = heavy_shape(h, dtype, streams, kv_heads, kv_heads, d, dv, recent, kept)) return st;
  const int64_t tiles = static_cast<int64_t>(h.r.streams) * h.r.kv * h.r.tiles;
  sizes[0] = tiles * sta::ring_tile_bytes(h.r.nbk, dtype);
  sizes[1] = tiles * sta::ring_tile_bytes(h.r.nbv, dtype);
  sizes[2] = h.pitch;
  return STA_OK;
}

int64_t sta_heavy_attention_bytes(int dtype, int64_t streams, int heads, int kv_heads, int d, int dv, int64_t recent,
                                  int64_t kept, int64_t sets, int64_t p) {
  sta::HeavyArgs h;
  if (heavy_shape(h, dtype, streams, heads, kv_heads, d, dv, recent, kept) != STA_OK) return -1;
  if (p < 0) return -1;
  if (p == 0) {
    plan_heavy(h, dtype, 0);
    return workspace_of(h, nullptr, 0).total();
  }
  sta::PrefixArgs x;
  if (prefix_of(x, h.r, dtype, sets, p, 1.f) != STA_OK) return -1;
  const int parts = plan_prefix(x, dtype, false).parts;
  plan_heavy(h, dtype, parts);
  return workspace_of(h, &x, parts).total();
}

int sta_heavy_attention(const void* q, const void* k, const void* v, int dtype, int64_t streams, int heads, int kv_heads,
                        int d, int dv, const int64_t* strides, float scale, int64_t recent, int64_t kept,
                        const void* prefix_k, const void* prefix_v, int64_t sets, int64_t p,
                        const int64_t* prefix_strides, const int32_t* prefix_lengths, void* keys, void* values,
                        int64_t* counts, float* weights, int64_t* positions, uint64_t* lowest, void* out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || !out || !strides || !k != !v || !std::isfinite(scale) || p < 0 ||
      (p > 0 && (!prefix_k || !prefix_v || !prefix_strides)))
    return STA_ERR_ARG;
  sta::HeavyArgs h;
  if (const int st = heavy_shape(h, dtype, streams, heads, kv_heads, d, dv, recent, kept)) return st;
  if (const int st = state_of(h, keys, values, counts, weights, positions, lowest)) return st;
  sta::RingArgs& a = h.r;
  a.q = rows_of(q, strides[0], strides[1], 0);
  a.append = k != nullptr;
  if (a.append) {
    a.k = rows_of(k, strides[2], strides[3], 0);
    a.v = rows_of(v, strides[4], strides[5], 0);
  }
  a.scale = scale;
  // above 0: what a wave without tiles has, -3e38, stays far below a logit times c
  a.c = std::fmax(std::fabs(scale) * 1.44269504088896340736f, 1e-37f);
  a.out = out;
  sta::PrefixArgs x;
  PrefixPlan plan{};
  if (p > 0) {
    if (const int st = prefix_of(x, a, dtype, sets, p, scale)) return st;
    if (!prefix_strides_ok(prefix_strides, 2, dtype)) return STA_ERR_UNSUPPORTED;
    plan = plan_prefix(x, dtype, false);
  }
  plan_heavy(h, dtype, plan.parts);
  const Workspace w = workspace_of(h, p > 0 ? &x : nullptr, plan.parts);
  if (w.total() > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < w.total())) return STA_ERR_SCRATCH;
  char* room = static_cast<char*>(workspace);
  h.logits = reinterpret_cast<float*>(room);
  h.moves = reinterpret_cast<sta::HeavyMove*>(room + w.logits);
  a.part = reinterpret_cast<float*>(room + w.logits + w.moves);
  h.stat = a.part + round16(4 * static_cast<int64_t>(a.streams) * a.heads * a.nsplit * h.part_pitch) / 4;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p > 0) {
    x.q = rows_of(q, strides[0], strides[1], 0);
    x.pk = prefix_rows_of(prefix_k, prefix_strides);
    x.pv = prefix_rows_of(prefix_v, prefix_strides + 3);
    x.prefix_lengths = prefix_lengths;
    set_parts(x, room + w.logits + w.moves + w.part, plan.parts);
    h.prefix = x.part;
    h.prefix_stat = x.stat;
    h.prefix_lengths = prefix_lengths;
    h.prefix_rows = x.p;
    h.per_set = x.per_set;
    if (const int st = run_prefix(x, plan, dtype, 1, s)) return st;
  }
  int st = STA_OK;
  by_type(dtype, [&](auto t) { st = by_keys<decltype(t)::value>(h, s); });
  return st;
}

int sta_heavy_update(const void* k, const void* v, int dtype, int64_t streams, int kv_heads, int d, int dv,
                     const int64_t* strides, int64_t recent, int64_t kept, void* keys, void* values, int64_t* counts,
                     float* weights, int64_t* positions, uint64_t* lowest, void* stream) {
  if (!k || !v || !strides) return STA_ERR_ARG;
  sta::HeavyArgs h;
  if (const int st = heavy_shape(h, dtype, streams, kv_heads, kv_heads, d, dv, recent, kept)) return st;
  if (const int st = state_of(h, keys, values, counts, weights, positions, lowest)) return st;
  h.r.k = rows_of(k, strides[0], strides[1], 0);
  h.r.v = rows_of(v, strides[2], strides[3], 0);
  dim3 g;
  if (!head_grid(h.r, 256, g)) return STA_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((sta::heavy_update_kernel<decltype(t)::value>), g, dim3(256), 0, s, h);
  });
  return check_launch();
}

int64_t sta_heavy_start_bytes(int64_t streams, int kv_heads, int64_t recent, int64_t kept) {
  sta::HeavyArgs h;
  if (heavy_shape(h, STA_F32, streams, kv_heads, kv_heads, 1, 1, recent, kept) != STA_OK) return -1;
  return 4 * static_cast<int64_t>(h.r.streams) * h.r.kv * h.pitch;
}

int sta_heavy_start(const void* k, const void* v, const float* given, int dtype, int64_t streams, int kv_heads, int64_t rows,
                    int d, int dv, const int64_t* strides, int64_t recent, int64_t kept, const int32_t* take, void* keys,
                    void* values, int64_t* counts, float* weights, int64_t* positions, uint64_t* lowest,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  if (!k || !v || !given || !strides) return STA_ERR_ARG;
  sta::HeavyFill f{};
  if (const int st = heavy_shape(f.h, dtype, streams, kv_heads, kv_heads, d, dv, recent, kept)) return st;
  if (const int st = state_of(f.h, keys, values, counts, weights, positions, lowest)) return st;
  if (rows < 1) return STA_ERR_SHAPE;
  if (rows > kMaxHeavySlots) return STA_ERR_UNSUPPORTED;
  if (!workspace || !aligned16(workspace) || workspace_bytes < sta_heavy_start_bytes(streams, kv_heads, recent, kept))
    return STA_ERR_SCRATCH;
  f.h.r.k = prefix_rows_of(k, strides);
  f.h.r.v = prefix_rows_of(v, strides + 3);
  f.rows = static_cast<int>(rows);
  f.take = take;
  f.given = given;
  f.token = static_cast<int*>(workspace);
  dim3 g, heads;
  if (!tile_grid(f.h.r, g) || !head_grid(f.h.r, 1024, heads)) return STA_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // up to a tile a compute unit (3 x 2 key heads of 1025 rows, 66 tiles: 13.2 us in two launches, 12.2 in one; 8 x 2000, 256
  // tiles 14.0 and 13.0, 512 tiles 14.5 and 23.6)
  if (static_cast<int64_t>(g.x) * g.y <= 256) {
    by_type(dtype, [&](auto t) {
      hipLaunchKernelGGL((sta::heavy_start_kernel<decltype(t)::value>), g, dim3(1024), 0, s, f);
    });
    return check_launch();
  }
  hipLaunchKernelGGL(sta::heavy_select_kernel, heads, dim3(1024), 0, s, f);
  by_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((sta::heavy_fill_kernel<decltype(t)::value>), g, dim3(256), 0, s, f);
  });
  return check_launch();
}

int sta_heavy_items(int dtype, int64_t streams, int kv_heads, int d, int dv, int64_t recent, int64_t kept,
                    const void* keys, const void* values, const float* weights, const int64_t* positions,
                    void* keys_out, void* values_out, float* weights_out, int64_t* positions_out, void* stream) {
  if (!keys || !values || !weights || !positions || !keys_out || !values_out || !weights_out || !positions_out ||
      !aligned16(keys) || !aligned16(values) || !aligned16(keys_out) || !aligned16(values_out))
    return STA_ERR_ARG;
  sta::HeavyArgs h;
  if (const int st = heavy_shape(h, dtype, streams, kv_heads, kv_heads, d, dv, recent, kept)) return st;
  h.r.keys = static_cast<uint8_t*>(const_cast<void*>(keys));
  h.r.values = static_cast<uint8_t*>(const_cast<void*>(values));
  h.weights = const_cast<float*>(weights);
  h.positions = const_cast<int64_t*>(positions);
  const sta::HeavyItems to{keys_out, values_out, positions_out, weights_out};
  dim3 g;
  if (!tile_grid(h.r, g)) return STA_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_type(dtype, [&](auto t) {
    hipLaunchKernelGGL((sta::heavy_items_kernel<decltype(t)::value>), g, dim3(256), 0, s, h, to);
  });
  return check_launch();
}

}  // extern "C"
