// Entry points of the token cache (see include/streamattn.h): argument checks, the split of a query, launches.
#include <cmath>

#include "api_common.hpp"
#include "ring_cache.hip"

using namespace sta_api;

namespace sta_api {
template <int ST, int Q, int NBK>
int launch_ring(const sta::RingArgs& a, hipStream_t s);
}  // namespace sta_api

namespace {

constexpr int kMaxRingD = 128;
constexpr int64_t kMaxRingSlots = int64_t(1) << 30;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

sta::Rows rows_of(const void* p, const int64_t* strides) { return sta::Rows{p, strides[0], strides[1], strides[2], 0}; }

// storage: the element type's own code, or 4 bits
bool storage_ok(int storage, int dtype) { return storage == dtype || storage == sta::RING_F4; }

int ring_shape(sta::RingArgs& a, int64_t streams, int heads, int kv_heads, int d, int dv, int64_t window,
               int64_t sinks) {
  a = sta::RingArgs{};
  if (streams < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || d < 1 || dv < 1) return STA_ERR_SHAPE;
  if (window < 1 || sinks < 0) return STA_ERR_ARG;
  if (d > kMaxRingD || dv > kMaxRingD || window > kMaxRingSlots || sinks > kMaxRingSlots - window ||
      streams > 0x7fffffff / kv_heads || streams > 0x7fffffff / heads)
    return STA_ERR_UNSUPPORTED;
  a.streams = static_cast<int>(streams);
  a.heads = heads;
  a.kv = kv_heads;
  a.group = heads / kv_heads;
  a.chunks = (a.group + 15) / 16;
  a.d = d;
  a.dv = dv;
  a.nbk = (d + 31) / 32;
  a.nbv = (dv + 31) / 32;
  a.window = static_cast<int>(window);
  a.sinks = static_cast<int>(sinks);
  a.slots = a.window + a.sinks;
  a.tiles = (a.slots + 31) / 32;
  a.nsplit = 1;
  return STA_OK;
}

// Workgroups that share a key head's slots.  A compute unit holds 2 to 4 at a time and the card has 256: up to 1536 keep
// them busy to the end (64 x 8 key heads of 32772 tokens in 4 bits: 2 workgroups a head 397 us, 3 388, 4 392).  Each has
// at least 16 tiles of 32 slots: shorter ones cost the second launch more than they save the first (one key head of
// 65552: 257 workgroups 7.6 + 6.4 us, 128 8.2 + 4.2; 260 tokens in one 8.0, in two 6.3 + 2.5).
int splits_of(const sta::RingArgs& a) {
  const int64_t blocks = static_cast<int64_t>(a.streams) * a.kv * a.chunks;
  int64_t want = 1536 / blocks;
  if (want > a.tiles / 16) want = a.tiles / 16;
  if (want > sta::RING_SPLITS) want = sta::RING_SPLITS;
  return static_cast<int>(want < 1 ? 1 : want);
}

// A workgroup a tile of the cache, in rows of 2^20 (a million tokens of 512 key heads are 2^24 tiles, whose threads one
// dimension of a launch does not take).
bool tile_grid(const sta::RingArgs& a, dim3& g) {
  const int64_t tiles = static_cast<int64_t>(a.streams) * a.kv * a.tiles, x = tiles < 1 << 20 ? tiles : 1 << 20;
  const int64_t y = (tiles + x - 1) / x;
  g = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
  return y <= 65535;
}

template <int ST, int Q>
int by_keys(const sta::RingArgs& a, hipStream_t s) {
  switch (a.nbk) {
    case 1: return launch_ring<ST, Q, 1>(a, s);
    case 2: return launch_ring<ST, Q, 2>(a, s);
    case 3: return launch_ring<ST, Q, 3>(a, s);
    default: return launch_ring<ST, Q, 4>(a, s);
  }
}

int dispatch(const sta::RingArgs& a, int dtype, int storage, hipStream_t s) {
  if (storage == sta::RING_F4) {
    if (dtype == STA_F32) return by_keys<sta::RING_F4, sta::F32>(a, s);
    if (dtype == STA_BF16) return by_keys<sta::RING_F4, sta::BF16>(a, s);
    return by_keys<sta::RING_F4, sta::F16>(a, s);
  }
  if (dtype == STA_F32) return by_keys<sta::F32, sta::F32>(a, s);
  if (dtype == STA_BF16) return by_keys<sta::BF16, sta::BF16>(a, s);
  return by_keys<sta::F16, sta::F16>(a, s);
}

bool cache_ok(const void* keys, const void* values, const void* kexp, const void* vexp, int storage) {
  if (!keys || !values || !aligned16(keys) || !aligned16(values)) return false;
  return storage != sta::RING_F4 || (kexp && vexp && aligned16(kexp) && aligned16(vexp));
}

}  // namespace

extern "C" {

int sta_ring_layout(int dtype, int storage, int64_t streams, int kv_heads, int d, int dv, int64_t window,
                    int64_t sinks, int64_t* bytes) {
  if (!bytes) return STA_ERR_ARG;
  if (!dtype_ok(dtype) || !storage_ok(storage, dtype)) return STA_ERR_DTYPE;
  sta::RingArgs a;
  if (const int st = ring_shape(a, streams, kv_heads, kv_heads, d, dv, window, sinks)) return st;
  const int64_t tiles = static_cast<int64_t>(a.streams) * a.kv * a.tiles;
  bytes[0] = tiles * sta::ring_tile_bytes(a.nbk, storage);
  bytes[1] = tiles * sta::ring_tile_bytes(a.nbv, storage);
  bytes[2] = tiles * sta::ring_key_exp_bytes(a.nbk, storage);
  bytes[3] = tiles * sta::ring_value_exp_bytes(a.nbv, storage);
  return STA_OK;
}

int64_t sta_ring_attention_bytes(int64_t streams, int heads, int kv_heads, int d, int dv, int64_t window,
                                 int64_t sinks) {
  sta::RingArgs a;
  if (ring_shape(a, streams, heads, kv_heads, d, dv, window, sinks) != STA_OK) return -1;
  const int n = splits_of(a);
  return n == 1 ? 0 : 4 * static_cast<int64_t>(a.streams) * heads * n * (dv + 2);
}

int sta_ring_attention(const void* q, const void* k, const void* v, int dtype, int storage, int64_t streams, int heads,
                       int kv_heads, int d, int dv, const int64_t* strides, float scale, int64_t window,
                       int64_t sinks, void* keys, void* values, void* key_exponents, void* value_exponents,
                       int32_t* counts, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || !out || !counts || !strides || !k != !v || !std::isfinite(scale)) return STA_ERR_ARG;
  if (!dtype_ok(dtype) || !storage_ok(storage, dtype)) return STA_ERR_DTYPE;
  if (!cache_ok(keys, values, key_exponents, value_exponents, storage)) return STA_ERR_ARG;
  sta::RingArgs a;
  if (const int st = ring_shape(a, streams, heads, kv_heads, d, dv, window, sinks)) return st;
  const int64_t need = sta_ring_attention_bytes(streams, heads, kv_heads, d, dv, window, sinks);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return STA_ERR_SCRATCH;
  const int64_t qs[3] = {strides[0], strides[1], 0}, ks[3] = {strides[2], strides[3], 0},
                vs[3] = {strides[4], strides[5], 0};
  a.q = rows_of(q, qs);
  a.append = k != nullptr;
  if (a.append) {
    a.k = rows_of(k, ks);
    a.v = rows_of(v, vs);
  }
  a.scale = scale;
  // above 0: what a wave without tiles has, -3e38, stays far below a logit times c
  a.c = std::fmax(std::fabs(scale) * 1.44269504088896340736f, 1e-37f);
  a.keys = static_cast<uint8_t*>(keys);
  a.values = static_cast<uint8_t*>(values);
  a.kexp = static_cast<uint8_t*>(key_exponents);
  a.vexp = static_cast<uint8_t*>(value_exponents);
  a.counts = counts;
  a.nsplit = splits_of(a);
  a.part = static_cast<float*>(workspace);
  a.out = out;
  return dispatch(a, dtype, storage, static_cast<hipStream_t>(stream));
}

int sta_ring_extend(const void* k, const void* v, int dtype, int storage, int64_t streams, int kv_heads, int64_t rows,
                    int d, int dv, const int64_t* strides, int64_t window, int64_t sinks, const int32_t* take,
                    void* keys, void* values, void* key_exponents, void* value_exponents, int32_t* counts,
                    void* stream) {
  if (!k || !v || !strides || !counts) return STA_ERR_ARG;
  if (!dtype_ok(dtype) || !storage_ok(storage, dtype)) return STA_ERR_DTYPE;
  if (!cache_ok(keys, values, key_exponents, value_exponents, storage)) return STA_ERR_ARG;
  sta::RingFill f{};
  if (const int st = ring_shape(f.a, streams, kv_heads, kv_heads, d, dv, window, sinks)) return st;
  if (rows < 1) return STA_ERR_SHAPE;
  if (rows > kMaxRingSlots) return STA_ERR_UNSUPPORTED;
  f.a.k = rows_of(k, strides);
  f.a.v = rows_of(v, strides + 3);
  f.a.keys = static_cast<uint8_t*>(keys);
  f.a.values = static_cast<uint8_t*>(values);
  f.a.kexp = static_cast<uint8_t*>(key_exponents);
  f.a.vexp = static_cast<uint8_t*>(value_exponents);
  f.a.counts = counts;
  f.rows = static_cast<int>(rows);
  f.take = take;
  dim3 g;
  if (!tile_grid(f.a, g)) return STA_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define STA_RING_EXTEND(ST, Q) hipLaunchKernelGGL((sta::ring_extend_kernel<ST, Q>), g, dim3(256), 0, s, f)
  if (storage == sta::RING_F4 && dtype == STA_F32) STA_RING_EXTEND(sta::RING_F4, sta::F32);
  else if (storage == sta::RING_F4 && dtype == STA_BF16) STA_RING_EXTEND(sta::RING_F4, sta::BF16);
  else if (storage == sta::RING_F4) STA_RING_EXTEND(sta::RING_F4, sta::F16);
  else if (dtype == STA_F32) STA_RING_EXTEND(sta::F32, sta::F32);
  else if (dtype == STA_BF16) STA_RING_EXTEND(sta::BF16, sta::BF16);
  else STA_RING_EXTEND(sta::F16, sta::F16);
#undef STA_RING_EXTEND
  hipLaunchKernelGGL(sta::ring_count_kernel, dim3((f.a.streams * f.a.kv + 255) / 256), dim3(256), 0, s, f);
  return check_launch();
}

int sta_ring_items(int dtype, int storage, int64_t streams, int kv_heads, int d, int dv, int64_t window,
                   int64_t sinks, const void* keys, const void* values, const void* key_exponents,
                   const void* value_exponents, const int32_t* counts, void* keys_out, void* values_out,
                   int32_t* positions, void* stream) {
  if (!counts || !keys_out || !values_out || !positions || !aligned16(keys_out) || !aligned16(values_out))
    return STA_ERR_ARG;
  if (!dtype_ok(dtype) || !storage_ok(storage, dtype)) return STA_ERR_DTYPE;
  if (!cache_ok(keys, values, key_exponents, value_exponents, storage)) return STA_ERR_ARG;
  sta::RingArgs a;
  if (const int st = ring_shape(a, streams, kv_heads, kv_heads, d, dv, window, sinks)) return st;
  a.keys = static_cast<uint8_t*>(const_cast<void*>(keys));
  a.values = static_cast<uint8_t*>(const_cast<void*>(values));
  a.kexp = static_cast<uint8_t*>(const_cast<void*>(key_exponents));
  a.vexp = static_cast<uint8_t*>(const_cast<void*>(value_exponents));
  a.counts = const_cast<int32_t*>(counts);
  dim3 g;
  if (!tile_grid(a, g)) return STA_ERR_SHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define STA_RING_ITEMS(ST, Q) \
  hipLaunchKernelGGL((sta::ring_items_kernel<ST, Q>), g, dim3(256), 0, s, a, keys_out, values_out, positions)
  if (storage == sta::RING_F4 && dtype == STA_F32) STA_RING_ITEMS(sta::RING_F4, sta::F32);
  else if (storage == sta::RING_F4 && dtype == STA_BF16) STA_RING_ITEMS(sta::RING_F4, sta::BF16);
  else if (storage == sta::RING_F4) STA_RING_ITEMS(sta::RING_F4, sta::F16);
  else if (dtype == STA_F32) STA_RING_ITEMS(sta::F32, sta::F32);
  else if (dtype == STA_BF16) STA_RING_ITEMS(sta::BF16, sta::BF16);
  else STA_RING_ITEMS(sta::F16, sta::F16);
#undef STA_RING_ITEMS
  return check_launch();
}

}  // extern "C"
