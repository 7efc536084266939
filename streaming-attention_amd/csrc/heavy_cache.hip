// The cache that keeps the most attended tokens, and the single-token attention over it.
//
// A (stream, key head) holds the last `recent` tokens in a ring of recent + 1 slots, token p in slot p % (recent + 1), and
// in `kept` slots behind them older ones, each slot with its position and its weight W, the attention weights that the
// token has received.  Token n of a stream sends token n - recent out of the ring: into the next kept slot while there
// is one, else into the kept slot of the lowest W (of equal ones the first) unless its own W is lower.  The ring's one
// slot more than it holds lets the token that leaves be read from its slot while the new one is written: the slot is
// empty from then on until the next token takes it.
//   p_hj = exp(s q_h.k_j - L_h), L_h = log of the sum over the tokens held (and the rows of a shared prefix),
//   o_h = sum_j p_hj v_j,   W_j += sum over the query heads of the key head of p_hj
// Increments that are not finite are left out, so that a token held with an infinity or NaN does not make its
// neighbours' weights NaN.  A token whose logit is +inf or NaN with a finite query makes that row's weights NaN, all of them,
// as long as it is held: its own weight becomes the lowest finite one, so that of the kept tokens it leaves first (its
// increments left out alone, tokens that come after it have weights of 0 and take each other's place, the first slot of equal
// ones, beside it).
//
// Keys and values lie as in the token cache of windowed attention (ring_cache.hip).  The slot of the lowest W is part of
// the state: whoever changes weights looks for it, in the pass that it makes over them anyway, so that a step knows it
// without one.  Two entries take turns (by the parity of the count that they are for), since workgroups of a step that
// read one may run beside another that clears the other.
#include "prefix_attn.hip"
#include "ring_cache.hip"

namespace sta {

struct HeavyArgs {
  RingArgs r;            // q, new tokens, sizes, cache, part, out; counts unused
  int recent, kept, ring, pitch;  // ring = recent + 1; pitch: slots of a row of weights and positions, whole tiles
  int64_t* counts;       // [streams][kv]: tokens so far
  float* weights;        // [streams][kv][pitch]
  int64_t* positions;    // [streams][kv][pitch], -1: no token
  unsigned long long* lowest;  // [streams][kv][2]: order of the lowest weight of the kept slots, and the slot
  float* logits;         // [streams][heads][pitch]: this step's; unused by workgroups that keep them in LDS
  struct HeavyMove* moves;  // [streams][kv], of steps that several workgroups share
  // partials, of splits (r.part: sums) and of a shared prefix: sums [streams][heads][parts][part_pitch], maximum and sum of
  // weights [streams][heads][parts][2]
  float* stat;
  const float *prefix, *prefix_stat;
  int prefix_parts, part_pitch;
  const int* prefix_lengths;  // [sets] or null: rows of the prefix that count, of prefix_rows
  int prefix_rows, per_set;   // per_set: streams that share one
  int alone;             // a workgroup has a key head to itself and finishes it: one split, up to 16 query heads, no prefix
  int local;             // such a workgroup keeps the logits in LDS
};

// What a step does to the slots of a key head.
struct HeavyMove {
  int64_t n;             // tokens before it
  int from, to;          // the slot that a token leaves (-1: none), the kept slot that it takes (-1: it is forgotten)
  int slot;              // of the new token (-1: none comes)
  int hole;              // the empty slot of a full ring (-1: none)
  int held;              // slots [0, held) but the hole hold a token
  float weight;          // of the token that leaves its slot
};

// weights in the order of unsigned numbers (none is NaN)
__device__ __forceinline__ uint32_t heavy_order(float w) {
  const uint32_t u = __float_as_uint(w);
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ unsigned long long heavy_key(float w, int slot) {
  return static_cast<unsigned long long>(heavy_order(w)) << 32 | static_cast<uint32_t>(slot);
}
constexpr unsigned long long HEAVY_NONE = ~0ull;

__device__ __forceinline__ unsigned long long heavy_min(unsigned long long a, unsigned long long b) { return a < b ? a : b; }
// the least of a workgroup's keys, for every thread (a barrier before red is used again is the caller's)
template <int THREADS>
__device__ __forceinline__ unsigned long long heavy_least(unsigned long long x, unsigned long long* red) {
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long y = static_cast<unsigned long long>(__shfl_xor(static_cast<long long>(x), o));
    x = heavy_min(x, y);
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  for (int i = 0; i < THREADS / 64; ++i) x = heavy_min(x, red[i]);
  return x;
}

// What a step of a key head with count n does: its slots, and once the leaving token's weight and the lowest kept ones (of
// even and of odd counts) are there, where it goes.
__device__ __forceinline__ HeavyMove heavy_slots(const HeavyArgs& a, bool append, int64_t n) {
  HeavyMove m;
  m.n = n < 0 ? 0 : n;
  const int64_t after = m.n + (append ? 1 : 0), older = after - a.recent;
  m.hole = older > 0 ? static_cast<int>((older - 1) % a.ring) : -1;
  m.held = older > 0 ? a.ring + static_cast<int>(older < a.kept ? older : a.kept) : static_cast<int>(after);
  m.slot = append ? static_cast<int>(m.n % a.ring) : -1;
  m.from = append ? m.hole : -1;
  m.to = -1;
  m.weight = 0.f;
  return m;
}
__device__ __forceinline__ float heavy_weight(const HeavyArgs& a, int sh, int slot) {
  return a.weights[static_cast<int64_t>(sh) * a.pitch + (slot < 0 ? 0 : slot)];
}
__device__ __forceinline__ void heavy_goes(const HeavyArgs& a, HeavyMove& m, float weight, unsigned long long even,
                                           unsigned long long odd) {
  const int64_t gone = m.n - a.recent;
  const unsigned long long low = m.n & 1 ? odd : even;
  const int lowest = static_cast<int>(low & 0xffffffffu);
  const bool free = gone < a.kept;
  const bool better = heavy_order(weight) >= static_cast<uint32_t>(low >> 32) && lowest >= a.ring && lowest < a.r.slots;
  if (m.from >= 0) {
    m.weight = weight;
    m.to = free ? a.ring + static_cast<int>(gone) : (better ? lowest : -1);
  }
}

// A thread's piece of a token's row, of the first 4 nbk threads 8 dimensions of the key, of threads 64 .. 64 + 32 nbv - 1
// a column of the value: from the call or a slot, into a slot.
template <int ST>
struct HeavyPiece {
  static constexpr int ES = ST == F32 ? 4 : 2;
  uint4 k[ES / 2];
  uint32_t v;

  __device__ __forceinline__ static bool key(const RingArgs& a) { return static_cast<int>(threadIdx.x) < 4 * a.nbk; }
  __device__ __forceinline__ static bool value(const RingArgs& a) {
    return threadIdx.x >= 64 && static_cast<int>(threadIdx.x) < 64 + 32 * a.nbv;
  }
  __device__ __forceinline__ static uint8_t* key_at(const RingArgs& a, int sh, int slot) {
    return a.keys + (static_cast<int64_t>(sh) * a.tiles + (slot >> 5)) * ring_tile_bytes(a.nbk, ST) +
           ring_key_at(slot & 31, 8 * threadIdx.x, a.nbk, ST);
  }
  __device__ __forceinline__ static uint8_t* value_at(const RingArgs& a, int sh, int slot) {
    return a.values + (static_cast<int64_t>(sh) * a.tiles + (slot >> 5)) * ring_tile_bytes(a.nbv, ST) +
           ring_value_at(slot & 31, threadIdx.x - 64, a.nbv, ST);
  }
  __device__ __forceinline__ void load_new(const RingArgs& a, int s, int hk) {
    if (key(a)) {
      const char* row = rows_at<ES>(a.k, s, hk, 0);
#pragma unroll
      for (int i = 0; i < ES / 2; ++i) k[i] = rows_chunk<ES>(row, 8 * threadIdx.x + (16 / ES) * i, a.d);
    } else if (value(a)) {
      const char* row = rows_at<ES>(a.v, s, hk, 0);
      const int col = threadIdx.x - 64;
      v = 0u;
      if (col < a.dv) {
        if constexpr (ES == 4)
          v = reinterpret_cast<const uint32_t*>(row)[col];
        else
          v = reinterpret_cast<const uint16_t*>(row)[col];
      }
    }
  }
  __device__ __forceinline__ void load(const RingArgs& a, int sh, int slot) {
    if (key(a)) {
#pragma unroll
      for (int i = 0; i < ES / 2; ++i) k[i] = reinterpret_cast<const uint4*>(key_at(a, sh, slot))[i];
    } else if (value(a)) {
      if constexpr (ES == 4)
        v = *reinterpret_cast<const uint32_t*>(value_at(a, sh, slot));
      else
        v = *reinterpret_cast<const uint16_t*>(value_at(a, sh, slot));
    }
  }
  __device__ __forceinline__ void store(const RingArgs& a, int sh, int slot) const {
    if (key(a)) {
#pragma unroll
      for (int i = 0; i < ES / 2; ++i) reinterpret_cast<uint4*>(key_at(a, sh, slot))[i] = k[i];
    } else if (value(a)) {
      if constexpr (ES == 4)
        *reinterpret_cast<uint32_t*>(value_at(a, sh, slot)) = v;
      else
        *reinterpret_cast<uint16_t*>(value_at(a, sh, slot)) = static_cast<uint16_t>(v);
    }
  }
};

// A slot's weight and position after the step, before its query adds to the weight.
__device__ __forceinline__ float heavy_base(const HeavyMove& m, int slot, float w) {
  if (slot == m.to) return m.weight;
  return slot == m.slot || slot == m.hole ? 0.f : w;
}

constexpr float HEAVY_LEAST = -3.4028235e38f;  // of a token whose logits are not finite
// A query beyond it, infinite or NaN is itself what makes a logit so.  (Keys of 128 columns up to 2^57 give finite logits below.)
constexpr float HEAVY_QUERY = 0x1p64f;

// four slots' weights
__device__ __forceinline__ floatx4* heavy_weights(const HeavyArgs& a, int sh, int at) {
  return reinterpret_cast<floatx4*>(a.weights + static_cast<int64_t>(sh) * a.pitch + 4 * at);
}
// Slots 4 at, .. + 3 of weights w grow by `queries` heads' logits (`pitch` floats each); what that does to the lowest kept
// weight.  stat: the heads' maxima, and their sums' inverses `stats` behind them.
template <int ST, typename Logits>
__device__ __forceinline__ unsigned long long heavy_grow(const HeavyArgs& a, const HeavyMove& m, int sh, int at,
                                                         const floatx4& w, Logits logits, int64_t pitch, int queries,
                                                         const float* stat, int stats) {
  constexpr float lift = win_weight_lift<ST>();
  floatx4 grown = floatx4{0.f, 0.f, 0.f, 0.f};
  bool wrong = false, lost[4] = {};
  auto add = [&](const floatx4& x, float top, float inv) {
#pragma unroll
    for (int j = 0; j < 4; ++j) grown[j] += __builtin_amdgcn_exp2f(fmaf(x[j] - top, a.r.c, lift)) * inv;
  };
  for (int i = 0; i < queries; ++i) {
    const float inv = stat[stats + i];
    wrong |= !win_finite(inv);
    add(*reinterpret_cast<const floatx4*>(logits + i * pitch + 4 * at), stat[i], inv);
  }
  if (wrong) {  // a row's sum is 0, or not finite: once more with the others, and is it by one of these tokens
    grown = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < queries; ++i) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(logits + i * pitch + 4 * at);
      const float inv = stat[stats + i];
      if (win_finite(inv)) add(x, stat[i], inv);
#pragma unroll
      for (int j = 0; j < 4; ++j) lost[j] |= !(x[j] < __builtin_inff());
    }
  }
  unsigned long long low = HEAVY_NONE;
  floatx4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int slot = 4 * at + j;
    const bool in = slot < m.held && slot != m.hole;
    const float base = heavy_base(m, slot, w[j]);
    y[j] = in ? (lost[j] ? fminf(base, HEAVY_LEAST) : base + grown[j]) : 0.f;
    if (in && slot >= a.ring) low = heavy_min(low, heavy_key(y[j], slot));
  }
  *heavy_weights(a, sh, at) = y;
  return low;
}

// positions of the slots that a step changes
__device__ __forceinline__ void heavy_positions(const HeavyArgs& a, const HeavyMove& m, int sh) {
  int64_t* row = a.positions + static_cast<int64_t>(sh) * a.pitch;
  if (m.to >= 0) row[m.to] = m.n - a.recent;
  if (m.from >= 0) row[m.from] = -1;
  if (m.slot >= 0) row[m.slot] = m.n;
}

__host__ __device__ constexpr int heavy_red_pitch(int nbv) { return 32 * nbv + 4; }
// rows of logits in LDS, four banks apart
__host__ __device__ constexpr int heavy_kept_pitch(int pitch) { return pitch + 4; }
// dynamic LDS of a workgroup of heavy_attention_kernel
__host__ __device__ constexpr int64_t heavy_lds_bytes(int group, int nbv, int pitch, bool local) {
  const int64_t rows = group < 16 ? group : 16;
  return 4 * rows * (4 * heavy_red_pitch(nbv) + (local ? heavy_kept_pitch(pitch) : 0));
}

// The walk of ring_attention_kernel over the slots that hold a token, with the logits put down for the weights' growth.  A
// workgroup that is alone with a key head finishes it: outputs, weights, the next lowest one; else heavy_join_kernel does.
template <int NBK, int NBV, int ST>
__global__ __launch_bounds__(256, ST == F32 ? 1 : 2) void heavy_attention_kernel(const HeavyArgs h) {
  const RingArgs& a = h.r;
  constexpr int PP = ST == F32 ? 1 : 2;  // planes of the weights, see ring_cache.hip (a prefix has one, see prefix_attn.hip)
  constexpr int ES = ST == F32 ? 4 : 2, CT = 2 * NBV, W = RingTile<NBK, NBV, ST>::W;
  constexpr int PITCH = heavy_red_pitch(NBV);
  extern __shared__ float heavy_lds[];  // [4][queries][PITCH] for the waves' sums, then the logits if they are kept here
  __shared__ float red_m[4 * 16], red_l[4 * 16], stat[2 * 16];
  __shared__ unsigned long long red_low[4];
  int id = blockIdx.x;
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int chunk = id % a.chunks, sh = id / a.chunks;
  const int s = sh / a.kv, hk = sh - s * a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
  const int rows = min(16, a.group);  // of red
  float *const red = heavy_lds, *const kept = heavy_lds + 4 * rows * PITCH;
  const int kept_pitch = heavy_kept_pitch(h.pitch);

  // Loads come one after the other only where one needs what another gave: what no count is needed for first, then the
  // leaving token, the first tile and the weights.
  const int64_t n = h.counts[sh];
  const unsigned long long low_even = h.lowest[2 * static_cast<int64_t>(sh)], low_odd = h.lowest[2 * static_cast<int64_t>(sh) + 1];
  HeavyPiece<ST> fresh{}, old{};
  if (a.append) fresh.load_new(a, s, hk);
  const int queries = min(16, a.group - 16 * chunk);
  const int64_t head0 = static_cast<int64_t>(s) * a.heads + hk * a.group + 16 * chunk;
  uint4 q_row[NBK][ES / 2];
  {
    const char* row = rows_at<ES>(a.q, s, hk * a.group + 16 * chunk + (li < queries ? li : 0), 0);
#pragma unroll
    for (int b = 0; b < NBK; ++b)
#pragma unroll
      for (int i = 0; i < ES / 2; ++i) q_row[b][i] = rows_chunk<ES>(row, 32 * b + 8 * lg + 16 / ES * i, a.d);
  }
  HeavyMove move = heavy_slots(h, a.append, n);
  const float leaving = heavy_weight(h, sh, move.from);
  if (move.from >= 0) old.load(a, sh, move.from);
  const bool alone = h.alone;
  const int all = (move.held + 31) >> 5, per = (all + a.nsplit - 1) / a.nsplit;
  const int t0 = split * per, t1 = t0 + per < all ? t0 + per : all, count = t1 - t0;
  const int hole_tile = move.hole >= 0 ? move.hole >> 5 : -1;
  const int64_t tile0 = static_cast<int64_t>(sh) * a.tiles;
  // Key heads begin at different tiles of their share: caches of equal lengths, walked in step, would else ask the same
  // memory channels at a time.
  const int turn = count > 0 ? (sh * 29) % count : 0;
  auto tile = [&](int i) {
    const int t = i + turn;
    return t0 + (t < count ? t : t - count);
  };
  // a wave's first tile, before the new token is in
  RingTile<NBK, NBV, ST> even;
  const int first = wave < count ? tile(wave) : -1;
  if (first >= 0) even.load(a, tile0 + first, lane);
  constexpr int HOLD = 4;
  floatx4 weights[HOLD];
#pragma unroll
  for (int j = 0; j < HOLD; ++j) {
    const int at = threadIdx.x + 256 * j;
    weights[j] = alone && 4 * at < move.held ? *heavy_weights(h, sh, at) : floatx4{0.f, 0.f, 0.f, 0.f};
  }
  heavy_goes(h, move, leaving, low_even, low_odd);
  if (a.append) {
    if (move.to >= 0 && (move.to >> 5) >= t0 && (move.to >> 5) < t1) old.store(a, sh, move.to);
    if ((move.slot >> 5) >= t0 && (move.slot >> 5) < t1) fresh.store(a, sh, move.slot);
    __syncthreads();
    if (first >= 0 && (first == move.to >> 5 || first == move.slot >> 5)) even.load(a, tile0 + first, lane);  // again
  }
  if (!alone && split == 0 && chunk == 0 && threadIdx.x == 0) {
    h.moves[sh] = move;
    h.lowest[2 * static_cast<int64_t>(sh) + ((move.n + a.append) & 1)] = HEAVY_NONE;
  }

  RingFrag<ST> qf[NBK];
#pragma unroll
  for (int b = 0; b < NBK; ++b) {
    constexpr int E = 16 / ES;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8 / E; ++i) {
      float y[E];
      rows_unpack<ST>(q_row[b][i], y);
#pragma unroll
      for (int e = 0; e < E; ++e) x[E * i + e] = li < queries ? (a.scale < 0.f ? -y[e] : y[e]) : 0.f;
    }
    RingFrag<ST> planes[1];
    ring_planes<ST, 1>(x, planes);
    qf[b] = planes[0];
  }

  floatx4 acc[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) acc[ct] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -3.4028235e38f, limit = m, l = 0.f;
  constexpr float lift = win_weight_lift<ST>();  // fp16 weights, see ring_cache.hip
  const float room = win_weight_room<ST>() / a.c;

  float* const logits = h.logits + (head0 + li) * h.pitch + 4 * lg;
  // a tile's part of the sums
  auto take = [&](RingTile<NBK, NBV, ST>& cur, int t) {
    floatx4 x[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      x[half] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NBK; ++b) {
        RingFrag<ST> k;
#pragma unroll
        for (int i = 0; i < W; ++i) k.w[i] = cur.k[half][b * W + i];
        x[half] = ring_mma<ST>(k, qf[b], x[half]);
      }
    }
    // not all of the tile's slots hold a token: this lane's do below `left`, but `hole`
    if (t == hole_tile || 32 * t + 32 > move.held) {
      const int left = move.held - 32 * t - 4 * lg, hole = move.hole - 32 * t - 4 * lg;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 16 * (i >> 2) + (i & 3);
        const bool out = at >= left || at == hole;
        x[i >> 2][i & 3] = out ? -__builtin_inff() : x[i >> 2][i & 3];
        // values: whatever the slot holds
        const uint32_t keep = out ? 0u : 0xffffffffu;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if constexpr (ST == F32)
            cur.v[ct * W + i] &= keep;
          else
            cur.v[ct * W + (i >> 1)] &= i & 1 ? keep | 0x0000ffffu : keep | 0xffff0000u;
        }
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i >> 2][i & 3]);
    if (li < queries) {
      if (h.local) {
        float* to = kept + li * kept_pitch + 4 * lg + 32 * t;
        *reinterpret_cast<floatx4*>(to) = x[0];
        *reinterpret_cast<floatx4*>(to + 16) = x[1];
      } else {
        *reinterpret_cast<floatx4*>(logits + 32 * t) = x[0];
        *reinterpret_cast<floatx4*>(logits + 32 * t + 16) = x[1];
      }
    }
    // the maximum moves, for all lanes of a query at once, when a weight would exceed 2^room
    if (__any(top > limit)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float shrink = __builtin_amdgcn_exp2f((m - top) * a.c);
      l *= shrink;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) acc[ct] *= shrink;
      m = top;
      limit = top + room;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(x[i >> 2][i & 3] - m, a.c, lift));
      l += p[i];
    }
    RingFrag<ST> pf[PP];
    ring_planes<ST, PP>(p, pf);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      RingFrag<ST> v;
#pragma unroll
      for (int i = 0; i < W; ++i) v.w[i] = cur.v[ct * W + i];
#pragma unroll
      for (int k = PP - 1; k >= 0; --k) acc[ct] = ring_mma<ST>(v, pf[k], acc[ct]);
    }
  };
  // every fourth tile a wave, one ahead in registers, the two buffers in turn
  {
    RingTile<NBK, NBV, ST> odd;
    int i = wave;
    while (i < count) {
      if (i + 4 < count) odd.load(a, tile0 + tile(i + 4), lane);
      take(even, tile(i));
      i += 4;
      if (i >= count) break;
      if (i + 4 < count) even.load(a, tile0 + tile(i + 4), lane);
      take(odd, tile(i));
      i += 4;
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  // A row with a logit of +inf or NaN: where the query is at fault no token is, and the wave puts what it has put down of such
  // a query down once more.
  if (__any(!win_finite(l))) {
    constexpr int E = 16 / ES;
    const char* row = rows_at<ES>(a.q, s, hk * a.group + 16 * chunk + (li < queries ? li : 0), 0);
    bool sane = true;
#pragma unroll 1
    for (int i = 0; i < NBK * ES / 2; ++i) {
      float y[E];
      rows_unpack<ST>(rows_chunk<ES>(row, 32 * (i / (ES / 2)) + 8 * lg + E * (i % (ES / 2)), a.d), y);
#pragma unroll
      for (int e = 0; e < E; ++e) sane &= fabsf(y[e]) < HEAVY_QUERY;
    }
    const unsigned long long odd = __ballot(!sane && li < queries);
    if (odd >> li & 0x1000100010001ull) {
      for (int i = wave; i < count; i += 4) {
        float* const to = h.local ? kept + li * kept_pitch + 4 * lg + 32 * tile(i) : logits + 32 * tile(i);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          floatx4 x = *reinterpret_cast<floatx4*>(to + 16 * half);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = win_finite(x[j]) ? x[j] : -__builtin_inff();
          *reinterpret_cast<floatx4*>(to + 16 * half) = x;
        }
      }
    }
  }

  // the four waves' sums
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    if (li < queries) *reinterpret_cast<floatx4*>(&red[(wave * rows + li) * PITCH + 16 * ct + 4 * lg]) = acc[ct];
  if (lg == 0) {
    red_m[wave * 16 + li] = prefix_top(m, l);
    red_l[wave * 16 + li] = l;
  }
  __syncthreads();
  for (int at = threadIdx.x; at < queries * a.dv; at += 256) {
    const int i = at / a.dv, col = at - i * a.dv;
    float top = red_m[i], sum = 0.f, den = 0.f;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, red_m[16 * w + i]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float lw = red_l[16 * w + i], f = lw == 0.f ? 0.f : __builtin_amdgcn_exp2f((red_m[16 * w + i] - top) * a.c);
      if (lw != 0.f) sum = fmaf(f, red[(w * rows + i) * PITCH + col], sum);
      den = fmaf(f, lw, den);
    }
    if (alone) {
      store_elem(a.out, (head0 + i) * a.dv + col, ST, move.held ? sum / den : 0.f);
      if (col == 0) {
        stat[i] = top;
        stat[16 + i] = 1.f / den;
      }
    } else {
      const int64_t part = (head0 + i) * a.nsplit + split;
      a.part[part * h.part_pitch + col] = sum;
      if (col == 0) *reinterpret_cast<floatx2*>(h.stat + 2 * part) = floatx2{prefix_top(top, den), den};
    }
  }
  if (!alone) return;
  __syncthreads();  // the logits of all waves, too
  unsigned long long low = HEAVY_NONE;
  auto grow = [&](int at, const floatx4& w) {
    if (4 * at >= move.held) return;
    const unsigned long long x =
        h.local ? heavy_grow<ST>(h, move, sh, at, w, static_cast<const float*>(kept), kept_pitch, queries, stat, 16)
                : heavy_grow<ST>(h, move, sh, at, w, static_cast<const float*>(h.logits + head0 * h.pitch), h.pitch, queries,
                                 stat, 16);
    low = heavy_min(low, x);
  };
#pragma unroll
  for (int j = 0; j < HOLD; ++j) grow(threadIdx.x + 256 * j, weights[j]);
  for (int at = threadIdx.x + 256 * HOLD; 4 * at < move.held; at += 256) grow(at, *heavy_weights(h, sh, at));
  low = heavy_least<256>(low, red_low);
  if (threadIdx.x == 0) {
    heavy_positions(h, move, sh);
    h.lowest[2 * static_cast<int64_t>(sh) + ((move.n + a.append) & 1)] = low;
    h.counts[sh] = move.n + a.append;
  }
}

__device__ __forceinline__ int heavy_prefix_rows(const HeavyArgs& a, int s) {
  return a.prefix_lengths ? prefix_clamp(a.prefix_lengths[s / a.per_set], a.prefix_rows) : a.prefix_rows;
}

// Steps that several workgroups share: outputs, 4 groups of 128 threads (a column each) over the partials of a query head,
// then in workgroups of their own the weights, 2048 slots of a key head each.
constexpr int HEAVY_SPLITS = 1024, HEAVY_SLOTS = 2048, HEAVY_HEADS = 512;
template <int ST>
__global__ __launch_bounds__(512) void heavy_join_kernel(const HeavyArgs h, int outputs, int ranges) {
  const RingArgs& a = h.r;
  constexpr int AHEAD = 16;
  __shared__ float weight[HEAVY_SPLITS], red[4 * 128], wave_red[8], stat[2 * HEAVY_HEADS];
  __shared__ unsigned long long red_low[8];
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const int total = a.nsplit + h.prefix_parts;
  // maximum and sum of weights of a head's partial, and a column of its sums; partials behind the last have none
  auto stat_of = [&](int64_t head, int j) {
    const float* at = j < a.nsplit ? h.stat + 2 * (head * a.nsplit + j) : h.prefix_stat + 2 * (head * h.prefix_parts + j - a.nsplit);
    return j < total ? *reinterpret_cast<const floatx2*>(at) : floatx2{-__builtin_inff(), 0.f};
  };
  auto sum_of = [&](int64_t head, int j, int col) {
    return j < a.nsplit ? a.part[(head * a.nsplit + j) * h.part_pitch + col]
                        : h.prefix[(head * h.prefix_parts + j - a.nsplit) * h.part_pitch + col];
  };
  if (static_cast<int>(blockIdx.x) < outputs) {
    const int64_t head = blockIdx.x;
    const int s = blockIdx.x / a.heads, hh = blockIdx.x - s * a.heads, sh = s * a.kv + hh / a.group;
    const int col = t & 127, group = t >> 7;
    // the partials' loads are under way before their weights are known
    float ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = col < a.dv && group + 4 * i < total ? sum_of(head, group + 4 * i, col) : 0.f;
    const floatx2 mine[2] = {stat_of(head, t), stat_of(head, t + 512)};
    const int held = h.moves[sh].held;
    float top = fmaxf(mine[0][0], mine[1][0]), den = 0.f;
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) wave_red[wave] = top;
    __syncthreads();
    for (int i = 0; i < 8; ++i) top = fmaxf(top, wave_red[i]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float f = mine[k][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f((mine[k][0] - top) * a.c);
      weight[t + 512 * k] = f;
      den = fmaf(f, mine[k][1], den);
    }
    for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
    __syncthreads();
    if (lane == 0) wave_red[wave] = den;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) sum = fmaf(weight[group + 4 * i], ahead[i], sum);
    if (col < a.dv) {
#pragma unroll 8
      for (int i = group + 4 * AHEAD; i < total; i += 4) sum = fmaf(weight[i], sum_of(head, i, col), sum);
    }
    red[t] = sum;
    __syncthreads();
    if (t < a.dv) {
      den = 0.f;
      for (int i = 0; i < 8; ++i) den += wave_red[i];
      sum = red[t] + red[128 + t] + red[256 + t] + red[384 + t];
      const bool sees = held || den != 0.f || (h.prefix_parts && heavy_prefix_rows(h, s));
      store_elem(a.out, head * a.dv + t, ST, sees ? sum / den : 0.f);  // logits of -inf alone: NaN
    }
    return;
  }
  const int id = blockIdx.x - outputs, sh = id / ranges, range = id - sh * ranges;
  const int s = sh / a.kv, hk = sh - s * a.kv;
  const int64_t head0 = static_cast<int64_t>(s) * a.heads + hk * a.group;
  const int at = range * (HEAVY_SLOTS / 4) + t;
  const floatx4 w = 4 * at < h.pitch ? *heavy_weights(h, sh, at) : floatx4{0.f, 0.f, 0.f, 0.f};
  const HeavyMove move = h.moves[sh];
  unsigned long long low = HEAVY_NONE;
  if (range * HEAVY_SLOTS < move.held) {
    for (int i = wave; i < a.group; i += 8) {  // a wave a head: its maximum and sum
      float top = -__builtin_inff(), den = 0.f;
      for (int j = lane; j < total; j += 64) {
        const floatx2 x = stat_of(head0 + i, j);
        const float up = fmaxf(top, x[0]);
        den = (den == 0.f ? 0.f : den * __builtin_amdgcn_exp2f((top - up) * a.c)) +
              (x[1] == 0.f ? 0.f : x[1] * __builtin_amdgcn_exp2f((x[0] - up) * a.c));
        top = up;
      }
      float up = top;
      for (int o = 32; o > 0; o >>= 1) up = fmaxf(up, __shfl_xor(up, o));
      den = den == 0.f ? 0.f : den * __builtin_amdgcn_exp2f((top - up) * a.c);
      for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
      if (lane == 0) {
        stat[i] = up;
        stat[HEAVY_HEADS + i] = 1.f / den;
      }
    }
    __syncthreads();
    if (4 * at < move.held)
      low = heavy_grow<ST>(h, move, sh, at, w, static_cast<const float*>(h.logits + head0 * h.pitch), h.pitch, a.group, stat,
                           HEAVY_HEADS);
  }
  low = heavy_least<512>(low, red_low);
  if (threadIdx.x == 0) {
    if (low != HEAVY_NONE) atomicMin(&h.lowest[2 * static_cast<int64_t>(sh) + ((move.n + a.append) & 1)], low);
    if (range == 0) {
      heavy_positions(h, move, sh);
      h.counts[sh] = move.n + a.append;
    }
  }
}

// One token of every stream into the cache, without a query: a workgroup a key head.
template <int ST>
__global__ __launch_bounds__(256) void heavy_update_kernel(const HeavyArgs h) {
  const RingArgs& a = h.r;
  __shared__ unsigned long long red_low[4];
  const int sh = blockIdx.x, s = sh / a.kv, hk = sh - s * a.kv;
  HeavyPiece<ST> fresh{}, old{};
  fresh.load_new(a, s, hk);
  HeavyMove move = heavy_slots(h, true, h.counts[sh]);
  if (move.from >= 0) old.load(a, sh, move.from);
  heavy_goes(h, move, heavy_weight(h, sh, move.from), h.lowest[2 * static_cast<int64_t>(sh)],
             h.lowest[2 * static_cast<int64_t>(sh) + 1]);
  if (move.to >= 0) old.store(a, sh, move.to);
  fresh.store(a, sh, move.slot);
  float* row = h.weights + static_cast<int64_t>(sh) * h.pitch;
  unsigned long long low = HEAVY_NONE;
  for (int slot = h.ring + threadIdx.x; slot < move.held; slot += 256)
    low = heavy_min(low, heavy_key(heavy_base(move, slot, row[slot]), slot));
  low = heavy_least<256>(low, red_low);  // with a barrier: every thread has read the count and its weights
  if (threadIdx.x == 0) {
    if (move.to >= 0) row[move.to] = move.weight;
    if (move.from >= 0) row[move.from] = 0.f;
    row[move.slot] = 0.f;
    heavy_positions(h, move, sh);
    h.lowest[2 * static_cast<int64_t>(sh) + ((move.n + 1) & 1)] = low;
    h.counts[sh] = move.n + 1;
  }
}

struct HeavyFill {
  HeavyArgs h;           // r.k, r.v: [streams][kv][rows][d | dv]
  int rows;
  const int* take;       // [streams] or null: rows of a stream that are tokens; a stream with none keeps what it holds
  const float* given;    // [streams][kv][rows]: the rows' weights
  int* token;            // [streams][kv][pitch]: the row of every slot, or -1
};

__device__ __forceinline__ int heavy_take(const HeavyFill& f, int s) {
  const int t = f.take ? f.take[s] : f.rows;
  return t < 0 ? 0 : (t > f.rows ? f.rows : t);
}
// a weight as the cache takes it: NaN and -0 as 0
__device__ __forceinline__ float heavy_given(float w) { return w == w ? w + 0.f : 0.f; }

// Which rows stay, by a workgroup of 1024 threads a key head: the last `recent`, and of the others the `kept` of the
// largest weights, of equal ones the first.  Three passes over the weights find the smallest that stays, 11 bits of its
// order at a time (the highest first, among those that agree with it so far): the weights of a prompt lie within a few powers
// of two, so that bins of 8 bits, the sign and 7 of the exponent's, would all be added to in one place.  One more pass puts the
// rows that stay down in their order: put_row(slot, row or -1, weight) once for every slot.  Bound by its barriers.  The first
// 8192 weights are held in registers.  16 x 8 key heads of 8192 rows: 16 us (the last pass 1024 at a time: 20; 8 x 65536 79
// and 111).  first_of_head: the workgroup writes what a key head has one of.
template <typename Put>
__device__ __forceinline__ void heavy_select(const HeavyFill& f, int sh, int n, bool first_of_head, Put put_row) {
  const HeavyArgs& h = f.h;
  constexpr int HOLD = 8, BINS = 2048;
  __shared__ int bins[BINS], wave_sum[16], chosen[2], cells[16 * HOLD];
  __shared__ unsigned long long red_low[16];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const float* given = f.given + static_cast<int64_t>(sh) * f.rows;
  const int older = n > h.recent ? n - h.recent : 0;
  float hold[HOLD];
#pragma unroll
  for (int j = 0; j < HOLD; ++j) hold[j] = t + 1024 * j < older ? heavy_given(given[t + 1024 * j]) : 0.f;

  uint32_t least = 0u;  // the order of the smallest weight that stays
  int equal = 0x7fffffff;  // how many of those equal to it stay
  if (older > h.kept) {
    int want = h.kept;  // among those that agree so far
    for (int shift = 21; shift >= -1; shift -= 11) {
      const int low = shift < 0 ? 0 : shift, bits = shift < 0 ? 10 : 11;  // 11 + 11 + 10 bits
      const uint32_t mask = (1u << bits) - 1u;
      bins[t] = bins[t + 1024] = 0;
      __syncthreads();
      auto put = [&](float w) {
        const uint32_t u = heavy_order(w);
        if (low + bits == 32 || u >> (low + bits) == least >> (low + bits)) atomicAdd(&bins[(u >> low) & mask], 1);
      };
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        if (1024 * j < older) {
          if (t + 1024 * j < older) put(hold[j]);
        }
      }
      for (int i = t + 1024 * HOLD; i < older; i += 1024) put(heavy_given(given[i]));
      __syncthreads();
      // the highest bin with `want` at or above it: sums from above, two bins a thread
      const int first = BINS - 1 - 2 * t, part[2] = {bins[first], bins[first - 1]};
      int before = part[0] + part[1];
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(before, o);
        if (lane >= o) before += y;
      }
      if (lane == 63) wave_sum[wave] = before;
      __syncthreads();
      before -= part[0] + part[1];
      for (int j = 0; j < wave; ++j) before += wave_sum[j];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (before < want && before + part[j] >= want) {
          chosen[0] = first - j;
          chosen[1] = want - before;
        }
        before += part[j];
      }
      __syncthreads();
      least |= static_cast<uint32_t>(chosen[0]) << low;
      want = chosen[1];
      __syncthreads();
    }
    equal = want;
  }
  // The rows that stay, in their order, 8192 at a time: counts by 64 rows of those equal to the smallest, then of those that
  // stay, each summed up by one wave.
  unsigned long long low = HEAVY_NONE;
  int taken = 0, ties = 0;
  const unsigned long long below = (1ull << lane) - 1ull;
  auto sum_up = [&](int& total) {  // cells become what is before them, and total's old value with it
    __syncthreads();
    if (wave == 0) {
      int part[HOLD / 4], sum = 0;
#pragma unroll
      for (int j = 0; j < HOLD / 4; ++j) {
        part[j] = cells[HOLD / 4 * lane + j];
        sum += part[j];
      }
      int before = sum;
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(before, o);
        if (lane >= o) before += y;
      }
      if (lane == 63) chosen[0] = before;
      before -= sum;
#pragma unroll
      for (int j = 0; j < HOLD / 4; ++j) {
        cells[HOLD / 4 * lane + j] = total + before;
        before += part[j];
      }
    }
    __syncthreads();
    total += chosen[0];
  };
  for (int i0 = 0; i0 < older; i0 += 1024 * HOLD) {
    uint32_t stays = 0u;
    const int live = min(HOLD, (older - i0 + 1023) / 1024);  // of hold
    if (i0 > 0) {
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        const int i = i0 + 1024 * j + t;
        hold[j] = i < older ? heavy_given(given[i]) : 0.f;
      }
    }
    if (equal != 0x7fffffff) {
      uint32_t tie = 0u;
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        bool in = false;
        if (j < live) in = i0 + 1024 * j + t < older && heavy_order(hold[j]) == least;
        const unsigned long long ballot = __ballot(in);
        if (lane == 0) cells[16 * j + wave] = __popcll(ballot);
        tie |= static_cast<uint32_t>(in) << j;
      }
      sum_up(ties);
#pragma unroll
      for (int j = 0; j < HOLD; ++j) {
        if (j < live) {
          const bool in = tie >> j & 1u;
          const int rank = cells[16 * j + wave] + __popcll(__ballot(in) & below);
          const bool stay = i0 + 1024 * j + t < older && (heavy_order(hold[j]) > least || (in && rank < equal));
          stays |= static_cast<uint32_t>(stay) << j;
        }
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int j = 0; j < HOLD; ++j) stays |= static_cast<uint32_t>(i0 + 1024 * j + t < older) << j;
    }
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      const unsigned long long ballot = __ballot(stays >> j & 1u);
      if (lane == 0) cells[16 * j + wave] = __popcll(ballot);
    }
    sum_up(taken);
#pragma unroll
    for (int j = 0; j < HOLD; ++j) {
      if (j < live) {
        const bool stay = stays >> j & 1u;
        const int slot = h.ring + cells[16 * j + wave] + __popcll(__ballot(stay) & below);
        if (stay) {
          put_row(slot, i0 + 1024 * j + t, hold[j]);
          low = heavy_min(low, heavy_key(hold[j], slot));
        }
      }
    }
    __syncthreads();
  }
  for (int slot = h.ring + taken + t; slot < h.pitch; slot += 1024) put_row(slot, -1, 0.f);
  for (int slot = t; slot < h.ring; slot += 1024) {
    const int p = n - 1 - static_cast<int>((static_cast<int64_t>(n) - 1 - slot + h.ring) % h.ring);
    const bool in = p >= 0 && p >= older;
    put_row(slot, in ? p : -1, in ? heavy_given(given[p]) : 0.f);
  }
  low = heavy_least<1024>(low, red_low);
  if (t == 0 && first_of_head) {
    h.lowest[2 * static_cast<int64_t>(sh) + (n & 1)] = low;
    h.counts[sh] = n;
  }
}

__global__ __launch_bounds__(1024) static void heavy_select_kernel(const HeavyFill f) {
  const int sh = blockIdx.x, n = heavy_take(f, sh / f.h.r.kv);
  if (n == 0) return;
  const int64_t at = static_cast<int64_t>(sh) * f.h.pitch;
  heavy_select(f, sh, n, true, [&](int slot, int row, float weight) {
    f.token[at + slot] = row;
    f.h.weights[at + slot] = weight;
    f.h.positions[at + slot] = row;
  });
}

// The rows that stay into their slots: a workgroup a tile.
template <int ST>
__global__ __launch_bounds__(256) void heavy_fill_kernel(const HeavyFill f) {
  const RingArgs& a = f.h.r;
  __shared__ int token[32];
  int sh, tile;
  if (!ring_place(a, sh, tile)) return;
  const int s = sh / a.kv, hk = sh - s * a.kv;
  if (heavy_take(f, s) == 0) return;
  if (threadIdx.x < 32) token[threadIdx.x] = f.token[static_cast<int64_t>(sh) * f.h.pitch + 32 * tile + threadIdx.x];
  if (!__syncthreads_or(threadIdx.x < 32 && token[threadIdx.x] >= 0)) return;
  ring_fill<ST, ST>(a, s, hk, tile, token);
}

// Both in one launch, for few tiles: the workgroup of each selects for itself and keeps what falls into its tile.
template <int ST>
__global__ __launch_bounds__(1024) void heavy_start_kernel(const HeavyFill f) {
  const RingArgs& a = f.h.r;
  __shared__ int token[32];
  const int sh = blockIdx.x / a.tiles, tile = blockIdx.x - sh * a.tiles, s = sh / a.kv;
  const int n = heavy_take(f, s);
  if (n == 0) return;
  const int64_t at = static_cast<int64_t>(sh) * f.h.pitch;
  heavy_select(f, sh, n, tile == 0, [&](int slot, int row, float weight) {
    if (slot >> 5 != tile) return;
    token[slot & 31] = row;
    f.h.weights[at + slot] = weight;
    f.h.positions[at + slot] = row;
  });
  __syncthreads();
  if (!__syncthreads_or(threadIdx.x < 32 && token[threadIdx.x & 31] >= 0)) return;
  ring_fill<ST, ST, 1024>(a, s, sh - s * a.kv, tile, token);
}

// The slots as they are: rows, positions and weights.
struct HeavyItems {
  void *keys, *values;   // [streams][kv][slots][d | dv]
  int64_t* positions;    // [streams][kv][slots]
  float* weights;
};
template <int ST>
__global__ __launch_bounds__(256) void heavy_items_kernel(const HeavyArgs h, const HeavyItems to) {
  int sh, tile;
  if (!ring_place(h.r, sh, tile)) return;
  const int64_t at = static_cast<int64_t>(sh) * h.pitch + 32 * tile;
  __shared__ int there[32];
  if (threadIdx.x < 32) {
    const int64_t p = h.positions[at + threadIdx.x];
    there[threadIdx.x] = p >= 0;
    if (32 * tile + static_cast<int>(threadIdx.x) < h.r.slots) {
      const int64_t slot = static_cast<int64_t>(sh) * h.r.slots + 32 * tile + threadIdx.x;
      to.positions[slot] = p;
      to.weights[slot] = h.weights[at + threadIdx.x];
    }
  }
  const bool some = __syncthreads_or(threadIdx.x < 32 && there[threadIdx.x]);
  ring_rows_out<ST, ST>(h.r, sh, tile, some, [&](int r) { return there[r] != 0; }, to.keys, to.values);
}

}  // namespace sta
