// Attention of a batch's new rows over a prefix that its sequences share and over each sequence's own tokens, and the
// weights that own tokens receive.
//
// Sequence b has lengths[b] own tokens, the last counts[b] of which have their queries in rows i < counts[b] of q.  Row i
// sees its set's prefix whole and the own tokens j <= lim(i) = lengths[b] - counts[b] + i:
//   x_j = s q_i.k_j,  L_i = log(sum_prefix exp(x_j) + sum_{own j <= lim(i)} exp(x_j)),  o_i = sum_j exp(x_j - L_i) v_j
//   received weights: W_j = sum over the rows i with lim(i) >= j, and the key head's query heads, of exp(x_ij - L_i)
// The sequences of a set (batch / sets neighbours) read one prefix.
//
// The rows of a "unit" of `span` sequences and one key head lie in the order (sequence, row, query head of the group): the
// query heads of a key head, and with span > 1 the sequences of a set, are rows of one product with the keys that
// they share.  A workgroup takes 128 (shared tiles: 32) rows and a share of the unit's key tiles; its walk is the one of
// window_forward_kernel, whose tiles, layouts and second pass for results that are not finite it uses.  Weights of 16-bit rows
// are rounded to their type for the value product (half a step each; sums of weights and received weights are not): outputs
// are off by 0.0023 of their deviation in bf16, 0.0017 with fp32 weights, which is the output's own rounding; fp16 2.9e-4 and
// 2.1e-4.  A second plane of the weights would make three products of two, and products are what bounds large calls.
#pragma once
#include "window_attn.hip"

namespace sta {

struct PrefixArgs {
  Rows q, k, v, pk, pv;  // q [batch][heads][n][d], own k, v [batch][kv][m][d | dv], prefix pk, pv [sets][kv][p][d | dv]
  int batch, heads, kv, group, sets, per_set;
  int n, m, p, d, dv;
  float scale, c;        // c = |scale| log2(e)
  const int *lengths, *counts, *prefix_lengths;  // [batch], [batch], [sets], or null
  void* out;             // [batch][heads][n][dv]
  float* lse;            // [batch][heads][n]: log2 of the row's sum of weights, or null
  float* part;           // [batch][heads][n][parts][pitch]: sums, on 16 bytes
  float* stat;           // [batch][heads][n][parts][2]: maximum and sum of weights
  int parts, pitch;      // parts 0: rows are finished by one workgroup; pitch: dv in whole units of 4
};

// One launch: which rows lie together, what they see, how their keys are dealt out.
struct PrefixWalk {
  int span;              // sequences of a unit
  int tiles, nsplit;     // row tiles of a unit, workgroups a tile
  int first;             // its first partial
  int prefix, own;       // segments
};

__device__ __forceinline__ int prefix_clamp(int x, int most) { return x < 0 ? 0 : (x > most ? most : x); }
__device__ __forceinline__ int prefix_length(const PrefixArgs& a, int b) {
  return a.lengths ? prefix_clamp(a.lengths[b], a.m) : a.m;
}
// rows of a sequence that are tokens
__device__ __forceinline__ int prefix_count(const PrefixArgs& a, int b, int length) {
  const int most = length < a.n ? length : a.n;
  return a.counts ? prefix_clamp(a.counts[b], most) : most;
}
__device__ __forceinline__ int prefix_rows(const PrefixArgs& a, int set) {
  return a.prefix_lengths ? prefix_clamp(a.prefix_lengths[set], a.p) : a.p;
}

// a partial of a row without weights: a maximum of -inf
__device__ __forceinline__ float prefix_top(float m, float l) { return l == 0.f ? -__builtin_inff() : m; }

// log2 of a row's sum of weights.  The sum's power of two goes into the whole number, so that the logarithm is taken near 1
// and rounds at its size there: of a sum of 2^13 it is off by up to 1e-6, much the same for neighbouring rows, so that it
// stays in the sums over them (received weights of 16384 rows: errors of 2.9e-7, so 5e-8).
template <int IN>
__device__ __forceinline__ float prefix_lse(float top, float den, float c) {
  const int e = __builtin_amdgcn_frexp_expf(den);
  return fmaf(top, c, static_cast<float>(e) - win_weight_lift<IN>()) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(den));
}

template <int P, int IN, bool SHARE, bool VALUES, bool CAREFUL>
__device__ __forceinline__ int prefix_pass(const PrefixArgs& a, const PrefixWalk& w, int id, uint4* key_lds, uint4* value_lds,
                                           int again) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), BK = win_keys<IN, SHARE>(), NSUB = BK / 32,
                MT = P / 32, STEP = SHARE ? 4 : 1;
  // the tiles of a unit, then the units of a key head next to each other: they read the same keys
  const int tile = w.tiles - 1 - id % w.tiles;
  id /= w.tiles;
  const int split = id % w.nsplit;
  id /= w.nsplit;
  const int units = a.batch / w.span, hk = id / units, b0 = (id - hk * units) * w.span;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  uint4 *const ks = key_lds + (SHARE ? wave * 2 * BK * CH : 0), *const vs = value_lds + (SHARE ? wave * 2 * BK * CH : 0);
  const int r0 = tile * win_rows<SHARE>(), w0 = r0 + (SHARE ? 0 : 32 * wave);
  const int per = a.n * a.group;  // rows of a sequence

  // a unit's row: its sequence, row and head; whether it is one; the last own token that it sees
  struct Place {
    int64_t at;  // in [batch][heads][n]
    int b, h, i, lim;
    bool in, live;
  };
  auto place = [&](int r) {
    Place x;
    x.in = r < w.span * per;
    const int y = x.in ? r : 0, bl = y / per, z = y - bl * per;
    x.b = b0 + bl;
    x.i = z / a.group;
    x.h = hk * a.group + z - x.i * a.group;
    x.at = (static_cast<int64_t>(x.b) * a.heads + x.h) * a.n + x.i;
    const int length = prefix_length(a, x.b), count = prefix_count(a, x.b, length);
    x.live = x.in && x.i < count;
    x.lim = length - count + x.i;
    return x;
  };
  const Place mine = place(w0 + (lane & 31));

  constexpr bool AHEAD = !CAREFUL && win_ahead<P, IN, SHARE>();
  int bad = 0;
  floatx16 acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[mt][i] = 0.f;
  // finite: see window_forward_pass
  float m = CAREFUL ? -3.4e38f : -1e30f, limit = m, l = 0.f;
  const float room = win_weight_room<IN>() / a.c;

  // key tiles of the prefix, then of the own tokens that the tile's rows see (own: span 1)
  const int rows_p = w.prefix ? prefix_rows(a, b0 / a.per_set) : 0;
  int own_end = 0, base = 0, count = a.n;
  if (w.own) {
    const int length = prefix_length(a, b0);
    count = prefix_count(a, b0, length);
    base = length - count;
    const int last = (r0 + win_rows<SHARE>() - 1) / a.group;
    own_end = r0 / a.group < count ? base + (last < count ? last + 1 : count) : 0;
  }
  // a wave without a live row (a padded batch has many) leaves its products out; four that share their rows, their loads too
  const bool awake = __any(mine.live), any = (!SHARE || awake) && (w.own ? own_end > 0 : r0 < w.span * per);
  const int tiles_p = any ? (rows_p + BK - 1) / BK : 0, all_tiles = any ? tiles_p + (own_end + BK - 1) / BK : 0;
  // Every nsplit-th tile: workgroups that walk in step are at neighbouring rows, and not at round distances, which would
  // ask the same memory channels at a time.
  const int own_first = (split + w.nsplit - tiles_p % w.nsplit) % w.nsplit;  // of the own tokens' tiles

  if (split < all_tiles) {
    WinFrag<IN> qf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* qrow = rows_at<ES>(a.q, mine.b, mine.h, mine.i);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      qf[s] = win_load_row<IN>(qrow, s, hh, a.d, flip);
      win_keep<IN>(qf[s], mine.live);
    }
#pragma unroll 1
    for (int seg = 0; seg < 2; ++seg) {
      const Rows kr = seg ? a.k : a.pk, vr = seg ? a.v : a.pv;
      const int rb = seg ? b0 : b0 / a.per_set, end = seg ? own_end : rows_p;
      const int lo = seg ? own_first : split, hi = seg ? all_tiles - tiles_p : tiles_p, step = STEP * w.nsplit;
      if (lo >= hi) continue;
      // the last key that a lane's row, the wave's first and its last one see
      const int lim = seg ? mine.lim : rows_p - 1;
      const int lim_lo = seg ? base + w0 / a.group : rows_p - 1;
      const int lim_hi = seg ? base + min((w0 + 31) / a.group, count - 1) : rows_p - 1;
      WinStage<P, IN, BK, SHARE ? 64 : 256> kst, vst;
      kst.init(kr, a.d);
      if constexpr (VALUES) vst.init(vr, a.dv);
      auto load = [&](int it) {
        const int row = it * BK;
        kst.load(rows_at<ES>(kr, rb, hk, row), end - row);
        if constexpr (VALUES) vst.load(rows_at<ES>(vr, rb, hk, row), end - row);
      };
      const int start = lo + (SHARE ? wave * w.nsplit : 0);
      if (AHEAD && start < hi) load(start);
      for (int it = start; it < hi; it += step) {
        if (!AHEAD) load(it);
        win_sync<SHARE>();
        const int key0 = it * BK;
        kst.put(ks, end - key0);
        if constexpr (VALUES) vst.put(vs, end - key0);
        win_sync<SHARE>();
        if (AHEAD && it + step < hi) load(it + step);
        if (key0 > lim_hi || !awake) continue;
        const bool all = key0 + BK - 1 <= lim_lo;
        floatx16 x[NSUB];
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) x[sub][i] = 0.f;
#pragma unroll
        for (int s = 0; s < P / 16; ++s)
#pragma unroll
          for (int sub = 0; sub < NSUB; ++sub)
            win_mma<IN>(x[sub], win_read_row<P, IN>(ks, 32 * sub + (lane & 31), s, hh), qf[s]);
        uint32_t pairs[NSUB] = {};
        if (!all) {
          const int ahead = lim - key0 - 4 * hh;
#pragma unroll
          for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const bool seen = 32 * sub + 8 * (i >> 2) + (i & 3) <= ahead;
              x[sub][i] = seen ? x[sub][i] : -__builtin_inff();
              if constexpr (CAREFUL) pairs[sub] |= static_cast<uint32_t>(seen) << i;
            }
        }
        float top = m;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, x[sub][i]);
        // the maximum moves, for both lanes of a row at once, when a weight would exceed 2^room
        if (__any(top > limit)) {
          top = fmaxf(top, __shfl_xor(top, 32));
          const float shrink = __builtin_amdgcn_exp2f((m - top) * a.c);
          l *= shrink;
          if constexpr (VALUES) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[mt][i] *= shrink;
          }
          m = top;
          limit = m + room;
        }
        const float mc = m * a.c - win_weight_lift<IN>();
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            // see window_forward_pass
            if constexpr (CAREFUL)
              x[sub][i] = __builtin_amdgcn_exp2f(fmaf(x[sub][i] - m, a.c, win_weight_lift<IN>()));
            else
              x[sub][i] = __builtin_amdgcn_exp2f(fmaf(x[sub][i], a.c, -mc));
          }
        // a tile's weights first: long rows' sums lose less
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub) {
          float sum = x[sub][0];
#pragma unroll
          for (int i = 1; i < 16; ++i) sum += x[sub][i];
          l += sum;
        }
        if constexpr (VALUES) {
          if (CAREFUL && !all) {
#pragma unroll
            for (int sub = 0; sub < NSUB; ++sub) win_add_seen<P, IN>(acc, x[sub], pairs[sub], vs, 32 * sub, lane);
            continue;
          }
#pragma unroll
          for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const WinFrag<IN> p = win_operand<IN>(x[sub], t);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
                win_mma<IN>(acc[mt], win_read_columns<P, IN>(vs, 32 * sub + 16 * t, mt, lane), p);
            }
        }
      }
    }
    l += __shfl_xor(l, 32);
  }

  // four sums of a row at column col (below dv), its maximum and sum of weights
  auto store4 = [&](const Place& x, int col, float inv, const floatx4& y) {
    if (a.parts)
      *reinterpret_cast<floatx4*>(a.part + (x.at * a.parts + w.first + split) * a.pitch + col) = y;
    else
      win_store4<IN>(a.out, x.at * a.dv, col, a.dv, x.live ? y[0] * inv : 0.f, x.live ? y[1] * inv : 0.f,
                     x.live ? y[2] * inv : 0.f, x.live ? y[3] * inv : 0.f);
  };
  auto store_sums = [&](const Place& x, float top, float den) {
    if (a.parts) {
      *reinterpret_cast<floatx2*>(a.stat + (x.at * a.parts + w.first + split) * 2) = floatx2{prefix_top(top, den), den};
    } else if (a.lse) {
      a.lse[x.at] = x.live ? prefix_lse<IN>(top, den, a.c) : 0.f;
    }
  };
  // a sum of weights that is not finite, or none though the row sees a key of the workgroup's share
  auto wrong = [&](const Place& x, float den) {
    const bool sees = split < tiles_p || (split < all_tiles && own_first * BK <= x.lim);
    return !win_finite(den) || (sees && !(den > 0.f));
  };

  if constexpr (SHARE) {
    float *red = reinterpret_cast<float*>(key_lds), *red_m = red + win_join_floats<P>(), *red_l = red_m + 4 * 32;
    __syncthreads();
    if constexpr (VALUES) win_join_put<P>(red, acc, wave, lane);
    if (hh == 0) {
      red_m[32 * wave + lane] = prefix_top(m, l);
      red_l[32 * wave + lane] = l;
    }
    __syncthreads();
    const int r = threadIdx.x / 8;
    const Place x = place(r0 + r);
    float top = red_m[r], den = 0.f, f[4];
#pragma unroll
    for (int i = 1; i < 4; ++i) top = fmaxf(top, red_m[32 * i + r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float li = red_l[32 * i + r];
      f[i] = li == 0.f ? 0.f : __builtin_amdgcn_exp2f((red_m[32 * i + r] - top) * a.c);
      den = fmaf(f[i], li, den);
    }
    bad = wrong(x, den);
    if (CAREFUL && !a.parts && !(den > 0.f)) den = __builtin_nanf("");  // no logit above -inf
    const float inv = 1.f / den;
    floatx4 o[MT];
    if constexpr (VALUES) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        o[j] = win_join_get<P>(red, 32 * j + 4 * (threadIdx.x & 7), f);
        bad |= win_bad4(o[j]);
      }
    }
    bad = x.live ? bad : 0;
#pragma unroll
    for (int y = 1; y < 8; y <<= 1) bad |= __shfl_xor(bad, y);
    if (x.in && (CAREFUL ? again : !bad)) {
      if constexpr (VALUES) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const int col = 32 * j + 4 * (threadIdx.x & 7);
          if (col < a.dv) store4(x, col, inv, o[j]);
        }
      }
      if ((threadIdx.x & 7) == 0) store_sums(x, top, den);
    }
    return bad;
  }

  float inv = 0.f;
  if (mine.live) {
    bad = wrong(mine, l);
    if (CAREFUL && !a.parts && !(l > 0.f)) l = __builtin_nanf("");
    inv = 1.f / l;
    if constexpr (VALUES) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad |= !win_finite(acc[mt][i]);
    }
  }
  bad |= __shfl_xor(bad, 32);
  const bool store = mine.in && (CAREFUL ? again : !bad);
  if (VALUES && a.parts) {
    // Partials by whole rows, through LDS: stored from the lanes that have them, 16 bytes here and there, they cost as much
    // as eight tiles of keys (64 x 32 heads over 32768 rows, 32 shares: 77 us, so 56)
    float* red = reinterpret_cast<float*>(key_lds);
    __syncthreads();
    win_join_put<P>(red, acc, wave, lane);
    win_sync<true>();
    constexpr int UNITS = P / 4;
#pragma unroll 4
    for (int i = 0; i < UNITS / 2; ++i) {
      const int unit = 64 * i + lane, r = unit / UNITS, col = 4 * (unit % UNITS);
      const int lo = __shfl(static_cast<int>(mine.at), r), hi = __shfl(static_cast<int>(mine.at >> 32), r);
      const bool row = __shfl(static_cast<int>(store), r);
      Place x = mine;
      x.at = static_cast<int64_t>(hi) << 32 | static_cast<uint32_t>(lo);
      if (row && col < a.dv) store4(x, col, 1.f, *reinterpret_cast<floatx4*>(&red[(wave * 32 + r) * (P + 4) + col]));
    }
  } else if (VALUES && store) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * mt + 8 * r + 4 * hh;
        if (col < a.dv)
          store4(mine, col, inv, floatx4{acc[mt][4 * r], acc[mt][4 * r + 1], acc[mt][4 * r + 2], acc[mt][4 * r + 3]});
      }
  }
  if (store && hh == 0) store_sums(mine, m, l);
  return bad;
}

// A wave's 32 rows over a tile of staged keys: the running maximum and sum of weights, and the value sums.
template <int P, int IN, int NSUB>
struct PrefixRows {
  floatx16 acc[P / 32];
  float m, limit, l, room;

  // low: where no logit is below it
  __device__ __forceinline__ void init(float low, float c) {
#pragma unroll
    for (int mt = 0; mt < P / 32; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mt][i] = 0.f;
    m = limit = low;
    l = 0.f;
    room = win_weight_room<IN>() / c;
  }
  __device__ __forceinline__ static void logits(floatx16 (&x)[NSUB], const uint4* ks, const WinFrag<IN> (&qf)[P / 16], int lane) {
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[sub][i] = 0.f;
#pragma unroll
    for (int s = 0; s < P / 16; ++s)
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub)
        win_mma<IN>(x[sub], win_read_row<P, IN>(ks, 32 * sub + (lane & 31), s, lane >> 5), qf[s]);
  }
  // logits to weights; all: every row sees every key, else the lane's row sees key k up to `ahead`
  template <bool VALUES>
  __device__ __forceinline__ void weights(floatx16 (&x)[NSUB], bool all, int ahead, float c) {
    if (!all) {
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool seen = 32 * sub + 8 * (i >> 2) + (i & 3) <= ahead;
          x[sub][i] = seen ? x[sub][i] : -__builtin_inff();
        }
    }
    float top = m;
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, x[sub][i]);
    // the maximum moves, for both lanes of a row at once, when a weight would exceed 2^room
    if (__any(top > limit)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float shrink = __builtin_amdgcn_exp2f((m - top) * c);
      l *= shrink;
      if constexpr (VALUES) {
#pragma unroll
        for (int mt = 0; mt < P / 32; ++mt)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[mt][i] *= shrink;
      }
      m = top;
      limit = m + room;
    }
    const float mc = m * c - win_weight_lift<IN>();
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[sub][i] = __builtin_amdgcn_exp2f(fmaf(x[sub][i], c, -mc));
      }
    // a tile's weights first: long rows' sums lose less
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub) {
      float sum = x[sub][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) sum += x[sub][i];
      l += sum;
    }
  }
  __device__ __forceinline__ void values(const floatx16 (&x)[NSUB], const uint4* vs, int lane) {
#pragma unroll
    for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const WinFrag<IN> p = win_operand<IN>(x[sub], t);
#pragma unroll
        for (int mt = 0; mt < P / 32; ++mt)
          win_mma<IN>(acc[mt], win_read_columns<P, IN>(vs, 32 * sub + 16 * t, mt, lane), p);
      }
  }
};

// The first pass for 16-bit heads of whole 16 bytes, wide tiles: that of prefix_pass with tiles that go from memory to LDS
// directly, keys and values of even and of odd tiles in buffers of their own, so that one barrier a tile is enough and a
// tile's value products run into the next one's logits.  The buffers are restrict arguments: the compiler then sees that
// reads of one need not wait for loads to another.  32 x 512 rows of 8 sequences behind 16384, 128 wide, 1.29 -> 1.12 ms
// (1000 TFLOP/s; a large matrix product 1200), 64 wide 0.38 -> 0.35 ms; 32 heads' statistics of 16384 rows 1.25 -> 1.06 ms.
// Widths between (their tiles padded to P): 8 x 32 heads of 512 rows behind 4096, 80 and 72 wide, 279 -> 249 us, 112 wide 362 -> 310.
typedef const __attribute__((address_space(1))) void* stream_global;
typedef __attribute__((address_space(3))) void* stream_lds;

// Where a lane's units of a tile lie in memory, from its first row: unit (NJ wave + j) 64 + lane of the tile's order in LDS
template <int P>
struct StreamTile {
  static constexpr int CH = P / 8, NJ = 64 * CH / 256;
  int pitch, at[NJ];

  __device__ __forceinline__ static int unit(int j) { return static_cast<int>(NJ * (threadIdx.x >> 6) + j) * 64 + (threadIdx.x & 63); }
  // units behind the rows' width are read as the last one: they meet zeros, or give columns that are not stored
  __device__ __forceinline__ void init(int64_t row_elements, int width) {
    pitch = static_cast<int>(row_elements) * 2;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int u = unit(j), r = u / CH;
      at[j] = r * pitch + min((u % CH) ^ win_swizzle<CH>(r), width / 8 - 1) * 16;
    }
  }
  // rows behind the last are read as the last one: their logits are hidden, their weights 0
  __device__ __forceinline__ void load(const char* row, int left, uint4* lds) const {
    const int first = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * NJ * 64;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      uint32_t off = at[j];
      if (left < 64) off -= max(0, unit(j) / CH - left + 1) * pitch;
      __builtin_amdgcn_global_load_lds((stream_global)(row + off), (stream_lds)(lds + first + 64 * j), 16, 0, 0);
    }
  }
};

// a barrier behind the wave's loads to LDS and its LDS reads
__device__ __forceinline__ void stream_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0), lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int P, bool VALUES>
__host__ __device__ constexpr int prefix_stream_bytes() { return (VALUES ? 4 : 2) * 64 * P * 2; }

template <int P, int IN, bool VALUES>
__device__ __forceinline__ int prefix_stream_pass(const PrefixArgs& a, const PrefixWalk& w, int id, float* red,
                                                  uint4* __restrict__ ks0, uint4* __restrict__ ks1,
                                                  uint4* __restrict__ vs0, uint4* __restrict__ vs1) {
  constexpr int MT = P / 32, BK = 64, NSUB = 2;
  const int tile = w.tiles - 1 - id % w.tiles;
  id /= w.tiles;
  const int split = id % w.nsplit;
  id /= w.nsplit;
  const int units = a.batch / w.span, hk = id / units, b0 = (id - hk * units) * w.span;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int r0 = tile * WIN_ROWS, w0 = r0 + 32 * wave, per = a.n * a.group;

  // the lane's row
  const int row = w0 + (lane & 31);
  const bool in = row < w.span * per;
  const int bl = (in ? row : 0) / per, z = (in ? row : 0) - bl * per, b = b0 + bl, i = z / a.group, h = hk * a.group + z - i * a.group;
  const int64_t at = (static_cast<int64_t>(b) * a.heads + h) * a.n + i;
  const int my_length = prefix_length(a, b), my_count = prefix_count(a, b, my_length);
  const bool live = in && i < my_count;
  const int my_lim = my_length - my_count + i;

  const int set = b0 / a.per_set, rows_p = w.prefix ? prefix_rows(a, set) : 0;
  int own_end = 0, base = 0, count = a.n;
  if (w.own) {
    const int length = prefix_length(a, b0);
    count = prefix_count(a, b0, length);
    base = length - count;
    const int last = (r0 + WIN_ROWS - 1) / a.group;
    own_end = r0 / a.group < count ? base + (last < count ? last + 1 : count) : 0;
  }
  const bool awake = __any(live), any = w.own ? own_end > 0 : r0 < w.span * per;  // awake: see prefix_pass
  const int tiles_p = any ? (rows_p + BK - 1) / BK : 0, all_tiles = tiles_p + (own_end + BK - 1) / BK;
  const int own_first = (split + w.nsplit - tiles_p % w.nsplit) % w.nsplit;

  PrefixRows<P, IN, NSUB> sums;
  sums.init(-1e30f, a.c);
  if (split < all_tiles) {
    WinFrag<IN> qf[P / 16];
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    const char* qrow = rows_at<2>(a.q, b, h, i);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      qf[s] = win_load_row<IN>(qrow, s, hh, a.d, flip);
      win_keep<IN>(qf[s], live);
    }
#pragma unroll 1
    for (int seg = 0; seg < 2; ++seg) {
      const Rows kr = seg ? a.k : a.pk, vr = seg ? a.v : a.pv;
      const int rb = seg ? b0 : set, end = seg ? own_end : rows_p;
      const int lo = seg ? own_first : split, hi = seg ? all_tiles - tiles_p : tiles_p, step = w.nsplit;
      if (lo >= hi) continue;
      const int lim = seg ? my_lim : rows_p - 1;
      const int lim_lo = seg ? base + w0 / a.group : rows_p - 1;
      const int lim_hi = seg ? base + min((w0 + 31) / a.group, count - 1) : rows_p - 1;
      StreamTile<P> kt, vt;
      kt.init(kr.sn, a.d);
      if constexpr (VALUES) vt.init(vr.sn, a.dv);
      const char *const kp = rows_at<2>(kr, rb, hk, 0), *const vp = VALUES ? rows_at<2>(vr, rb, hk, 0) : nullptr;
      // nothing behind the last tile
      auto keys = [&](int it, uint4* to) {
        if (it < hi) kt.load(kp + static_cast<int64_t>(it) * BK * kt.pitch, end - it * BK, to);
      };
      auto values = [&](int it, uint4* to) {
        if constexpr (VALUES) {
          if (it < hi) vt.load(vp + static_cast<int64_t>(it) * BK * vt.pitch, end - it * BK, to);
        }
      };
      // a tile, from keys and values that are there when it begins and when its weights are taken
      auto turn = [&](int it, uint4* ks, const uint4* vs, uint4* next) {
        const int key0 = it * BK, active = key0 <= lim_hi && awake;
        floatx16 x[NSUB];
        if (active) {
          sums.logits(x, ks, qf, lane);
          sums.template weights<VALUES>(x, key0 + BK - 1 <= lim_lo, lim - key0 - 4 * hh, a.c);
        }
        // these keys and the values before are done with; the next keys and these values are there
        stream_barrier();
        keys(it + 2 * step, ks);
        values(it + step, next);
        if (VALUES && active) sums.values(x, vs, lane);
      };
      keys(lo, ks0);
      keys(lo + step, ks1);
      values(lo, vs0);
      stream_barrier();
#pragma unroll 1
      for (int it = lo; it < hi; it += 2 * step) {
        turn(it, ks0, vs0, vs1);
        if (it + step < hi) turn(it + step, ks1, vs1, vs0);
      }
      stream_barrier();
    }
    sums.l += __shfl_xor(sums.l, 32);
  }

  int bad = 0;
  if (live) {
    const bool sees = split < tiles_p || (split < all_tiles && own_first * BK <= my_lim);
    bad = !win_finite(sums.l) || (sees && !(sums.l > 0.f));
    if constexpr (VALUES) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 16; ++e) bad |= !win_finite(sums.acc[mt][e]);
    }
  }
  bad |= __shfl_xor(bad, 32);
  const bool store = in && !bad;
  if (a.parts) {
    const int64_t part = at * a.parts + w.first + split;
    if constexpr (VALUES) {  // by whole rows, see prefix_pass
      __syncthreads();
      win_join_put<P>(red, sums.acc, wave, lane);
      win_sync<true>();
      constexpr int UNITS = P / 4;
#pragma unroll 4
      for (int u = 0; u < UNITS / 2; ++u) {
        const int unit = 64 * u + lane, r = unit / UNITS, col = 4 * (unit % UNITS);
        const int lo = __shfl(static_cast<int>(part), r), hi = __shfl(static_cast<int>(part >> 32), r);
        const int64_t to = static_cast<int64_t>(hi) << 32 | static_cast<uint32_t>(lo);
        if (__shfl(static_cast<int>(store), r) && col < a.dv)
          *reinterpret_cast<floatx4*>(a.part + to * a.pitch + col) = *reinterpret_cast<floatx4*>(&red[(wave * 32 + r) * (P + 4) + col]);
      }
    }
    if (store && hh == 0)
      *reinterpret_cast<floatx2*>(a.stat + 2 * part) = floatx2{prefix_top(sums.m, sums.l), sums.l};
  } else if (store) {
    const float inv = 1.f / sums.l;
    if constexpr (VALUES) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = 32 * mt + 8 * r + 4 * hh;
          if (col < a.dv)
            win_store4<IN>(a.out, at * a.dv, col, a.dv, live ? sums.acc[mt][4 * r] * inv : 0.f,
                           live ? sums.acc[mt][4 * r + 1] * inv : 0.f, live ? sums.acc[mt][4 * r + 2] * inv : 0.f,
                           live ? sums.acc[mt][4 * r + 3] * inv : 0.f);
        }
    }
    if (a.lse && hh == 0) a.lse[at] = live ? prefix_lse<IN>(sums.m, sums.l, a.c) : 0.f;
  }
  return bad;
}

// both passes over a walk, see win_passes
template <int P, int IN, bool SHARE, bool VALUES, bool STREAM>
__device__ __forceinline__ void prefix_passes(const PrefixArgs& a, const PrefixWalk& w, int id, uint4* lds) {
  constexpr int VALUE_UNITS = win_keys<IN, SHARE>() * win_chunks<IN == F32 ? 4 : 2>(P);
  win_passes([&](auto second, int again) {
    constexpr bool CAREFUL = decltype(second)::value;
    if constexpr (STREAM && !CAREFUL) {
      constexpr int UNITS = 64 * P / 8;
      return prefix_stream_pass<P, IN, VALUES>(a, w, id, reinterpret_cast<float*>(lds), lds, lds + UNITS, lds + 2 * UNITS,
                                               lds + 3 * UNITS);
    } else {
      return prefix_pass<P, IN, SHARE, VALUES, CAREFUL>(a, w, id, lds, lds + VALUE_UNITS, again);
    }
  });
}
// waves a SIMD
template <int P, int IN, bool SHARE, bool VALUES, bool STREAM>
__host__ __device__ constexpr int prefix_waves() {
  return STREAM ? (VALUES ? (P > 64 ? 2 : 3) : 4) : win_row_waves<P, IN, SHARE>();
}

template <int P, int IN, bool SHARE, bool VALUES, bool STREAM>
__global__ __launch_bounds__(256, (prefix_waves<P, IN, SHARE, VALUES, STREAM>())) void prefix_attention_kernel(
    const PrefixArgs a, const PrefixWalk w) {
  extern __shared__ uint4 win_lds[];
  prefix_passes<P, IN, SHARE, VALUES, STREAM>(a, w, xcd_remap(blockIdx.x, gridDim.x), win_lds);
}

// Both walks of a batch of few rows in one launch: that over the prefix is bound by products and by latency, that over the
// own tokens by memory.  64 x 32 heads, 128 wide, 32768 shared and up to 1024 own rows: 74 us, that over the prefix by itself
// 63; the prefix's workgroups first (with the two in turn 98 us, 78 then).
template <int P, int IN, bool SHARE_A, bool SHARE_B, bool STREAM>
__global__ __launch_bounds__(256, (prefix_waves<P, IN, SHARE_B, true, false>() < prefix_waves<P, IN, SHARE_A, true, STREAM>()
                                       ? prefix_waves<P, IN, SHARE_B, true, false>()
                                       : prefix_waves<P, IN, SHARE_A, true, STREAM>())) void
prefix_walks_kernel(const PrefixArgs a, const PrefixWalk wa, const PrefixWalk wb, int grid_a, int grid_b) {
  extern __shared__ uint4 win_lds[];
  // each walk's neighbours on one XCD, the first walk's workgroups before the second's
  const int xcds = grid_a % 8 == 0 && grid_b % 8 == 0 ? 8 : 1, xcd = blockIdx.x % xcds, slot = blockIdx.x / xcds;
  const int ga = grid_a / xcds, gb = grid_b / xcds;
  if (slot < ga)
    prefix_passes<P, IN, SHARE_A, true, STREAM>(a, wa, xcd * ga + slot, win_lds);
  else
    prefix_passes<P, IN, SHARE_B, true, false>(a, wb, xcd * gb + slot - ga, win_lds);
}

// The partials of a row: a workgroup of 128 threads a row, a thread a column.  Bound by latency, so that the partials' loads
// are under way before their weights are known.
template <int IN>
__global__ __launch_bounds__(128) void prefix_join_kernel(const PrefixArgs a) {
  __shared__ float weight[256], red[2];
  constexpr int AHEAD = 32;
  const int64_t row = blockIdx.x + static_cast<int64_t>(blockIdx.y) * gridDim.x;
  if (row >= static_cast<int64_t>(a.batch) * a.heads * a.n) return;
  const int t = threadIdx.x, b = static_cast<int>(row / (static_cast<int64_t>(a.heads) * a.n)), i = static_cast<int>(row % a.n);
  const int length = prefix_length(a, b);
  if (i >= prefix_count(a, b, length)) {
    if (t < a.dv && a.out) store_elem(a.out, row * a.dv + t, IN, 0.f);
    if (t == 0 && a.lse) a.lse[row] = 0.f;
    return;
  }
  const float* part = a.part + row * a.parts * a.pitch + t;
  const floatx2* stat = reinterpret_cast<const floatx2*>(a.stat) + row * a.parts;
  const bool column = t < a.dv && a.out;
  float ahead[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) ahead[j] = column && j < a.parts ? part[j * a.pitch] : 0.f;
  floatx2 mine[2];
  float top = -__builtin_inff(), den = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    mine[k] = t + 128 * k < a.parts ? stat[t + 128 * k] : floatx2{-__builtin_inff(), 0.f};
    top = fmaxf(top, mine[k][0]);
  }
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((t & 63) == 0) red[t >> 6] = top;
  __syncthreads();
  top = fmaxf(red[0], red[1]);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float f = mine[k][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f((mine[k][0] - top) * a.c);
    weight[t + 128 * k] = f;
    den = fmaf(f, mine[k][1], den);
  }
  for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
  if ((t & 63) == 0) red[t >> 6] = den;
  __syncthreads();
  den = red[0] + red[1];
  if (!(den > 0.f)) den = __builtin_nanf("");
  if (column) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) sum = fmaf(weight[j], ahead[j], sum);
#pragma unroll 8
    for (int j = AHEAD; j < a.parts; ++j) sum = fmaf(weight[j], part[j * a.pitch], sum);
    store_elem(a.out, row * a.dv + t, IN, sum / den);
  }
  if (t == 0 && a.lse) a.lse[row] = prefix_lse<IN>(top, den, a.c);
}

// The same for up to 16 partials a row: a thread takes four columns of a row, and its statistics by itself, without LDS or
// barriers (16384 rows of two partials: 32 -> 14 us with their walks; 32 rows of 16 of one walk 10.4 and 10.6, of 32
// partials fp32 12.9 and 13.9).
constexpr int PREFIX_FEW_PARTS = 16;
template <int IN>
__global__ __launch_bounds__(256) void prefix_join_few_kernel(const PrefixArgs a) {
  const int units = a.out ? a.pitch / 4 : 1, rows = 256 / units, t = threadIdx.x / units, col = 4 * (threadIdx.x - t * units);
  const int64_t row = (blockIdx.x + static_cast<int64_t>(blockIdx.y) * gridDim.x) * rows + t;
  if (t >= rows || row >= static_cast<int64_t>(a.batch) * a.heads * a.n) return;
  const int b = static_cast<int>(row / (static_cast<int64_t>(a.heads) * a.n)), i = static_cast<int>(row % a.n);
  const floatx2* stat = reinterpret_cast<const floatx2*>(a.stat) + row * a.parts;
  const float* part = a.part + row * a.parts * a.pitch + col;
  floatx2 stats[PREFIX_FEW_PARTS];
  floatx4 parts[PREFIX_FEW_PARTS];
#pragma unroll
  for (int j = 0; j < PREFIX_FEW_PARTS; ++j) {
    stats[j] = floatx2{-__builtin_inff(), 0.f};
    parts[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (j < a.parts) {
      stats[j] = stat[j];
      if (a.out) parts[j] = *reinterpret_cast<const floatx4*>(part + j * a.pitch);
    }
  }
  float top = -__builtin_inff(), den = 0.f;
#pragma unroll
  for (int j = 0; j < PREFIX_FEW_PARTS; ++j) top = fmaxf(top, stats[j][0]);
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < PREFIX_FEW_PARTS; ++j) {
    const float f = stats[j][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f((stats[j][0] - top) * a.c);
    den = fmaf(f, stats[j][1], den);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = fmaf(f, parts[j][k], sum[k]);
  }
  if (!(den > 0.f)) den = __builtin_nanf("");
  const bool live = i < prefix_count(a, b, prefix_length(a, b));
  if (a.out)
    for (int k = 0; k < 4; ++k)
      if (col + k < a.dv) store_elem(a.out, row * a.dv + col + k, IN, live ? sum[k] / den : 0.f);
  if (col == 0 && a.lse) a.lse[row] = live ? prefix_lse<IN>(top, den, a.c) : 0.f;
}

struct ReceivedArgs {
  PrefixArgs a;          // q, own k; lse: the rows' statistics
  int few;               // up to RECEIVED_FEW rows: received_few_kernel
  int stream;            // rows on 16 bytes
  int tiles, nsplit;     // workgroups of a key head along its keys, and along the rows (few: 1)
  float* sums;           // [nsplit][batch][kv][m], or the weights themselves with one
  float* weights;        // [batch][kv][m]
};

constexpr int RECEIVED_FEW = 128;
template <int IN>
__host__ __device__ constexpr int received_rows() { return IN == F32 ? 32 : 64; }
// blocks of 32 keys a wave: two share what a wave reads of the rows, which one block's products wait for (LDS reads 128 bytes
// a cycle; 32 heads of 16384 rows, 128 wide, 1.77 ms with one, 1.32 with two).  fp32 operands leave no room for two.
template <int IN>
__host__ __device__ constexpr int received_blocks() { return IN == F32 ? 1 : 2; }

// A row's statistic as its weights take it.  A row whose sum of weights is not finite has none that are; no row, no weights.
__device__ __forceinline__ float received_stat(float lse, bool row) {
  return row ? (win_finite(lse) ? -lse : __builtin_nanf("")) : -__builtin_inff();
}

// Weights of 32 staged rows from r0 (a multiple of 32) with a wave's keys.  (Products that start from the statistics would
// save 4 % and round their sums at the statistics' size: errors of 5e-7, so 5e-8.)
template <int P, int IN, int NB>
__device__ __forceinline__ void received_weights(floatx16 (&x)[NB], const uint4* qs, const float* stat, int r0,
                                                 const WinFrag<IN> (&kf)[NB][P / 16], float c, int lane) {
  const int hh = lane >> 5;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) x[n][e] = 0.f;
#pragma unroll
  for (int s = 0; s < P / 16; ++s) {
    const WinFrag<IN> q = win_read_row<P, IN>(qs, r0 + (lane & 31), s, hh);
#pragma unroll
    for (int n = 0; n < NB; ++n) win_mma<IN>(x[n], q, kf[n][s]);
  }
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    const floatx4 y = *reinterpret_cast<const floatx4*>(&stat[r0 + 8 * (e >> 2) + 4 * hh]);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[n][e + j] = __builtin_amdgcn_exp2f(fmaf(x[n][e + j], c, y[j]));
  }
}
__device__ __forceinline__ void received_add(float& total, float& lost, const floatx16& x) {
  float sum = x[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) sum += x[e];
  const float y = sum - lost, z = total + y;
  lost = (z - total) - y;
  total = z;
}

// The weights that keys receive.  A workgroup holds 32 to 64 keys a wave as operands and walks over its share of the rows
// that see one of them, head by head of the group; with X = Q K^T a lane has 16 rows of one key, whose weights it sums: no
// exchange between lanes until the end.  Sums of 16 go into a compensated total (16384 x 4 rows).  32 heads of 16384 rows,
// 128 wide: 1.04 to 1.10 ms by card, 1000 to 1060 TFLOP/s (a large matrix product 1200 to 1390); 64 wide 0.75 ms, bound by the
// exponentials.
// STREAM: 16-bit rows of whole 16 bytes go from memory to LDS directly, a tile ahead in two buffers, with one
// barrier a tile, and leave room for a third wave a SIMD (on one card 1.32 -> 1.22 -> 1.14 ms).
template <int P, int IN, bool STREAM>
__device__ __forceinline__ void received_walk(const ReceivedArgs& w, int id, uint4* __restrict__ qs0, uint4* __restrict__ qs1,
                                              float* __restrict__ stat0, float* __restrict__ stat1) {
  constexpr int ES = IN == F32 ? 4 : 2, BQ = received_rows<IN>(), NB = received_blocks<IN>();
  const PrefixArgs& a = w.a;
  // a tile's workgroups, then the tiles of a key head next to each other, those that most rows see first
  const int split = id % w.nsplit;
  id /= w.nsplit;
  const int tile = id % w.tiles, unit = id / w.tiles, b = unit / a.kv, hk = unit - b * a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int length = prefix_length(a, b), count = prefix_count(a, b, length), base = length - count;
  const int key0 = tile * 128 * NB, w0 = key0 + 32 * NB * wave;

  float total[NB], lost[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) total[n] = lost[n] = 0.f;
  const int i0 = (key0 > base ? key0 - base : 0) / BQ * BQ;  // the first row that sees one of the keys
  const int row_tiles = key0 < length && i0 < count ? (count - i0 + BQ - 1) / BQ : 0, all = row_tiles * a.group;
  const int share = (all + w.nsplit - 1) / w.nsplit, t0 = split * share, t1 = t0 + share < all ? t0 + share : all;
  if (t0 < t1) {
    WinFrag<IN> kf[NB][P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int key = w0 + 32 * n + (lane & 31);
      const char* row = rows_at<ES>(a.k, b, hk, key < length ? key : 0);
#pragma unroll
      for (int s = 0; s < P / 16; ++s) {
        kf[n][s] = win_load_row<IN>(row, s, hh, a.d, flip);
        win_keep<IN>(kf[n][s], key < length);
      }
    }
    // a tile of rows: head g of the group, rows from i on
    struct At {
      int g, i;
    };
    At next{t0 / row_tiles, i0 + (t0 % row_tiles) * BQ};  // of the tile that is loaded next
    auto advance = [&]() {
      const At x = next;
      next.i += BQ;
      if (next.i >= count) {
        next.i = i0;
        ++next.g;
      }
      return x;
    };
    auto stat_of = [&](const At& x) {
      const int h = hk * a.group + x.g, r = x.i + static_cast<int>(threadIdx.x % BQ);
      return received_stat(a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.n + (r < count ? r : count - 1)], r < count);
    };
    auto rows_of = [&](const At& x) { return rows_at<ES>(a.q, b, hk * a.group + x.g, x.i); };
    auto take = [&](int row, const uint4* qs, const float* stat) {
      // Every row sees every key, and there is one in every place: zeros that fill up the last tile give NaN with an infinite key
      // (straight to LDS the last row fills it up, whose logits are its own).
      const bool every = base + row >= w0 + 32 * NB - 1 && (STREAM || row + BQ <= count);
#pragma unroll
      for (int sub = 0; sub < BQ / 32; ++sub) {
        floatx16 x[NB];
        received_weights<P, IN, NB>(x, qs, stat, 32 * sub, kf, a.c, lane);
        if (!every) {
          const int end = count - row - 32 * sub - 4 * hh;  // of the lane's rows
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            // the first of the lane's rows that sees its key
            const int from = w0 + 32 * n + (lane & 31) - base - row - 32 * sub - 4 * hh;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int at = 8 * (e >> 2) + (e & 3);
              x[n][e] = at >= from && (STREAM || at < end) ? x[n][e] : 0.f;
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) received_add(total[n], lost[n], x[n]);
      }
    };
    if constexpr (STREAM) {
      StreamTile<P> qt;
      qt.init(a.q.sn, a.d);
      At x = advance();
      qt.load(rows_of(x), count - x.i, qs0);
      if (threadIdx.x < BQ) stat0[threadIdx.x] = stat_of(x);
      int row = x.i, coming = 0;
      float stat = 0.f;
      auto load = [&](int it, uint4* qs) {  // the tile behind `it`, if there is one
        if (it + 1 >= t1) return;
        x = advance();
        qt.load(rows_of(x), count - x.i, qs);
        stat = stat_of(x);
        coming = x.i;
      };
      // a tile; then the next one is there
      auto turn = [&](int it, const uint4* qs, const float* st, uint4* after, float* after_stat) {
        load(it, after);
        take(row, qs, st);
        if (it + 1 < t1 && threadIdx.x < BQ) after_stat[threadIdx.x] = stat;
        row = coming;
        stream_barrier();
      };
      stream_barrier();
#pragma unroll 1
      for (int it = t0; it < t1; it += 2) {
        turn(it, qs0, stat0, qs1, stat1);
        if (it + 1 < t1) turn(it + 1, qs1, stat1, qs0, stat0);
      }
    } else {
      WinStage<P, IN, BQ, 256> stage;
      stage.init(a.q, a.d);
      At x = advance();
      stage.load(rows_of(x), count - x.i);
      float stat = stat_of(x);
      for (int it = t0; it < t1; ++it) {
        const int row = x.i;
        __syncthreads();
        stage.put(qs0, count - row);
        if (threadIdx.x < BQ) stat0[threadIdx.x] = stat;
        __syncthreads();
        if (it + 1 < t1) {
          x = advance();
          stage.load(rows_of(x), count - x.i);
          stat = stat_of(x);
        }
        take(row, qs0, stat0);
      }
    }
  }
  float* const to = (w.nsplit == 1 ? w.weights : w.sums + static_cast<int64_t>(split) * a.batch * a.kv * a.m) +
                    static_cast<int64_t>(unit) * a.m;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    total[n] += __shfl_xor(total[n], 32);
    const int key = w0 + 32 * n + (lane & 31);
    if (hh == 0 && key < a.m) to[key] = key < length ? total[n] : 0.f;
  }
}

template <int P, int IN, bool STREAM>
__global__ __launch_bounds__(256, (STREAM ? 3 : 2)) void received_kernel(const ReceivedArgs w) {
  constexpr int UNITS = received_rows<IN>() * win_chunks<IN == F32 ? 4 : 2>(P), BQ = received_rows<IN>();
  __shared__ uint4 qs[(STREAM ? 2 : 1) * UNITS];
  __shared__ __attribute__((aligned(16))) float stat[2 * BQ];
  received_walk<P, IN, STREAM>(w, xcd_remap(blockIdx.x, gridDim.x), qs, qs + (STREAM ? UNITS : 0), stat, stat + BQ);
}

// The same for up to RECEIVED_FEW rows, those of the group's heads together (row i of head g at i group + g): they stay in
// LDS, and the waves walk over the keys, 32 at a time and the next two blocks on their way, each by itself.  Keys go
// through LDS too: as operands they are loaded in pieces of 32 bytes a row and instruction.  Bound by reading the keys.
template <int P, int IN>
__host__ __device__ constexpr int received_few_bytes(int rows) {  // of LDS
  return (rows + 4 * 32) * P * (IN == F32 ? 4 : 2) + 8 * rows;
}
template <int P, int IN>
__global__ __launch_bounds__(256, 2) void received_few_kernel(const ReceivedArgs w) {
  constexpr int ES = IN == F32 ? 4 : 2, E = 16 / ES, CH = win_chunks<ES>(P);
  extern __shared__ uint4 win_lds[];
  const PrefixArgs& a = w.a;
  const int id = xcd_remap(blockIdx.x, gridDim.x), part = id % w.tiles, unit = id / w.tiles;
  const int b = unit / a.kv, hk = unit - b * a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int length = prefix_length(a, b), count = prefix_count(a, b, length), base = length - count;
  const int rows = count * a.group, blocks = (rows + 31) / 32;  // rows, and blocks of 32 of them
  const int room = (a.n * a.group + 31) / 32 * 32;
  uint4 *const qs = win_lds, *const ks = qs + room * CH + wave * 32 * CH;
  float* const stat = reinterpret_cast<float*>(qs + (room + 4 * 32) * CH);
  int* const seen = reinterpret_cast<int*>(stat + room);  // the last token that a row sees
  float* const to = w.weights + static_cast<int64_t>(unit) * a.m;

  const int step = 4 * w.tiles, first = 4 * part + wave;  // blocks of keys
  const int key_blocks = rows > 0 ? (length + 31) / 32 : 0;
  WinStage<P, IN, 32, 64> even, odd;
  even.init(a.k, a.d);
  odd.init(a.k, a.d);
  auto load = [&](auto& stage, int block) {
    if (block < key_blocks) stage.load(rows_at<ES>(a.k, b, hk, 32 * block), length - 32 * block);
  };
  load(even, first);
  load(odd, first + step);

  for (int u = threadIdx.x; u < 32 * blocks * CH; u += 256) {
    const int r = u / CH, c = u - r * CH, i = min(r, rows - 1) / a.group, h = hk * a.group + min(r, rows - 1) - i * a.group;
    // the last row fills up the last block: it sees every key, and zeros would give NaN with an infinite one
    qs[r * CH + (c ^ win_swizzle<CH>(r))] = rows_unit<ES>(rows_at<ES>(a.q, b, h, i), c * E, a.d);
  }
  for (int r = threadIdx.x; r < 32 * blocks; r += 256) {
    const int i = min(r, rows - 1) / a.group, h = hk * a.group + min(r, rows - 1) - i * a.group;
    stat[r] = received_stat(a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.n + i], r < rows);
    seen[r] = base + i;
  }
  __syncthreads();

  const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
  auto take = [&](auto& stage, int block) {
    const int key = 32 * block + (lane & 31);
    float total = 0.f, lost = 0.f;
    if (block < key_blocks) {
      win_sync<true>();
      stage.put(ks, length - 32 * block);
      load(stage, block + 2 * step);
      win_sync<true>();
      WinFrag<IN> kf[1][P / 16];
#pragma unroll
      for (int s = 0; s < P / 16; ++s) {
        kf[0][s] = win_read_row<P, IN>(ks, lane & 31, s, hh);
#pragma unroll
        for (int j = 0; j < (IN == F32 ? 2 : 1); ++j) {
          uint4& u = kf[0][s].w[j];
          u = uint4{u.x ^ flip, u.y ^ flip, u.z ^ flip, u.w ^ flip};
        }
      }
      for (int r0 = 0; r0 < 32 * blocks; r0 += 32) {
        floatx16 x[1];
        received_weights<P, IN, 1>(x, qs, stat, r0, kf, a.c, lane);
        if (32 * block + 31 > base) {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[0][e] = key <= seen[r0 + 8 * (e >> 2) + 4 * hh + (e & 3)] ? x[0][e] : 0.f;
        }
        received_add(total, lost, x[0]);
      }
    }
    total += __shfl_xor(total, 32);
    if (hh == 0 && key < a.m) to[key] = key < length ? total : 0.f;
  };
  const int end = (a.m + 31) / 32;
  for (int block = first; block < end; block += 2 * step) {
    take(even, block);
    if (block + step < end) take(odd, block + step);
  }
}

// the splits' sums
__global__ __launch_bounds__(256) static void received_join_kernel(const ReceivedArgs w) {
  const int64_t count = static_cast<int64_t>(w.a.batch) * w.a.kv * w.a.m;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= count) return;
  float sum = 0.f;
  for (int j = 0; j < w.nsplit; ++j) sum += w.sums[j * count + i];
  w.weights[i] = sum;
}

}  // namespace sta
