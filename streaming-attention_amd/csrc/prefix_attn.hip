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
// window_forward_kernel, whose tiles, layouts and second pass for results that are not finite it uses.
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
  float* part;           // [batch][heads][n][parts][dv + 2]: sums, then maximum and sum of weights
  int parts;             // 0: rows are finished by one workgroup
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

template <int P, int IN, bool SHARE, bool VALUES, bool CAREFUL>
__device__ __forceinline__ int prefix_pass(const PrefixArgs& a, const PrefixWalk& w, int again) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), BK = win_keys<IN, SHARE>(), NSUB = BK / 32,
                MT = P / 32, STEP = SHARE ? 4 : 1;
  extern __shared__ uint4 win_lds[];
  // the tiles of a unit, then the units of a key head next to each other: they read the same keys
  int id = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = w.tiles - 1 - id % w.tiles;
  id /= w.tiles;
  const int split = id % w.nsplit;
  id /= w.nsplit;
  const int units = a.batch / w.span, hk = id / units, b0 = (id - hk * units) * w.span;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  uint4 *const ks = win_lds + (SHARE ? wave * 2 * BK * CH : 0), *const vs = ks + BK * CH;
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
  const bool any = w.own ? own_end > 0 : r0 < w.span * per;
  const int tiles_p = any ? (rows_p + BK - 1) / BK : 0, all_tiles = tiles_p + (own_end + BK - 1) / BK;
  const int share = (all_tiles + w.nsplit - 1) / w.nsplit;
  const int t0 = split * share, t1 = t0 + share < all_tiles ? t0 + share : all_tiles;

  if (t0 < t1) {
    WinFrag<IN> qf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* qrow = rows_at<ES>(a.q, mine.b, mine.h, mine.i);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      qf[s] = win_load_row<IN>(qrow, s, hh, a.d, flip);
      win_keep<IN>(qf[s], mine.live);
    }
#pragma unroll 1
    for (int seg = t0 < tiles_p ? 0 : 1; seg < (t1 > tiles_p ? 2 : 1); ++seg) {
      const Rows kr = seg ? a.k : a.pk, vr = seg ? a.v : a.pv;
      const int rb = seg ? b0 : b0 / a.per_set, end = seg ? own_end : rows_p;
      const int lo = seg ? (t0 > tiles_p ? t0 - tiles_p : 0) : t0, hi = seg ? t1 - tiles_p : (t1 < tiles_p ? t1 : tiles_p);
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
      const int start = lo + (SHARE ? wave : 0);
      if (AHEAD && start < hi) load(start);
      for (int it = start; it < hi; it += STEP) {
        if (!AHEAD) load(it);
        win_sync<SHARE>();
        const int key0 = it * BK;
        kst.put(ks, end - key0);
        if constexpr (VALUES) vst.put(vs, end - key0);
        win_sync<SHARE>();
        if (AHEAD && it + STEP < hi) load(it + STEP);
        if (key0 > lim_hi) continue;
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
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) l += x[sub][i];
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

  // four sums of a row at column col, its maximum and sum of weights
  auto store4 = [&](const Place& x, int col, float inv, float y0, float y1, float y2, float y3) {
    if (col >= a.dv) return;
    if (a.parts) {
      float* to = a.part + (x.at * a.parts + w.first + split) * (a.dv + 2) + col;
      to[0] = y0;
      if (col + 1 < a.dv) to[1] = y1;
      if (col + 2 < a.dv) to[2] = y2;
      if (col + 3 < a.dv) to[3] = y3;
    } else {
      win_store4<IN>(a.out, x.at * a.dv, col, a.dv, x.live ? y0 * inv : 0.f, x.live ? y1 * inv : 0.f,
                     x.live ? y2 * inv : 0.f, x.live ? y3 * inv : 0.f);
    }
  };
  auto store_sums = [&](const Place& x, float top, float den) {
    if (a.parts) {
      float* to = a.part + (x.at * a.parts + w.first + split) * (a.dv + 2) + a.dv;
      to[0] = prefix_top(top, den);
      to[1] = den;
    } else if (a.lse) {
      a.lse[x.at] = x.live ? top * a.c - win_weight_lift<IN>() + __builtin_amdgcn_logf(den) : 0.f;
    }
  };
  // a sum of weights that is not finite, or none though the row sees a key of the workgroup's share
  auto wrong = [&](const Place& x, float den) {
    const bool sees = t0 < tiles_p || (t0 < t1 && (t0 - tiles_p) * BK <= x.lim);
    return !win_finite(den) || (sees && !(den > 0.f));
  };

  if constexpr (SHARE) {
    float *red = reinterpret_cast<float*>(win_lds), *red_m = red + win_join_floats<P>(), *red_l = red_m + 4 * 32;
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
        for (int j = 0; j < MT; ++j)
          store4(x, 32 * j + 4 * (threadIdx.x & 7), inv, o[j][0], o[j][1], o[j][2], o[j][3]);
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
  if (mine.in && (CAREFUL ? again : !bad)) {
    if constexpr (VALUES) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          store4(mine, 32 * mt + 8 * r + 4 * hh, inv, acc[mt][4 * r], acc[mt][4 * r + 1], acc[mt][4 * r + 2],
                 acc[mt][4 * r + 3]);
    }
    if (hh == 0) store_sums(mine, m, l);
  }
  return bad;
}

template <int P, int IN, bool SHARE, bool VALUES>
__global__ __launch_bounds__(256, (win_row_waves<P, IN, SHARE>())) void prefix_attention_kernel(const PrefixArgs a,
                                                                                               const PrefixWalk w) {
  win_passes([&](auto second, int again) {
    return prefix_pass<P, IN, SHARE, VALUES, decltype(second)::value>(a, w, again);
  });
}

// The partials of a row: a workgroup of 128 threads a row, a thread a column.
template <int IN>
__global__ __launch_bounds__(128) void prefix_join_kernel(const PrefixArgs a) {
  __shared__ float weight[256], red[2];
  const int64_t row = blockIdx.x + static_cast<int64_t>(blockIdx.y) * gridDim.x;
  if (row >= static_cast<int64_t>(a.batch) * a.heads * a.n) return;
  const int b = static_cast<int>(row / (static_cast<int64_t>(a.heads) * a.n)), i = static_cast<int>(row % a.n);
  const int length = prefix_length(a, b);
  const bool live = i < prefix_count(a, b, length);
  const int pitch = a.dv + 2;
  const float* part = a.part + row * a.parts * pitch;
  if (live) {
    float top = -__builtin_inff(), den = 0.f;
    for (int j = threadIdx.x; j < a.parts; j += 128) top = fmaxf(top, part[j * pitch + a.dv]);
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(red[0], red[1]);
    __syncthreads();
    for (int j = threadIdx.x; j < a.parts; j += 128) {
      const float lj = part[j * pitch + a.dv + 1];
      const float f = lj == 0.f ? 0.f : __builtin_amdgcn_exp2f((part[j * pitch + a.dv] - top) * a.c);
      weight[j] = f;
      den = fmaf(f, lj, den);
    }
    for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = den;
    __syncthreads();
    den = red[0] + red[1];
    if (!(den > 0.f)) den = __builtin_nanf("");
    if (static_cast<int>(threadIdx.x) < a.dv && a.out) {
      float sum = 0.f;
#pragma unroll 8
      for (int j = 0; j < a.parts; ++j) sum = fmaf(weight[j], part[j * pitch + threadIdx.x], sum);
      store_elem(a.out, row * a.dv + threadIdx.x, IN, sum / den);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[row] = top * a.c - win_weight_lift<IN>() + __builtin_amdgcn_logf(den);
  } else {
    if (static_cast<int>(threadIdx.x) < a.dv && a.out) store_elem(a.out, row * a.dv + threadIdx.x, IN, 0.f);
    if (threadIdx.x == 0 && a.lse) a.lse[row] = 0.f;
  }
}

struct ReceivedArgs {
  PrefixArgs a;          // q, own k; lse: the rows' statistics
  int tiles, nsplit;     // tiles of 128 keys, workgroups a tile
  float* sums;           // [nsplit][batch][kv][m], or the weights themselves with one
  float* weights;        // [batch][kv][m]
};

template <int IN>
__host__ __device__ constexpr int received_rows() { return IN == F32 ? 32 : 64; }

// The weights that keys receive.  A workgroup holds 128 keys of a key head as operands, 32 a wave, and walks over the
// rows that see one of them, head by head of the group; with X = Q K^T a lane has 16 rows of one key, whose weights
// it sums: no exchange between lanes until the end.  Sums of 16 go into a compensated total (16384 x 4 rows).
template <int P, int IN>
__global__ __launch_bounds__(256, 2) void received_kernel(const ReceivedArgs w) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), BQ = received_rows<IN>(), NSUB = BQ / 32;
  __shared__ uint4 qs[BQ * CH];
  __shared__ __attribute__((aligned(16))) float stat[BQ];
  const PrefixArgs& a = w.a;
  int id = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = id % w.tiles;
  id /= w.tiles;
  const int split = id % w.nsplit, unit = id / w.nsplit, b = unit / a.kv, hk = unit - b * a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int length = prefix_length(a, b), count = prefix_count(a, b, length), base = length - count;
  const int key0 = tile * WIN_ROWS, w0 = key0 + 32 * wave, key = w0 + (lane & 31);

  float total = 0.f, lost = 0.f;
  const int i0 = (key0 > base ? key0 - base : 0) / BQ * BQ;  // the first row that sees one of the keys
  const int row_tiles = key0 < length && i0 < count ? (count - i0 + BQ - 1) / BQ : 0, all = row_tiles * a.group;
  const int share = (all + w.nsplit - 1) / w.nsplit, t0 = split * share, t1 = t0 + share < all ? t0 + share : all;
  if (t0 < t1) {
    WinFrag<IN> kf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* krow = rows_at<ES>(a.k, b, hk, key < length ? key : 0);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      kf[s] = win_load_row<IN>(krow, s, hh, a.d, flip);
      win_keep<IN>(kf[s], key < length);
    }
    WinStage<P, IN, BQ, 256> stage;
    stage.init(a.q, a.d);
    float next = 0.f;
    auto load = [&](int it) {
      const int g = it / row_tiles, i = i0 + (it - g * row_tiles) * BQ, h = hk * a.group + g;
      stage.load(rows_at<ES>(a.q, b, h, i), count - i);
      const int r = i + static_cast<int>(threadIdx.x % BQ);
      next = a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.n + (r < count ? r : count - 1)];
      // behind the last row: no weights; a row whose sum of weights is not finite has none that are
      next = r < count ? (win_finite(next) ? next : __builtin_nanf("")) : __builtin_inff();
    };
    load(t0);
    for (int it = t0; it < t1; ++it) {
      const int i = i0 + it % row_tiles * BQ;
      __syncthreads();
      stage.put(qs, count - i);
      if (threadIdx.x < BQ) stat[threadIdx.x] = next;
      __syncthreads();
      if (it + 1 < t1) load(it + 1);
      const bool every = base + i >= w0 + 31;
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub) {
        floatx16 x;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.f;
#pragma unroll
        for (int s = 0; s < P / 16; ++s)
          win_mma<IN>(x, win_read_row<P, IN>(qs, 32 * sub + (lane & 31), s, hh), kf[s]);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const floatx4 y = *reinterpret_cast<const floatx4*>(&stat[32 * sub + 8 * (e >> 2) + 4 * hh]);
          x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], a.c, -y[e & 3]));
        }
        if (!every) {
          const int from = key - base - i - 32 * sub - 4 * hh;  // the first of the lane's rows that sees its key
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = 8 * (e >> 2) + (e & 3) >= from ? x[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += x[e];
        const float y = sum - lost, z = total + y;
        lost = (z - total) - y;
        total = z;
      }
    }
  }
  total += __shfl_xor(total, 32);
  if (hh == 0 && key < a.m) {
    float* to = w.nsplit == 1 ? w.weights : w.sums + static_cast<int64_t>(split) * a.batch * a.kv * a.m;
    to[static_cast<int64_t>(unit) * a.m + key] = key < length ? total : 0.f;
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
