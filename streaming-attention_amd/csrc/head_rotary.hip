// Norm and rotation of query and key heads in one pass: for every row x of a head, with weight w and position p,
//   h = x rsqrt(mean(x^2) + eps) w,   y = R(p) h,
// R(p) turning the pairs (h_a, h_b) of the first r columns by the angle whose cos and sin the table's row p holds:
//   y_a = h_a cos - h_b sin,   y_b = h_b cos + h_a sin      (pairs (i, i + r/2), or (2 i, 2 i + 1) interleaved)
// and backwards, with g = R(-p) dy:   dw = sum over rows of g x inv,   dx = inv (g w - x inv mean(g w x inv)).
// Everything is fp32, rounded once into the output.
//
// Memory-bound: a row is read once and written once (backward: x and dy read, dx written).  A lane holds two
// 16-byte units of a row that turn into each other (columns c and c + r/2, or 2 neighbouring units), so a row of 64 16-bit
// columns takes 4 lanes and nothing is exchanged but the sums of squares.  A lane keeps its position's cos and sin and its
// columns' weights over several heads: the table's row is twice a 16-bit row.  Rows whose width, alignment or
// rotated part do not fall into 16-byte units take head_rotary_any_kernel, a wave a row, element by element.
// A position outside the table turns its rows into NaN.
#include "rows.hpp"

namespace sta {

struct RotArgs {
  Rows x[2], g[2];      // q, k and the gradients of their results
  void* y[2];           // results, or dx: [batch][heads][n][d] dense
  const void* w[2];     // weights [d] or null (1)
  int wtype[2];
  int heads[2], segs[2];  // heads, and workgroup rows (blockIdx.y) that walk over them, per_seg heads each
  int per_seg;
  int n, d, r, items;   // items = batch n
  int lanes;            // lanes a row, a power of two
  const float* table;   // [limit][r]: r/2 cos, r/2 sin
  int limit;
  const void* positions;  // [batch][n] (pos_sb 0: [n]) or null: 0 .. n-1
  int pos64;
  int64_t pos_sb, pos_sn;
  float eps, inv_d;
  int interleaved;
  float* part[2];       // backward: sums of dw [segs gridDim.x][d]
};

// 2^-70: the squares of 256 of fp32's largest values times it stay in fp32
constexpr float ROT_SMALL = 8.470329472543003e-22f;

__device__ __forceinline__ int64_t rot_position(const RotArgs& a, int b, int n) {
  if (!a.positions) return n;
  const int64_t at = b * a.pos_sb + n * a.pos_sn;
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
}

__device__ __forceinline__ float rot_weight(const RotArgs& a, int which, int col) {
  return a.w[which] ? load_elem(a.w[which], col, a.wtype[which]) : 1.f;
}

// Loads past the caches' usual policy: 8 x 16 x 4096 x 64 bf16, queries and keys, forward 102 -> 74 us, backward
// 166 -> 98 us.
__device__ __forceinline__ uint4 rot_load(const char* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  const u4 x = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  return uint4{x[0], x[1], x[2], x[3]};
}

template <int IN, bool INTER, bool BACK>
__global__ __launch_bounds__(256) void head_rotary_kernel(const RotArgs a) {
  constexpr int ES = IN == F32 ? 4 : 2, E = 16 / ES;
  __shared__ float red[BACK ? 256 * 2 * E : 1];
  const int which = static_cast<int>(blockIdx.y) < a.segs[0] ? 0 : 1;
  const int seg = blockIdx.y - (which ? a.segs[0] : 0);
  const int h0 = seg * a.per_seg, h1 = min(h0 + a.per_seg, a.heads[which]);
  const int u = threadIdx.x & (a.lanes - 1), slot = threadIdx.x / a.lanes, per = 256 / a.lanes;
  const int pairs = a.r / 2, turning = INTER ? 0 : pairs / E;
  int ca, cb;
  if (INTER) {
    ca = 2 * E * u;
    cb = ca + E;
  } else if (u < turning) {
    ca = E * u;
    cb = pairs + E * u;
  } else {
    ca = a.r + 2 * E * (u - turning);
    cb = ca + E;
  }
  const bool has_a = ca < a.d, has_b = cb < a.d;
  float wa[E], wb[E], da[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    wa[e] = has_a ? rot_weight(a, which, ca + e) : 0.f;
    wb[e] = has_b ? rot_weight(a, which, cb + e) : 0.f;
    da[e] = db[e] = 0.f;
  }
  const uint4 zero = uint4{0u, 0u, 0u, 0u};
  for (int item = blockIdx.x * per + slot; item < a.items; item += gridDim.x * per) {
    const int b = item / a.n, n = item - b * a.n;
    // the next head's units are loaded while this one's are turned
    uint4 na, nb, nga, ngb;
    auto load = [&](int h) {
      const char* xr = rows_at<ES>(a.x[which], b, h, n);
      na = has_a ? rot_load(xr + ca * ES) : zero;
      nb = has_b ? rot_load(xr + cb * ES) : zero;
      if constexpr (BACK) {
        const char* gr = rows_at<ES>(a.g[which], b, h, n);
        nga = has_a ? rot_load(gr + ca * ES) : zero;
        ngb = has_b ? rot_load(gr + cb * ES) : zero;
      }
    };
    load(h0);
    const int64_t p = rot_position(a, b, n);
    const bool known = p >= 0 && p < a.limit;
    const float* row = a.table + (known ? p : 0) * a.r;
    // cos and sin of the pairs: half-split (a_e, b_e); interleaved the E / 2 pairs of each unit
    float c[E], s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = INTER ? (e < E / 2 ? ca / 2 + e : cb / 2 + e - E / 2) : ca + e;
      const bool turn = INTER ? i < pairs : u < turning;
      c[e] = turn ? row[i] : 1.f;
      s[e] = turn ? row[pairs + i] : 0.f;
      if (!known) c[e] = __builtin_nanf("");
    }
    for (int h = h0; h < h1; ++h) {
      float xa[E], xb[E], ga[E], gb[E];
      const uint4 ua = na, ub = nb;
      if constexpr (BACK) {
        rows_unpack<IN>(nga, ga);
        rows_unpack<IN>(ngb, gb);
      }
      if (h + 1 < h1) load(h + 1);
      rows_unpack<IN>(ua, xa);
      rows_unpack<IN>(ub, xb);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(xa[e], xa[e], fmaf(xb[e], xb[e], ss));
      for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
      float inv = 1.f / sqrtf(fmaf(ss, a.inv_d, a.eps));
      if (!(ss < __builtin_inff())) {  // squares past fp32: of the row times a power of two
        ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float ya = xa[e] * ROT_SMALL, yb = xb[e] * ROT_SMALL;
          ss = fmaf(ya, ya, fmaf(yb, yb, ss));
        }
        for (int o = a.lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        inv = ROT_SMALL / sqrtf(fmaf(ss, a.inv_d, a.eps * ROT_SMALL * ROT_SMALL));
      }
      float ya[E], yb[E];
      // (a column that does not turn takes nothing of its neighbour, not even 0 times an infinity)
      auto turn = [&](const float (&fa)[E], const float (&fb)[E], float sign) {
        if constexpr (INTER) {
#pragma unroll
          for (int i = 0; i < E / 2; ++i) {
            const float sa = sign * s[i], sb = sign * s[E / 2 + i];
            const bool ta = ca / 2 + i < pairs, tb = cb / 2 + i < pairs;
            ya[2 * i] = fa[2 * i] * c[i] - (ta ? fa[2 * i + 1] * sa : 0.f);
            ya[2 * i + 1] = fa[2 * i + 1] * c[i] + (ta ? fa[2 * i] * sa : 0.f);
            yb[2 * i] = fb[2 * i] * c[E / 2 + i] - (tb ? fb[2 * i + 1] * sb : 0.f);
            yb[2 * i + 1] = fb[2 * i + 1] * c[E / 2 + i] + (tb ? fb[2 * i] * sb : 0.f);
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            ya[e] = fa[e] * c[e] - (u < turning ? fb[e] * (sign * s[e]) : 0.f);
            yb[e] = fb[e] * c[e] + (u < turning ? fa[e] * (sign * s[e]) : 0.f);
          }
        }
      };
      if constexpr (!BACK) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          xa[e] *= inv * wa[e];
          xb[e] *= inv * wb[e];
        }
        turn(xa, xb, 1.f);
      } else {
        turn(ga, gb, -1.f);
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          xa[e] *= inv;
          xb[e] *= inv;
          da[e] = fmaf(ya[e], xa[e], da[e]);
          db[e] = fmaf(yb[e], xb[e], db[e]);
          ya[e] *= wa[e];
          yb[e] *= wb[e];
          m = fmaf(ya[e], xa[e], fmaf(yb[e], xb[e], m));
        }
        for (int o = a.lanes >> 1; o > 0; o >>= 1) m += __shfl_xor(m, o);
        m *= a.inv_d;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          ya[e] = inv * (ya[e] - xa[e] * m);
          yb[e] = inv * (yb[e] - xb[e] * m);
        }
      }
      char* yr = static_cast<char*>(a.y[which]) +
                 ((static_cast<int64_t>(b) * a.heads[which] + h) * a.n + n) * a.d * ES;
      if (has_a) *reinterpret_cast<uint4*>(yr + ca * ES) = rows_pack<IN>(ya);
      if (has_b) *reinterpret_cast<uint4*>(yr + cb * ES) = rows_pack<IN>(yb);
    }
  }
  if constexpr (BACK) {
    if (!a.part[which]) return;
    // red[slot][column]: per d <= 256 2 E, since lanes 2 E >= d
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (has_a) red[slot * a.d + ca + e] = da[e];
      if (has_b) red[slot * a.d + cb + e] = db[e];
    }
    __syncthreads();
    for (int col = threadIdx.x; col < a.d; col += 256) {
      float sum = 0.f;
      for (int i = 0; i < per; ++i) sum += red[i * a.d + col];
      a.part[which][(static_cast<int64_t>(seg) * gridDim.x + blockIdx.x) * a.d + col] = sum;
    }
  }
}

// A wave a row, lane l columns l, l + 64, ...
template <int IN, bool BACK>
__global__ __launch_bounds__(256) void head_rotary_any_kernel(const RotArgs a) {
  constexpr int ES = IN == F32 ? 4 : 2, C = 4;
  __shared__ float red[BACK ? 4 * 64 * C : 1];
  const int which = static_cast<int>(blockIdx.y) < a.segs[0] ? 0 : 1;
  const int seg = blockIdx.y - (which ? a.segs[0] : 0);
  const int h0 = seg * a.per_seg, h1 = min(h0 + a.per_seg, a.heads[which]);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pairs = a.r / 2;
  int other[C];    // the column that a column turns with; itself where it does not turn
  float sign[C], w[C], wo[C], dw[C];
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int col = lane + 64 * k;
    const bool first = a.interleaved ? (col & 1) == 0 : col < pairs;
    other[k] = col >= a.r ? col : (a.interleaved ? col ^ 1 : (first ? col + pairs : col - pairs));
    sign[k] = col >= a.r ? 0.f : (first ? -1.f : 1.f);
    w[k] = col < a.d ? rot_weight(a, which, col) : 0.f;
    wo[k] = col < a.d ? rot_weight(a, which, other[k]) : 0.f;
    dw[k] = 0.f;
  }
  for (int item = blockIdx.x * 4 + wave; item < a.items; item += gridDim.x * 4) {
    const int b = item / a.n, n = item - b * a.n;
    const int64_t p = rot_position(a, b, n);
    const bool known = p >= 0 && p < a.limit;
    const float* row = a.table + (known ? p : 0) * a.r;
    float c[C], s[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int col = lane + 64 * k;
      c[k] = 1.f;
      s[k] = 0.f;
      if (col < a.r) {
        const int i = a.interleaved ? col >> 1 : (col < pairs ? col : col - pairs);
        c[k] = row[i];
        s[k] = row[pairs + i] * sign[k];
      }
      if (!known) c[k] = __builtin_nanf("");
    }
    for (int h = h0; h < h1; ++h) {
      const char* xr = rows_at<ES>(a.x[which], b, h, n);
      float x[C], y[C];
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < C; ++k) {
        x[k] = lane + 64 * k < a.d ? load_elem(xr, lane + 64 * k, IN) : 0.f;
        ss = fmaf(x[k], x[k], ss);
      }
      for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
      float inv = 1.f / sqrtf(fmaf(ss, a.inv_d, a.eps));
      if (!(ss < __builtin_inff())) {
        ss = 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k) ss = fmaf(x[k] * ROT_SMALL, x[k] * ROT_SMALL, ss);
        for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
        inv = ROT_SMALL / sqrtf(fmaf(ss, a.inv_d, a.eps * ROT_SMALL * ROT_SMALL));
      }
      if constexpr (!BACK) {
#pragma unroll
        for (int k = 0; k < C; ++k)
          if (lane + 64 * k < a.d)
            y[k] = x[k] * (inv * w[k]) * c[k] + load_elem(xr, other[k], IN) * (inv * wo[k]) * s[k];
      } else {
        const char* gr = rows_at<ES>(a.g[which], b, h, n);
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k)
          if (lane + 64 * k < a.d) {
            y[k] = load_elem(gr, lane + 64 * k, IN) * c[k] - load_elem(gr, other[k], IN) * s[k];
            x[k] *= inv;
            dw[k] = fmaf(y[k], x[k], dw[k]);
            y[k] *= w[k];
            m = fmaf(y[k], x[k], m);
          }
        for (int o = 32; o > 0; o >>= 1) m += __shfl_xor(m, o);
        m *= a.inv_d;
#pragma unroll
        for (int k = 0; k < C; ++k)
          if (lane + 64 * k < a.d) y[k] = inv * (y[k] - x[k] * m);
      }
      const int64_t at = ((static_cast<int64_t>(b) * a.heads[which] + h) * a.n + n) * a.d;
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (lane + 64 * k < a.d) store_elem(a.y[which], at + lane + 64 * k, IN, y[k]);
    }
  }
  if constexpr (BACK) {
    if (!a.part[which]) return;
#pragma unroll
    for (int k = 0; k < C; ++k) red[(wave * C + k) * 64 + lane] = dw[k];
    __syncthreads();
    for (int col = threadIdx.x; col < a.d; col += 256) {
      const int k = col >> 6, l = col & 63;
      float sum = 0.f;
      for (int i = 0; i < 4; ++i) sum += red[(i * C + k) * 64 + l];
      a.part[which][(static_cast<int64_t>(seg) * gridDim.x + blockIdx.x) * a.d + col] = sum;
    }
  }
}

// dw from the workgroups' sums: 4 columns a workgroup, 64 threads a column over the rows, then in order
__global__ __launch_bounds__(256) static void head_rotary_weight_kernel(const float* part0, const float* part1, int rows0,
                                                                        int rows1, int d, void* dw0, void* dw1,
                                                                        int type) {
  __shared__ float red[256];
  const float* part = blockIdx.y ? part1 : part0;
  const int rows = blockIdx.y ? rows1 : rows0;
  if (!part) return;
  const int col = blockIdx.x * 4 + (threadIdx.x & 3);
  float s = 0.f;
  if (col < d) {
#pragma unroll 16
    for (int r = threadIdx.x >> 2; r < rows; r += 64) s += part[static_cast<int64_t>(r) * d + col];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 4 && col < d) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += red[4 * i + threadIdx.x];
    store_elem(blockIdx.y ? dw1 : dw0, col, type, sum);
  }
}

}  // namespace sta
