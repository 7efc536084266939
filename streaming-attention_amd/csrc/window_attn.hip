// Exact causal attention over a sliding window and a few first tokens (sinks), with its gradients.
//
// Row i of a sequence sees the keys V(i) = {j <= i : i - j < window or j < sinks}:
//   p_ij = exp(s q_i.k_j - L_i), L_i = log sum_{j in V(i)} exp(s q_i.k_j),   o_i = sum_{j in V(i)} p_ij v_j
//   dv_j = sum_i p_ij do_i,   D_i = do_i.o_i,   ds_ij = s p_ij (do_i.v_j - D_i)
//   dq_i = sum_j ds_ij k_j,   dk_j = sum_i ds_ij q_i
// Query heads share a key head in groups of heads / kv_heads; dk and dv are the sums over the group.  Rows at or
// behind a sequence's length are no part of it: outputs and gradients there are zero, whatever the inputs hold.
//
// Matrix-core layout (v_mfma_f32_32x32x16 for 16-bit rows, 32x32x2_f32 eight times over the same operands for
// fp32): lane l = 32 h + i holds A[i][8 h + j], B[8 h + j][i], j = 0..7, and D[8 (r / 4) + 4 h + r % 4][i] in
// accumulator element r.  The logits are taken transposed where the next product contracts over keys (X^T = K Q^T: a
// lane holds 16 keys of one row) and plain where it contracts over rows (X = Q K^T: 16 rows of one key), so that
// the weights in accumulator elements 8 t .. 8 t + 7 are the B operand of the next product as they stand, for the
// contraction order {4 h + 0..3, 8 + 4 h + 0..3} of 16 keys (rows); the A operand in that order is a transposed
// read of the staged rows (ds_read_b64_tr_b16: 4 rows x 16 columns a 16-lane group; 32-bit reads for fp32).
//
// LDS rows are P elements wide without padding; 16-byte chunk c of row r sits at c ^ win_swizzle(r), which spreads
// both 16 consecutive rows at one chunk (row reads) and 4 rows at 4 chunks (transposed reads) over all 64 banks.
//
// Hidden pairs are left out by selects, never by arithmetic on their logits.  A tile's products still multiply hidden
// pairs' zero weights with their values, so an infinity or NaN in a value that some rows of a tile see would reach
// those that do not: a workgroup with a result that is not finite goes over its tiles once more, taking the partly visible ones
// pair by pair (win_add_seen), and stores that result from there.
#pragma once
#include <type_traits>

#include "rows.hpp"

namespace sta {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 win_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 win_half2 __attribute__((ext_vector_type(2)));
typedef short win_short4 __attribute__((ext_vector_type(4)));

struct WinArgs {
  Rows q, k, v, go;     // go: the output's gradient
  int heads, group;        // query heads, query heads per key head
  int batch, n, d, dv;
  int window, sinks;       // 1 <= window <= n, 0 <= sinks <= n (the host clamps both to n)
  float c;                 // |scale| log2(e): weights are exp2(c x - lse), x of queries with the scale's sign
  float scale;             // the scale itself
  const int* lengths;      // [batch] or null
  void* out;               // [batch][heads][n][dv]
  void* rest;              // [batch][heads][n][dv]: what the rounding of out left, rounded; or null
  float* lse;              // [batch][heads][n]: log2 of the row's sum of weights, or null
  float* delta;            // [batch][heads][n]: D_i
  void *dq, *dk, *dv_out;  // [batch][heads][n][d], [batch][kv heads][n][d | dv]
  int share, key_share;    // tiles of 32 rows (keys) instead of 128, see win_rows
  int tiles, key_tiles;
  // gradients of sinks behind their window: rows [j + window, n) of the first sink_tiles key tiles, far_chunks
  // workgroups a tile with far_rows rows each; sums part [batch kv_heads][far_chunks + 1][sink_rows][d + dv]
  int sink_tiles, far_chunks, far_rows, sink_rows;
  float* part;
  float lift, drop;        // 2^e and 2^-e: the weights' scale in fp16 gradients
};

constexpr int WIN_ROWS = 128;

template <int ES>
__host__ __device__ constexpr int win_chunks(int p) { return p * ES / 16; }

// see the top of the file; needs only bits 0..3 of the row
template <int CH>
__device__ __forceinline__ int win_swizzle(int row) {
  if constexpr (CH % 16 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
  if constexpr (CH % 8 == 0) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  return (row >> 2) & 3;
}

template <int IN>
struct WinFrag {  // 8 contraction elements of a lane
  uint4 w[IN == F32 ? 2 : 1];
};

template <int IN>
__device__ __forceinline__ void win_mma(floatx16& acc, const WinFrag<IN>& a, const WinFrag<IN>& b) {
  if constexpr (IN == F32) {
    const float* x = reinterpret_cast<const float*>(a.w);
    const float* y = reinterpret_cast<const float*>(b.w);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], acc, 0, 0, 0);
  } else if constexpr (IN == F16) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(win_half8, a.w[0]),
                                                 __builtin_bit_cast(win_half8, b.w[0]), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.w[0]),
                                                  __builtin_bit_cast(bf16x8, b.w[0]), acc, 0, 0, 0);
  }
}

// accumulator elements 8 t .. 8 t + 7 as an operand (16 bits: each rounded to nearest even)
template <int IN>
__device__ __forceinline__ WinFrag<IN> win_operand(const floatx16& x, int t) {
  WinFrag<IN> f;
  if constexpr (IN == F32) {
    f.w[0] = uint4{__float_as_uint(x[8 * t]), __float_as_uint(x[8 * t + 1]), __float_as_uint(x[8 * t + 2]),
                   __float_as_uint(x[8 * t + 3])};
    f.w[1] = uint4{__float_as_uint(x[8 * t + 4]), __float_as_uint(x[8 * t + 5]), __float_as_uint(x[8 * t + 6]),
                   __float_as_uint(x[8 * t + 7])};
  } else {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const floatx2 y = floatx2{x[8 * t + 2 * j], x[8 * t + 2 * j + 1]};
      if constexpr (IN == F16)
        u[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, win_half2));
      else
        u[j] = pk_bf16(y[0], y[1]);
    }
    f.w[0] = uint4{u[0], u[1], u[2], u[3]};
  }
  return f;
}

// Staging of ROWS rows of a tile by a workgroup (256 threads) or a wave: registers first (load), LDS when the tile before is done with (put).
// The loads are free of branches, so that they stay in flight while a tile computes: rows behind the last are read as the
// last one and a row's last 16 bytes in the place of a unit that would reach over its end; put zeroes the ones and
// moves the others into place.
template <int P, int IN, int ROWS, int THREADS>
struct WinStage {
  static constexpr int ES = IN == F32 ? 4 : 2, E = 16 / ES, CH = win_chunks<ES>(P);
  static constexpr int COUNT = (ROWS * CH + THREADS - 1) / THREADS;
  static constexpr bool EVEN = THREADS % CH == 0;  // a thread's units lie in one column, THREADS / CH rows apart
  uint4 u[COUNT];
  uint32_t at[EVEN ? 1 : COUNT];  // bytes from the tile's first row (the host keeps 64 rows below 2^31 bytes)
  int pitch, width;

  __device__ __forceinline__ static int unit(int i) { return (threadIdx.x % THREADS) + THREADS * i; }
  __device__ __forceinline__ void init(const Rows& t, int w) {
    pitch = static_cast<int>(t.sn) * ES;
    width = w;
#pragma unroll
    for (int i = 0; i < (EVEN ? 1 : COUNT); ++i) {
      const int x = unit(i);
      at[i] = min(x / CH, ROWS - 1) * pitch + min(x % CH * E, width - E) * ES;
    }
  }
  // the tile at `row`, `left` >= 1 of its rows being there; a row has at least 16 bytes
  __device__ __forceinline__ void load(const char* row, int left) {
    uint32_t off[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) off[i] = at[EVEN ? 0 : i];
    if (left < ROWS) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i)
        off[i] -= static_cast<uint32_t>(max(0, min(unit(i) / CH, ROWS - 1) - left + 1) * pitch);
    }
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const char* from = EVEN ? row + static_cast<int64_t>(i * (THREADS / CH)) * pitch : row;
      u[i] = rows_load16(from + static_cast<int32_t>(off[i]));
    }
  }
  __device__ __forceinline__ void put(uint4* lds, int left) const {
    auto to = [&](int i, const uint4& x) {
      const int k = unit(i), r = k / CH, c = k % CH;
      if (ROWS * CH % THREADS == 0 || k < ROWS * CH) lds[r * CH + (c ^ win_swizzle<CH>(r))] = x;
    };
    if (left >= ROWS && width == P) {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) to(i, u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        const int k = unit(i), r = k / CH, c = k % CH;
        uint4 x = u[i];
        if (width % E) x = rows_shift(x, max(0, c * E + E - width) * ES & 15);
        const bool in = r < left && c * E < width;
        to(i, uint4{in ? x.x : 0u, in ? x.y : 0u, in ? x.z : 0u, in ? x.w : 0u});
      }
    }
  }
};

// A (or B) operand of 16 dimensions [16 s, 16 s + 16) of staged row r
template <int P, int IN>
__device__ __forceinline__ WinFrag<IN> win_read_row(const uint4* lds, int r, int s, int h) {
  constexpr int CH = win_chunks<IN == F32 ? 4 : 2>(P);
  WinFrag<IN> f;
  const int x = win_swizzle<CH>(r);
  if constexpr (IN == F32) {
    f.w[0] = lds[r * CH + ((4 * s + 2 * h) ^ x)];
    f.w[1] = lds[r * CH + ((4 * s + 2 * h + 1) ^ x)];
  } else {
    f.w[0] = lds[r * CH + ((2 * s + h) ^ x)];
  }
  return f;
}

// A operand of columns [32 mt, 32 mt + 32) over staged rows [r0, r0 + 16) (a multiple of 16) in the contraction order
// of the accumulators
template <int P, int IN>
__device__ __forceinline__ WinFrag<IN> win_read_columns(const uint4* lds, int r0, int mt, int lane) {
  constexpr int CH = win_chunks<IN == F32 ? 4 : 2>(P);
  const int h = lane >> 5;
  WinFrag<IN> f;
  if constexpr (IN == F32) {
    uint32_t u[8];
    const int col = 32 * mt + (lane & 31);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = r0 + 8 * (j >> 2) + 4 * h + (j & 3);
      u[j] = reinterpret_cast<const uint32_t*>(lds)[4 * (r * CH + ((col >> 2) ^ win_swizzle<CH>(r))) + (col & 3)];
    }
    f.w[0] = uint4{u[0], u[1], u[2], u[3]};
    f.w[1] = uint4{u[4], u[5], u[6], u[7]};
  } else {
    const int col = 32 * mt + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    uint32_t u[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = r0 + 8 * t + 4 * h + ((lane & 15) >> 2);
      const int at = 8 * (r * CH + ((col >> 3) ^ win_swizzle<CH>(r))) + (col & 7);
      typedef __attribute__((address_space(3))) win_short4* lds_ptr;
      const win_short4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_ptr)(reinterpret_cast<short*>(const_cast<uint4*>(lds)) + at));
      const uint2 y = __builtin_bit_cast(uint2, x);
      u[2 * t] = y.x;
      u[2 * t + 1] = y.y;
    }
    f.w[0] = uint4{u[0], u[1], u[2], u[3]};
  }
  return f;
}

// acc += weights times values of 32 staged rows from r0 (a multiple of 32), over the seen pairs alone: bit i of a lane's `seen`
// stands for its element i, whose row win_mma's layout gives.  By vector instructions, row after row, which only results that
// are not finite ask for: backward, bf16, one NaN in the gradient of 32 heads of 16384 x 128, window 4096, 10 ms (4.2 without it; 900
// with rows and keys taken alone by a wave each), a gradient that is NaN throughout of 8 x 16 heads of 4096 x 64, window 1024, 2.5
// ms (0.87; 344).
template <int P, int IN>
__device__ __forceinline__ void win_add_seen(floatx16 (&acc)[P / 32], const floatx16& weights, uint32_t seen, const uint4* lds,
                                             int r0, int lane) {
  constexpr int ES = IN == F32 ? 4 : 2, E = 16 / ES, CH = win_chunks<ES>(P);
  floatx16 w = weights;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = r0 + 8 * (i >> 2) + 4 * half + (i & 3), from = (lane & 31) + 32 * half;
      const float p = __shfl(w[0], from);
      const bool in = __shfl(static_cast<int>(seen), from) & 1;
#pragma unroll
      for (int mt = 0; mt < P / 32; ++mt) {
        // the columns of the lane's accumulator elements, four neighbours at a time
        uint32_t v[4][ES];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = 32 * mt + 8 * c + 4 * (lane >> 5);
          const uint4* unit = lds + r * CH + ((col / E) ^ win_swizzle<CH>(r));
          __builtin_memcpy(v[c], __builtin_assume_aligned(reinterpret_cast<const char*>(unit) + col % E * ES, 4 * ES), 4 * ES);
        }
        if (in) {
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[mt][e] = fmaf(p, load_elem(v[e >> 2], e & 3, IN), acc[mt][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < 15; ++j) w[j] = w[j + 1];
    seen >>= 1;
  }
}

// 8 dimensions at column 16 s + 8 h of a row in memory (none of a row of width 0), with the sign of the scale in `flip`
template <int IN>
__device__ __forceinline__ WinFrag<IN> win_load_row(const char* row, int s, int h, int width, uint32_t flip) {
  constexpr int ES = IN == F32 ? 4 : 2;
  WinFrag<IN> f;
#pragma unroll
  for (int i = 0; i < (IN == F32 ? 2 : 1); ++i) {
    const uint4 u = rows_unit<ES>(row, 16 * s + 8 * h + 4 * i, width);
    f.w[i] = uint4{u.x ^ flip, u.y ^ flip, u.z ^ flip, u.w ^ flip};
  }
  return f;
}

// Keeps the operands of a lane whose row is one; others are zero.
template <int IN>
__device__ __forceinline__ void win_keep(WinFrag<IN>& f, bool row) {
#pragma unroll
  for (int i = 0; i < (IN == F32 ? 2 : 1); ++i)
    f.w[i] = uint4{row ? f.w[i].x : 0u, row ? f.w[i].y : 0u, row ? f.w[i].z : 0u, row ? f.w[i].w : 0u};
}

// waves a SIMD of window_dkv_kernel
template <int P, int IN>
__host__ __device__ constexpr int win_dkv_waves() { return IN != F32 && P <= 64 ? (P > 32 ? 2 : 3) : 1; }
// whether its instructions are laid out by hand
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr bool win_pipe() { return !SHARE && IN != F32 && win_dkv_waves<P, IN>() == 1; }

// keeps x in accumulation registers, where a kernel has both kinds (the compiler else moves sums there and back)
template <bool PIN>
__device__ __forceinline__ void win_pin(floatx16& x) {
  if constexpr (PIN) asm volatile("" : "+a"(x));
}

// fp16's gradients of logits, p (do.v - D), are carried times a power of two: at first the weights' `lift`, and where one of a
// row (dq; of a key: dk) would pass 65504 a lower one for that row alone, from there on, with what was summed before
// lowered too.  Then the largest is between 2^11 and 2^12, so what the others lose below fp16's normal range is at most 2^-36
// of it.  (With the lift alone such rows and keys came out infinite and were taken again one by one: 8 x 16 heads of 4096 x 64,
// window 1024, unit normal gradients times 1 / 64 / 1024: 0.78 / 13.8 / 338 ms; so 0.79 / 0.75 / 0.80.)
// The factor by which operands up to `big` are lowered; infinities stay.
__device__ __forceinline__ float win_lower(float big) {
  const uint32_t e = __float_as_uint(big) >> 23;
  return big > 65504.f && e < 255u ? __uint_as_float((265u - e) << 23) : 1.f;
}
// the largest magnitude of a lane's elements (NaN left out)
__device__ __forceinline__ float win_largest(const floatx16& x) {
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(x[i]));
  return big;
}

__device__ __forceinline__ bool win_finite(float x) { return fabsf(x) < __builtin_inff(); }

// four values of a row at column col (a multiple of 4) of a dense [.., width] tensor
template <int IN>
__device__ __forceinline__ void win_store4(void* base, int64_t row_at, int col, int width, float a, float b, float c,
                                           float d) {
  const int64_t at = row_at + col;
  if (col + 4 <= width && (width & 3) == 0) {
    if constexpr (IN == F32) {
      *reinterpret_cast<floatx4*>(static_cast<float*>(base) + at) = floatx4{a, b, c, d};
    } else {
      uint2 u;
      if constexpr (IN == F16) {
        u.x = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{a, b}), win_half2));
        u.y = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{c, d}), win_half2));
      } else {
        u.x = pk_bf16(a, b);
        u.y = pk_bf16(c, d);
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = u;
    }
    return;
  }
  if (col < width) store_elem(base, at, IN, a);
  if (col + 1 < width) store_elem(base, at + 1, IN, b);
  if (col + 2 < width) store_elem(base, at + 2, IN, c);
  if (col + 3 < width) store_elem(base, at + 3, IN, d);
}

// what the rounding of x to the rows' type leaves (0 of an infinity or NaN)
template <int IN>
__device__ __forceinline__ float win_rest(float x) {
  float y;
  if constexpr (IN == F16)
    y = static_cast<float>(static_cast<_Float16>(x));
  else
    y = __uint_as_float(pk_bf16(x, 0.f) << 16);
  return win_finite(y) ? x - y : 0.f;
}

// four values of a row of out, and of what their rounding leaves
template <int IN>
__device__ __forceinline__ void win_store_out(const WinArgs& a, int64_t row_at, int col, float x0, float x1, float x2,
                                              float x3) {
  win_store4<IN>(a.out, row_at, col, a.dv, x0, x1, x2, x3);
  if constexpr (IN != F32) {
    if (a.rest)
      win_store4<IN>(a.rest, row_at, col, a.dv, win_rest<IN>(x0), win_rest<IN>(x1), win_rest<IN>(x2), win_rest<IN>(x3));
  }
}

__device__ __forceinline__ int win_length(const WinArgs& a, int b) {
  if (!a.lengths) return a.n;
  const int len = a.lengths[b];
  return len < 0 ? 0 : (len > a.n ? a.n : len);
}

// Two ways to deal out a head's rows.  Wide: 128 rows (keys) a workgroup, 32 a wave, which share the staged tiles of the
// other side.  Shared, for grids that would leave compute units idle: 32 rows a workgroup, whose four waves stage and
// take every fourth tile of the other side by themselves and are joined through LDS: four times the workgroups, each a
// quarter as long.
template <bool SHARE>
__host__ __device__ constexpr int win_rows() { return SHARE ? 32 : WIN_ROWS; }
// whether a tile's rows are loaded while the one before computes: not where a wave would hold 128 registers of them
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr bool win_ahead() { return !(SHARE && IN == F32 && P > 64); }
template <bool SHARE>
__device__ __forceinline__ void win_sync() {
  if constexpr (SHARE) {  // a wave's LDS accesses are in order; the fences keep the compiler's order
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  } else {
    __syncthreads();
  }
}

// The accumulators of the four waves in LDS, [wave][32 rows][P + 4], and their sums with weights f: 4 columns (a
// multiple of 4 from col) of row threadIdx.x / 8
template <int P>
__host__ __device__ constexpr int win_join_floats() { return 4 * 32 * (P + 4); }
template <int P>
__device__ __forceinline__ void win_join_put(float* red, const floatx16 (&acc)[P / 32], int wave, int lane) {
#pragma unroll
  for (int mt = 0; mt < P / 32; ++mt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<floatx4*>(&red[(wave * 32 + (lane & 31)) * (P + 4) + 32 * mt + 8 * r + 4 * (lane >> 5)]) =
          floatx4{acc[mt][4 * r], acc[mt][4 * r + 1], acc[mt][4 * r + 2], acc[mt][4 * r + 3]};
}
template <int P>
__device__ __forceinline__ floatx4 win_join_get(const float* red, int col, const float (&f)[4]) {
  floatx4 s = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 4; ++w)
    s += *reinterpret_cast<const floatx4*>(&red[(w * 32 + threadIdx.x / 8) * (P + 4) + col]) * f[w];
  return s;
}
__device__ __forceinline__ int win_bad4(const floatx4& x) {
  return !(win_finite(x[0]) && win_finite(x[1]) && win_finite(x[2]) && win_finite(x[3]));
}

// Results that are finite are stored by a first pass over the tiles, the others by a second, careful one, which every thread of
// the workgroup takes if one result is not.  A pass is told which lanes' results were left, and tells.  It costs the first
// pass up to 4 % (registers, a barrier at its end).
template <typename Pass>
__device__ __forceinline__ void win_passes(Pass pass) {
  __shared__ int more;
  if (threadIdx.x == 0) more = 0;  // a barrier lies between this and a result
  const int bad = pass(std::false_type{}, 0);
  if (__any(bad)) more = 1;
  __syncthreads();
  if (more) pass(std::true_type{}, bad);
}

// Which (batch, query head, tile) a workgroup takes: the heads of a group and the neighbouring tiles of a head on one
// XCD, whose L2 then holds the keys they share; the last tiles (most keys) first.
__device__ __forceinline__ void win_place(const WinArgs& a, int& b, int& h, int& tile) {
  int id = xcd_remap(blockIdx.x, gridDim.x);
  const int g = id % a.group;
  id /= a.group;
  tile = a.tiles - 1 - id % a.tiles;
  id /= a.tiles;
  const int kv = a.heads / a.group;
  h = id % kv * a.group + g;
  b = id / kv;
}

// waves a SIMD of the forward and the dq kernel: what their first pass has room for (the second one may spill)
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr int win_row_waves() {
  return P > 64 ? (IN == F32 ? 1 : 2) : (IN == F32 && SHARE ? 2 : (P == 64 ? 3 : 4));
}
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr int win_dq_waves() {
  if (IN == F32) return P > 64 || (SHARE && P > 32) ? 1 : (P > 32 || SHARE ? 2 : 3);
  return SHARE && P > 96 ? 1 : (SHARE || P > 64 ? 2 : (P > 32 ? 3 : 4));
}
template <int IN, bool SHARE>
__host__ __device__ constexpr int win_keys() { return IN == F32 || SHARE ? 32 : 64; }
// LDS of the forward and the dq kernel
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr int win_lds_bytes() {
  const int stage = 2 * win_keys<IN, SHARE>() * P * (IN == F32 ? 4 : 2);
  if (!SHARE) return stage;
  const int join = 4 * (win_join_floats<P>() + 2 * 4 * 32);
  return 4 * stage > join ? 4 * stage : join;
}

// The forward kernel's weights relative to the running maximum: at most 2^room, before it moves, and carried times 2^lift.
// fp16 ends at 2^16, and below 2^-14 it holds steps of 2^-24 only: with 2^11 a weight loses at most 2^-36 of the row's largest,
// less than the output's rounding for up to 2^24 keys (2^-25 as they are: any number of keys of weight 2^-26 next to one
// of weight 1 would be lost).
template <int IN>
__host__ __device__ constexpr float win_weight_room() { return IN == F16 ? 4.f : 8.f; }
template <int IN>
__host__ __device__ constexpr float win_weight_lift() { return IN == F16 ? 11.f : 0.f; }

// Row tiles: keys staged win_keys at a time, the next tile's rows in registers while this one computes, softmax in one
// pass.  The weights of 16-bit rows enter the second product rounded to their type (half a step each, errors that
// average over the keys and end below the output's own rounding); their sum is taken before that, in fp32.
// Measured, bf16: 32 heads of 16384 rows, 128 wide, window 4096: 1.10 ms, 880 TFLOP/s, bound by the products (a large
// matrix product reaches 1180).  8 x 16 heads of 4096 rows, 64 wide, window 1024: 0.20 ms, 600 TFLOP/s, bound by the vector
// unit: a tile of 64 keys takes 16 products (512 cycles of the matrix unit) but 32 exponentials, a quarter of the rate,
// and about 150 other instructions (1100 cycles); 4 waves a SIMD instead of 3 change nothing.
template <int P, int IN, bool SHARE, bool CAREFUL>
__device__ __forceinline__ int window_forward_pass(const WinArgs& a, int again) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), BK = win_keys<IN, SHARE>(), NSUB = BK / 32,
                MT = P / 32, STEP = SHARE ? 4 : 1;
  extern __shared__ uint4 win_lds[];
  int b, h, tile;
  win_place(a, b, h, tile);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  uint4 *const ks = win_lds + (SHARE ? wave * 2 * BK * CH : 0), *const vs = ks + BK * CH;
  const int len = win_length(a, b), hk = h / a.group;
  const int r0 = tile * win_rows<SHARE>(), w0 = r0 + (SHARE ? 0 : 32 * wave), row = w0 + (lane & 31);
  const int64_t head_row = (static_cast<int64_t>(b) * a.heads + h) * a.n;

  constexpr bool AHEAD = !CAREFUL && win_ahead<P, IN, SHARE>();
  int bad = 0;
  floatx16 acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[mt][i] = 0.f;
  // finite: exp2(m_old - m_new) is 0 or at most 1, never a NaN; rows whose logits are all below have no weights, and are bad
  float m = CAREFUL ? -3.4e38f : -1e30f, limit = m, l = 0.f;
  const float room = win_weight_room<IN>() / a.c;

  if (r0 < len) {
    WinFrag<IN> qf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* qrow = rows_at<ES>(a.q, b, h, row < len ? row : 0);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      qf[s] = win_load_row<IN>(qrow, s, hh, a.d, flip);
      win_keep<IN>(qf[s], row < len);
    }

    const int last = (r0 + win_rows<SHARE>() < len ? r0 + win_rows<SHARE>() : len) - 1;
    const int t_lo = (r0 - a.window + 1 > 0 ? r0 - a.window + 1 : 0) / BK;
    int n_sink = (a.sinks + BK - 1) / BK;
    if (n_sink > t_lo) n_sink = t_lo;
    const int count = n_sink + last / BK - t_lo + 1;
    WinStage<P, IN, BK, SHARE ? 64 : 256> kst, vst;
    auto first_key = [&](int it) { return (it < n_sink ? it : t_lo + it - n_sink) * BK; };
    kst.init(a.k, a.d);
    vst.init(a.v, a.dv);
    auto load = [&](int it) {
      const int row = first_key(it);
      kst.load(rows_at<ES>(a.k, b, hk, row), len - row);
      vst.load(rows_at<ES>(a.v, b, hk, row), len - row);
    };
    const int start = SHARE ? wave : 0;
    if (AHEAD && start < count) load(start);
    for (int it = start; it < count; it += STEP) {
      if (!AHEAD) load(it);
      win_sync<SHARE>();
      const int key0 = first_key(it);
      kst.put(ks, len - key0);
      vst.put(vs, len - key0);
      win_sync<SHARE>();
      if (AHEAD && it + STEP < count) load(it + STEP);
      // of the wave's rows, does one see one of the keys; do all see all of them
      const bool some = key0 <= w0 + 31 && w0 < len && (w0 - (key0 + BK - 1) < a.window || key0 < a.sinks);
      if (!some) continue;
      const bool all = (key0 + BK - 1 <= w0) & ((w0 + 31 - key0 < a.window) | (key0 + BK <= a.sinks));
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
        // key <= row within the window in one comparison; of the sinks those up to the row
        const int ahead = row - key0 - 4 * hh, sinks = min(a.sinks, row + 1) - key0 - 4 * hh;
        const bool far = key0 < a.sinks;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 32 * sub + 8 * (i >> 2) + (i & 3);
            bool seen = static_cast<uint32_t>(ahead - k) < static_cast<uint32_t>(a.window);
            if (far) seen = seen | (k < sinks);
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
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[mt][i] *= shrink;
        m = top;
        limit = m + room;
      }
      const float mc = m * a.c - win_weight_lift<IN>();
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          // a product m c of more than 2^31 is off by more than an exponent holds: such rows are bad too
          if constexpr (CAREFUL)
            x[sub][i] = __builtin_amdgcn_exp2f(fmaf(x[sub][i] - m, a.c, win_weight_lift<IN>()));
          else
            x[sub][i] = __builtin_amdgcn_exp2f(fmaf(x[sub][i], a.c, -mc));
        }
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) l += x[sub][i];
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
    l += __shfl_xor(l, 32);
  }

  if constexpr (SHARE) {
    float *red = reinterpret_cast<float*>(win_lds), *red_m = red + win_join_floats<P>(), *red_l = red_m + 4 * 32;
    __syncthreads();
    win_join_put<P>(red, acc, wave, lane);
    if (hh == 0) {
      red_m[32 * wave + lane] = m;
      red_l[32 * wave + lane] = l;
    }
    __syncthreads();
    const int r = threadIdx.x / 8, at_row = r0 + r;
    float top = red_m[r], den = 0.f, f[4];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, red_m[32 * w + r]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = __builtin_amdgcn_exp2f((red_m[32 * w + r] - top) * a.c);
      den = fmaf(f[w], red_l[32 * w + r], den);
    }
    const bool in = at_row < len;
    if (CAREFUL && !(den > 0.f)) den = __builtin_nanf("");  // no logit above -inf
    const float inv = in ? 1.f / den : 0.f;
    floatx4 o[MT];
    bad = !(den > 0.f && win_finite(den));
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      o[j] = win_join_get<P>(red, 32 * j + 4 * (threadIdx.x & 7), f);
      bad |= win_bad4(o[j]);
    }
    bad = in ? bad : 0;
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) bad |= __shfl_xor(bad, x);
    if (at_row < a.n && (CAREFUL ? again : !bad)) {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int col = 32 * j + 4 * (threadIdx.x & 7);
        if (col < a.dv)
          win_store_out<IN>(a, (head_row + at_row) * a.dv, col, in ? o[j][0] * inv : 0.f, in ? o[j][1] * inv : 0.f,
                            in ? o[j][2] * inv : 0.f, in ? o[j][3] * inv : 0.f);
      }
      if (a.lse && (threadIdx.x & 7) == 0)
        a.lse[head_row + at_row] = in ? top * a.c - win_weight_lift<IN>() + __builtin_amdgcn_logf(den) : 0.f;
    }
    return bad;
  }

  const bool in = row < len;
  float inv = 0.f;
  if (in) {
    if (CAREFUL && !(l > 0.f)) l = __builtin_nanf("");
    inv = 1.f / l;
    bad = !(l > 0.f && win_finite(l));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) bad |= !win_finite(acc[mt][i]);
  }
  bad |= __shfl_xor(bad, 32);
  if (row < a.n && (CAREFUL ? again : !bad)) {
    const int64_t at = (head_row + row) * a.dv;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * mt + 8 * r + 4 * hh;
        if (col < a.dv)
          win_store_out<IN>(a, at, col, in ? acc[mt][4 * r] * inv : 0.f, in ? acc[mt][4 * r + 1] * inv : 0.f,
                            in ? acc[mt][4 * r + 2] * inv : 0.f, in ? acc[mt][4 * r + 3] * inv : 0.f);
      }
    if (a.lse && hh == 0) a.lse[head_row + row] = in ? m * a.c - win_weight_lift<IN>() + __builtin_amdgcn_logf(l) : 0.f;
  }
  return bad;
}

template <int P, int IN, bool SHARE>
__global__ __launch_bounds__(256, (win_row_waves<P, IN, SHARE>())) void window_forward_kernel(const WinArgs a) {
  win_passes([&](auto second, int again) { return window_forward_pass<P, IN, SHARE, decltype(second)::value>(a, again); });
}

// dq and D: the forward kernel's walk over the keys with the rows' statistics given.  D of a rounded out is off by do.(out -
// o), the same for all keys of a row, which adds about a tenth to the gradients' rounding errors (a third with windows of 16
// keys); with what the rounding left (rest) it is not.  ds is rounded to the rows' type for
// its product with the keys like the weights of the forward kernel.  32 heads of 16384 rows, 128 wide, window 4096,
// bf16: 1.48 ms, three products at 975 TFLOP/s, bound by them; 8 x 16 heads of 4096 rows, 64 wide, window 1024: 291 us with
// three waves a SIMD (one register less a lane than the compiler takes by itself), 316 with two.
template <int P, int IN, bool SHARE, bool CAREFUL>
__device__ __forceinline__ int window_dq_pass(const WinArgs& a, int again) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), BK = win_keys<IN, SHARE>(), NSUB = BK / 32,
                MT = P / 32, STEP = SHARE ? 4 : 1;
  extern __shared__ uint4 win_lds[];
  int b, h, tile;
  win_place(a, b, h, tile);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  uint4 *const ks = win_lds + (SHARE ? wave * 2 * BK * CH : 0), *const vs = ks + BK * CH;
  const int len = win_length(a, b), hk = h / a.group;
  const int r0 = tile * win_rows<SHARE>(), w0 = r0 + (SHARE ? 0 : 32 * wave), row = w0 + (lane & 31);
  const int64_t head_row = (static_cast<int64_t>(b) * a.heads + h) * a.n;
  const bool in = row < len;

  constexpr bool AHEAD = !CAREFUL && win_ahead<P, IN, SHARE>();
  int bad = 0;
  floatx16 acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[mt][i] = 0.f;
  float delta = 0.f, drop = a.drop;
  bool lost = false;  // the row's statistics are NaN, and with them all of its gradient

  if (r0 < len) {
    WinFrag<IN> qf[P / 16], gf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* qrow = rows_at<ES>(a.q, b, h, in ? row : 0);
    const char* grow = rows_at<ES>(a.go, b, h, in ? row : 0);
    const int64_t orow_at = (head_row + (in ? row : 0)) * a.dv * ES;
    const char* orow = static_cast<const char*>(a.out) + orow_at;
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      qf[s] = win_load_row<IN>(qrow, s, hh, a.d, flip);
      gf[s] = win_load_row<IN>(grow, s, hh, a.dv, 0u);
      WinFrag<IN> o = win_load_row<IN>(orow, s, hh, a.dv, 0u);
      win_keep<IN>(qf[s], in);
      win_keep<IN>(gf[s], in);
      win_keep<IN>(o, in);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(load_elem(&gf[s], j, IN), load_elem(&o, j, IN), delta);
      if constexpr (IN != F32) {
        if (a.rest) {
          o = win_load_row<IN>(static_cast<const char*>(a.rest) + orow_at, s, hh, a.dv, 0u);
          win_keep<IN>(o, in);
#pragma unroll
          for (int j = 0; j < 8; ++j) delta = fmaf(load_elem(&gf[s], j, IN), load_elem(&o, j, IN), delta);
        }
      }
    }
    delta += __shfl_xor(delta, 32);
    const float lse = in ? a.lse[head_row + row] : 0.f;
    lost = delta != delta || lse != lse;
    if (in && hh == 0 && (!SHARE || wave == 0)) a.delta[head_row + row] = delta;

    const int last = (r0 + win_rows<SHARE>() < len ? r0 + win_rows<SHARE>() : len) - 1;
    const int t_lo = (r0 - a.window + 1 > 0 ? r0 - a.window + 1 : 0) / BK;
    int n_sink = (a.sinks + BK - 1) / BK;
    if (n_sink > t_lo) n_sink = t_lo;
    const int count = n_sink + last / BK - t_lo + 1;
    WinStage<P, IN, BK, SHARE ? 64 : 256> kst, vst;
    auto first_key = [&](int it) { return (it < n_sink ? it : t_lo + it - n_sink) * BK; };
    kst.init(a.k, a.d);
    vst.init(a.v, a.dv);
    auto load = [&](int it) {
      const int row = first_key(it);
      kst.load(rows_at<ES>(a.k, b, hk, row), len - row);
      vst.load(rows_at<ES>(a.v, b, hk, row), len - row);
    };
    const int start = SHARE ? wave : 0;
    if (AHEAD && start < count) load(start);
    float shift = __builtin_amdgcn_logf(a.lift) - lse;
    for (int it = start; it < count; it += STEP) {
      if (!AHEAD) load(it);
      win_sync<SHARE>();
      const int key0 = first_key(it);
      kst.put(ks, len - key0);
      vst.put(vs, len - key0);
      win_sync<SHARE>();
      if (AHEAD && it + STEP < count) load(it + STEP);
      const bool some = key0 <= w0 + 31 && w0 < len && (w0 - (key0 + BK - 1) < a.window || key0 < a.sinks);
      if (!some) continue;
      const bool all = (key0 + BK - 1 <= w0) & ((w0 + 31 - key0 < a.window) | (key0 + BK <= a.sinks));
#pragma unroll
      for (int sub = 0; sub < NSUB; ++sub) {
        floatx16 x, g;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = g[i] = 0.f;
#pragma unroll
        for (int s = 0; s < P / 16; ++s) {
          win_mma<IN>(x, win_read_row<P, IN>(ks, 32 * sub + (lane & 31), s, hh), qf[s]);
          win_mma<IN>(g, win_read_row<P, IN>(vs, 32 * sub + (lane & 31), s, hh), gf[s]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], a.c, shift)) * (g[i] - delta);
        uint32_t pairs = 0;
        if (!all) {
          const int ahead = row - key0 - 4 * hh, sinks = min(a.sinks, row + 1) - key0 - 4 * hh;
          const bool far = key0 < a.sinks;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = 32 * sub + 8 * (i >> 2) + (i & 3);
            bool seen = static_cast<uint32_t>(ahead - k) < static_cast<uint32_t>(a.window);
            if (far) seen = seen | (k < sinks);
            x[i] = seen ? x[i] : 0.f;
            if constexpr (CAREFUL) pairs |= static_cast<uint32_t>(seen) << i;
          }
        }
        if constexpr (IN == F16) {
          float big = win_largest(x);
          if (__any(big > 65504.f)) {
            big = fmaxf(big, __shfl_xor(big, 32));
            const float f = win_lower(big);
            drop /= f;
            shift += __builtin_amdgcn_logf(f);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[mt][i] *= f;
          }
        }
        if (CAREFUL && !all) {
          win_add_seen<P, IN>(acc, x, pairs, ks, 32 * sub, lane);
          continue;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const WinFrag<IN> p = win_operand<IN>(x, t);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            win_mma<IN>(acc[mt], win_read_columns<P, IN>(ks, 32 * sub + 16 * t, mt, lane), p);
        }
      }
    }
  }

  if constexpr (SHARE) {
    float *red = reinterpret_cast<float*>(win_lds), *red_d = red + win_join_floats<P>();
    float weight[4] = {1.f, 1.f, 1.f, 1.f};
    __syncthreads();
    win_join_put<P>(red, acc, wave, lane);
    if (IN == F16 && hh == 0) red_d[32 * wave + lane] = drop;
    __syncthreads();
    if constexpr (IN == F16) {
#pragma unroll
      for (int w = 0; w < 4; ++w) weight[w] = red_d[32 * w + threadIdx.x / 8];
    }
    const int at_row = r0 + threadIdx.x / 8;
    lost = __shfl(static_cast<int>(lost), threadIdx.x / 8);
    const float f = lost ? __builtin_nanf("") : a.scale;
    floatx4 o[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      o[j] = win_join_get<P>(red, 32 * j + 4 * (threadIdx.x & 7), weight);
      bad |= win_bad4(o[j]);
    }
    bad = at_row < len && !lost ? bad : 0;
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) bad |= __shfl_xor(bad, x);
    if (at_row < a.n && (CAREFUL ? again : !bad)) {
      const bool real = at_row < len;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int col = 32 * j + 4 * (threadIdx.x & 7);
        if (col < a.d)
          win_store4<IN>(a.dq, (head_row + at_row) * a.d, col, a.d, real ? o[j][0] * f : 0.f, real ? o[j][1] * f : 0.f,
                         real ? o[j][2] * f : 0.f, real ? o[j][3] * f : 0.f);
      }
    }
    return bad;
  }

  if (in && !lost) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) bad |= !win_finite(acc[mt][i]);
  }
  bad |= __shfl_xor(bad, 32);
  if (row < a.n && (CAREFUL ? again : !bad)) {
    const int64_t at = (head_row + row) * a.d;
    const float f = lost ? __builtin_nanf("") : a.scale * drop;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * mt + 8 * r + 4 * hh;
        if (col < a.d)
          win_store4<IN>(a.dq, at, col, a.d, in ? acc[mt][4 * r] * f : 0.f, in ? acc[mt][4 * r + 1] * f : 0.f,
                         in ? acc[mt][4 * r + 2] * f : 0.f, in ? acc[mt][4 * r + 3] * f : 0.f);
      }
  }
  return bad;
}

template <int P, int IN, bool SHARE>
__global__ __launch_bounds__(256, (win_dq_waves<P, IN, SHARE>())) void window_dq_kernel(const WinArgs a) {
  win_passes([&](auto second, int again) { return window_dq_pass<P, IN, SHARE, decltype(second)::value>(a, again); });
}

// Rows that window_dkv_kernel stages at a time, and its LDS: two stages of query and gradient rows and their statistics
// (shared: one stage a wave).
template <int IN, bool SHARE>
__host__ __device__ constexpr int win_staged_rows() { return IN == F32 || SHARE ? 32 : 64; }
template <int P, int IN, bool SHARE>
__host__ __device__ constexpr int win_dkv_lds() {
  const int rows = win_staged_rows<IN, SHARE>(), stage = 2 * rows * P * (IN == F32 ? 4 : 2) + 2 * rows * 4;
  if (!SHARE) return (win_pipe<P, IN, SHARE>() ? 3 : 2) * stage;
  const int join = 4 * (win_join_floats<P>() + 4 * 32);
  return 4 * stage > join ? 4 * stage : join;
}

// dk and dv: one workgroup per 128 keys of a key head (32 a wave) walks over the rows that see them within the window,
// for every head of the group; the rows behind the window of a sink go to workgroups of their own (far), whose
// sums, like those of the sinks' own tiles, are added by window_sink_kernel in their order.  p and ds are rounded to
// the rows' type for their products like the weights of the forward kernel.
// dk and dv of 32 keys of 128 columns take 128 registers a lane and the keys' operands 64, so a compute unit holds one wave
// a SIMD above 64 columns.  PIPE (16-bit rows): that wave's instructions are laid out by hand, see below; without it (SHARE) the
// operands are at least read ahead.  32 heads of 16384 rows over 8 key heads, 128 wide,
// window 4096, bf16: 2.44 ms, four products at 790 TFLOP/s (before it had a second pass 2.37, and 3.03 without PIPE; operands
// read two steps ahead 2.48, three 2.37, four 2.33; dk and dv in kernels of their own, 5 products but two waves a SIMD, 3.45; 93
// wide, 4 x 16 heads of 4096 rows, window 1024, with dq 841 us, 923 without PIPE).  What is left: about 300
// instructions a wave issues for 32 rows, one at a time, against 1024 cycles of the matrix unit.
// Up to 64 columns two waves a SIMD fill each other's waits better than PIPE does: 8 x 16 heads of 4096 rows, 64 wide, window
// 1024, 515 us (PIPE with one wave 722, with two, which spill, 714); 32 heads of 16384 over 8 key heads, window 4096, 1.36
// ms (1.73); 32 wide 265 us (314); 96 wide the other way round: 4 x 16 heads over 4 key heads 359 us with PIPE, 411 with two waves.
// FULL: both widths are the padded one (with PIPE).
template <int P, int IN, bool SHARE, bool FULL, bool CAREFUL>
__device__ __forceinline__ int window_dkv_pass(const WinArgs& a, int again) {
  constexpr int ES = IN == F32 ? 4 : 2, CH = win_chunks<ES>(P), MT = P / 32, BQ = win_staged_rows<IN, SHARE>(),
                NSUB = BQ / 32, TILE = win_rows<SHARE>(), THREADS = SHARE ? 64 : 256;
  constexpr int STAGE = 2 * BQ * CH;  // 16-byte units of a stage
  constexpr int WAVES = win_dkv_waves<P, IN>();
  constexpr bool PIPE = win_pipe<P, IN, SHARE>();
  extern __shared__ uint4 win_lds[];
  constexpr int STAGES = SHARE ? 4 : (PIPE ? 3 : 2);  // of the waves, or of tiles
  float* const stats = reinterpret_cast<float*>(win_lds + STAGES * STAGE);  // [stage][lift - lse, delta][BQ]
  const int kv = a.heads / a.group;
  const int far_items = a.sink_tiles * a.far_chunks, items = far_items + a.key_tiles;
  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int item = id % items, bh = id / items, b = bh / kv, hk = bh % kv;
  const bool far = item < far_items;
  const int chunk = far ? item / a.sink_tiles : -1;
  const int tile = far ? item % a.sink_tiles : item - far_items;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hh = lane >> 5;
  const int len = win_length(a, b);
  const int k0 = tile * TILE, kw = k0 + (SHARE ? 0 : 32 * wave), key = kw + (lane & 31);

  // rows [lo, hi] to walk over
  int lo, hi;
  if (far) {
    lo = a.window + chunk * a.far_rows;
    hi = lo + a.far_rows - 1;
    if (lo < k0 + a.window) lo = k0 + a.window;
  } else {
    lo = k0;
    hi = k0 + TILE - 1 < a.n - a.window ? k0 + TILE - 1 + a.window - 1 : a.n - 1;
  }
  if (hi > len - 1) hi = len - 1;

  constexpr bool AHEAD = !SHARE || (!CAREFUL && win_ahead<P, IN, SHARE>());
  int bad = 0;
  floatx16 dk[MT], dv[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[mt][i] = dv[mt][i] = 0.f;
  // by what the key's gradients of logits are lowered (see win_lower), and what they are looked at above: 65504, or any once one
  // of the wave's keys has been lowered
  float lower = 1.f, limit = 65504.f;
  // g as it fits
  auto fit = [&](floatx16& g) {
    if constexpr (IN == F16) {
      if (__any(win_largest(g) > limit)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] *= lower;
        float big = win_largest(g);
        big = fmaxf(big, __shfl_xor(big, 32));
        const float f = win_lower(big);
        if (!__any(f < 1.f)) return;
        lower *= f;
        limit = -1.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] *= f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          win_pin<WAVES == 1>(dk[mt]);
#pragma unroll
          for (int i = 0; i < 16; ++i) dk[mt][i] *= f;
          win_pin<WAVES == 1>(dk[mt]);
        }
      }
    }
  };

  if (lo <= hi) {
    WinFrag<IN> kf[P / 16], vf[P / 16];
    const uint32_t flip = a.scale < 0.f ? (IN == F32 ? 0x80000000u : 0x80008000u) : 0u;
    const char* krow = rows_at<ES>(a.k, b, hk, key < len ? key : 0);
    const char* vrow = rows_at<ES>(a.v, b, hk, key < len ? key : 0);
#pragma unroll
    for (int s = 0; s < P / 16; ++s) {
      kf[s] = win_load_row<IN>(krow, s, hh, a.d, flip);
      vf[s] = win_load_row<IN>(vrow, s, hh, a.dv, 0u);
      win_keep<IN>(kf[s], key < len);
      win_keep<IN>(vf[s], key < len);
    }
    const int first = lo / BQ * BQ, per_head = hi / BQ - lo / BQ + 1, count = per_head * a.group;
    const float lift = __builtin_amdgcn_logf(a.lift);
    // does the lane's key take part in row i here
    auto sees = [&](int i) {
      if (far) return i - key >= a.window && i >= lo && i <= hi && key < a.sinks;
      return static_cast<uint32_t>(i - key) < static_cast<uint32_t>(a.window);
    };
    // hidden pairs' weights and gradients
    auto hide = [&](floatx16& x, floatx16& g, int base) {
      const int ahead = base - key, from = lo - base, last = key < a.sinks ? hi - base : -1;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 8 * (i >> 2) + (i & 3);
        bool seen = static_cast<uint32_t>(ahead + r) < static_cast<uint32_t>(a.window);
        if (far) seen = (ahead + r >= a.window) & (r >= from) & (r <= last);
        x[i] = seen ? x[i] : 0.f;
        g[i] = seen ? g[i] : 0.f;
      }
    };
    // of the wave's keys, does none or do all see each of the rows [q0, q0 + rows)
    auto none = [&](int q0, int rows) {
      return far ? kw >= a.sinks || q0 + rows - 1 - kw < a.window : q0 + rows - 1 < kw || q0 - (kw + 31) >= a.window;
    };
    auto whole = [&](int q0, int rows) {
      const bool behind = (kw + 32 <= a.sinks) & (q0 - (kw + 31) >= a.window) & (q0 >= lo) & (q0 + rows - 1 <= hi);
      const bool within = (q0 >= kw + 31) & (q0 + rows - 1 - kw < a.window);
      return far ? behind : within;
    };
    if constexpr (PIPE && !CAREFUL) {
      // One wave a SIMD has nothing else to do while it waits, so its own matrix and vector instructions are interleaved:
      // the products of the next 32 rows' logits with the weights of these, the next tiles' way into LDS with the
      // sums (the barriers of the schedule keep that order).  Three stages: tile `it` and the next are written, the third is
      // being written; one __syncthreads a tile.  Rows behind the last are read as the last one, their weights are
      // exp2(-inf).  No tile is left out for a wave that sees none of it: the others' barrier waits for it anyway.
      constexpr int U = MT, E = 16 / ES;  // 16-byte units of a tensor's tile a thread, their elements
      static_assert(!PIPE || (U == BQ * CH / 256 && NSUB == 2));
      uint4 uq[U], ug[U];
      uint32_t to[U], off[2][U];
      const int pitch_q = static_cast<int>(a.q.sn) * ES, pitch_g = static_cast<int>(a.go.sn) * ES;
      const int srow = threadIdx.x % BQ;
      const bool of_lse = threadIdx.x % (2 * BQ) < BQ;
      float stat;
      int next = 0, lrow = first, lhead = hk * a.group;  // the tile to be read, its first row and head
      bool cut = true;                                   // off is not that of whole tiles
      const char *qp, *gp;
      const float* sp;
      bool srow_in;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int k = threadIdx.x + 256 * i, row = k / CH;
        to[i] = row * CH + ((k % CH) ^ win_swizzle<CH>(row));
      }
      auto aim = [&]() {
        const int left = len - lrow;
        if (cut || left < BQ) {
          cut = left < BQ;
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int k = threadIdx.x + 256 * i, row = min(k / CH, left - 1);
            off[0][i] = row * pitch_q + (FULL ? k % CH * E : min(k % CH * E, a.d - E)) * ES;
            off[1][i] = row * pitch_g + (FULL ? k % CH * E : min(k % CH * E, a.dv - E)) * ES;
          }
        }
        qp = rows_at<ES>(a.q, b, lhead, lrow);
        gp = rows_at<ES>(a.go, b, lhead, lrow);
        sp = (of_lse ? a.lse : a.delta) + (static_cast<int64_t>(b) * a.heads + lhead) * a.n + min(lrow + srow, len - 1);
        srow_in = lrow + srow < len;
        // the tile after; behind the last one, that again
        if (++next < count) {
          lrow += BQ;
          if (lrow > hi) {
            lrow = first;
            ++lhead;
          }
        }
      };
      auto read = [&](int i) {
        uq[i] = rows_load16(qp + off[0][i]);
        ug[i] = rows_load16(gp + off[1][i]);
        if (i == 0) stat = *sp;
      };
      bool stat_in;
      // a unit into its place: a row's last one moved down where it reaches over the end, none behind it
      auto place = [&](int at, uint4 x, int col, int width) {
        if (width % E) x = rows_shift(x, max(0, col + E - width) * ES & 15);
        if (col < width) win_lds[at] = x;
      };
      auto write = [&](int i, int st) {
        if constexpr (FULL) {
          win_lds[st * STAGE + to[i]] = uq[i];
          win_lds[st * STAGE + BQ * CH + to[i]] = ug[i];
        } else {
          const int col = (threadIdx.x + 256 * i) % CH * E;
          place(st * STAGE + to[i], uq[i], col, a.d);
          place(st * STAGE + BQ * CH + to[i], ug[i], col, a.dv);
        }
        if (i == 0) {
          const float x = of_lse ? lift - stat : stat;
          stats[st * 2 * BQ + threadIdx.x % (2 * BQ)] = stat_in ? x : (of_lse ? -__builtin_inff() : 0.f);
        }
      };
      if constexpr (!FULL) {  // the columns behind the widths
        for (int i = threadIdx.x; i < 3 * STAGE; i += 256) win_lds[i] = uint4{0u, 0u, 0u, 0u};
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        aim();
#pragma unroll
        for (int i = 0; i < U; ++i) read(i);
        stat_in = srow_in;
        if (j < 2) {
#pragma unroll
          for (int i = 0; i < U; ++i) write(i, j);
        }
      }
      int stage = 0;
      auto rows_of_stage = [&](int st) { return win_lds + st * STAGE; };
      floatx16 x[2], g[2];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i) x[0][i] = g[0][i] = 0.f;
#pragma unroll
      for (int s = 0; s < P / 16; ++s) {
        win_mma<IN>(x[0], win_read_row<P, IN>(win_lds, lane & 31, s, hh), kf[s]);
        win_mma<IN>(g[0], win_read_row<P, IN>(win_lds + BQ * CH, lane & 31, s, hh), vf[s]);
      }
      int q0 = first;
      for (int it = 0; it < count; ++it) {
        if (it) __syncthreads();
        const int after = stage == 2 ? 0 : stage + 1, third = after == 2 ? 0 : after + 1;
        aim();
        const uint4 *qs = rows_of_stage(stage), *gs = qs + BQ * CH;
        const floatx4* st = reinterpret_cast<const floatx4*>(stats + stage * 2 * BQ);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          win_pin<WAVES == 1>(dk[mt]);
          win_pin<WAVES == 1>(dv[mt]);
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          floatx16 &x0 = x[sub], &g0 = g[sub], &x1 = x[sub ^ 1], &g1 = g[sub ^ 1];
          // the rows after these (behind the last tile: of whatever the stage holds, not used)
          const uint4 *nq = sub ? rows_of_stage(after) : qs, *ng = nq + BQ * CH;
          const int nrow = 32 * (sub ^ 1) + (lane & 31);
          floatx4 shift[4], delta[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            shift[r] = st[8 * sub + 2 * r + hh];
            delta[r] = st[BQ / 4 + 8 * sub + 2 * r + hh];
          }
          constexpr int STEPS = P / 16, LEAD = STEPS < 3 ? STEPS : 3;
          WinFrag<IN> qa[STEPS], ga[STEPS], qc[2][MT], gc[2][MT];
#pragma unroll
          for (int i = 0; i < 16; ++i) x1[i] = g1[i] = 0.f;
#pragma unroll
          for (int s = 0; s < LEAD; ++s) {
            qa[s] = win_read_row<P, IN>(nq, nrow, s, hh);
            ga[s] = win_read_row<P, IN>(ng, nrow, s, hh);
          }
          __builtin_amdgcn_sched_barrier(0);
          auto weigh = [&](int i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(x0[i], a.c, shift[i >> 2][i & 3]));
            g0[i] = p * (g0[i] - delta[i >> 2][i & 3]);
            x0[i] = p;
          };
#pragma unroll
          for (int s = 0; s < STEPS; ++s) {
            if (s + LEAD < STEPS) {
              qa[s + LEAD] = win_read_row<P, IN>(nq, nrow, s + LEAD, hh);
              ga[s + LEAD] = win_read_row<P, IN>(ng, nrow, s + LEAD, hh);
            }
            if (s == STEPS - 2) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) gc[0][mt] = win_read_columns<P, IN>(gs, 32 * sub, mt, lane);
            }
            if (s == STEPS - 1) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) qc[0][mt] = win_read_columns<P, IN>(qs, 32 * sub, mt, lane);
            }
            win_mma<IN>(x1, qa[s], kf[s]);
            const int from = 16 * s / STEPS, to = 16 * (s + 1) / STEPS, half = (from + to) / 2;
#pragma unroll
            for (int i = from; i < half; ++i) weigh(i);
            __builtin_amdgcn_sched_barrier(0);
            win_mma<IN>(g1, ga[s], vf[s]);
#pragma unroll
            for (int i = half; i < to; ++i) weigh(i);
            __builtin_amdgcn_sched_barrier(0);
          }
          asm volatile("" : "+v"(x0), "+v"(g0));
          if (__builtin_expect(!whole(q0 + 32 * sub, 32), 0)) hide(x0, g0, q0 + 32 * sub + 4 * hh);
          fit(g0);
          WinFrag<IN> p[2], ds[2];
          p[0] = win_operand<IN>(x0, 0);
          ds[0] = win_operand<IN>(g0, 0);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            gc[1][mt] = win_read_columns<P, IN>(gs, 32 * sub + 16, mt, lane);
            qc[1][mt] = win_read_columns<P, IN>(qs, 32 * sub + 16, mt, lane);
            win_mma<IN>(dv[mt], gc[0][mt], p[0]);
            win_mma<IN>(dk[mt], qc[0][mt], ds[0]);
            if (mt == 0) {
              p[1] = win_operand<IN>(x0, 1);
              ds[1] = win_operand<IN>(g0, 1);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            win_mma<IN>(dv[mt], gc[1][mt], p[1]);
            win_mma<IN>(dk[mt], qc[1][mt], ds[1]);
            if (sub == 0) {
              write(mt, third);
              read(mt);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (sub == 0) stat_in = srow_in;
        }
        stage = after;
        q0 += BQ;
        if (q0 > hi) q0 = first;
      }
    } else {
      WinStage<P, IN, BQ, THREADS> qst, gst;
      qst.init(a.q, a.d);
      gst.init(a.go, a.dv);
      float stat = 0.f;
      const int self = threadIdx.x % THREADS;
      auto row_of = [&](int it) { return first + it % per_head * BQ; };
      auto load = [&](int it) {
        const int row0 = row_of(it), h = hk * a.group + it / per_head;
        qst.load(rows_at<ES>(a.q, b, h, row0), len - row0);
        gst.load(rows_at<ES>(a.go, b, h, row0), len - row0);
        if (self < 2 * BQ) {
          const int row = row0 + self % BQ;
          const float* from = self < BQ ? a.lse : a.delta;
          stat = row < len ? from[(static_cast<int64_t>(b) * a.heads + h) * a.n + row] : 0.f;
          if (self < BQ) stat = lift - stat;
        }
      };
      auto put = [&](int it, int stage) {
        qst.put(win_lds + stage * STAGE, len - row_of(it));
        gst.put(win_lds + stage * STAGE + BQ * CH, len - row_of(it));
        if (self < 2 * BQ) stats[stage * 2 * BQ + self] = stat;
      };
      const int start = SHARE ? wave : 0, step = SHARE ? 4 : 1;
      if (AHEAD && start < count) load(start);
      if constexpr (!SHARE) {
        put(0, 0);
        if (count > 1) load(1);
      }
      for (int it = start; it < count; it += step) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          win_pin<WAVES == 1>(dk[mt]);
          win_pin<WAVES == 1>(dv[mt]);
        }
        int stage = wave;
        if (!AHEAD) load(it);
        win_sync<SHARE>();
        if constexpr (SHARE) {
          put(it, wave);
          win_sync<SHARE>();
          if (AHEAD && it + step < count) load(it + step);
        } else {  // stage `it` is written, the other one read
          stage = it & 1;
          if (it + 1 < count) put(it + 1, stage ^ 1);
          if (it + 2 < count) load(it + 2);
        }
        const uint4 *qs = win_lds + stage * STAGE, *gs = qs + BQ * CH;
        const floatx4* st = reinterpret_cast<const floatx4*>(stats + stage * 2 * BQ);
        const int q0 = row_of(it);
        if (none(q0, BQ)) continue;
        const bool all = whole(q0, BQ);
#pragma unroll 1
        for (int sub = 0; sub < NSUB; ++sub) {
          // one wave a SIMD: every operand is read well before its product, there is nothing else to do while it waits (fp32
          // products take eight times as long as their operands' reads: those are read as they come)
          constexpr bool EARLY = IN != F32 && WAVES == 1 && !CAREFUL;
          WinFrag<IN> qa[EARLY ? P / 16 : 1], ga[EARLY ? P / 16 : 1], qc[MT], gc[MT];
          floatx16 x, g;
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = g[i] = 0.f;
          if constexpr (EARLY) {
#pragma unroll
            for (int s = 0; s < P / 16; ++s) {
              qa[s] = win_read_row<P, IN>(qs, 32 * sub + (lane & 31), s, hh);
              ga[s] = win_read_row<P, IN>(gs, 32 * sub + (lane & 31), s, hh);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int s = 0; s < P / 16; ++s) {
            if constexpr (!EARLY) {
              qa[0] = win_read_row<P, IN>(qs, 32 * sub + (lane & 31), s, hh);
              ga[0] = win_read_row<P, IN>(gs, 32 * sub + (lane & 31), s, hh);
            }
            win_mma<IN>(x, qa[EARLY ? s : 0], kf[s]);
            win_mma<IN>(g, ga[EARLY ? s : 0], vf[s]);
          }
          floatx4 shift[4], delta[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            shift[r] = st[8 * sub + 2 * r + hh];
            delta[r] = st[BQ / 4 + 8 * sub + 2 * r + hh];
          }
          if constexpr (EARLY) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              gc[mt] = win_read_columns<P, IN>(gs, 32 * sub, mt, lane);
              qc[mt] = win_read_columns<P, IN>(qs, 32 * sub, mt, lane);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(x[i], a.c, shift[i >> 2][i & 3]));
            g[i] = p * (g[i] - delta[i >> 2][i & 3]);
            x[i] = p;
          }
          if (!all) hide(x, g, q0 + 32 * sub + 4 * hh);
          fit(g);
          if (CAREFUL && !all) {
            uint32_t pairs = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) pairs |= static_cast<uint32_t>(sees(q0 + 32 * sub + 4 * hh + 8 * (i >> 2) + (i & 3))) << i;
            win_add_seen<P, IN>(dv, x, pairs, gs, 32 * sub, lane);
            win_add_seen<P, IN>(dk, g, pairs, qs, 32 * sub, lane);
            continue;
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const WinFrag<IN> p = win_operand<IN>(x, t), ds = win_operand<IN>(g, t);
            WinFrag<IN> gn[EARLY ? MT : 1], qn[EARLY ? MT : 1];
            if constexpr (EARLY) {
              if (t == 0) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  gn[mt] = win_read_columns<P, IN>(gs, 32 * sub + 16, mt, lane);
                  qn[mt] = win_read_columns<P, IN>(qs, 32 * sub + 16, mt, lane);
                }
              }
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              if constexpr (!EARLY) {
                gc[mt] = win_read_columns<P, IN>(gs, 32 * sub + 16 * t, mt, lane);
                qc[mt] = win_read_columns<P, IN>(qs, 32 * sub + 16 * t, mt, lane);
              }
              win_mma<IN>(dv[mt], gc[mt], p);
              win_mma<IN>(dk[mt], qc[mt], ds);
            }
            if constexpr (EARLY) {
              if (t == 0) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  gc[mt] = gn[mt];
                  qc[mt] = qn[mt];
                }
              }
            }
          }
        }
      }
    }
  }

  // sums to be added to others' (the sinks of a call with rows behind their window)
  const float f = a.scale * a.drop / (SHARE ? 1.f : lower);
  auto part_at = [&](int j) {
    return ((static_cast<int64_t>(bh) * (a.far_chunks + 1) + chunk + 1) * a.sink_rows + j) * (a.d + a.dv);
  };
  auto is_part = [&](int j) { return a.far_chunks > 0 && j < a.sink_rows; };
  // 4 columns of key j's dk (value 0) or dv (1), where this workgroup has any to give; zero behind the last key (a zero
  // weight times a row that is not finite may have left a NaN there)
  auto store4 = [&](int j, int value, int col, float x0, float x1, float x2, float x3) {
    const int width = value ? a.dv : a.d;
    if (col >= width) return;
    if (j >= len) x0 = x1 = x2 = x3 = 0.f;
    if (is_part(j)) {
      float* to = a.part + part_at(j) + (value ? a.d : 0);
      to[col] = x0;
      if (col + 1 < width) to[col + 1] = x1;
      if (col + 2 < width) to[col + 2] = x2;
      if (col + 3 < width) to[col + 3] = x3;
    } else if (!far && j < a.n) {
      win_store4<IN>(value ? a.dv_out : a.dk, (static_cast<int64_t>(bh) * a.n + j) * width, col, width, x0, x1, x2, x3);
    }
  };
  if constexpr (SHARE) {
    float *red = reinterpret_cast<float*>(win_lds), *red_f = red + win_join_floats<P>();
    const int j = k0 + threadIdx.x / 8;
    floatx4 o[2][MT];
#pragma unroll
    for (int value = 0; value < 2; ++value) {
      __syncthreads();
      win_join_put<P>(red, value ? dv : dk, wave, lane);
      if (IN == F16 && value == 0 && hh == 0) red_f[32 * wave + lane] = 1.f / lower;
      __syncthreads();
      float weight[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (IN == F16) {
#pragma unroll
        for (int w = 0; w < 4; ++w) weight[w] = value ? 1.f : red_f[32 * w + threadIdx.x / 8];
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        o[value][mt] = win_join_get<P>(red, 32 * mt + 4 * (threadIdx.x & 7), weight);
        bad |= win_bad4(o[value][mt]);
      }
    }
    bad = j < len ? bad : 0;
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) bad |= __shfl_xor(bad, x);
    if (CAREFUL ? again : !bad) {
#pragma unroll
      for (int value = 0; value < 2; ++value)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const floatx4 y = o[value][mt] * (value ? a.drop : f);
          store4(j, value, 32 * mt + 4 * (threadIdx.x & 7), y[0], y[1], y[2], y[3]);
        }
    }
    return bad;
  }

#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad |= !(win_finite(dk[mt][i]) && win_finite(dv[mt][i]));
  bad = key < len ? bad : 0;
  bad |= __shfl_xor(bad, 32);
  if (CAREFUL ? again : !bad) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = 32 * mt + 8 * r + 4 * hh;
        store4(key, 0, col, dk[mt][4 * r] * f, dk[mt][4 * r + 1] * f, dk[mt][4 * r + 2] * f, dk[mt][4 * r + 3] * f);
        store4(key, 1, col, dv[mt][4 * r] * a.drop, dv[mt][4 * r + 1] * a.drop, dv[mt][4 * r + 2] * a.drop,
               dv[mt][4 * r + 3] * a.drop);
      }
  }
  return bad;
}

template <int P, int IN, bool SHARE, bool FULL>
__global__ __launch_bounds__(256, (win_dkv_waves<P, IN>())) void window_dkv_kernel(const WinArgs a) {
  win_passes([&](auto second, int again) { return window_dkv_pass<P, IN, SHARE, FULL, decltype(second)::value>(a, again); });
}

// dk and dv of the sinks: their tile's sums and the far chunks', in order.  One thread a column.
template <int IN>
__global__ __launch_bounds__(256) void window_sink_kernel(const WinArgs a) {
  const int width = a.d + a.dv;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = static_cast<int64_t>(a.sink_rows) * width;
  const int64_t bh = at / per;
  if (bh >= static_cast<int64_t>(a.batch) * (a.heads / a.group)) return;
  const int64_t in = at % per;
  float s = 0.f;
#pragma unroll 8
  for (int c = 0; c <= a.far_chunks; ++c) s += a.part[(bh * (a.far_chunks + 1) + c) * per + in];
  const int64_t row = bh * a.n + in / width;
  const int col = static_cast<int>(in % width);
  if (col < a.d)
    store_elem(a.dk, row * a.d + col, IN, s);
  else
    store_elem(a.dv_out, row * a.dv + col - a.d, IN, s);
}

}  // namespace sta
