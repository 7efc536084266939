// The token cache of windowed attention and the single-token attention over it.
//
// A (stream, key head) holds sinks + window slots: token p < sinks sits in slot p, the others in a ring, token p in
// slot sinks + (p - sinks) % window, so that after n tokens the first min(n, sinks + window) slots hold what the next
// query sees, in an order that softmax does not mind.  counts[stream][head] is n.
//
// Slots lie in tiles of 32, each laid out in the order in which the matrix instructions take it (v_mfma_f32_16x16x32,
// 16x16x4_f32 eight times for fp32), so that a wave loads operands straight from memory, in whole lines and without
// LDS.  With lane l = 16 g + i:
//   keys    [2 halves of 16 slots][d / 32][lane][8]: lane holds slot i of the half, dimensions 32 b + 8 g + 0..7
//   values  [dv / 16][lane][8]: lane holds column 16 c + i of slots {4 g + 0..3, 16 + 4 g + 0..3}
// X^T = K Q^T leaves lane (query i, g) with slots 4 g + 0..3 of each half: the B operand of O^T += V^T P^T as it stands.
//
// Storage in 4 bits (fp4): values in blocks of 32 columns of a token, each 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign,
// times 2^(floor(log2(largest)) - 2), which one byte holds as an exponent (biased by 127; at least 2^-126).  Values
// are rounded to the nearest, ties to the even code, above 6 down to 6; a block that holds a value that is not finite
// is NaN as a whole (exponent byte 255, which the conversion turns into NaN whatever the code).
//   keys    [half][lane][d / 32] words of 8 codes, exponents [slot 16][half][d / 32 or next power of two]
//   values  [lane][dv / 32][8 slots] bytes, columns 32 b + i and 32 b + 16 + i of a slot in the halves of a byte (so that
//           both take one exponent in one conversion, and a token writes whole bytes), exponents [g][dv / 32][8 slots]
// Codes become bf16 with their powers (exact); queries of more than 8 bits and the weights are carried as bf16 planes (fp16
// queries 2, fp32 3; weights 2, 3 for fp32), of 16-bit caches as 2 planes of their type: the products keep the accuracy
// of the output's type, and a step is bound by reading the cache.
#include <type_traits>

#include "rows.hpp"

namespace sta {

constexpr int RING_F4 = 3;  // storage code beside the element types F32, BF16, F16

struct RingArgs {
  Rows q, k, v;  // q [streams][heads][d], the new tokens k, v [streams][kv][d | dv] (sn unused)
  int streams, heads, kv, group, chunks;  // chunks: groups of 16 query heads of a key head
  int d, dv, nbk, nbv;   // blocks of 32 columns
  int sinks, window, slots, tiles;
  float scale, c;        // c = |scale| log2(e)
  uint8_t *keys, *values, *kexp, *vexp;
  int* counts;           // [streams][kv]
  int append, nsplit;
  float* part;           // [streams][heads][nsplit][dv + 2]: sums, then maximum and sum of weights
  void* out;             // [streams][heads][dv]
};

__host__ __device__ constexpr int ring_exps(int nb) { return nb < 3 ? nb : 4; }  // exponent bytes of a slot
__host__ __device__ constexpr int64_t ring_tile_bytes(int nb, int storage) {
  return storage == RING_F4 ? 512 * nb : 1024 * nb * (storage == F32 ? 4 : 2);
}
__host__ __device__ constexpr int64_t ring_key_exp_bytes(int nb, int storage) {
  return storage == RING_F4 ? 32 * ring_exps(nb) : 0;
}
__host__ __device__ constexpr int64_t ring_value_exp_bytes(int nb, int storage) {
  return storage == RING_F4 ? 32 * nb : 0;
}

__device__ __forceinline__ int ring_slot(const RingArgs& a, int p) {
  return p < a.sinks ? p : a.sinks + (p - a.sinks) % a.window;
}

// tokens that a key head has taken
__device__ __forceinline__ int ring_count(const RingArgs& a, int sh) {
  const int n = a.counts[sh];
  return n < 0 ? 0 : n;
}
// The count after `take` more tokens.  One that would pass 31 bits goes back by whole windows: the slots keep their turn
// (window and sinks + window are at most 2^30, so it stays above them).
__device__ __forceinline__ int ring_after(const RingArgs& a, int n, int take) {
  constexpr int64_t most = 0x7fffffff;
  int64_t end = static_cast<int64_t>(n) + take;
  if (end > most) end -= (end - most + a.window - 1) / a.window * a.window;
  return static_cast<int>(end);
}

// the key head and tile of a workgroup of a launch over tiles
__device__ __forceinline__ bool ring_place(const RingArgs& a, int& sh, int& tile) {
  const int64_t id = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  sh = static_cast<int>(id / a.tiles);
  tile = static_cast<int>(id - static_cast<int64_t>(sh) * a.tiles);
  return sh < a.streams * a.kv;
}

// byte of dimension col (keys) or column col (values) of slot r of a tile; of 4-bit caches the byte that holds the
// code (keys: low half for even dimensions, values: for the first 16 columns of a block)
__device__ __forceinline__ int ring_key_at(int r, int col, int nb, int storage) {
  const int half = r >> 4, b = col >> 5, g = (col >> 3) & 3, j = col & 7, lane = 16 * g + (r & 15);
  if (storage == RING_F4) return ((half * 64 + lane) * nb + b) * 4 + (j >> 1);
  return (((half * nb + b) * 64 + lane) * 8 + j) * (storage == F32 ? 4 : 2);
}
__device__ __forceinline__ int ring_value_at(int r, int col, int nb, int storage) {
  const int g = (r >> 2) & 3, j = 4 * (r >> 4) + (r & 3), lane = 16 * g + (col & 15), ct = col >> 4;
  if (storage == RING_F4) return (lane * nb + (ct >> 1)) * 8 + j;
  return ((ct * 64 + lane) * 8 + j) * (storage == F32 ? 4 : 2);
}
__device__ __forceinline__ int ring_key_exp_at(int r, int b, int nb) {
  return ((r & 15) * 2 + (r >> 4)) * ring_exps(nb) + b;
}
__device__ __forceinline__ int ring_value_exp_at(int r, int b, int nb) {
  return (((r >> 2) & 3) * nb + b) * 8 + 4 * (r >> 4) + (r & 3);
}

__device__ __forceinline__ float ring_power(uint32_t byte) { return __uint_as_float(byte << 23); }

// the exponent byte of a block whose largest magnitude has these bits
__device__ __forceinline__ int ring_exponent(uint32_t largest) {
  if (largest >= 0x7f800000u) return 255;
  const int e = static_cast<int>(largest >> 23) - 2;
  return e < 1 ? 1 : e;
}
// the 4-bit codes of two values in a block with exponent byte e: rounded to the nearest, ties to even, 6 at most
__device__ __forceinline__ uint32_t ring_codes(float x, float y, int e) {
  if (e == 255) return 0u;
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x, y, ring_power(e), 0);
}
// and of eight, in order
__device__ __forceinline__ uint32_t ring_codes(const float (&x)[8], int e) {
  if (e == 255) return 0u;
  const float power = ring_power(e);
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], power, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], power, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], power, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], power, 3);
}
__device__ __forceinline__ float ring_decode(uint32_t code) {
  const float m[8] = {0.f, 0.5f, 1.f, 1.5f, 2.f, 3.f, 4.f, 6.f};
  const float x = m[code & 7u];
  return code & 8u ? -x : x;
}

// N words in the widest loads that N allows, past the caches' usual policy: a step reads each tile once (reading 2 GiB
// 7.0 TB/s that way, 6.4 with plain loads)
template <int N>
__device__ __forceinline__ void ring_load(uint32_t (&w)[N], const uint8_t* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u4 u = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = u[j];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u2 u = __builtin_nontemporal_load(reinterpret_cast<const u2*>(p) + i);
#pragma unroll
      for (int j = 0; j < 2; ++j) w[2 * i + j] = u[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p) + i);
  }
}

// Operands of the products.  TYPE: F32 (8 floats a lane), BF16, F16 (8 16-bit values a lane).
typedef _Float16 ring_half8 __attribute__((ext_vector_type(8)));
typedef _Float16 ring_half2 __attribute__((ext_vector_type(2)));

template <int TYPE>
struct RingFrag {
  uint32_t w[TYPE == F32 ? 8 : 4];
};

template <int TYPE>
__device__ __forceinline__ floatx4 ring_mma(const RingFrag<TYPE>& a, const RingFrag<TYPE>& b, floatx4 c) {
  if constexpr (TYPE == F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = mfma4(__uint_as_float(a.w[j]), __uint_as_float(b.w[j]), c);
    return c;
  } else if constexpr (TYPE == F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ring_half8, a.w),
                                                  __builtin_bit_cast(ring_half8, b.w), c, 0, 0, 0);
  } else {
    return mfma_bf16(__builtin_bit_cast(bf16x8, a.w), __builtin_bit_cast(bf16x8, b.w), c);
  }
}

// 8 floats as NP planes, each the rounding of what the planes before it leave
template <int TYPE, int NP>
__device__ __forceinline__ void ring_planes(const float (&x)[8], RingFrag<TYPE> (&f)[NP]) {
  if constexpr (TYPE == F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[0].w[j] = __float_as_uint(x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        if constexpr (TYPE == F16) {
          const ring_half2 h = __builtin_convertvector((floatx2{a, b}), ring_half2);
          f[p].w[j] = __builtin_bit_cast(uint32_t, h);
          a -= static_cast<float>(h[0]);
          b -= static_cast<float>(h[1]);
        } else {
          const uint32_t u = pk_bf16(a, b);
          f[p].w[j] = u;
          a -= __uint_as_float(u << 16);
          b -= __uint_as_float(u & 0xffff0000u);
        }
      }
    }
  }
}

// 8 codes as bf16 values times one power
__device__ __forceinline__ RingFrag<BF16> ring_key_values(uint32_t codes, float power) {
  RingFrag<BF16> f;
  f.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 0));
  f.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 1));
  f.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 2));
  f.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 3));
  return f;
}

// 4 slots' pairs of columns (a byte each) times their powers, and the two columns' words of 4 slots each
__device__ __forceinline__ void ring_value_words(uint32_t codes, const float (&power)[4], uint32_t (&first)[2],
                                                 uint32_t (&second)[2]) {
  uint32_t r[4];
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power[0], 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power[1], 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power[2], 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power[3], 3));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    first[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x05040100u);
    second[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x07060302u);
  }
}

// One token into its slot, by a workgroup of at least 64 + 32 nbv threads (the caller's barrier follows).
template <int ST, int Q>
__device__ void ring_put(const RingArgs& a, int s, int hk, int slot) {
  constexpr int ES = Q == F32 ? 4 : 2;
  const int64_t tile = (static_cast<int64_t>(s) * a.kv + hk) * a.tiles + (slot >> 5);
  const int r = slot & 31, t = threadIdx.x;
  if (t < 4 * a.nbk) {
    const char* row = rows_at<ES>(a.k, s, hk, 0);
    const int col = 8 * t;  // block t / 4, g = t % 4
    uint8_t* at = a.keys + tile * ring_tile_bytes(a.nbk, ST) + ring_key_at(r, col, a.nbk, ST);
    if constexpr (ST == RING_F4) {
      float x[8];
      uint32_t top = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = col + j < a.d ? load_elem(row, col + j, Q) : 0.f;
        top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
      const int e = ring_exponent(top);
      *reinterpret_cast<uint32_t*>(at) = ring_codes(x, e);
      if ((t & 3) == 0)
        a.kexp[tile * ring_key_exp_bytes(a.nbk, ST) + ring_key_exp_at(r, t >> 2, a.nbk)] = static_cast<uint8_t>(e);
    } else {
#pragma unroll
      for (int i = 0; i < ES / 2; ++i)
        reinterpret_cast<uint4*>(at)[i] = rows_chunk<ES>(row, col + (16 / ES) * i, a.d);
    }
  } else if (t >= 64 && t < 64 + (ST == RING_F4 ? 16 : 32) * a.nbv) {
    const char* row = rows_at<ES>(a.v, s, hk, 0);
    uint8_t* values = a.values + tile * ring_tile_bytes(a.nbv, ST);
    if constexpr (ST == RING_F4) {
      const int b = (t - 64) >> 4, c0 = 32 * b + (t & 15), c1 = c0 + 16;
      const float x0 = c0 < a.dv ? load_elem(row, c0, Q) : 0.f, x1 = c1 < a.dv ? load_elem(row, c1, Q) : 0.f;
      uint32_t top = max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o)));
      const int e = ring_exponent(top);
      values[ring_value_at(r, c0, a.nbv, ST)] = static_cast<uint8_t>(ring_codes(x0, x1, e));
      if ((t & 15) == 0)
        a.vexp[tile * ring_value_exp_bytes(a.nbv, ST) + ring_value_exp_at(r, b, a.nbv)] = static_cast<uint8_t>(e);
    } else {
      const int col = t - 64;
      uint8_t* at = values + ring_value_at(r, col, a.nbv, ST);
      if constexpr (ES == 4)
        *reinterpret_cast<uint32_t*>(at) = col < a.dv ? reinterpret_cast<const uint32_t*>(row)[col] : 0u;
      else
        *reinterpret_cast<uint16_t*>(at) = col < a.dv ? reinterpret_cast<const uint16_t*>(row)[col] : uint16_t(0);
    }
  }
}

// A tile's operands as they lie in memory, for one lane
template <int NBK, int NBV, int ST>
struct RingTile {
  static constexpr int W = ST == RING_F4 ? 1 : (ST == F32 ? 8 : 4);  // words of 8 elements
  uint32_t k[2][NBK * W], v[2 * NBV * W];
  static constexpr int KE = ring_exps(NBK) == 4 ? 2 : 1;  // words of a slot pair's exponents
  uint32_t ke[KE], ve[2 * NBV];

  __device__ __forceinline__ void load(const RingArgs& a, int64_t tile, int lane) {
    const uint8_t* kp = a.keys + tile * ring_tile_bytes(NBK, ST);
    const uint8_t* vp = a.values + tile * ring_tile_bytes(NBV, ST);
    if constexpr (ST == RING_F4) {
#pragma unroll
      for (int half = 0; half < 2; ++half) ring_load(k[half], kp + (half * 64 + lane) * NBK * 4);
      ring_load(v, vp + lane * 2 * NBV * 4);
      const uint8_t* ep = a.kexp + tile * ring_key_exp_bytes(NBK, ST) + (lane & 15) * 2 * ring_exps(NBK);
      if constexpr (NBK == 1)
        ke[0] = *reinterpret_cast<const uint16_t*>(ep);
      else
        ring_load(ke, ep);
      ring_load(ve, a.vexp + tile * ring_value_exp_bytes(NBV, ST) + (lane >> 4) * 8 * NBV);
    } else {
      uint32_t w[W];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int b = 0; b < NBK; ++b) {
          ring_load(w, kp + (((half * NBK + b) * 64 + lane) * W) * 4);
#pragma unroll
          for (int i = 0; i < W; ++i) k[half][b * W + i] = w[i];
        }
#pragma unroll
      for (int ct = 0; ct < 2 * NBV; ++ct) {
        ring_load(w, vp + ((ct * 64 + lane) * W) * 4);
#pragma unroll
        for (int i = 0; i < W; ++i) v[ct * W + i] = w[i];
      }
    }
  }
};

// the power of two in byte i of exponent words
__device__ __forceinline__ float ring_power_of(const uint32_t* w, int i) {
  return ring_power((w[i >> 2] >> (8 * (i & 3))) & 0xffu);
}

// A workgroup a share of a key head's tiles, its four waves every fourth tile, joined through LDS at the end.  The
// matrix instructions have 16 columns for the query heads of a key head; with fewer they idle, which costs nothing: bound
// by reading the cache, for 4 bits nearly as much by the conversions (285 VALU instructions a tile of 128 + 128 columns,
// 69 % of the cycles at 4.7 TB/s).  64 x 32 heads x 4100 tokens of 64 + 64 bf16 (2.15 GB): 345 us, 6.2 TB/s; 64 x 8 key
// heads x 32772 tokens of 128 + 128 in 4 bits (2.28 GB): 388 us, 5.9 TB/s (558 us with the exponents multiplied into
// logits and weights, 480 with a check for the last tile in every tile); plain reads reach 7.0 TB/s.
template <int NBK, int NBV, int ST, int Q>
__global__ __launch_bounds__(256, ST == F32 ? 1 : 2) void ring_attention_kernel(const RingArgs a) {
  constexpr int XT = ST == RING_F4 ? BF16 : ST;                                   // type of the products
  constexpr int QP = ST == RING_F4 ? (Q == F32 ? 3 : (Q == F16 ? 2 : 1)) : 1;     // planes of the queries
  constexpr int PP = ST == F32 ? 1 : (Q == F32 ? 3 : 2);                          // and of the weights
  constexpr int ES = Q == F32 ? 4 : 2, CT = 2 * NBV, W = RingTile<NBK, NBV, ST>::W;
  constexpr int PITCH = 32 * NBV + 4;
  __shared__ float red[4 * 16 * PITCH], red_m[4 * 16], red_l[4 * 16];
  int id = blockIdx.x;
  const int split = id % a.nsplit;
  id /= a.nsplit;
  const int chunk = id % a.chunks, sh = id / a.chunks;
  const int s = sh / a.kv, hk = sh - s * a.kv;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;

  const int n = ring_count(a, sh);
  const int held = n < a.slots - a.append ? n + a.append : a.slots;
  const int all = (held + 31) >> 5, per = (all + a.nsplit - 1) / a.nsplit;
  const int t0 = split * per, t1 = t0 + per < all ? t0 + per : all;
  if (a.append) {
    const int slot = ring_slot(a, n);
    if ((slot >> 5) >= t0 && (slot >> 5) < t1) ring_put<ST, Q>(a, s, hk, slot);
    __syncthreads();
  }

  const int queries = min(16, a.group - 16 * chunk);
  RingFrag<XT> qf[NBK][QP];
  {
    const bool in = li < queries;
    const char* row = rows_at<ES>(a.q, s, hk * a.group + 16 * chunk + (in ? li : 0), 0);
#pragma unroll
    for (int b = 0; b < NBK; ++b) {
      constexpr int E = 16 / ES;
      float x[8];
#pragma unroll
      for (int i = 0; i < 8 / E; ++i) {
        float y[E];
        rows_unpack<Q>(rows_chunk<ES>(row, 32 * b + 8 * lg + E * i, a.d), y);
#pragma unroll
        for (int e = 0; e < E; ++e) x[E * i + e] = in ? (a.scale < 0.f ? -y[e] : y[e]) : 0.f;
      }
      ring_planes<XT, QP>(x, qf[b]);
    }
  }

  floatx4 acc[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) acc[ct] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -3.4028235e38f, limit = m, l = 0.f;
  // fp16 weights are carried times 2^11, at most 2^15: below 2^-14 fp16 holds steps of 2^-24 only, of which a long cache has
  // many; so a weight loses at most 2^-36 of the largest
  constexpr bool LIFT = XT == F16;
  const float room = (LIFT ? 4.f : 8.f) / a.c;

  const int64_t tile0 = static_cast<int64_t>(sh) * a.tiles;
  // a tile's part of the sums; PART: not all of its slots hold a token
  auto take = [&](const RingTile<NBK, NBV, ST>& cur, int t, auto part) {
    constexpr bool PART = decltype(part)::value;
    floatx4 x[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      x[half] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < NBK; ++b) {
        if constexpr (ST == RING_F4) {
          const RingFrag<XT> k = ring_key_values(cur.k[half][b], ring_power_of(cur.ke, half * ring_exps(NBK) + b));
#pragma unroll
          for (int p = QP - 1; p >= 0; --p) x[half] = ring_mma<XT>(k, qf[b][p], x[half]);
        } else {
          RingFrag<XT> k;
#pragma unroll
          for (int i = 0; i < W; ++i) k.w[i] = cur.k[half][b * W + i];
          x[half] = ring_mma<XT>(k, qf[b][0], x[half]);
        }
      }
    }
    // slots of this lane that hold a token
    const int left = held - 32 * t - 4 * lg;
    float top = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (PART && 16 * (i >> 2) + (i & 3) >= left) x[i >> 2][i & 3] = -__builtin_inff();
      top = fmaxf(top, x[i >> 2][i & 3]);
    }
    // the maximum moves, for all lanes of a query at once, when a weight would exceed 2^8 (fp16: 2^4)
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
      const float y = x[i >> 2][i & 3] - m;
      p[i] = __builtin_amdgcn_exp2f(LIFT ? fmaf(y, a.c, 11.f) : y * a.c);
      if (PART && 16 * (i >> 2) + (i & 3) >= left) p[i] = 0.f;
      l += p[i];
    }
    RingFrag<XT> pf[PP];
    ring_planes<XT, PP>(p, pf);
    if constexpr (ST == RING_F4) {
#pragma unroll
      for (int b = 0; b < NBV; ++b) {
        RingFrag<XT> v[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float power[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            power[i] = ring_power_of(cur.ve, 8 * b + 4 * half + i);
            if (PART && 16 * half + i >= left) power[i] = 0.f;  // a slot without a token, whatever it holds
          }
          uint32_t first[2], second[2];
          ring_value_words(cur.v[2 * b + half], power, first, second);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            v[0].w[2 * half + i] = first[i];
            v[1].w[2 * half + i] = second[i];
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = PP - 1; k >= 0; --k) acc[2 * b + h] = ring_mma<XT>(v[h], pf[k], acc[2 * b + h]);
      }
    } else {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        RingFrag<XT> v;
#pragma unroll
        for (int i = 0; i < W; ++i) v.w[i] = cur.v[ct * W + i];
        if constexpr (PART) {  // slots without a token: whatever they hold
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (16 * (i >> 2) + (i & 3) >= left) {
              if constexpr (ST == F32)
                v.w[i] = 0u;
              else
                v.w[i >> 1] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
            }
        }
#pragma unroll
        for (int k = PP - 1; k >= 0; --k) acc[ct] = ring_mma<XT>(v, pf[k], acc[ct]);
      }
    }
  };
  // whole tiles, one ahead in registers, the two buffers in turn; then the last tile if it is not whole
  {
    const int end = t1 < (held >> 5) ? t1 : held >> 5;
    RingTile<NBK, NBV, ST> even, odd;
    int t = t0 + wave;
    if (t < end) even.load(a, tile0 + t, lane);
    while (t < end) {
      if (t + 4 < end) odd.load(a, tile0 + t + 4, lane);
      take(even, t, std::false_type{});
      t += 4;
      if (t >= end) break;
      if (t + 4 < end) even.load(a, tile0 + t + 4, lane);
      take(odd, t, std::false_type{});
      t += 4;
    }
    if (t < t1) {
      even.load(a, tile0 + t, lane);
      take(even, t, std::true_type{});
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // the four waves' sums
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    *reinterpret_cast<floatx4*>(&red[(wave * 16 + li) * PITCH + 16 * ct + 4 * lg]) = acc[ct];
  if (lg == 0) {
    red_m[wave * 16 + li] = m;
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
      const float f = __builtin_amdgcn_exp2f((red_m[16 * w + i] - top) * a.c);
      sum = fmaf(f, red[(w * 16 + i) * PITCH + col], sum);
      den = fmaf(f, red_l[16 * w + i], den);
    }
    const int64_t head = static_cast<int64_t>(s) * a.heads + hk * a.group + 16 * chunk + i;
    if (a.nsplit == 1) {
      store_elem(a.out, head * a.dv + col, Q, held ? sum / den : 0.f);
    } else {
      float* part = a.part + (head * a.nsplit + split) * (a.dv + 2);
      part[col] = sum;
      if (col == 0) {
        part[a.dv] = top;
        part[a.dv + 1] = den;
      }
    }
  }
  // every thread has read the count; other workgroups read it only where ring_join_kernel counts
  if (a.append && a.nsplit == 1 && a.chunks == 1 && threadIdx.x == 0) a.counts[sh] = ring_after(a, n, 1);
}

// The splits' sums of a query head, 4 groups of 128 threads (a column each) over the splits, and the count of a step
// that several workgroups share.  Bound by latency: 8 heads x 257 splits of 80 columns 6.4 us (113 us with one thread a
// column over all splits, each load waiting for the one before), 128 splits 4.2 us.
constexpr int RING_SPLITS = 1024;
template <int Q>
__global__ __launch_bounds__(512) void ring_join_kernel(const RingArgs a) {
  __shared__ float weight[RING_SPLITS], red[4 * 128], wave_red[8];
  const int64_t head = blockIdx.x;
  const int s = blockIdx.x / a.heads, h = blockIdx.x - s * a.heads, sh = s * a.kv + h / a.group;
  const int col = threadIdx.x & 127, group = threadIdx.x >> 7, wave = threadIdx.x >> 6;
  if (a.nsplit > 1) {
    const int pitch = a.dv + 2;
    const float* part = a.part + head * a.nsplit * pitch;
    float top = -3.4028235e38f, den = 0.f;
    for (int i = threadIdx.x; i < a.nsplit; i += 512) {
      weight[i] = part[i * pitch + a.dv];
      top = fmaxf(top, weight[i]);
    }
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) wave_red[wave] = top;
    __syncthreads();
    for (int i = 0; i < 8; ++i) top = fmaxf(top, wave_red[i]);
    for (int i = threadIdx.x; i < a.nsplit; i += 512) {
      const float f = __builtin_amdgcn_exp2f((weight[i] - top) * a.c);
      weight[i] = f;
      den = fmaf(f, part[i * pitch + a.dv + 1], den);
    }
    for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) wave_red[wave] = den;
    float sum = 0.f;
    if (col < a.dv) {
#pragma unroll 8
      for (int i = group; i < a.nsplit; i += 4) sum = fmaf(weight[i], part[i * pitch + col], sum);
    }
    red[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < a.dv) {
      den = 0.f;
      for (int i = 0; i < 8; ++i) den += wave_red[i];
      sum = red[threadIdx.x] + red[128 + threadIdx.x] + red[256 + threadIdx.x] + red[384 + threadIdx.x];
      const bool empty = !a.append && ring_count(a, sh) == 0;
      store_elem(a.out, head * a.dv + threadIdx.x, Q, empty ? 0.f : sum / den);
    }
  }
  if (a.append && h % a.group == 0 && threadIdx.x == 0) a.counts[sh] = ring_after(a, ring_count(a, sh), 1);
}

struct RingFill {
  RingArgs a;          // k, v: [streams][kv][rows][d | dv] with row strides
  int rows;
  const int* take;     // [streams] or null: rows of a stream that are tokens
};

// The token (an index into the call's rows) that slot gets from rows 0 .. take-1 after n tokens, or -1.
__device__ __forceinline__ int ring_token(const RingArgs& a, int slot, int n, int take) {
  const int64_t end = static_cast<int64_t>(n) + take;  // positions [n, end)
  int64_t p = slot;
  if (slot >= a.sinks) {
    if (end - 1 < slot) return -1;
    p = slot + (end - 1 - slot) / a.window * a.window;
  }
  return p >= n && p < end ? static_cast<int>(p - n) : -1;
}

__device__ __forceinline__ int ring_take(const RingFill& f, int s) {
  const int t = f.take ? f.take[s] : f.rows;
  return t < 0 ? 0 : (t > f.rows ? f.rows : t);
}

// A workgroup a tile of 32 slots: the last token that falls into each slot.
template <int ST, int Q>
__global__ __launch_bounds__(256) void ring_extend_kernel(const RingFill f) {
  constexpr int ES = Q == F32 ? 4 : 2;
  const RingArgs& a = f.a;
  __shared__ uint32_t vals[32 * 132];  // the tile's values (bits, or codes), 32 nbv + 1 a slot
  __shared__ int token[32];
  int sh, tile;
  if (!ring_place(a, sh, tile)) return;
  const int s = sh / a.kv, hk = sh - s * a.kv, n = ring_count(a, sh), take = ring_take(f, s);
  if (threadIdx.x < 32) {
    const int slot = 32 * tile + threadIdx.x;
    token[threadIdx.x] = slot < a.slots ? ring_token(a, slot, n, take) : -1;
  }
  if (!__syncthreads_or(threadIdx.x < 32 && token[threadIdx.x] >= 0)) return;  // no token falls into this tile
  const int64_t at = static_cast<int64_t>(sh) * a.tiles + tile;
  uint8_t* keys = a.keys + at * ring_tile_bytes(a.nbk, ST);
  uint8_t* values = a.values + at * ring_tile_bytes(a.nbv, ST);
  const int pitch = 32 * a.nbv + 1;
  // 8 columns of a slot's key a thread, 4 neighbouring threads a block
  for (int i = threadIdx.x; i < 32 * 4 * a.nbk; i += 256) {
    const int r = i / (4 * a.nbk), u = i - r * 4 * a.nbk, col = 8 * u, p = token[r];
    const char* row = rows_at<ES>(a.k, s, hk, p < 0 ? 0 : p);
    uint8_t* to = keys + ring_key_at(r, col, a.nbk, ST);
    if constexpr (ST == RING_F4) {
      float x[8];
      uint32_t top = 0u;
      constexpr int E = 16 / ES;
#pragma unroll
      for (int c = 0; c < 8 / E; ++c) {
        float y[E];
        rows_unpack<Q>(p < 0 ? uint4{0u, 0u, 0u, 0u} : rows_chunk<ES>(row, col + E * c, a.d), y);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[E * c + e] = y[e];
          top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        }
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
      const int e = ring_exponent(top);
      if (p >= 0) {
        *reinterpret_cast<uint32_t*>(to) = ring_codes(x, e);
        if ((u & 3) == 0)
          a.kexp[at * ring_key_exp_bytes(a.nbk, ST) + ring_key_exp_at(r, u >> 2, a.nbk)] = static_cast<uint8_t>(e);
      }
    } else if (p >= 0) {
#pragma unroll
      for (int c = 0; c < ES / 2; ++c)
        reinterpret_cast<uint4*>(to)[c] = rows_chunk<ES>(row, col + (16 / ES) * c, a.d);
    }
  }
  // values: the rows (codes) of the tile's slots, then 8 slots of a column a thread
  for (int i = threadIdx.x; i < 32 * 4 * a.nbv; i += 256) {
    const int r = i / (4 * a.nbv), u = i - r * 4 * a.nbv, col = 8 * u, p = token[r];
    const char* row = rows_at<ES>(a.v, s, hk, p < 0 ? 0 : p);
    constexpr int E = 16 / ES;
    uint32_t* to = vals + r * pitch + col;
    float x[8];
    uint32_t top = 0u;
#pragma unroll
    for (int c = 0; c < 8 / E; ++c) {
      const uint4 w = p < 0 ? uint4{0u, 0u, 0u, 0u} : rows_chunk<ES>(row, col + E * c, a.dv);
      if constexpr (ST == RING_F4) {
        float y[E];
        rows_unpack<Q>(w, y);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[E * c + e] = y[e];
          top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
        }
      } else {
        const uint32_t z[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < E; ++e) to[E * c + e] = ES == 4 ? z[e & 3] : (z[(e >> 1) & 3] >> (16 * (e & 1))) & 0xffffu;
      }
    }
    if constexpr (ST == RING_F4) {
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
      const int e = ring_exponent(top);
      const uint32_t codes = ring_codes(x, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = (codes >> (4 * j)) & 15u;
      if (p >= 0 && (u & 3) == 0)
        a.vexp[at * ring_value_exp_bytes(a.nbv, ST) + ring_value_exp_at(r, u >> 2, a.nbv)] = static_cast<uint8_t>(e);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * (ST == RING_F4 ? a.nbv : 2 * a.nbv); i += 256) {
    const int lane = i & 63, ct = i >> 6, g = lane >> 4;
    const int col = ST == RING_F4 ? 32 * ct + (lane & 15) : 16 * ct + (lane & 15);
    uint32_t w[8];
    bool all = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = 16 * (j >> 2) + 4 * g + (j & 3);
      w[j] = vals[r * pitch + col];
      if constexpr (ST == RING_F4) w[j] |= vals[r * pitch + col + 16] << 4;
      all = all && token[r] >= 0;
    }
    uint8_t* to = values + (ST == RING_F4 ? (lane * a.nbv + ct) * 8 : (ct * 64 + lane) * 8 * (ST == F32 ? 4 : 2));
    if (all) {
      if constexpr (ST == RING_F4) {
        *reinterpret_cast<uint2*>(to) = uint2{w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24,
                                              w[4] | w[5] << 8 | w[6] << 16 | w[7] << 24};
      } else if constexpr (ST == F32) {
        reinterpret_cast<uint4*>(to)[0] = uint4{w[0], w[1], w[2], w[3]};
        reinterpret_cast<uint4*>(to)[1] = uint4{w[4], w[5], w[6], w[7]};
      } else {
        *reinterpret_cast<uint4*>(to) = uint4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
      }
      continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (token[16 * (j >> 2) + 4 * g + (j & 3)] < 0) continue;
      if constexpr (ST == RING_F4)
        to[j] = static_cast<uint8_t>(w[j]);
      else if constexpr (ST == F32)
        reinterpret_cast<uint32_t*>(to)[j] = w[j];
      else
        reinterpret_cast<uint16_t*>(to)[j] = static_cast<uint16_t>(w[j]);
    }
  }
}

// counts += the tokens that ring_extend_kernel has put in
__global__ __launch_bounds__(256) static void ring_count_kernel(const RingFill f) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < f.a.streams * f.a.kv) f.a.counts[i] = ring_after(f.a, ring_count(f.a, i), ring_take(f, i / f.a.kv));
}

// The slots' rows as they stand for: keys [streams][kv][slots][d], values [..][dv] in the element type, zero where no
// token is; positions [streams][slots], -1 there.  A workgroup a tile: the tile's words in their order into LDS rows, then
// whole rows out.
template <int ST, int Q>
__global__ __launch_bounds__(256) void ring_items_kernel(const RingArgs a, void* keys, void* values, int* positions) {
  constexpr int PITCH = 129;
  __shared__ uint32_t rows[32 * PITCH];  // values: floats (4-bit), or the elements' bits
  int sh, tile;
  if (!ring_place(a, sh, tile)) return;
  const int s = sh / a.kv, hk = sh - s * a.kv, n = ring_count(a, sh);
  const int64_t at = static_cast<int64_t>(sh) * a.tiles + tile;
  const uint8_t* kp = a.keys + at * ring_tile_bytes(a.nbk, ST);
  const uint8_t* vp = a.values + at * ring_tile_bytes(a.nbv, ST);
  const int live = min(32, a.slots - 32 * tile);  // slots of the tile
  const bool some = 32 * tile < n;                // one of them holds a token
  auto elem = [&](const uint8_t* p, int e) -> uint32_t {
    if constexpr (ST == F32) return reinterpret_cast<const uint32_t*>(p)[e];
    return reinterpret_cast<const uint16_t*>(p)[e];
  };
  auto store_rows = [&](void* out, int width) {
    constexpr int ES = Q == F32 ? 4 : 2, E = 16 / ES;
    const int64_t base = (static_cast<int64_t>(sh) * a.slots + 32 * tile) * width;
    if (width % E == 0) {  // 16 bytes a thread
      const int units = width / E;
      for (int i = threadIdx.x; i < live * units; i += 256) {
        const int r = i / units, col = (i - r * units) * E;
        const bool held = 32 * tile + r < n;
        uint4 w;
        if constexpr (ST == RING_F4) {
          float f[E];
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = held ? __uint_as_float(rows[r * PITCH + col + e]) : 0.f;
          w = rows_pack<Q>(f);
        } else {
          uint32_t f[E];
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] = held ? rows[r * PITCH + col + e] : 0u;
          if constexpr (ES == 4)
            w = uint4{f[0], f[1], f[2], f[3]};
          else
            w = uint4{f[0] | f[1] << 16, f[2] | f[3] << 16, f[4] | f[5] << 16, f[6] | f[7] << 16};
        }
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));  // past the caches: 16 x 8 heads of 4100 x 64 40 -> 37.5 us
        __builtin_nontemporal_store(u4{w.x, w.y, w.z, w.w}, reinterpret_cast<u4*>(static_cast<char*>(out) + base * ES) + i);
      }
      return;
    }
    for (int i = threadIdx.x; i < live * width; i += 256) {
      const int r = i / width, col = i - r * width;
      const uint32_t w = 32 * tile + r < n ? rows[r * PITCH + col] : 0u;
      if constexpr (ST == RING_F4)
        store_elem(out, base + i, Q, __uint_as_float(w));
      else if constexpr (ST == F32)
        static_cast<uint32_t*>(out)[base + i] = w;
      else
        static_cast<uint16_t*>(out)[base + i] = static_cast<uint16_t>(w);
    }
  };
  for (int i = threadIdx.x; some && i < 128 * a.nbk; i += 256) {  // 8 dimensions of a slot a thread, in the cache's order
    const int lane = i & 63, u = i >> 6, half = u / a.nbk, b = u - half * a.nbk;
    const int r = 16 * half + (lane & 15), col = 32 * b + 8 * (lane >> 4);
    if constexpr (ST == RING_F4) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(kp)[(half * 64 + lane) * a.nbk + b];
      const float e = ring_power(a.kexp[at * ring_key_exp_bytes(a.nbk, ST) + ring_key_exp_at(r, b, a.nbk)]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        rows[r * PITCH + col + j] = __float_as_uint(ring_decode((w >> (4 * j)) & 15u) * e);
    } else {
      const uint8_t* p = kp + (u * 64 + lane) * 8 * (ST == F32 ? 4 : 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) rows[r * PITCH + col + j] = elem(p, j);
    }
  }
  __syncthreads();
  store_rows(keys, a.d);
  __syncthreads();
  for (int i = threadIdx.x; some && i < 64 * (ST == RING_F4 ? a.nbv : 2 * a.nbv); i += 256) {  // 8 slots of a column a thread
    const int lane = i & 63, ct = i >> 6, g = lane >> 4;
    const int col = ST == RING_F4 ? 32 * ct + (lane & 15) : 16 * ct + (lane & 15);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = 16 * (j >> 2) + 4 * g + (j & 3);
      if constexpr (ST == RING_F4) {
        const uint32_t w = vp[(lane * a.nbv + ct) * 8 + j];
        const float e = ring_power(a.vexp[at * ring_value_exp_bytes(a.nbv, ST) + ring_value_exp_at(r, ct, a.nbv)]);
        rows[r * PITCH + col] = __float_as_uint(ring_decode(w & 15u) * e);
        rows[r * PITCH + col + 16] = __float_as_uint(ring_decode(w >> 4) * e);
      } else {
        rows[r * PITCH + col] = elem(vp + (ct * 64 + lane) * 8 * (ST == F32 ? 4 : 2), j);
      }
    }
  }
  __syncthreads();
  store_rows(values, a.dv);
  if (hk == 0 && static_cast<int>(threadIdx.x) < live) {
    const int slot = 32 * tile + threadIdx.x;
    int p = -1;
    if (slot < n) p = slot < a.sinks ? slot : slot + (n - 1 - slot) / a.window * a.window;
    positions[static_cast<int64_t>(s) * a.slots + slot] = p;
  }
}

}  // namespace sta
