// Rows of strided [batch][heads][n][width] tensors, read in units of 16 bytes.
#pragma once
#include "common.hpp"

namespace sta {

// workgroups of 256 threads in one dimension of a launch, whose threads have to stay below 2^32
constexpr int64_t MAX_GROUPS = (int64_t(1) << 24) - 1;

// element strides; `aligned`: every row starts on 16 bytes (set for the kernels that ask for it)
struct Rows {
  const void* p;
  int64_t sb, sh, sn;
  int aligned;
};

template <int ES>
__device__ __forceinline__ const char* rows_at(const Rows& t, int64_t b, int64_t h, int64_t row) {
  return static_cast<const char*>(t.p) + (b * t.sb + h * t.sh + row * t.sn) * ES;
}

// 16 bytes at any element's address (gfx950 reads them in one load whatever the alignment)
__device__ __forceinline__ uint4 rows_load16(const char* p) {
  uint4 u;
  __builtin_memcpy(&u, p, 16);
  return u;
}

// u moved down by `bytes` (0 .. 15), zeros coming in above
__device__ __forceinline__ uint4 rows_shift(const uint4& u, int bytes) {
  uint64_t lo = u.x | static_cast<uint64_t>(u.y) << 32, hi = u.z | static_cast<uint64_t>(u.w) << 32;
  if (bytes & 8) {
    lo = hi;
    hi = 0;
  }
  const int s = 8 * (bytes & 7);
  lo = s ? (lo >> s) | (hi << (64 - s)) : lo;
  hi >>= s;
  return uint4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
               static_cast<uint32_t>(hi >> 32)};
}

// 16 bytes at column `col` of a row of at least 16 bytes, columns at or behind `width` zero: where the unit reaches over
// the row's end, the row's last 16 bytes, moved into place
template <int ES>
__device__ __forceinline__ uint4 rows_unit(const char* row, int col, int width) {
  constexpr int E = 16 / ES;
  uint4 u = rows_load16(row + min(col, width - E) * ES);
  if (width % E) u = rows_shift(u, max(0, col + E - width) * ES & 15);
  return col < width ? u : uint4{0u, 0u, 0u, 0u};
}

// the same of a row of any width
template <int ES>
__device__ __forceinline__ uint4 rows_chunk(const char* row, int col, int width) {
  constexpr int E = 16 / ES;
  if (width >= E) return rows_unit<ES>(row, col, width);
  uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (col + e < width) {
      if constexpr (ES == 4)
        u[e] = reinterpret_cast<const uint32_t*>(row)[col + e];
      else
        u[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[col + e]) << (16 * (e & 1));
    }
  return uint4{u[0], u[1], u[2], u[3]};
}

// the elements of a 16-byte unit as floats, and back (rounded to nearest even)
template <int IN>
__device__ __forceinline__ void rows_unpack(const uint4& u, float (&f)[IN == F32 ? 4 : 8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (IN == F32) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (IN == BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] & 0xffffu)));
      f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
    }
  }
}

template <int IN>
__device__ __forceinline__ uint4 rows_pack(const float (&f)[IN == F32 ? 4 : 8]) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (IN == F32)
      w[i] = __float_as_uint(f[i]);
    else if constexpr (IN == BF16)
      w[i] = pk_bf16(f[2 * i], f[2 * i + 1]);
    else
      w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{f[2 * i], f[2 * i + 1]}), half2_t));
  }
  return uint4{w[0], w[1], w[2], w[3]};
}

}  // namespace sta
