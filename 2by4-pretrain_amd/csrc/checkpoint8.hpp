// Activations kept in 8 bits for the backward pass: the format, and what encodes and decodes it inside a kernel.
//
// A matrix of rows x cols is kept as ceil(cols / 32) blocks a row, 32 adjacent columns each (the last one filled up with zeros): 32 bytes
// of OCP e4m3 and one byte b of scale, of which the values are e4m3 * 2^(b - 127).  All blocks of a row follow each other, then those of the
// next row; the scales are a matrix of their own in the same order.
//
// The scale is the power of two for which the largest magnitude of the block lies in (224, 448] scales: 448 is e4m3's largest number, so nothing
// saturates, and multiplying by a power of two is exact, so every value is off by at most half a step of its own (2^-4 of it; below 2^-6
// scales, 2^-10 scales).  Two details:
//   - magnitudes that would round past the largest number of the matrix's type (more than 1.9375 * 2^Emax) are held at 1.875 * 2^Emax;
//   - scales end at 2^-117, so that what is kept is a normal float32 or zero.
// An infinity or a NaN is kept as a NaN and leaves the scale of its block alone.
#pragma once
#include "tf24_common.hpp"

namespace tf24 {
namespace {

constexpr int kKeptBlock = 32;      // columns that share a scale
constexpr int kKeptUnit = 8;        // columns of a lane; the four lanes of a block are adjacent
constexpr int kKeptLanes = kKeptBlock / kKeptUnit;

__host__ __device__ inline int64_t kept_blocks(int64_t cols) { return (cols + kKeptBlock - 1) / kKeptBlock; }

// 4-, 8- and 16-byte accesses at any element: global memory takes them unaligned, in the same instruction
typedef unsigned int any1 __attribute__((aligned(2)));
typedef unsigned int any2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int any4 __attribute__((ext_vector_type(4), aligned(2)));

// The `n` <= 8 elements at p as float32, zeros behind them.  Fewer than eight are four, two and one, as far as there are.
template <typename T>
__device__ __forceinline__ void load_up_to_8(const T* p, int n, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    any4 w = {0, 0, 0, 0};
    if (n == 8) w = *reinterpret_cast<const any4*>(p);
    else if (n > 0) {
      any2 four = {0, 0};
      uint32_t two = 0, one = 0;
      if (n & 4) four = *reinterpret_cast<const any2*>(p);
      if (n & 2) two = *reinterpret_cast<const any1*>(p + (n & 4));
      if (n & 1) one = p[n - 1].bits;
      const uint32_t r0 = n & 2 ? two : one, r1 = n & 2 ? one : 0;
      w = n & 4 ? any4{four.x, four.y, r0, r1} : any4{r0, r1, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = to_float(T{(uint16_t)(w[e >> 1] >> (16 * (e & 1)))});
  } else {
    any4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (n & 12) a = *reinterpret_cast<const any4*>(p);
    if (n == 8) b = *reinterpret_cast<const any4*>(p + 4);
    else if (n > 0) {
      any2 two = {0, 0};
      uint32_t one = 0;
      if (n & 2) two = *reinterpret_cast<const any2*>(p + (n & 4));
      if (n & 1) one = __builtin_bit_cast(uint32_t, p[n - 1]);
      const any4 rest = n & 2 ? any4{two.x, two.y, one, 0} : any4{one, 0, 0, 0};
      if (n & 4) b = rest;
      else a = rest;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t lo = a[e], hi = b[e];                       // (a bit cast of a vector's element itself takes the first one)
      v[e] = __builtin_bit_cast(float, lo);
      v[4 + e] = __builtin_bit_cast(float, hi);
    }
  }
}
// v rounded to T; the values as they are stored are left in v
template <typename T>
__device__ __forceinline__ void round_8(float (&v)[8], any4 (&w)[sizeof(T) / 2]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const T lo = from_float<T>(v[e]), hi = from_float<T>(v[e + 1]);
      w[0][e >> 1] = (uint32_t)lo.bits | ((uint32_t)hi.bits << 16);
      v[e] = to_float(lo);
      v[e + 1] = to_float(hi);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) w[e >> 2][e & 3] = __builtin_bit_cast(uint32_t, v[e]);
  }
}
// v, rounded to T, to the first n <= 8 elements at p; the values as they are stored are left in v
template <typename T>
__device__ __forceinline__ void store_up_to_8(T* p, int n, float (&v)[8]) {
  any4 w[sizeof(T) / 2];
  round_8<T>(v, w);
  if (n == 8) {
    *reinterpret_cast<any4*>(p) = w[0];
    if constexpr (sizeof(T) == 4) *reinterpret_cast<any4*>(p + 4) = w[1];
  } else if (n > 0) {                                            // four, two and one, as far as there are
    if constexpr (sizeof(T) == 2) {
      uint32_t r0 = w[0][0], r1 = w[0][1];
      if (n & 4) {
        *reinterpret_cast<any2*>(p) = any2{r0, r1};
        r0 = w[0][2];
        r1 = w[0][3];
      }
      if (n & 2) {
        *reinterpret_cast<any1*>(p + (n & 4)) = r0;
        r0 = r1;
      }
      if (n & 1) p[n - 1].bits = (uint16_t)r0;
    } else {
      any4 r = w[0];
      if (n & 4) {
        *reinterpret_cast<any4*>(p) = r;
        r = w[1];
      }
      if (n & 2) {
        *reinterpret_cast<any2*>(p + (n & 4)) = any2{r[0], r[1]};
        r[0] = r[2];
      }
      const uint32_t one = r[0];
      if (n & 1) p[n - 1] = __builtin_bit_cast(float, one);
    }
  }
}

// The eight columns of a lane, whose block are it and its three neighbours (lanes 4i .. 4i + 3, all of which enter).  T: type of the matrix.
struct Kept8 { uint2 values; uint32_t scale; };
template <typename T>
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));      // quad_perm [1,0,3,2]
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));   // [2,3,0,1]
}
template <typename T>
__device__ __forceinline__ Kept8 keep_8(const float (&x)[8]) {
  constexpr uint32_t LIMIT = std::is_same<T, f16_t>::value ? 0x47700000u : 0x7f700000u;       // 1.875 * 2^Emax
  constexpr uint32_t INF = 0x7f800000u;
  float v[8];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    v[e] = x[e];
    top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
  }
  if (__builtin_expect(top > LIMIT, 0)) {
    top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, v[e]), magnitude = bits & 0x7fffffffu;
      const uint32_t held = magnitude > LIMIT ? LIMIT : magnitude;
      v[e] = __builtin_bit_cast(float, magnitude >= INF ? 0x7fc00000u : held | (bits & 0x80000000u));
      top = max(top, magnitude >= INF ? 0u : held);
    }
  }
  top = quad_max<T>(top);
  // the largest magnitude's exponent, one more where its mantissa is over 1.75, less 8
  const uint32_t exponent = (top + 0x1fffffu) >> 23;
  Kept8 k;
  k.scale = max(exponent, 18u) - 8u;
  const float by = __builtin_bit_cast(float, (254u - k.scale) << 23);
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * by, v[1] * by, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * by, v[3] * by, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * by, v[5] * by, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * by, v[7] * by, hi, true);
  k.values = make_uint2((uint32_t)lo, (uint32_t)hi);
  return k;
}
// eight kept values and their block's scale as float32 (exact)
__device__ __forceinline__ void kept_to_float(uint2 values, uint32_t scale, float (&v)[8]) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  const float s = __builtin_bit_cast(float, scale << 23);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t w = h ? values.y : values.x;
    const float2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true);
    v[4 * h] = a.x; v[4 * h + 1] = a.y; v[4 * h + 2] = b.x; v[4 * h + 3] = b.y;
  }
}

// Unit u (eight columns) of a kept matrix -> its row; units_per_row is a multiple of 4.  Division by a constant of the launch as a product
// (u < 2^31): exact for every u with multiplier = floor(2^(31 + l) / d) + 1, l = ceil(log2 d).
struct UnitRows {
  uint32_t units, multiplier, shift;      // of a row; of the division
};
inline UnitRows unit_rows(int64_t cols) {
  const uint32_t d = (uint32_t)(kept_blocks(cols) * kKeptLanes);
  uint32_t l = 0;
  while (((uint64_t)1 << l) < d) l++;
  return {d, (uint32_t)((((uint64_t)1 << (31 + l)) / d) + 1), l - 1};         // (d >= 4, so l >= 2)
}
inline bool too_many_units(int64_t rows, int64_t cols) { return rows > 0x7fffffffLL / (kept_blocks(cols) * kKeptLanes); }
__device__ __forceinline__ uint32_t row_of_unit(const UnitRows& r, uint32_t u) { return __umulhi(u, r.multiplier) >> r.shift; }

}  // namespace
}  // namespace tf24
