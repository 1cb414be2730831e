// What the two directions of the block norms share: the places and loads of rows, sums over the threads of a row, dispatch.
#pragma once
#include "checkpoint8.hpp"

namespace tf24 {
namespace {

constexpr int kMaxCols = 16384;
constexpr int kNarrowCols = 8192, kWideThreads = 1024;           // wider rows have kernels of their own

// GROUP threads share a row, each with UNITS units of 8 columns; a workgroup has at least THREADS threads, and works on ROWS rows at once
template <int GROUP_, int UNITS_, int THREADS_>
struct ShapeT {
  static constexpr int GROUP = GROUP_, UNITS = UNITS_, THREADS = GROUP > THREADS_ ? GROUP : THREADS_, ROWS = THREADS / GROUP, WAVES = GROUP / 64;
  static constexpr int MAX_COLS = GROUP * UNITS * 8;
};

__device__ __forceinline__ float wave_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));       // quad_perm [1,0,3,2]
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));       // [2,3,0,1]
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));      // row_half_mirror
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));      // row_mirror
  const auto rows = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  v = __builtin_bit_cast(float, (uint32_t)rows[0]) + __builtin_bit_cast(float, (uint32_t)rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
  return __builtin_bit_cast(float, (uint32_t)halves[0]) + __builtin_bit_cast(float, (uint32_t)halves[1]);
}

// Sums over the threads of a row.  More than one wave: through LDS, in two buffers by turns, so that one barrier a sum is enough (who writes
// a buffer again has passed the barrier that every reader of its last use arrived at afterwards).  All rows of a workgroup take their sums together.
template <typename S>
struct RowSum {
  float (*lds)[S::ROWS][S::WAVES][2];
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (S::WAVES > 1) {
      const int group = threadIdx.x / S::GROUP, wave = threadIdx.x % S::GROUP / 64;
      if ((threadIdx.x & 63) == 0) { lds[turn][group][wave][0] = a; lds[turn][group][wave][1] = b; }
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int w = 0; w < S::WAVES; w++) { a += lds[turn][group][w][0]; b += lds[turn][group][w][1]; }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ void operator()(float& a) {
    a = wave_sum(a);
    if constexpr (S::WAVES > 1) {
      const int group = threadIdx.x / S::GROUP, wave = threadIdx.x % S::GROUP / 64;
      if ((threadIdx.x & 63) == 0) lds[turn][group][wave][0] = a;
      __syncthreads();
      a = 0.0f;
#pragma unroll
      for (int w = 0; w < S::WAVES; w++) a += lds[turn][group][w][0];
      turn ^= 1;
    }
  }
};

// p + i, as an address that all lanes share and 32 bits of a lane's own (i elements are less than 2^32 bytes)
template <typename T>
__device__ __forceinline__ T* lane_at(T* p, uint32_t i) {
  using Byte = std::conditional_t<std::is_const<T>::value, const char, char>;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(p) + i * (uint32_t)sizeof(T));
}

template <int UNITS> struct Cells { float v[UNITS][8]; };

// Where a lane's units lie in a row: unit u is `count[u]` columns (8, fewer in the row's last unit, or none) from `col[u]` on.  RAGGED: the last
// unit may hold fewer; kernels for rows of whole units do without what that takes.
template <int UNITS_, bool RAGGED_>
struct Place {
  static constexpr int UNITS = UNITS_;
  static constexpr bool RAGGED = RAGGED_;
  uint32_t col[UNITS], from[UNITS];                              // `from`: where eight columns are loaded that hold them
  int count[UNITS];
  int cols;
  __device__ __forceinline__ Place(int t, int group, int cols) : cols(cols) {
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      col[u] = (uint32_t)(t + u * group) * 8;
      count[u] = min(max(cols - (int)col[u], 0), 8);
      from[u] = (uint32_t)max(min((int)col[u], cols - 8), 0);
    }
  }
  __device__ __forceinline__ bool has(int u, int e) const { return RAGGED ? e < count[u] : count[u] > 0; }
  // The same, as if it were another: addresses formed with it are not kept in registers from row to row.
  __device__ __forceinline__ Place another() const {
    Place p = *this;
#pragma unroll
    for (int u = 0; u < UNITS; u++) asm volatile("" : "+v"(p.col[u]), "+v"(p.from[u]), "+v"(p.count[u]));
    return p;
  }
  // v, rounded to T, to unit u of a row; the values as they are stored are left in v
  template <typename T>
  __device__ __forceinline__ void store(T* row, int u, float (&v)[8]) const {
    if (RAGGED) store_up_to_8(lane_at(row, col[u]), count[u], v);
    else if (count[u] > 0) store_up_to_8(lane_at(row, col[u]), 8, v);
    else {
      any4 unused[sizeof(T) / 2];
      round_8<T>(v, unused);
    }
  }
};

// A lane's part of a row as it lies in memory, where it has no columns zeros, or with OTHERS values of other columns of the row.  The last unit of a row, if it is
// not a whole one, is loaded with the columns in front of it (settle moves them out, with OTHERS behind the unit's own): one load whatever the
// size, which nothing waits for before the row's turn.
template <typename T, int UNITS, bool OTHERS = false>
struct Raw {
  static constexpr int WORDS = (int)sizeof(T) * 2;               // of 32 bits in a unit
  any4 w[UNITS][WORDS / 4];
  template <typename P>
  __device__ __forceinline__ void load(const T* row, const P& at) {
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
#pragma unroll
      for (int q = 0; q < WORDS / 4; q++) w[u][q] = any4{0, 0, 0, 0};
      if (!P::RAGGED || at.cols >= 8) {
        if (OTHERS || at.count[u] > 0) {
#pragma unroll
          for (int q = 0; q < WORDS / 4; q++) w[u][q] = *(reinterpret_cast<const any4*>(lane_at(row, at.from[u])) + q);
        }
      } else {                                                   // rows shorter than a load
#pragma unroll 1
        for (int e = 0; e < (OTHERS ? 8 : at.count[u]); e++) {
          uint32_t bits;
          if constexpr (sizeof(T) == 2) bits = (uint32_t)row[OTHERS ? min(e, at.cols - 1) : e].bits << (16 * (e & 1));
          else bits = __builtin_bit_cast(uint32_t, row[OTHERS ? min(e, at.cols - 1) : e]);
#pragma unroll
          for (int q = 0; q < WORDS; q++) w[u][q >> 2][q & 3] |= q == (sizeof(T) == 2 ? e >> 1 : e) ? bits : 0;
        }
      }
    }
  }
  // A row of eight columns or more, without branches: lanes that have no columns load the last ones, and without OTHERS drop them.
  template <typename P>
  __device__ __forceinline__ void load_all(const T* row, const P& at) {
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
      for (int q = 0; q < WORDS / 4; q++) w[u][q] = *(reinterpret_cast<const any4*>(lane_at(row, at.from[u])) + q);
    settle(at);
    if (OTHERS) return;
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
      for (int q = 0; q < WORDS; q++) w[u][q >> 2][q & 3] = at.count[u] > 0 ? w[u][q >> 2][q & 3] : 0;
  }
  // the columns of a unit that is not whole to its front, zeros (OTHERS: those in front of them) behind them
  template <typename P>
  __device__ __forceinline__ void settle(const P& at) {
    if (!P::RAGGED || (at.cols & 7) == 0 || at.cols < 8) return;
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      const int by = at.count[u] > 0 ? 8 - at.count[u] : 0;      // columns in front
      uint32_t v[2 * WORDS];                                     // the unit, and what moves in behind it
      const auto behind = [&] {
#pragma unroll
        for (int q = 0; q < WORDS; q++) v[WORDS + q] = OTHERS ? v[q] : 0;
      };
#pragma unroll
      for (int q = 0; q < WORDS; q++) v[q] = w[u][q >> 2][q & 3];
      if constexpr (sizeof(T) == 2) {
        behind();
#pragma unroll
        for (int q = 0; q < WORDS; q++) v[q] = by & 1 ? __builtin_amdgcn_alignbit(v[q + 1], v[q], 16) : v[q];
      }
#pragma unroll
      for (int step = 1; step < WORDS; step *= 2) {
        const bool move = by & (sizeof(T) == 2 ? 2 * step : step);
        behind();
#pragma unroll
        for (int q = 0; q < WORDS; q++) v[q] = move ? v[q + step] : v[q];
      }
#pragma unroll
      for (int q = 0; q < WORDS; q++) w[u][q >> 2][q & 3] = v[q];
    }
  }
  __device__ __forceinline__ float get(int u, int e) const {
    if constexpr (sizeof(T) == 2) return to_float(T{(uint16_t)(w[u][0][e >> 1] >> (16 * (e & 1)))});
    else {
      const uint32_t bits = w[u][e >> 2][e & 3];
      return __builtin_bit_cast(float, bits);
    }
  }
};

// Nothing is moved across: units one after the other, with the registers of one.
__device__ __forceinline__ void in_turn() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A lane's parameters, of a type known at the call, from element `first` on; without any `otherwise`.  Zeros where it has no columns.
template <typename T, typename P>
__device__ __forceinline__ void load_typed(const void* p, int64_t first, const P& at, Cells<P::UNITS>& c) {
  constexpr int UNITS = P::UNITS;
  Raw<T, UNITS> raw;
  raw.load((const T*)p + first, at);
  raw.settle(at);
#pragma unroll
  for (int u = 0; u < UNITS; u++)
#pragma unroll
    for (int e = 0; e < 8; e++) c.v[u][e] = raw.get(u, e);
}
template <typename P>
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t first, const P& at, float otherwise, Cells<P::UNITS>& c) {
  constexpr int UNITS = P::UNITS;
  if (!p) {
#pragma unroll
    for (int u = 0; u < UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) c.v[u][e] = (P::RAGGED ? e < at.count[u] : at.count[u] > 0) ? otherwise : 0.0f;
  } else if (dtype == TF24_F32) load_typed<float>(p, first, at, c);
  else if (dtype == TF24_F16) load_typed<f16_t>(p, first, at, c);
  else load_typed<bf16_t>(p, first, at, c);
}
// unit u of them alone
template <typename P>
__device__ __forceinline__ void load_unit(const void* p, int dtype, int64_t first, const P& at, int u, float otherwise, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (P::RAGGED ? e < at.count[u] : at.count[u] > 0) ? otherwise : 0.0f;
    return;
  }
  if (!P::RAGGED && at.count[u] <= 0) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    return;
  }
  const int n = P::RAGGED ? at.count[u] : 8;
  if (dtype == TF24_F32) load_up_to_8(lane_at((const float*)p + first, at.col[u]), n, v);
  else if (dtype == TF24_F16) load_up_to_8(lane_at((const f16_t*)p + first, at.col[u]), n, v);
  else load_up_to_8(lane_at((const bf16_t*)p + first, at.col[u]), n, v);
}
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t at, float otherwise) {
  if (!p) return otherwise;
  if (dtype == TF24_F32) return ((const float*)p)[at];
  return dtype == TF24_F16 ? to_float(((const f16_t*)p)[at]) : to_float(((const bf16_t*)p)[at]);
}

// ---------------------------------------------------------------- host
// the narrowest shape that holds a row of up to kNarrowCols; THREADS: the least number of a workgroup
template <int THREADS, typename F>
auto with_shape(int64_t cols, F&& f) {
  if (cols <= 512) return f(ShapeT<64, 1, THREADS>{});
  constexpr int WIDE = THREADS > 256 ? THREADS : 64;             // (forward: one row to a workgroup, whose barriers are its own)
  if (cols <= 1024) return f(ShapeT<128, 1, WIDE>{});
  if (cols <= 2048) return f(ShapeT<256, 1, WIDE>{});
  if (cols <= 4096) return f(ShapeT<512, 1, WIDE>{});
  return f(ShapeT<512, 2, WIDE>{});
}
constexpr int kForwardThreads = 256, kBackwardThreads = 512;
// What 256 compute units hold at once, so that no part of a round runs by itself: forward four waves a SIMD, backward a workgroup of eight
// waves a compute unit, two a SIMD (3003 rows of 1601 columns in 1502 workgroups and 259 pieces 56 us both passes, in 1001 and 252 43).
constexpr uint32_t kForwardWaves = 4096, kBackwardPieces = 256;

template <typename F>
auto with_types(int stream_dtype, int block_dtype, F&& f) {
  if (stream_dtype == TF24_F32) {
    if (block_dtype == TF24_F32) return f(float{}, float{});
    if (block_dtype == TF24_F16) return f(float{}, f16_t{});
    return f(float{}, bf16_t{});
  }
  if (stream_dtype == TF24_F16) return f(f16_t{}, f16_t{});
  return f(bf16_t{}, bf16_t{});
}

bool is_float(int dt) { return dt == TF24_F32 || dt == TF24_F16 || dt == TF24_BF16; }

int check_norm(const char* fn, int stream_dtype, int block_dtype, int param_dtype, int gate_dtype, int64_t rows, int64_t cols, bool gate, int64_t rows_per_gate,
               int post_kind, int pre_kind) {
  if (!is_float(stream_dtype) || !is_float(block_dtype) || (stream_dtype != TF24_F32 && block_dtype != stream_dtype))
    return fail(TF24_ERR_DTYPE, "%s: types %d (stream) and %d (block) are not supported together", fn, stream_dtype, block_dtype);
  if (!is_float(param_dtype) || (gate && !is_float(gate_dtype))) return fail(TF24_ERR_DTYPE, "%s: unsupported parameter or gate dtype %d, %d", fn, param_dtype, gate_dtype);
  if (rows < 0 || rows > 0x7fffffffLL - kForwardWaves || cols < 1 || cols > kMaxCols)
    return fail(TF24_ERR_SHAPE, "%s: shape (%lld, %lld) is not supported: 1 to %d columns", fn, (long long)rows, (long long)cols, kMaxCols);
  if (post_kind < 0 || post_kind > TF24_NORM_LAYER || pre_kind < 0 || pre_kind > TF24_NORM_LAYER) return fail(TF24_ERR_ARG, "%s: bad kind of norm %d, %d", fn, post_kind, pre_kind);
  if (gate && rows && (rows_per_gate < 1 || rows % rows_per_gate))
    return fail(TF24_ERR_SHAPE, "%s: %lld rows do not divide into gates of %lld", fn, (long long)rows, (long long)rows_per_gate);
  return TF24_OK;
}

}  // namespace
}  // namespace tf24
