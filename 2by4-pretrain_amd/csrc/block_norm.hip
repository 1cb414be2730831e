// What stands between the blocks of a transformer, in one pass over memory each way:
//
//     z = N_post(y)  (or y)         h = rho x + g z         n = N_pre(h)
//
// x is the residual stream (type R), y a block's output and n the next block's input (type T), g a gate: none, one per channel, per
// group of rows (a sequence) or per row.  N is a layer norm ((v - mean) r w + b, r = 1 / sqrt(var + eps)) or an rms norm (v r w + b, r = 1 /
// sqrt(mean v^2 + eps)).  h is rounded to R before it is normalised: what n is computed from is what the next block's
// addition and the backward pass read.  Without y this is the norm before the first block: n = N_pre(x).
//
// Backward, from dh and dn, with q = dn w_pre and hhat = (h - mean) r:
//     d  = dh + r (q - mean(q) - hhat mean(q hhat))           (rms: without mean(q))
//     dx = rho d        dy = N_post's backward of g d         the sums over rows: dn hhat, dn, d yhat, d
// of which the gradients of weights, biases and a gate that rows share are formed: with A = sum d yhat and B = sum d over the rows that
// share a gate, dg = w_post A + b_post B, dw_post = sum over gates g A, db_post = sum g B; without a norm of y, A = sum d y and dg = A.
//
// Bound by memory: a row is read once and kept in registers while its means are taken (the variance from the centred values: a
// second pass over registers, not over memory).  A row belongs to a wave (up to 1024 columns), or to 2 to 16 waves that
// exchange their sums through LDS; a lane holds one or two units of eight adjacent columns, so accesses are 16 bytes whatever the type
// and the alignment, and four adjacent lanes hold a block of what is kept in 8 bits (checkpoint8.hpp).  Workgroups take runs of rows, keep the
// parameters in registers, and load the next row while they compute on one.  In the backward pass a run ends in one partial sum per column, which a
// second launch adds in a fixed order: no atomics, the same bits every time.
#include "checkpoint8.hpp"

namespace tf24 {
namespace {

constexpr int kMaxCols = 16384;

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

// A lane's part of a row as it lies in memory, zeros behind the last column
template <typename T, int UNITS>
struct Raw {
  any4 w[UNITS][sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, const uint32_t (&col)[UNITS], const int (&n)[UNITS]) {
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
      const T* p = row + col[u];
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; q++) w[u][q] = any4{0, 0, 0, 0};
      if (n[u] == 8) {
#pragma unroll
        for (int q = 0; q < (int)sizeof(T) / 2; q++) w[u][q] = *(reinterpret_cast<const any4*>(p) + q);
      } else if (n[u] > 0) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e < n[u]) {
            if constexpr (sizeof(T) == 2) w[u][0][e >> 1] |= (uint32_t)p[e].bits << (16 * (e & 1));
            else w[u][e >> 2][e & 3] = __builtin_bit_cast(uint32_t, p[e]);
          }
      }
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

template <int UNITS> struct Cells { float v[UNITS][8]; };

// `n` <= 8 parameters from element `at` on, of a type known at the call, zeros behind them; `otherwise` without any
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t at, int n, float otherwise, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = e < n ? otherwise : 0.0f;
  } else if (dtype == TF24_F32) load_up_to_8((const float*)p + at, n, v);
  else if (dtype == TF24_F16) load_up_to_8((const f16_t*)p + at, n, v);
  else load_up_to_8((const bf16_t*)p + at, n, v);
}
__device__ __forceinline__ void store_result(void* p, int dtype, int64_t at, float v) {
  if (dtype == TF24_F32) ((float*)p)[at] = v;
  else if (dtype == TF24_F16) ((f16_t*)p)[at] = from_float<f16_t>(v);
  else ((bf16_t*)p)[at] = from_float<bf16_t>(v);
}

// mean (0 for an rms norm) and r of a row whose columns behind the last one hold 0; the row itself becomes what the mean leaves of it.
// The mean is off by some units of its last place, which next to a small deviation is a lot: the sum of the centred values (exact differences
// where that matters) shows by how much, and goes with the sum of their squares.
template <typename S>
__device__ __forceinline__ void statistics(Cells<S::UNITS>& c, const int (&n)[S::UNITS], int kind, float inv_cols, float eps, RowSum<S>& sum, float& mean, float& r) {
  mean = 0.0f;
  float s = 0.0f, left = 0.0f;
  if (kind == TF24_NORM_LAYER) {
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) s += c.v[u][e];
    sum(s);
    mean = s * inv_cols;
    s = 0.0f;
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        c.v[u][e] = e < n[u] ? c.v[u][e] - mean : 0.0f;
        s = __builtin_fmaf(c.v[u][e], c.v[u][e], s);
        left += c.v[u][e];
      }
    sum(s, left);
    left *= inv_cols;
    mean += left;
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) c.v[u][e] = e < n[u] ? c.v[u][e] - left : 0.0f;
  } else {
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) s = __builtin_fmaf(c.v[u][e], c.v[u][e], s);
    sum(s);
  }
  r = rsqrtf(__builtin_fmaf(s, inv_cols, eps) - left * left);
}

struct ForwardArgs {
  const void *x, *y, *gate, *post_weight, *post_bias, *pre_weight, *pre_bias;
  void *out, *n;
  float* stats;                     // [4][rows]: mean and r of the norm behind, of the norm before; NULL: not kept
  uint8_t *values, *scales;         // n in 8 bits; NULL: not kept
  int64_t ld_x, ld_y, ld_gate;
  uint32_t rows, rows_per_block, rows_per_gate;
  int cols, blocks;                 // blocks of 32 columns in a row
  int param_dtype, gate_dtype, post_kind, pre_kind;
  float scale, eps, inv_cols;
};

template <typename R, typename T, bool RESIDUAL, typename S>
__global__ void __launch_bounds__(S::THREADS)
block_norm_forward(const ForwardArgs a) {
  constexpr int U = S::UNITS;
  static_assert(S::ROWS == 1 || S::WAVES == 1, "rows of a workgroup end at different times: no barriers then");
  __shared__ float lds[2][S::ROWS][S::WAVES][2];
  RowSum<S> sum{lds};
  const int t = threadIdx.x % S::GROUP;
  const uint32_t last = min(a.rows, (blockIdx.x + 1) * a.rows_per_block);
  uint32_t row = blockIdx.x * a.rows_per_block + (S::ROWS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::GROUP) : 0);
  int n[U];
  uint32_t col[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    col[u] = (uint32_t)(t + u * S::GROUP) * 8;
    n[u] = min(max(a.cols - (int)col[u], 0), 8);
  }
  struct Row { Raw<R, U> x; Raw<T, U> y; };
  Row rows[2];
  auto load = [&](Row& r, uint32_t at) {
    r.x.load((const R*)a.x + (int64_t)at * a.ld_x, col, n);
    if (RESIDUAL) r.y.load((const T*)a.y + (int64_t)at * a.ld_y, col, n);
  };
  if (row < last) load(rows[0], row);
  Cells<U> post_w, post_b, pre_w, pre_b, gate;
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (RESIDUAL) {
      load_params(a.post_weight, a.param_dtype, col[u], n[u], 1.0f, post_w.v[u]);
      load_params(a.post_bias, a.param_dtype, col[u], n[u], 0.0f, post_b.v[u]);
    }
    load_params(a.pre_weight, a.param_dtype, col[u], n[u], 1.0f, pre_w.v[u]);
    load_params(a.pre_bias, a.param_dtype, col[u], n[u], 0.0f, pre_b.v[u]);
  }
  uint32_t gate_row = ~0u;
  // (columns behind the last one hold zeros throughout: their weights and biases are zeros)
  auto process = [&](const Row& r, uint32_t row) {
    Cells<U> h, v;
    if constexpr (RESIDUAL) {
      if (a.gate && row / a.rows_per_gate != gate_row) {
        gate_row = row / a.rows_per_gate;
#pragma unroll
        for (int u = 0; u < U; u++) load_params(a.gate, a.gate_dtype, gate_row * a.ld_gate + col[u], n[u], 1.0f, gate.v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) v.v[u][e] = r.y.get(u, e);
      if (a.post_kind) {
        float mean, scale;
        statistics<S>(v, n, a.post_kind, a.inv_cols, a.eps, sum, mean, scale);
        if (a.stats && t == 0) { a.stats[row] = mean; a.stats[a.rows + row] = scale; }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) v.v[u][e] = __builtin_fmaf(v.v[u][e] * scale, post_w.v[u][e], post_b.v[u][e]);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(a.scale, r.x.get(u, e), a.gate ? gate.v[u][e] * v.v[u][e] : v.v[u][e]);
        store_up_to_8((R*)a.out + (int64_t)row * a.cols + col[u], n[u], h.v[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = r.x.get(u, e);
    }
    if (a.pre_kind) {
      float mean, scale;
      statistics<S>(h, n, a.pre_kind, a.inv_cols, a.eps, sum, mean, scale);
      if (a.stats && t == 0) { a.stats[2 * (uint64_t)a.rows + row] = mean; a.stats[3 * (uint64_t)a.rows + row] = scale; }
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(h.v[u][e] * scale, pre_w.v[u][e], pre_b.v[u][e]);
        store_up_to_8((T*)a.n + (int64_t)row * a.cols + col[u], n[u], h.v[u]);
        if (a.values) {
          const Kept8 k = keep_8<T>(h.v[u]);
          if ((int)col[u] < a.blocks * kKeptBlock) {
            const uint64_t unit = (uint64_t)row * a.blocks * kKeptLanes + col[u] / 8;
            *reinterpret_cast<uint2*>(a.values + unit * 8) = k.values;
            if ((t & 3) == 0) a.scales[unit >> 2] = (uint8_t)k.scale;
          }
        }
      }
    }
  };
  while (row < last) {                                           // (by twos: a copy of a row's registers would wait for its loads)
    const uint32_t second = row + S::ROWS, third = second + S::ROWS;
    if (second < last) load(rows[1], second);
    process(rows[0], row);
    if (second >= last) break;
    if (third < last) load(rows[0], third);
    process(rows[1], second);
    row = third;
  }
}

// Rows of a backward workgroup: piece `sub` of the rows of a gate, or of all rows where no gate is shared by some of them
struct Pieces {
  uint32_t groups, per_group, rows_of_group;
  __host__ __device__ uint32_t count() const { return groups * per_group; }
};

struct BackwardArgs {
  const void *grad_out, *grad_n, *h, *y, *gate, *post_weight, *post_bias, *pre_weight;
  const float* stats;
  void *grad_x, *grad_y, *grad_gate;          // grad_gate: of a gate per row only
  float* partial;                             // [4][pieces][cols]: sums of d yhat, d, dn hhat, dn; NULL: none is wanted
  int64_t ld_grad_out, ld_grad_n, ld_h, ld_y, ld_gate;
  Pieces pieces;
  uint32_t rows;
  int cols, gate_per_row, param_dtype, gate_dtype, post_kind, pre_kind;
  float scale, inv_cols;
};

template <typename R, typename T, bool RESIDUAL, typename S>
__global__ void __launch_bounds__(S::THREADS)
block_norm_backward(const BackwardArgs a) {
  constexpr int U = S::UNITS;
  __shared__ float lds[2][S::ROWS][S::WAVES][2];
  __shared__ __attribute__((aligned(16))) float column_sums[S::ROWS > 1 ? S::ROWS : 1][S::ROWS > 1 ? S::MAX_COLS : 4];
  RowSum<S> sum{lds};
  const int t = threadIdx.x % S::GROUP;
  const uint32_t turn = S::ROWS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::GROUP) : 0;
  const uint32_t group = blockIdx.x / a.pieces.per_group, sub = blockIdx.x - group * a.pieces.per_group;
  const uint32_t start = group * a.pieces.rows_of_group;
  const uint32_t first = start + (uint32_t)((uint64_t)sub * a.pieces.rows_of_group / a.pieces.per_group);
  const uint32_t last = start + (uint32_t)((uint64_t)(sub + 1) * a.pieces.rows_of_group / a.pieces.per_group);
  int n[U];
  uint32_t col[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    col[u] = (uint32_t)(t + u * S::GROUP) * 8;
    n[u] = min(max(a.cols - (int)col[u], 0), 8);
  }
  struct Row { Raw<R, U> dout, h; Raw<T, U> dn, y; };
  Row rows[2] = {};
  auto load = [&](Row& r, uint32_t at) {
    if (a.grad_out) r.dout.load((const R*)a.grad_out + (int64_t)at * a.ld_grad_out, col, n);
    if (a.pre_kind) {
      r.dn.load((const T*)a.grad_n + (int64_t)at * a.ld_grad_n, col, n);
      r.h.load((const R*)a.h + (int64_t)at * a.ld_h, col, n);
    }
    if (RESIDUAL && a.y) r.y.load((const T*)a.y + (int64_t)at * a.ld_y, col, n);
  };
  if (first + turn < last) load(rows[0], first + turn);
  // Columns behind the last one have zeros for weights and gradients, and what their other terms are (hat: minus the mean) meets a zero before a sum.
  // `post_w` is the weight times the gate that the rows share.
  Cells<U> post_w, pre_w, sum_dy, sum_d, sum_nh, sum_n;
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (RESIDUAL) {
      load_params(a.post_weight, a.param_dtype, col[u], n[u], 1.0f, post_w.v[u]);
      if (a.gate && !a.gate_per_row) {
        float gate[8];
        load_params(a.gate, a.gate_dtype, group * a.ld_gate + col[u], n[u], 1.0f, gate);
#pragma unroll
        for (int e = 0; e < 8; e++) post_w.v[u][e] *= gate[e];
      }
    }
    load_params(a.pre_weight, a.param_dtype, col[u], n[u], 1.0f, pre_w.v[u]);
#pragma unroll
    for (int e = 0; e < 8; e++) sum_dy.v[u][e] = sum_d.v[u][e] = sum_nh.v[u][e] = sum_n.v[u][e] = 0.0f;
  }
  // One row of each of the workgroup's groups of threads; `here`: there is one (the others go along with zeros, for the barriers).
  auto process = [&](const Row& r, uint32_t row, bool here) {
    const uint32_t at = here ? row : first;
    Cells<U> d;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) d.v[u][e] = r.dout.get(u, e);
    if (a.pre_kind) {
      const float mean = a.stats[2 * (uint64_t)a.rows + at], scale = a.stats[3 * (uint64_t)a.rows + at], shift = -mean * scale;
      Cells<U> hat, q;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float g = r.dn.get(u, e);
          hat.v[u][e] = __builtin_fmaf(r.h.get(u, e), scale, shift);
          sum_nh.v[u][e] = __builtin_fmaf(g, hat.v[u][e], sum_nh.v[u][e]);
          sum_n.v[u][e] += g;
          q.v[u][e] = g * pre_w.v[u][e];
          s1 += q.v[u][e];
          s2 = __builtin_fmaf(q.v[u][e], hat.v[u][e], s2);
        }
      sum(s1, s2);
      s1 = a.pre_kind == TF24_NORM_LAYER ? s1 * a.inv_cols : 0.0f;
      s2 *= -a.inv_cols;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) d.v[u][e] = __builtin_fmaf(scale, __builtin_fmaf(hat.v[u][e], s2, q.v[u][e] - s1), d.v[u][e]);
    }
    if (a.grad_x && here) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        float dx[8];
#pragma unroll
        for (int e = 0; e < 8; e++) dx[e] = a.scale * d.v[u][e];
        store_up_to_8((R*)a.grad_x + (int64_t)row * a.cols + col[u], n[u], dx);
      }
    }
    if constexpr (RESIDUAL) {
      const float mean = a.post_kind ? a.stats[at] : 0.0f, scale = a.post_kind ? a.stats[a.rows + at] : 1.0f, shift = -mean * scale;
      if (a.gate_per_row) {                                      // d becomes that of z
#pragma unroll
        for (int u = 0; u < U; u++) {
          float gate[8];
          load_params(a.gate, a.gate_dtype, at * a.ld_gate + col[u], n[u], 1.0f, gate);
          if (a.grad_gate && here) {
            float dg[8], b[8];
            load_params(a.post_bias, a.param_dtype, col[u], n[u], 0.0f, b);
#pragma unroll
            for (int e = 0; e < 8; e++) dg[e] = d.v[u][e] * (a.post_kind ? __builtin_fmaf(__builtin_fmaf(r.y.get(u, e), scale, shift), post_w.v[u][e], b[e]) : r.y.get(u, e));
            if (a.gate_dtype == TF24_F32) store_up_to_8((float*)a.grad_gate + (int64_t)row * a.cols + col[u], n[u], dg);
            else if (a.gate_dtype == TF24_F16) store_up_to_8((f16_t*)a.grad_gate + (int64_t)row * a.cols + col[u], n[u], dg);
            else store_up_to_8((bf16_t*)a.grad_gate + (int64_t)row * a.cols + col[u], n[u], dg);
          }
#pragma unroll
          for (int e = 0; e < 8; e++) d.v[u][e] *= gate[e];
        }
      }
      Cells<U> hat;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          hat.v[u][e] = __builtin_fmaf(r.y.get(u, e), scale, shift);
          sum_dy.v[u][e] = __builtin_fmaf(d.v[u][e], hat.v[u][e], sum_dy.v[u][e]);
          sum_d.v[u][e] += d.v[u][e];
          d.v[u][e] *= post_w.v[u][e];
          s1 += d.v[u][e];
          s2 = __builtin_fmaf(d.v[u][e], hat.v[u][e], s2);
        }
      if (a.post_kind) {
        sum(s1, s2);
        s1 = a.post_kind == TF24_NORM_LAYER ? s1 * a.inv_cols : 0.0f;
        s2 *= -a.inv_cols;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) d.v[u][e] = scale * __builtin_fmaf(hat.v[u][e], s2, d.v[u][e] - s1);
      }
      if (a.grad_y && here) {
#pragma unroll
        for (int u = 0; u < U; u++) store_up_to_8((T*)a.grad_y + (int64_t)row * a.cols + col[u], n[u], d.v[u]);
      }
    }
  };
  for (uint32_t base = first; base < last; base += 2 * S::ROWS) {          // (by twos: a copy of a row's registers would wait for its loads)
    const uint32_t row = base + turn, second = row + S::ROWS, third = second + S::ROWS;
    if (second < last) load(rows[1], second);
    else rows[1] = {};
    process(rows[0], row, row < last);
    if (base + S::ROWS >= last) break;
    if (third < last) load(rows[0], third);
    else rows[0] = {};
    process(rows[1], second, second < last);
  }
  if (!a.partial) return;
  const uint32_t pieces = a.pieces.count();
#pragma unroll
  for (int k = RESIDUAL ? 0 : 2; k < 4; k++) {
    const Cells<U>& c = k == 0 ? sum_dy : k == 1 ? sum_d : k == 2 ? sum_nh : sum_n;
    float* to = a.partial + ((uint64_t)k * pieces + blockIdx.x) * a.cols;
    if constexpr (S::ROWS == 1) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = c.v[u][e];
        store_up_to_8(to + col[u], n[u], v);
      }
    } else {
      float* mine = column_sums[threadIdx.x / S::GROUP];
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) mine[(e >> 2) * (S::MAX_COLS / 2) + (t + u * S::GROUP) * 4 + (e & 3)] = c.v[u][e];
      __syncthreads();
      for (int i = threadIdx.x; i < a.cols; i += S::THREADS) {
        const int at = ((i >> 2) & 1) * (S::MAX_COLS / 2) + (i >> 3) * 4 + (i & 3);
        float v = column_sums[0][at];
#pragma unroll
        for (int w = 1; w < S::ROWS; w++) v += column_sums[w][at];
        to[i] = v;
      }
      __syncthreads();
    }
  }
}

// The gradients of the parameters from the pieces' sums.  Job 0: weight of the norm behind, 1: its bias, 2, 3: those of the norm before,
// from 4 on: the gates that rows share; a workgroup takes 32 columns of a job, 32 strands of pieces side by side, or where a gate has few pieces
// a gate for each strand.
struct FinishArgs {
  const float* partial;
  const void *gate, *post_weight, *post_bias;
  void *grad_post_weight, *grad_post_bias, *grad_pre_weight, *grad_pre_bias, *grad_gate;
  int64_t ld_gate;
  Pieces pieces;
  int cols, column_blocks, gate_per_row, param_dtype, gate_dtype, post_kind;
  __host__ __device__ bool strand_per_gate() const { return pieces.per_group < 16; }
};

constexpr int kStrands = 32;
__global__ void __launch_bounds__(32 * kStrands)
block_norm_finish(const FinishArgs a) {
  __shared__ float strands[kStrands][33];
  const uint32_t job = blockIdx.x / a.column_blocks;
  void* to = job == 0 ? a.grad_post_weight : job == 1 ? a.grad_post_bias : job == 2 ? a.grad_pre_weight : job == 3 ? a.grad_pre_bias : a.grad_gate;
  if (!to) return;
  const int c = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int col = (int)(blockIdx.x - job * a.column_blocks) * 32 + c;
  const uint32_t pieces = a.pieces.count();
  const bool alone = job >= 4 && a.strand_per_gate();
  const uint32_t gate = job < 4 ? 0 : alone ? (job - 4) * kStrands + strand : job - 4;
  const uint32_t begin = gate * a.pieces.per_group, end = job < 4 ? pieces : min(pieces, begin + a.pieces.per_group);
  const uint32_t step = alone ? 1 : kStrands;
  float total = 0.0f;
  if (col < a.cols) {
    const uint64_t one = (uint64_t)pieces * a.cols;
    const float* from = a.partial + (job < 4 ? job * one : 0) + col;
    const bool gated = job < 2 && a.gate && !a.gate_per_row, affine = job >= 4 && a.post_kind;
    float w[8], b[8];
    if (affine) {
      load_params(a.post_weight, a.param_dtype, col, 1, 1.0f, w);
      load_params(a.post_bias, a.param_dtype, col, 1, 0.0f, b);
    }
    for (uint32_t p0 = begin + (alone ? 0 : strand); p0 < end; p0 += 8 * step) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = p0 + i * step < end ? from[(uint64_t)(p0 + i * step) * a.cols] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t p = p0 + i * step;
        if (p < end) {
          if (gated) {
            float g[8];
            load_params(a.gate, a.gate_dtype, p / a.pieces.per_group * a.ld_gate + col, 1, 1.0f, g);
            v[i] *= g[0];
          } else if (affine) {
            v[i] = __builtin_fmaf(w[0], v[i], b[0] * from[one + (uint64_t)p * a.cols]);
          }
          total += v[i];
        }
      }
    }
  }
  if (alone) {
    if (gate < a.pieces.groups && col < a.cols) store_result(to, a.gate_dtype, (int64_t)gate * a.cols + col, total);
    return;
  }
  strands[strand][c] = total;
  __syncthreads();
  if (strand == 0 && col < a.cols) {
#pragma unroll
    for (int s = 1; s < kStrands; s++) total += strands[s][c];
    store_result(to, job < 4 ? a.param_dtype : a.gate_dtype, (int64_t)gate * a.cols + col, total);
  }
}

// ---------------------------------------------------------------- host
// the narrowest shape that holds a row; THREADS: the least number of a workgroup
template <int THREADS, typename F>
auto with_shape(int64_t cols, F&& f) {
  if (cols <= 512) return f(ShapeT<64, 1, THREADS>{});
  constexpr int WIDE = THREADS > 256 ? THREADS : 64;             // (forward: one row to a workgroup, whose barriers are its own)
  if (cols <= 1024) return f(ShapeT<128, 1, WIDE>{});
  if (cols <= 2048) return f(ShapeT<256, 1, WIDE>{});
  if (cols <= 4096) return f(ShapeT<512, 1, WIDE>{});
  if (cols <= 8192) return f(ShapeT<512, 2, WIDE>{});
  return f(ShapeT<1024, 2, WIDE>{});
}
constexpr int kForwardThreads = 256, kBackwardThreads = 512;

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

// What 256 compute units hold at once, so that no part of a round runs by itself: forward four waves a SIMD, backward a workgroup of eight
// waves a compute unit, two a SIMD (3003 rows of 1601 columns in 1502 workgroups and 259 pieces 56 us both passes, in 1001 and 252 40).
constexpr uint32_t kForwardWaves = 4096, kBackwardPieces = 256;

Pieces plan_pieces(int64_t rows, int64_t cols, int64_t rows_per_gate) {
  const uint32_t groups = rows_per_gate > 1 && rows_per_gate < rows ? (uint32_t)(rows / rows_per_gate) : 1;
  const uint32_t rows_of_group = (uint32_t)(rows / groups);
  const uint32_t at_once = with_shape<kBackwardThreads>(cols, [](auto s) { return (uint32_t)decltype(s)::ROWS; });
  const uint32_t wanted = groups < kBackwardPieces ? kBackwardPieces / groups : 1, most = (rows_of_group + at_once - 1) / at_once;
  return {groups, wanted < most ? wanted : most, rows_of_group};
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

extern "C" int tf24_block_norm_forward(const void* x, int64_t ld_x, const void* y, int64_t ld_y, int stream_dtype, int block_dtype, int64_t rows, int64_t cols,
                                       const void* gate, int gate_dtype, int64_t ld_gate, int64_t rows_per_gate, const void* post_weight, const void* post_bias,
                                       const void* pre_weight, const void* pre_bias, int param_dtype, int post_kind, int pre_kind, float scale, float eps, void* out,
                                       void* n, float* stats, void* values, void* scales, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_block_norm_forward";
  if (int rc = check_norm(fn, stream_dtype, block_dtype, param_dtype, gate_dtype, rows, cols, gate, rows_per_gate, post_kind, pre_kind)) return rc;
  if (!rows) return TF24_OK;
  if (!x || (y && !out) || (pre_kind && !n) || (!y && (!pre_kind || post_kind || gate || out)) || !values != !scales || (values && !pre_kind))
    return fail(TF24_ERR_ARG, "%s: null pointer, or one that nothing is read from or written to", fn);
  if (ld_x < 0 || ld_y < 0 || ld_gate < 0) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  if (int rc = check_aligned(fn, dtype_size(stream_dtype), {x, out})) return rc;
  if (int rc = check_aligned(fn, dtype_size(block_dtype), {y, n})) return rc;
  if (int rc = check_aligned(fn, dtype_size(param_dtype), {post_weight, post_bias, pre_weight, pre_bias})) return rc;
  if (int rc = check_aligned(fn, gate ? dtype_size(gate_dtype) : 1, {gate})) return rc;
  if (int rc = check_aligned(fn, 16, {values, stats})) return rc;
  return with_types(stream_dtype, block_dtype, [&](auto r, auto t) {
    return with_shape<kForwardThreads>(cols, [&](auto shape) {
      using S = decltype(shape);
      constexpr uint32_t most = kForwardWaves / (S::THREADS / 64);
      const uint32_t each = (uint32_t)((rows + most - 1) / most);
      const uint32_t per_block = (each + S::ROWS - 1) / S::ROWS * S::ROWS;
      ForwardArgs a{x, y, gate, post_weight, post_bias, pre_weight, pre_bias, out, n, stats, (uint8_t*)values, (uint8_t*)scales, ld_x, ld_y, ld_gate, (uint32_t)rows,
                    per_block, (uint32_t)(gate ? rows_per_gate : 1), (int)cols, (int)kept_blocks(cols), param_dtype, gate_dtype, post_kind, pre_kind, scale, eps,
                    1.0f / (float)cols};
      auto* kernel = y ? block_norm_forward<decltype(r), decltype(t), true, S> : block_norm_forward<decltype(r), decltype(t), false, S>;
      hipLaunchKernelGGL(kernel, dim3(((uint32_t)rows + per_block - 1) / per_block), dim3(S::THREADS), 0, (hipStream_t)stream, a);
      return check_launch("tf24_block_norm_forward");
    });
  });
}

extern "C" int64_t tf24_block_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int64_t rows_per_gate) {
  using namespace tf24;
  if (rows < 1 || cols < 1 || cols > kMaxCols) return 0;
  return (int64_t)plan_pieces(rows, cols, rows_per_gate).count() * cols * 16;
}

extern "C" int tf24_block_norm_backward(const void* grad_out, int64_t ld_grad_out, const void* grad_n, int64_t ld_grad_n, const void* h, int64_t ld_h, const void* y,
                                        int64_t ld_y, int stream_dtype, int block_dtype, int64_t rows, int64_t cols, const void* gate, int gate_dtype, int64_t ld_gate,
                                        int64_t rows_per_gate, const void* post_weight, const void* post_bias, const void* pre_weight, int param_dtype, int post_kind,
                                        int pre_kind, int residual, float scale, const float* stats, void* grad_x, void* grad_y, void* grad_gate,
                                        void* grad_post_weight, void* grad_post_bias, void* grad_pre_weight, void* grad_pre_bias, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_block_norm_backward";
  if (int rc = check_norm(fn, stream_dtype, block_dtype, param_dtype, gate_dtype, rows, cols, gate, rows_per_gate, post_kind, pre_kind)) return rc;
  if (!rows) return fail(TF24_ERR_SHAPE, "%s: no rows", fn);      // (the caller's gradients are zeros)
  const bool post_grads = grad_post_weight || grad_post_bias, wants_gate = grad_gate;
  if ((pre_kind && (!grad_n || !h)) || ((pre_kind || post_kind) && !stats) || (!pre_kind && (!grad_out || grad_pre_weight || grad_pre_bias)) ||
      (!residual && (!pre_kind || y || gate || post_kind || grad_y || post_grads || wants_gate)) || (wants_gate && !gate) ||
      (post_grads && !post_kind) || (!y && (post_kind || wants_gate)))
    return fail(TF24_ERR_ARG, "%s: null pointer, or one that nothing is read from or written to", fn);
  if (ld_grad_out < 0 || ld_grad_n < 0 || ld_h < 0 || ld_y < 0 || ld_gate < 0) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  if (int rc = check_aligned(fn, dtype_size(stream_dtype), {grad_out, h, grad_x})) return rc;
  if (int rc = check_aligned(fn, dtype_size(block_dtype), {grad_n, y, grad_y})) return rc;
  if (int rc = check_aligned(fn, dtype_size(param_dtype), {post_weight, post_bias, pre_weight, grad_post_weight, grad_post_bias, grad_pre_weight, grad_pre_bias})) return rc;
  if (int rc = check_aligned(fn, gate ? dtype_size(gate_dtype) : 1, {gate, grad_gate})) return rc;
  if (int rc = check_aligned(fn, 16, {workspace, stats})) return rc;
  const bool per_row = gate && rows_per_gate == 1 && rows > 1;
  const Pieces pieces = plan_pieces(rows, cols, gate ? rows_per_gate : rows);
  const bool sums = post_grads || grad_pre_weight || grad_pre_bias || (wants_gate && !per_row);
  if (sums && (!workspace || workspace_bytes < (int64_t)pieces.count() * cols * 16))
    return fail(TF24_ERR_ARG, "%s: a workspace of %lld bytes is needed", fn, (long long)pieces.count() * cols * 16);
  const int column_blocks = (int)((cols + 31) / 32);
  const FinishArgs f{(const float*)workspace, gate, post_weight, post_bias, grad_post_weight, grad_post_bias, grad_pre_weight, grad_pre_bias, per_row ? nullptr : grad_gate,
                     ld_gate, pieces, (int)cols, column_blocks, per_row, param_dtype, gate_dtype, post_kind};
  const int64_t gate_jobs = !f.grad_gate ? 0 : f.strand_per_gate() ? (pieces.groups + kStrands - 1) / kStrands : pieces.groups, jobs = 4 + gate_jobs;
  if (jobs * column_blocks > 0x7fffffffLL) return fail(TF24_ERR_SHAPE, "%s: too many gates (%lld)", fn, (long long)pieces.groups);
  const int rc = with_types(stream_dtype, block_dtype, [&](auto r, auto t) {
    return with_shape<kBackwardThreads>(cols, [&](auto shape) {
      using S = decltype(shape);
      BackwardArgs a{grad_out, grad_n, h, y, gate, post_weight, post_bias, pre_weight, stats, grad_x, grad_y, per_row ? grad_gate : nullptr,
                     sums ? (float*)workspace : nullptr, ld_grad_out, ld_grad_n, ld_h, ld_y, ld_gate, pieces, (uint32_t)rows, (int)cols, per_row, param_dtype,
                     gate_dtype, post_kind, pre_kind, scale, 1.0f / (float)cols};
      auto* kernel = residual ? block_norm_backward<decltype(r), decltype(t), true, S> : block_norm_backward<decltype(r), decltype(t), false, S>;
      hipLaunchKernelGGL(kernel, dim3(pieces.count()), dim3(S::THREADS), 0, (hipStream_t)stream, a);
      return check_launch("tf24_block_norm_backward");
    });
  });
  if (rc || !sums) return rc;
  hipLaunchKernelGGL(block_norm_finish, dim3((uint32_t)(jobs * column_blocks)), dim3(32 * kStrands), 0, (hipStream_t)stream, f);
  return check_launch(fn);
}
