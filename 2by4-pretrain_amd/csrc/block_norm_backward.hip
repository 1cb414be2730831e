// The backward pass of the block norms (block_norm.hip has the formulas).
//
// Four sums over the rows stay in registers (32 of a lane) while a workgroup goes through its piece of the rows: 256 pieces, a workgroup of eight waves on
// each compute unit, whose next rows are loaded while it computes on these.  More pieces than are at work at once would be a second round, and their
// partial sums (16 bytes a column and piece) more to write and to add.
// Measured (kernel time, bytes that it cannot do without): 12288 rows of 768, float32 stream and float16 blocks: 37 us = 4.6 TB/s; 8192 rows of 4096
// bf16: 85 us = 4.7 TB/s; block_norm_finish 5.0 and 7.2 us, of which the launch is 2.  The first kernels, without loads ahead: 47 and 146 us.
#include "block_norm_rows.hpp"

namespace tf24 {
namespace {

__device__ __forceinline__ void store_result(void* p, int dtype, int64_t at, float v) {
  if (dtype == TF24_F32) ((float*)p)[at] = v;
  else if (dtype == TF24_F16) ((f16_t*)p)[at] = from_float<f16_t>(v);
  else ((bf16_t*)p)[at] = from_float<bf16_t>(v);
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
  int cols, param_dtype, gate_dtype, post_kind, pre_kind;
  bool gate_per_row;
  float scale, inv_cols;
};

// MODE: rows of whole units; of any number of columns; and with a gate for every row as well
enum { WHOLE, ANY, ROW_GATES };
template <typename R, typename T, bool RESIDUAL, int MODE, typename S>
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
  const Place<U, MODE != WHOLE> place(t, S::GROUP, a.cols);
  struct Row { Raw<R, U> dout; Raw<R, U, true> h; Raw<T, U> dn; Raw<T, U, true> y; float pre_mean, pre_scale, post_mean, post_scale; };
  Row rows[2] = {};
  auto load = [&](Row& r, uint32_t at) {
    if (a.grad_out) r.dout.load((const R*)a.grad_out + (int64_t)at * a.ld_grad_out, place);
    if (a.pre_kind) {
      r.dn.load((const T*)a.grad_n + (int64_t)at * a.ld_grad_n, place);
      r.h.load((const R*)a.h + (int64_t)at * a.ld_h, place);
      r.pre_mean = a.stats[2 * (uint64_t)a.rows + at];
      r.pre_scale = a.stats[3 * (uint64_t)a.rows + at];
    }
    if (RESIDUAL && a.y) r.y.load((const T*)a.y + (int64_t)at * a.ld_y, place);
    if (RESIDUAL && a.post_kind) {
      r.post_mean = a.stats[at];
      r.post_scale = a.stats[a.rows + at];
    }
  };
  if (first + turn < last) load(rows[0], first + turn);
  // Columns behind the last one have zeros for weights and gradients and another column's normed value, so that every term of theirs in a sum is a zero
  // (with zeros for h, its normed value would be minus the mean times r: an infinity in a row of one very large value, and NaN in the sums).
  // `post_w` is the weight times the gate that the rows share.
  Cells<U> post_w, pre_w, sum_dy = {}, sum_d = {}, sum_nh = {}, sum_n = {};
  if (RESIDUAL) {
    load_params(a.post_weight, a.param_dtype, 0, place, 1.0f, post_w);
    if (MODE != ROW_GATES && a.gate) {
      Cells<U> gate;
      load_params(a.gate, a.gate_dtype, group * a.ld_gate, place, 1.0f, gate);
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) post_w.v[u][e] *= gate.v[u][e];
    }
  }
  load_params(a.pre_weight, a.param_dtype, 0, place, 1.0f, pre_w);
  // One row of each of the workgroup's groups of threads; `here`: there is one (the others go along with zeros, for the barriers).
  auto process = [&](Row& r, uint32_t row, bool here) {
    r.dout.settle(place);
    r.h.settle(place);
    r.dn.settle(place);
    if (RESIDUAL) r.y.settle(place);
    Cells<U> d;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) d.v[u][e] = r.dout.get(u, e);
    if (a.pre_kind) {
      const float scale = r.pre_scale, mean = r.pre_mean;
      Cells<U> hat, q;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float g = r.dn.get(u, e);
          hat.v[u][e] = (r.h.get(u, e) - mean) * scale;           // (-mean * scale would be rounded where the mean is large)
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
        for (int e = 0; e < 8; e++) {
          d.v[u][e] = __builtin_fmaf(scale, __builtin_fmaf(hat.v[u][e], s2, q.v[u][e] - s1), d.v[u][e]);
          if (RESIDUAL && !place.has(u, e)) d.v[u][e] = 0.0f;
        }
    }
    if (a.grad_x && here) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        float dx[8];
#pragma unroll
        for (int e = 0; e < 8; e++) dx[e] = a.scale * d.v[u][e];
        place.store((R*)a.grad_x + (int64_t)row * a.cols, u, dx);
      }
    }
    if constexpr (RESIDUAL) {
      const float scale = a.post_kind ? r.post_scale : 1.0f, mean = a.post_kind ? r.post_mean : 0.0f;
      if (MODE == ROW_GATES && here) {                              // d becomes that of z
        Cells<U> gate, bias;
        load_params(a.gate, a.gate_dtype, row * a.ld_gate, place, 1.0f, gate);
        if (a.grad_gate) {
          load_params(a.post_bias, a.param_dtype, 0, place, 0.0f, bias);
#pragma unroll
          for (int u = 0; u < U; u++) {
            float dg[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
              dg[e] = d.v[u][e] * (a.post_kind ? __builtin_fmaf((r.y.get(u, e) - mean) * scale, post_w.v[u][e], bias.v[u][e]) : r.y.get(u, e));
            const int64_t to = (int64_t)row * a.cols;
            if (a.gate_dtype == TF24_F32) place.store((float*)a.grad_gate + to, u, dg);
            else if (a.gate_dtype == TF24_F16) place.store((f16_t*)a.grad_gate + to, u, dg);
            else place.store((bf16_t*)a.grad_gate + to, u, dg);
          }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) d.v[u][e] *= gate.v[u][e];
      }
      Cells<U> hat;
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          hat.v[u][e] = (r.y.get(u, e) - mean) * scale;
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
        for (int u = 0; u < U; u++) place.store((T*)a.grad_y + (int64_t)row * a.cols, u, d.v[u]);
      }
    }
  };
  if constexpr (U > 1) {                                         // (two rows of two units do not fit the registers)
    static_assert(S::ROWS == 1, "a workgroup to a row");
    for (uint32_t row = first; row < last; row++) {
      process(rows[0], row, true);
      if (row + 1 < last) load(rows[0], row + 1);
    }
  } else {
    for (uint32_t base = first; base < last; base += 2 * S::ROWS) {        // (by twos: a copy of a row's registers would wait for its loads)
      const uint32_t row = base + turn, second = row + S::ROWS, third = second + S::ROWS;
      if (second < last) load(rows[1], second);
      else rows[1] = {};
      process(rows[0], row, row < last);
      if (base + S::ROWS >= last) break;
      if (third < last) load(rows[0], third);
      else rows[0] = {};
      process(rows[1], second, second < last);
    }
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
        place.store(to, u, v);
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

// Rows of more columns than the registers above hold: a row to a workgroup of 16 waves with 128 registers a lane.  Parameters and gates are loaded where they
// are used (from the caches), centred values formed twice, and two of the four sums over the rows live in LDS, each lane's own 16 bytes at a time.  A row's
// registers are loaded when its turn comes: the next row's beside them would be spilled.
template <typename R, typename T, bool RESIDUAL, bool RAGGED>
__global__ void __launch_bounds__(kWideThreads)
block_norm_backward_wide(const BackwardArgs a, uint32_t rows_per_gate) {
  using S = ShapeT<kWideThreads, 2, kWideThreads>;
  constexpr int U = S::UNITS;
  typedef float float4w __attribute__((ext_vector_type(4)));
  __shared__ float lds[2][1][S::WAVES][2];
  __shared__ float4w column_sums[RESIDUAL ? 2 : 1][RESIDUAL ? U * 2 : 1][RESIDUAL ? kWideThreads : 1];
  RowSum<S> sum{lds};
  const int t = threadIdx.x;
  const uint32_t group = blockIdx.x / a.pieces.per_group, sub = blockIdx.x - group * a.pieces.per_group;
  const uint32_t start = group * a.pieces.rows_of_group;
  const uint32_t first = start + (uint32_t)((uint64_t)sub * a.pieces.rows_of_group / a.pieces.per_group);
  const uint32_t last = start + (uint32_t)((uint64_t)(sub + 1) * a.pieces.rows_of_group / a.pieces.per_group);
  const Place<U, RAGGED> own(t, S::GROUP, a.cols);
  Cells<U> sum_nh = {}, sum_n = {};
  if (RESIDUAL) {
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int q = 0; q < 2 * U; q++) column_sums[RESIDUAL ? k : 0][RESIDUAL ? q : 0][RESIDUAL ? t : 0] = float4w{0, 0, 0, 0};
  }
  for (uint32_t row = first; row < last; row++) {
    const auto place = own.another();
    Cells<U> d = {};
    if (a.grad_out) {
      Raw<R, U> dout;
      dout.load_all((const R*)a.grad_out + (int64_t)row * a.ld_grad_out, place);
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) d.v[u][e] = dout.get(u, e);
    }
    if (a.pre_kind) {
      const float mean = a.stats[2 * (uint64_t)a.rows + row], scale = a.stats[3 * (uint64_t)a.rows + row];
      float s1 = 0.0f, s2 = 0.0f;
      Raw<R, U, true> h;
      Raw<T, U> dn;
      h.load_all((const R*)a.h + (int64_t)row * a.ld_h, place);
      dn.load_all((const T*)a.grad_n + (int64_t)row * a.ld_grad_n, place);
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        float w[8];
        load_unit(a.pre_weight, a.param_dtype, 0, place, u, 1.0f, w);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float g = dn.get(u, e), hat = (h.get(u, e) - mean) * scale, q = g * w[e];
          sum_nh.v[u][e] = __builtin_fmaf(g, hat, sum_nh.v[u][e]);
          sum_n.v[u][e] += g;
          s1 += q;
          s2 = __builtin_fmaf(q, hat, s2);
        }
      }
      sum(s1, s2);
      s1 = a.pre_kind == TF24_NORM_LAYER ? s1 * a.inv_cols : 0.0f;
      s2 *= -a.inv_cols;
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        float w[8];
        load_unit(a.pre_weight, a.param_dtype, 0, place, u, 1.0f, w);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float hat = (h.get(u, e) - mean) * scale;
          d.v[u][e] = __builtin_fmaf(scale, __builtin_fmaf(hat, s2, dn.get(u, e) * w[e] - s1), d.v[u][e]);
          if (RESIDUAL && !place.has(u, e)) d.v[u][e] = 0.0f;
        }
      }
    }
    if (a.grad_x) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        float dx[8];
#pragma unroll
        for (int e = 0; e < 8; e++) dx[e] = a.scale * d.v[u][e];
        place.store((R*)a.grad_x + (int64_t)row * a.cols, u, dx);
      }
    }
    if constexpr (RESIDUAL) {
      const float mean = a.post_kind ? a.stats[row] : 0.0f, scale = a.post_kind ? a.stats[a.rows + row] : 1.0f;
      Raw<T, U, true> y = {};
      if (a.y) y.load_all((const T*)a.y + (int64_t)row * a.ld_y, place);
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        float w[8], g[8];
        load_unit(a.post_weight, a.param_dtype, 0, place, u, 1.0f, w);
        load_unit(a.gate, a.gate_dtype, row / rows_per_gate * a.ld_gate, place, u, 1.0f, g);
        if (a.grad_gate) {                                         // a gate for every row
          float b[8], dg[8];
          load_unit(a.post_bias, a.param_dtype, 0, place, u, 0.0f, b);
#pragma unroll
          for (int e = 0; e < 8; e++) dg[e] = d.v[u][e] * (a.post_kind ? __builtin_fmaf((y.get(u, e) - mean) * scale, w[e], b[e]) : y.get(u, e));
          const int64_t to = (int64_t)row * a.cols;
          if (a.gate_dtype == TF24_F32) place.store((float*)a.grad_gate + to, u, dg);
          else if (a.gate_dtype == TF24_F16) place.store((f16_t*)a.grad_gate + to, u, dg);
          else place.store((bf16_t*)a.grad_gate + to, u, dg);
        }
#pragma unroll
        for (int half = 0; half < 2; half++) {
          float4w dy = column_sums[0][2 * u + half][t], dd = column_sums[1][2 * u + half][t];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int e = 4 * half + i;
            const float hat = (y.get(u, e) - mean) * scale;
            float v = d.v[u][e];
            if (a.gate_per_row) v *= g[e];                         // (the sums of gates that rows share are taken without them)
            dy[i] = __builtin_fmaf(v, hat, dy[i]);
            dd[i] += v;
            v *= a.gate_per_row ? w[e] : w[e] * g[e];
            s1 += v;
            s2 = __builtin_fmaf(v, hat, s2);
            d.v[u][e] = v;
          }
          column_sums[0][2 * u + half][t] = dy;
          column_sums[1][2 * u + half][t] = dd;
        }
      }
      if (a.post_kind) {
        sum(s1, s2);
        s1 = a.post_kind == TF24_NORM_LAYER ? s1 * a.inv_cols : 0.0f;
        s2 *= -a.inv_cols;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < 8; e++) d.v[u][e] = scale * __builtin_fmaf((y.get(u, e) - mean) * scale, s2, d.v[u][e] - s1);
      }
      if (a.grad_y) {
#pragma unroll
        for (int u = 0; u < U; u++) place.store((T*)a.grad_y + (int64_t)row * a.cols, u, d.v[u]);
      }
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int k = RESIDUAL ? 0 : 2; k < 4; k++) {
    float* to = a.partial + ((uint64_t)k * a.pieces.count() + blockIdx.x) * a.cols;
#pragma unroll
    for (int u = 0; u < U; u++) {
      in_turn();
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (RESIDUAL && k < 2) v[e] = column_sums[RESIDUAL ? k : 0][RESIDUAL ? 2 * u + (e >> 2) : 0][RESIDUAL ? t : 0][e & 3];
        else v[e] = k == 2 ? sum_nh.v[u][e] : sum_n.v[u][e];
      }
      own.store(to, u, v);
    }
  }
}

// The gradients of the parameters from the pieces' sums.  Job 0: weight of the norm behind, 1: its bias, 2, 3: those of the norm before,
// from 4 on: the gates that rows share; a workgroup takes 32 columns of a job, 32 strands of pieces side by side, or where a gate has few pieces
// a gate for each strand.  The pieces are added in float64: with millions of gates a strand has 10^5 of them, and float32 sums of so many are off by thousands of
// units (2^20 gates of two rows, equal terms: 4341), where everything else is off by a few.
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
  __shared__ double strands[kStrands][33];
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
  double total = 0.0;
  if (col < a.cols) {
    const uint64_t one = (uint64_t)pieces * a.cols;
    const float* from = a.partial + (job < 4 ? job * one : 0) + col;
    const bool gated = job < 2 && a.gate && !a.gate_per_row, affine = job >= 4 && a.post_kind;
    const float w = affine ? load_param(a.post_weight, a.param_dtype, col, 1.0f) : 0.0f, b = affine ? load_param(a.post_bias, a.param_dtype, col, 0.0f) : 0.0f;
    for (uint32_t p0 = begin + (alone ? 0 : strand); p0 < end; p0 += 8 * step) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = p0 + i * step < end ? from[(uint64_t)(p0 + i * step) * a.cols] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t p = p0 + i * step;
        if (p < end) {
          if (gated) {
            v[i] *= load_param(a.gate, a.gate_dtype, p / a.pieces.per_group * a.ld_gate + col, 1.0f);
          } else if (affine) {
            v[i] = __builtin_fmaf(w, v[i], b * from[one + (uint64_t)p * a.cols]);
          }
          total += v[i];
        }
      }
    }
  }
  if (alone) {
    if (gate < a.pieces.groups && col < a.cols) store_result(to, a.gate_dtype, (int64_t)gate * a.cols + col, (float)total);
    return;
  }
  strands[strand][c] = total;
  __syncthreads();
  if (strand == 0 && col < a.cols) {
#pragma unroll
    for (int s = 1; s < kStrands; s++) total += strands[s][c];
    store_result(to, job < 4 ? a.param_dtype : a.gate_dtype, (int64_t)gate * a.cols + col, (float)total);
  }
}

// The pieces of the rows: 256 of them (kBackwardPieces), cut at gates that rows share.
Pieces plan_pieces(int64_t rows, int64_t cols, int64_t rows_per_gate) {
  const uint32_t groups = rows_per_gate > 1 && rows_per_gate < rows ? (uint32_t)(rows / rows_per_gate) : 1;
  const uint32_t rows_of_group = (uint32_t)(rows / groups);
  const uint32_t at_once = cols > kNarrowCols ? 1 : with_shape<kBackwardThreads>(cols, [](auto s) { return (uint32_t)decltype(s)::ROWS; });
  const uint32_t most = (rows_of_group + at_once - 1) / at_once;
  if (groups < 16) return {groups, kBackwardPieces / groups < most ? kBackwardPieces / groups : most, rows_of_group};
  // The last round of workgroups should be a full one: with 4096 sequences or more it hardly counts, with 320 of them a piece each would leave three
  // quarters of the second round empty.  In rows, a piece costs those that it has and what begins and ends it.  (Both passes, 1152 columns: 130 gates of 256
  // rows 265 us with a piece each, 217 so; 320 of them 557 and 463.)
  const double ends = 3.0 + 4096.0 / (double)cols;
  uint32_t best = 1;
  double least = 0.0;
  for (uint32_t p = 1; p <= 16 && p <= most; p++) {
    const double rounds = (double)(((uint64_t)groups * p + kBackwardPieces - 1) / kBackwardPieces);
    const double time = rounds * ((double)((most + p - 1) / p * at_once) + ends);
    if (p == 1 || time < least) best = p, least = time;
  }
  return {groups, best, rows_of_group};
}

}  // namespace
}  // namespace tf24

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
  if ((int64_t)pieces.count() * kWideThreads > 0xffffffffLL || (sums && jobs * column_blocks * (32 * kStrands) > 0xffffffffLL))      // (threads of a launch)
    return fail(TF24_ERR_SHAPE, "%s: too many gates (%lld)", fn, (long long)pieces.groups);
  const BackwardArgs a{grad_out, grad_n, h, y, gate, post_weight, post_bias, pre_weight, stats, grad_x, grad_y, per_row ? grad_gate : nullptr,
                       sums ? (float*)workspace : nullptr, ld_grad_out, ld_grad_n, ld_h, ld_y, ld_gate, pieces, (uint32_t)rows, (int)cols, param_dtype,
                       gate_dtype, post_kind, pre_kind, per_row, scale, 1.0f / (float)cols};
  const int rc = with_types(stream_dtype, block_dtype, [&](auto r, auto t) {
    using R = decltype(r);
    using T = decltype(t);
    if (cols > kNarrowCols) {
      auto* kernel = cols % 8 ? (residual ? block_norm_backward_wide<R, T, true, true> : block_norm_backward_wide<R, T, false, true>)
                              : (residual ? block_norm_backward_wide<R, T, true, false> : block_norm_backward_wide<R, T, false, false>);
      hipLaunchKernelGGL(kernel, dim3(pieces.count()), dim3(kWideThreads), 0, (hipStream_t)stream, a, gate ? (uint32_t)rows_per_gate : (uint32_t)rows);
      return check_launch("tf24_block_norm_backward");
    }
    return with_shape<kBackwardThreads>(cols, [&](auto shape) {
      using S = decltype(shape);
      auto* kernel = per_row ? block_norm_backward<R, T, true, ROW_GATES, S>
                             : cols % 8 ? (residual ? block_norm_backward<R, T, true, ANY, S> : block_norm_backward<R, T, false, ANY, S>)
                                        : (residual ? block_norm_backward<R, T, true, WHOLE, S> : block_norm_backward<R, T, false, WHOLE, S>);
      hipLaunchKernelGGL(kernel, dim3(pieces.count()), dim3(S::THREADS), 0, (hipStream_t)stream, a);
      return check_launch("tf24_block_norm_backward");
    });
  });
  if (rc || !sums) return rc;
  hipLaunchKernelGGL(block_norm_finish, dim3((uint32_t)(jobs * column_blocks)), dim3(32 * kStrands), 0, (hipStream_t)stream, f);
  return check_launch(fn);
}
