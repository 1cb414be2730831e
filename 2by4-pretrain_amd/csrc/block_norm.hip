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
// second pass over registers, not over memory).  A row belongs to a wave (up to 512 columns), or to 2 to 16 waves that
// exchange their sums through LDS; a lane holds one or two units of eight adjacent columns, so accesses are 16 bytes whatever the type
// and the alignment, and four adjacent lanes hold a block of what is kept in 8 bits (checkpoint8.hpp).  Workgroups take runs of rows, keep the
// parameters in registers, and load the next row while they compute on one.  In the backward pass a run ends in one partial sum per column, which a
// second launch adds in a fixed order: no atomics, the same bits every time.
//
// Measured (kernel time, bytes that it cannot do without): 12288 rows of 768, float32 stream and float16 blocks, both norms and a gate: 26 us = 4.4 TB/s;
// 8192 rows of 4096 bf16: 53 us = 5.0 TB/s, where a copy of such a size reaches 5.2.  Rows of 1601 bf16, which begin at any even address and end in the middle of a unit:
// 14.4 us for 3003 of them = 2.7 TB/s: three rows to each of 1001 workgroups.  A row of 4096 by itself 3.4 us: the latency of one load, sums over eight
// waves and a store.  A lane's parameters are 40 registers, a row as it is loaded 8 to 16; the next row's keep the memory busy while the sums of one
// wait for each other (the first kernel, which loaded a row when its turn came, took 29.7 and 76.9 us).
#include "block_norm_rows.hpp"

namespace tf24 {
namespace {

// mean (0 for an rms norm) and r of a row whose columns behind the last one hold 0; the row itself becomes what the mean leaves of it.
// The mean is off by some units of its last place, which next to a small deviation is a lot: the sum of the centred values (exact differences
// where that matters) shows by how much, and goes with the sum of their squares.
template <typename S, typename P>
__device__ __forceinline__ void statistics(Cells<S::UNITS>& c, const P& at, int kind, float inv_cols, float eps, RowSum<S>& sum, float& mean, float& r) {
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
        c.v[u][e] = (P::RAGGED ? e < at.count[u] : at.count[u] > 0) ? c.v[u][e] - mean : 0.0f;
        s = __builtin_fmaf(c.v[u][e], c.v[u][e], s);
        left += c.v[u][e];
      }
    sum(s, left);
    left *= inv_cols;
    mean += left;
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) c.v[u][e] = (P::RAGGED ? e < at.count[u] : at.count[u] > 0) ? c.v[u][e] - left : 0.0f;
  } else {
#pragma unroll
    for (int u = 0; u < S::UNITS; u++)
#pragma unroll
      for (int e = 0; e < 8; e++) s = __builtin_fmaf(c.v[u][e], c.v[u][e], s);
    sum(s);
  }
  const float variance = __builtin_fmaf(s, inv_cols, -left * left);
  r = rsqrtf((variance < 0.0f ? 0.0f : variance) + eps);          // (of a row of one value rounding may leave less than nothing; a NaN stays)
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

// n, and what is kept of it in 8 bits
template <typename T, typename P>
__device__ __forceinline__ void store_normed(const ForwardArgs& a, const P& place, uint32_t row, int u, float (&n)[8]) {
  place.store((T*)a.n + (int64_t)row * a.cols, u, n);
  if (a.values) {
    const Kept8 k = keep_8<T>(n);
    if ((int)place.col[u] < a.blocks * kKeptBlock) {
      const uint64_t unit = (uint64_t)row * a.blocks * kKeptLanes + place.col[u] / 8;
      *reinterpret_cast<uint2*>(a.values + unit * 8) = k.values;
      if ((unit & 3) == 0) a.scales[unit >> 2] = (uint8_t)k.scale;
    }
  }
}

template <typename R, typename T, bool RESIDUAL, bool RAGGED, typename S>
__global__ void __launch_bounds__(S::THREADS)
block_norm_forward(const ForwardArgs a) {
  constexpr int U = S::UNITS;
  static_assert(S::ROWS == 1 || S::WAVES == 1, "rows of a workgroup end at different times: no barriers then");
  __shared__ float lds[2][S::ROWS][S::WAVES][2];
  RowSum<S> sum{lds};
  const int t = threadIdx.x % S::GROUP;
  const uint32_t last = min(a.rows, (blockIdx.x + 1) * a.rows_per_block);
  uint32_t row = blockIdx.x * a.rows_per_block + (S::ROWS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::GROUP) : 0);
  const Place<U, RAGGED> place(t, S::GROUP, a.cols);
  struct Row { Raw<R, U> x; Raw<T, U> y; };
  Row rows[2];
  auto load = [&](Row& r, uint32_t at) {
    r.x.load((const R*)a.x + (int64_t)at * a.ld_x, place);
    if (RESIDUAL) r.y.load((const T*)a.y + (int64_t)at * a.ld_y, place);
  };
  if (row < last) load(rows[0], row);
  Cells<U> post_w, post_b, pre_w, pre_b, gate;
  if (RESIDUAL) {
    load_params(a.post_weight, a.param_dtype, 0, place, 1.0f, post_w);
    load_params(a.post_bias, a.param_dtype, 0, place, 0.0f, post_b);
  }
  load_params(a.pre_weight, a.param_dtype, 0, place, 1.0f, pre_w);
  load_params(a.pre_bias, a.param_dtype, 0, place, 0.0f, pre_b);
  uint32_t gate_row = ~0u;
  // (columns behind the last one hold zeros throughout: their weights and biases are zeros)
  auto process = [&](Row& r, uint32_t row) {
    Cells<U> h, v;
    r.x.settle(place);
    if (RESIDUAL) r.y.settle(place);
    if constexpr (RESIDUAL) {
      if (a.gate && row / a.rows_per_gate != gate_row) {
        gate_row = row / a.rows_per_gate;
        load_params(a.gate, a.gate_dtype, gate_row * a.ld_gate, place, 1.0f, gate);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) v.v[u][e] = r.y.get(u, e);
      if (a.post_kind) {
        float mean, scale;
        statistics<S>(v, place, a.post_kind, a.inv_cols, a.eps, sum, mean, scale);
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
        place.store((R*)a.out + (int64_t)row * a.cols, u, h.v[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = r.x.get(u, e);
    }
    if (a.pre_kind) {
      float mean, scale;
      statistics<S>(h, place, a.pre_kind, a.inv_cols, a.eps, sum, mean, scale);
      if (a.stats && t == 0) { a.stats[2 * (uint64_t)a.rows + row] = mean; a.stats[3 * (uint64_t)a.rows + row] = scale; }
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(h.v[u][e] * scale, pre_w.v[u][e], pre_b.v[u][e]);
        store_normed<T>(a, place, row, u, h.v[u]);
      }
    }
  };
  if constexpr (U > 1) {                                         // (two rows of two units do not fit the registers)
    for (; row < last; row += S::ROWS) {
      process(rows[0], row);
      if (row + S::ROWS < last) load(rows[0], row + S::ROWS);
    }
    return;
  }
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

// Rows of more columns than the registers above hold: a row to a workgroup of 16 waves, 128 registers a lane.  Parameters and gates are loaded where they
// are used (from the caches: up to five times four bytes a column beside the eight or twelve of the row itself), the next row's registers when this row's
// have been used.  Both passes of 4000 x 12288 bf16 359 us and of 4000 x 16384 429 (2.2 and 2.4 TB/s); with everything in registers, most of it
// spilled, 990 and 1090.
template <typename R, typename T, bool RESIDUAL, bool RAGGED>
__global__ void __launch_bounds__(kWideThreads)
block_norm_forward_wide(const ForwardArgs a) {
  using S = ShapeT<kWideThreads, 2, kWideThreads>;
  constexpr int U = S::UNITS;
  __shared__ float lds[2][1][S::WAVES][2];
  RowSum<S> sum{lds};
  const int t = threadIdx.x;
  const uint32_t last = min(a.rows, (blockIdx.x + 1) * a.rows_per_block);
  const Place<U, RAGGED> own(t, S::GROUP, a.cols);
  Raw<R, U> x;
  Raw<T, U> y;
  auto load = [&](uint32_t row) {
    x.load((const R*)a.x + (int64_t)row * a.ld_x, own);
    if (RESIDUAL) y.load((const T*)a.y + (int64_t)row * a.ld_y, own);
  };
  const uint32_t first = blockIdx.x * a.rows_per_block;
  if (first < last) load(first);
  for (uint32_t row = first; row < last; row++) {
    const auto place = own.another();
    Cells<U> h;
    x.settle(place);
    if constexpr (RESIDUAL) {
      y.settle(place);
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = y.get(u, e);
      if (a.post_kind) {
        float mean, scale;
        statistics<S>(h, place, a.post_kind, a.inv_cols, a.eps, sum, mean, scale);
        if (a.stats && t == 0) { a.stats[row] = mean; a.stats[a.rows + row] = scale; }
#pragma unroll
        for (int u = 0; u < U; u++) {
          in_turn();
          float w[8], b[8];
          load_unit(a.post_weight, a.param_dtype, 0, place, u, 1.0f, w);
          load_unit(a.post_bias, a.param_dtype, 0, place, u, 0.0f, b);
#pragma unroll
          for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(h.v[u][e] * scale, w[e], b[e]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        if (a.gate) {
          float g[8];
          load_unit(a.gate, a.gate_dtype, row / a.rows_per_gate * a.ld_gate, place, u, 1.0f, g);
#pragma unroll
          for (int e = 0; e < 8; e++) h.v[u][e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(a.scale, x.get(u, e), h.v[u][e]);
        place.store((R*)a.out + (int64_t)row * a.cols, u, h.v[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = x.get(u, e);
    }
    if (row + 1 < last) load(row + 1);
    if (a.pre_kind) {
      float mean, scale;
      statistics<S>(h, place, a.pre_kind, a.inv_cols, a.eps, sum, mean, scale);
      if (a.stats && t == 0) { a.stats[2 * (uint64_t)a.rows + row] = mean; a.stats[3 * (uint64_t)a.rows + row] = scale; }
#pragma unroll
      for (int u = 0; u < U; u++) {
        in_turn();
        float w[8], b[8];
        load_unit(a.pre_weight, a.param_dtype, 0, place, u, 1.0f, w);
        load_unit(a.pre_bias, a.param_dtype, 0, place, u, 0.0f, b);
#pragma unroll
        for (int e = 0; e < 8; e++) h.v[u][e] = __builtin_fmaf(h.v[u][e] * scale, w[e], b[e]);
        store_normed<T>(a, place, row, u, h.v[u]);
      }
    }
  }
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
  if (values && too_many_units(rows, cols)) return fail(TF24_ERR_SHAPE, "%s: matrix too large to be kept (%lld x %lld)", fn, (long long)rows, (long long)cols);
  if (ld_x < 0 || ld_y < 0 || ld_gate < 0) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  if (int rc = check_aligned(fn, dtype_size(stream_dtype), {x, out})) return rc;
  if (int rc = check_aligned(fn, dtype_size(block_dtype), {y, n})) return rc;
  if (int rc = check_aligned(fn, dtype_size(param_dtype), {post_weight, post_bias, pre_weight, pre_bias})) return rc;
  if (int rc = check_aligned(fn, gate ? dtype_size(gate_dtype) : 1, {gate})) return rc;
  if (int rc = check_aligned(fn, 16, {values, stats})) return rc;
  return with_types(stream_dtype, block_dtype, [&](auto r, auto t) {
    using R = decltype(r);
    using T = decltype(t);
    const auto launch = [&](auto* kernel, int threads, int rows_at_once) {
      const uint32_t most = kForwardWaves / (uint32_t)(threads / 64), each = (uint32_t)((rows + most - 1) / most);
      const uint32_t per_block = (each + rows_at_once - 1) / rows_at_once * rows_at_once;
      const ForwardArgs a{x, y, gate, post_weight, post_bias, pre_weight, pre_bias, out, n, stats, (uint8_t*)values, (uint8_t*)scales, ld_x, ld_y, ld_gate, (uint32_t)rows,
                          per_block, (uint32_t)(gate ? rows_per_gate : 1), (int)cols, (int)kept_blocks(cols), param_dtype, gate_dtype, post_kind, pre_kind, scale, eps,
                          1.0f / (float)cols};
      hipLaunchKernelGGL(kernel, dim3(((uint32_t)rows + per_block - 1) / per_block), dim3(threads), 0, (hipStream_t)stream, a);
      return check_launch("tf24_block_norm_forward");
    };
    if (cols > kNarrowCols)
      return launch(cols % 8 ? (y ? block_norm_forward_wide<R, T, true, true> : block_norm_forward_wide<R, T, false, true>)
                             : (y ? block_norm_forward_wide<R, T, true, false> : block_norm_forward_wide<R, T, false, false>), kWideThreads, 1);
    return with_shape<kForwardThreads>(cols, [&](auto shape) {
      using S = decltype(shape);
      return launch(cols % 8 ? (y ? block_norm_forward<R, T, true, true, S> : block_norm_forward<R, T, false, true, S>)
                             : (y ? block_norm_forward<R, T, true, false, S> : block_norm_forward<R, T, false, false, S>), S::THREADS, S::ROWS);
    });
  });
}
