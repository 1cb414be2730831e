// GELU-GLU for gfx950: out = gelu_tanh(gate) * x with [x | gate] the two halves of the input's
// last dimension, and its backward pass; float32 arithmetic, one rounding to the storage type.
//
// Both memory orders of the reference's two code paths are one indexing scheme: element (i, j) of
// the x half at i*ld + j and its gate at the same place + gate_off.  Row-major input [rows, cols]:
// i = row, j = column < cols/2, gate_off = cols/2.  Column-major input (the reference's "fall back
// to 2D" path, memory [cols][ld]): i = column < cols/2, j = row, gate_off = (cols/2)*ld.
// A lane owns 8 consecutive j (16-byte accesses for 16-bit types) when the extents allow it.
//
// The second pair of kernels keeps the input in 8 bits only (checkpoint8.hpp: as a matrix of 2 * rows rows, x and gate of a row one after the
// other): the forward pass encodes what it reads, and on request what it writes, the backward pass decodes it.  Bound by memory: 12288 x 2 * 4096 float16,
// 405 MB in each pass, 68 us forward and 70 backward = 5.8 TB/s; forward where nothing is kept 302 MB in 49 us = 6.1 TB/s.
#include "checkpoint8.hpp"

namespace tf24 {
namespace {

constexpr int kThreads = 256;
constexpr float kBeta = 0.7978845608028654f;     // sqrt(2/pi)
constexpr float kKappa = 0.044715f;
constexpr float kExpLinear = (float)(-2.0 * 0.7978845608028654 * 1.4426950408889634);               // -2u as a power of two
constexpr float kExpCubic = (float)(-2.0 * 0.7978845608028654 * 1.4426950408889634 * 0.044715);

// 0.5 * (1 + tanh(u)) is the logistic function of 2u: one exponential and one reciprocal per
// element.  exp of a large argument gives +inf and the reciprocal 0, so no range split is needed.
// The vector ALUs are busy for more than half of the memory time, so instructions count: with the
// polynomials as multiply-adds (the factors of the exponent folded into their constants) an element
// takes 8 and 14 of them instead of 11 and 22, and with loads that may stay in the caches 12288 x 8192
// fp16 takes 45.5 + 77 instead of 48.4 + 81.7 us (forward + backward; streaming stores: 10 us less
// than plain ones).  Error against float64 as before: that of the rounding to 16 bits.
struct GluTerms {
  float gelu;      // gelu_tanh(gate) = gate * sig
  float dgelu;     // d gelu_tanh / d gate = sig + gate * sig * (1 - sig) * 2 * du/dgate
};
template <bool GRAD>
__device__ __forceinline__ GluTerms glu_terms(float gate) {
  const float g2 = gate * gate;
  const float sig = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gate * __builtin_fmaf(g2, kExpCubic, kExpLinear)));
  GluTerms r;
  r.gelu = gate * sig;
  r.dgelu = 0.0f;
  if constexpr (GRAD) r.dgelu = __builtin_fmaf(r.gelu * (1.0f - sig), __builtin_fmaf(g2, 6.0f * kBeta * kKappa, 2.0f * kBeta), sig);
  return r;
}

// V = elements per lane (8 or 1); blocks are numbered along j first
template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
gelu_glu_fwd(const T* __restrict__ in, int64_t ld_in, int64_t gate_off, int64_t ni, int64_t nj,
             T* __restrict__ out, int64_t ld_out) {
  const uint32_t chunks = (uint32_t)((nj / V + kThreads - 1) / kThreads);
  const int64_t i = blockIdx.x / chunks;
  const int64_t j = ((int64_t)(blockIdx.x - (uint32_t)i * chunks) * kThreads + threadIdx.x) * V;
  if (j >= nj) return;
  Pack<T, V> x, g, o;
  x.load(in + i * ld_in + j);
  g.load(in + i * ld_in + j + gate_off);
#pragma unroll
  for (int e = 0; e < V; e++) o.v[e] = from_float<T>(glu_terms<false>(to_float(g.v[e])).gelu * to_float(x.v[e]));
  o.store_stream(out + i * ld_out + j);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads)
gelu_glu_bwd(const T* __restrict__ grad_out, int64_t ld_go, const T* __restrict__ in, int64_t ld_in, int64_t gate_off,
             int64_t ni, int64_t nj, T* __restrict__ grad_in, int64_t ld_gi, int64_t gate_off_gi) {
  const uint32_t chunks = (uint32_t)((nj / V + kThreads - 1) / kThreads);
  const int64_t i = blockIdx.x / chunks;
  const int64_t j = ((int64_t)(blockIdx.x - (uint32_t)i * chunks) * kThreads + threadIdx.x) * V;
  if (j >= nj) return;
  Pack<T, V> go, x, g, gx, gg;
  go.load(grad_out + i * ld_go + j);
  x.load(in + i * ld_in + j);
  g.load(in + i * ld_in + j + gate_off);
#pragma unroll
  for (int e = 0; e < V; e++) {
    const GluTerms t = glu_terms<true>(to_float(g.v[e]));
    const float dy = to_float(go.v[e]);
    gx.v[e] = from_float<T>(dy * t.gelu);
    gg.v[e] = from_float<T>(dy * to_float(x.v[e]) * t.dgelu);
  }
  gx.store_stream(grad_in + i * ld_gi + j);
  gg.store_stream(grad_in + i * ld_gi + j + gate_off_gi);
}

// Row-major input, `half` columns of x and as many of gate in each row; a lane owns a unit of the output's columns.  What is kept of the
// input (KEEP: nothing where no backward pass will read it) has units and blocks of 2 * rows rows, that of the output of `rows` rows (numbered as
// the lanes are).
template <typename T, bool KEEP, bool KEEP_OUT>
__global__ void __launch_bounds__(kThreads)
gelu_glu_fwd_keep(const T* __restrict__ in, int64_t ld_in, int half, UnitRows by, uint32_t total, T* __restrict__ out, int64_t ld_out, uint8_t* __restrict__ values,
                  uint8_t* __restrict__ scales, uint8_t* __restrict__ out_values, uint8_t* __restrict__ out_scales) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= total) return;                                        // (a multiple of 4: whole blocks)
  const uint32_t row = row_of_unit(by, u), first = row * by.units, col = (u - first) * kKeptUnit;
  const int n = min(max(half - (int)col, 0), 8);
  float x[8], g[8], o[8];
  load_up_to_8(in + (int64_t)row * ld_in + col, n, x);
  load_up_to_8(in + (int64_t)row * ld_in + half + col, n, g);
#pragma unroll
  for (int e = 0; e < 8; e++) o[e] = glu_terms<false>(g[e]).gelu * x[e];
  store_up_to_8(out + (int64_t)row * ld_out + col, n, o);
  if constexpr (KEEP) {
    const Kept8 kx = keep_8<T>(x), kg = keep_8<T>(g);
    const uint64_t ux = (uint64_t)u + first, ug = ux + by.units;  // rows 2 row and 2 row + 1
    *reinterpret_cast<uint2*>(values + ux * 8) = kx.values;
    *reinterpret_cast<uint2*>(values + ug * 8) = kg.values;
    if ((u & 3) == 0) {
      scales[ux >> 2] = (uint8_t)kx.scale;
      scales[ug >> 2] = (uint8_t)kg.scale;
    }
  }
  if constexpr (KEEP_OUT) {
    const Kept8 ko = keep_8<T>(o);
    *reinterpret_cast<uint2*>(out_values + (uint64_t)u * 8) = ko.values;
    if ((u & 3) == 0) out_scales[u >> 2] = (uint8_t)ko.scale;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
gelu_glu_bwd_kept(const T* __restrict__ grad_out, int64_t ld_go, const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales, int half, UnitRows by,
                  uint32_t total, T* __restrict__ grad_in, int64_t ld_gi) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= total) return;
  const uint32_t row = row_of_unit(by, u), first = row * by.units, col = (u - first) * kKeptUnit;
  const int n = min(half - (int)col, 8);
  if (n <= 0) return;
  const uint64_t ux = (uint64_t)u + first, ug = ux + by.units;
  float go[8], x[8], g[8], gx[8], gg[8];
  load_up_to_8(grad_out + (int64_t)row * ld_go + col, n, go);
  kept_to_float(*reinterpret_cast<const uint2*>(values + ux * 8), scales[ux >> 2], x);
  kept_to_float(*reinterpret_cast<const uint2*>(values + ug * 8), scales[ug >> 2], g);
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const GluTerms t = glu_terms<true>(g[e]);
    gx[e] = go[e] * t.gelu;
    gg[e] = go[e] * x[e] * t.dgelu;
  }
  store_up_to_8(grad_in + (int64_t)row * ld_gi + col, n, gx);
  store_up_to_8(grad_in + (int64_t)row * ld_gi + half + col, n, gg);
}

struct View {
  int64_t ni, nj, gate_off;
};
// layout of the [rows, cols] input -> the (i, j) scheme above
View view_of(int layout, int64_t rows, int64_t cols, int64_t ld) {
  if (layout == TF24_ROW_MAJOR) return {rows, cols / 2, cols / 2};
  return {cols / 2, rows, (cols / 2) * ld};
}
bool vectorizable(int64_t nj, std::initializer_list<int64_t> offsets, std::initializer_list<const void*> ptrs) {
  if (nj % 8) return false;
  for (int64_t o : offsets) if (o % 8) return false;
  for (const void* p : ptrs) if ((uintptr_t)p % 16) return false;
  return true;
}

template <typename T>
int forward(const void* in, int layout, int64_t ld_in, int64_t rows, int64_t cols, void* out, int64_t ld_out, hipStream_t s) {
  const View v = view_of(layout, rows, cols, ld_in);
  if (vectorizable(v.nj, {ld_in, ld_out, v.gate_off}, {in, out})) {
    dim3 grid((unsigned)(v.ni * ((v.nj / 8 + kThreads - 1) / kThreads)));
    hipLaunchKernelGGL((gelu_glu_fwd<T, 8>), grid, dim3(kThreads), 0, s, (const T*)in, ld_in, v.gate_off, v.ni, v.nj, (T*)out, ld_out);
  } else {
    dim3 grid((unsigned)(v.ni * ((v.nj + kThreads - 1) / kThreads)));
    hipLaunchKernelGGL((gelu_glu_fwd<T, 1>), grid, dim3(kThreads), 0, s, (const T*)in, ld_in, v.gate_off, v.ni, v.nj, (T*)out, ld_out);
  }
  return check_launch("tf24_gelu_glu_forward");
}

template <typename T>
int backward(const void* go, int64_t ld_go, const void* in, int layout, int64_t ld_in, int64_t rows, int64_t cols,
             void* gi, int64_t ld_gi, hipStream_t s) {
  const View v = view_of(layout, rows, cols, ld_in);
  const int64_t gate_off_gi = view_of(layout, rows, cols, ld_gi).gate_off;
  if (vectorizable(v.nj, {ld_go, ld_in, ld_gi, v.gate_off, gate_off_gi}, {go, in, gi})) {
    dim3 grid((unsigned)(v.ni * ((v.nj / 8 + kThreads - 1) / kThreads)));
    hipLaunchKernelGGL((gelu_glu_bwd<T, 8>), grid, dim3(kThreads), 0, s, (const T*)go, ld_go, (const T*)in, ld_in, v.gate_off, v.ni, v.nj,
                       (T*)gi, ld_gi, gate_off_gi);
  } else {
    dim3 grid((unsigned)(v.ni * ((v.nj + kThreads - 1) / kThreads)));
    hipLaunchKernelGGL((gelu_glu_bwd<T, 1>), grid, dim3(kThreads), 0, s, (const T*)go, ld_go, (const T*)in, ld_in, v.gate_off, v.ni, v.nj,
                       (T*)gi, ld_gi, gate_off_gi);
  }
  return check_launch("tf24_gelu_glu_backward");
}

int check_args(const char* fn, int dtype, int layout, int64_t rows, int64_t cols, std::initializer_list<int64_t> lds_full,
               std::initializer_list<int64_t> lds_half) {
  if (dtype != TF24_F32 && dtype != TF24_F16 && dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (layout != TF24_ROW_MAJOR && layout != TF24_COL_MAJOR) return fail(TF24_ERR_ARG, "%s: bad layout %d", fn, layout);
  if (rows < 1 || cols < 2 || cols % 2) return fail(TF24_ERR_SHAPE, "%s: shape (%lld, %lld) is not supported: the last dimension must be even", fn, (long long)rows, (long long)cols);
  const int64_t ni = layout == TF24_ROW_MAJOR ? rows : cols / 2, nj = layout == TF24_ROW_MAJOR ? cols / 2 : rows;
  if (ni * ((nj + kThreads - 1) / kThreads) > 0x7fffffffLL) return fail(TF24_ERR_SHAPE, "%s: tensor too large", fn);
  // leading dimensions: the contiguous extent is cols (row-major) or rows (column-major) for the
  // full-width tensors, cols/2 or rows for the half-width ones
  for (int64_t ld : lds_full)
    if (ld < (layout == TF24_ROW_MAJOR ? cols : rows)) return fail(TF24_ERR_STRIDE, "%s: leading dimension %lld too small", fn, (long long)ld);
  for (int64_t ld : lds_half)
    if (ld < (layout == TF24_ROW_MAJOR ? cols / 2 : rows)) return fail(TF24_ERR_STRIDE, "%s: leading dimension %lld too small", fn, (long long)ld);
  return TF24_OK;
}

}  // namespace
}  // namespace tf24

extern "C" int tf24_gelu_glu_forward(const void* in, int dtype, int layout, int64_t ld_in, int64_t rows, int64_t cols,
                                     void* out, int64_t ld_out, void* stream) {
  using namespace tf24;
  int rc = check_args("tf24_gelu_glu_forward", dtype, layout, rows, cols, {ld_in}, {ld_out});
  if (rc != TF24_OK) return rc;
  if (!in || !out) return fail(TF24_ERR_ARG, "tf24_gelu_glu_forward: null pointer");
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TF24_F32: return forward<float>(in, layout, ld_in, rows, cols, out, ld_out, s);
    case TF24_F16: return forward<f16_t>(in, layout, ld_in, rows, cols, out, ld_out, s);
    default: return forward<bf16_t>(in, layout, ld_in, rows, cols, out, ld_out, s);
  }
}

extern "C" int tf24_gelu_glu_backward(const void* grad_out, int64_t ld_grad_out, const void* in, int dtype, int layout,
                                      int64_t ld_in, int64_t rows, int64_t cols, void* grad_in, int64_t ld_grad_in,
                                      void* stream) {
  using namespace tf24;
  int rc = check_args("tf24_gelu_glu_backward", dtype, layout, rows, cols, {ld_in, ld_grad_in}, {ld_grad_out});
  if (rc != TF24_OK) return rc;
  if (!grad_out || !in || !grad_in) return fail(TF24_ERR_ARG, "tf24_gelu_glu_backward: null pointer");
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TF24_F32: return backward<float>(grad_out, ld_grad_out, in, layout, ld_in, rows, cols, grad_in, ld_grad_in, s);
    case TF24_F16: return backward<f16_t>(grad_out, ld_grad_out, in, layout, ld_in, rows, cols, grad_in, ld_grad_in, s);
    default: return backward<bf16_t>(grad_out, ld_grad_out, in, layout, ld_in, rows, cols, grad_in, ld_grad_in, s);
  }
}

namespace tf24 {
namespace {

int check_kept(const char* fn, int dtype, int64_t rows, int64_t cols, int64_t ld_full, int64_t ld_half) {
  if (dtype != TF24_F32 && dtype != TF24_F16 && dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (rows < 0 || cols < 2 || cols % 2 || cols > (int64_t)1 << 30)
    return fail(TF24_ERR_SHAPE, "%s: shape (%lld, %lld) is not supported: the last dimension must be even", fn, (long long)rows, (long long)cols);
  if (too_many_units(rows, cols / 2)) return fail(TF24_ERR_SHAPE, "%s: tensor too large", fn);
  if (rows > 1 && (ld_full < cols || ld_half < cols / 2))
    return fail(TF24_ERR_STRIDE, "%s: leading dimensions %lld, %lld too small", fn, (long long)ld_full, (long long)ld_half);
  return TF24_OK;
}

template <typename T>
int forward_keep(const void* in, int64_t ld_in, int64_t rows, int64_t cols, void* out, int64_t ld_out, void* values, void* scales, void* out_values, void* out_scales,
                 hipStream_t s) {
  const UnitRows by = unit_rows(cols / 2);
  const uint32_t total = (uint32_t)rows * by.units;
  auto* kernel = values ? (out_values ? gelu_glu_fwd_keep<T, true, true> : gelu_glu_fwd_keep<T, true, false>)
                        : (out_values ? gelu_glu_fwd_keep<T, false, true> : gelu_glu_fwd_keep<T, false, false>);
  hipLaunchKernelGGL(kernel, dim3((total + kThreads - 1) / kThreads), dim3(kThreads), 0, s, (const T*)in, ld_in, (int)(cols / 2), by, total, (T*)out, ld_out,
                     (uint8_t*)values, (uint8_t*)scales, (uint8_t*)out_values, (uint8_t*)out_scales);
  return check_launch("tf24_gelu_glu_forward_checkpoint");
}

template <typename T>
int backward_kept(const void* go, int64_t ld_go, const void* values, const void* scales, int64_t rows, int64_t cols, void* gi, int64_t ld_gi, hipStream_t s) {
  const UnitRows by = unit_rows(cols / 2);
  const uint32_t total = (uint32_t)rows * by.units;
  hipLaunchKernelGGL(gelu_glu_bwd_kept<T>, dim3((total + kThreads - 1) / kThreads), dim3(kThreads), 0, s, (const T*)go, ld_go, (const uint8_t*)values,
                     (const uint8_t*)scales, (int)(cols / 2), by, total, (T*)gi, ld_gi);
  return check_launch("tf24_gelu_glu_backward_checkpoint");
}

}  // namespace
}  // namespace tf24

extern "C" int tf24_gelu_glu_forward_checkpoint(const void* in, int dtype, int64_t ld_in, int64_t rows, int64_t cols, void* out, int64_t ld_out, void* values,
                                                void* scales, void* out_values, void* out_scales, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_gelu_glu_forward_checkpoint";
  if (int rc = check_kept(fn, dtype, rows, cols, ld_in, ld_out)) return rc;
  if (!rows) return TF24_OK;
  if (!in || !out || !values != !scales || !out_values != !out_scales) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, dtype_size(dtype), {in, out})) return rc;
  if (int rc = check_aligned(fn, 16, {values, out_values})) return rc;
  auto* go = dtype == TF24_F32 ? forward_keep<float> : dtype == TF24_F16 ? forward_keep<f16_t> : forward_keep<bf16_t>;
  return go(in, ld_in, rows, cols, out, ld_out, values, scales, out_values, out_scales, (hipStream_t)stream);
}

extern "C" int tf24_gelu_glu_backward_checkpoint(const void* grad_out, int64_t ld_grad_out, const void* values, const void* scales, int dtype, int64_t rows,
                                                 int64_t cols, void* grad_in, int64_t ld_grad_in, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_gelu_glu_backward_checkpoint";
  if (int rc = check_kept(fn, dtype, rows, cols, ld_grad_in, ld_grad_out)) return rc;
  if (!rows) return TF24_OK;
  if (!grad_out || !values || !scales || !grad_in) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, dtype_size(dtype), {grad_out, grad_in})) return rc;
  if (int rc = check_aligned(fn, 16, {values})) return rc;
  auto* go = dtype == TF24_F32 ? backward_kept<float> : dtype == TF24_F16 ? backward_kept<f16_t> : backward_kept<bf16_t>;
  return go(grad_out, ld_grad_out, values, scales, rows, cols, grad_in, ld_grad_in, (hipStream_t)stream);
}
