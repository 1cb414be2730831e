// A matrix to 8 bits and back (checkpoint8.hpp has the format): one pass over memory either way.
//
// A lane owns eight adjacent columns, the four lanes of a block find its largest magnitude through data parallel primitives, and what is
// kept is written as it is numbered: unit u at byte 8 u, block b's scale at byte b.  Bound by memory: 16384 x 8192 bf16, 407 MB either way, is encoded in
// 71 to 78 us (5.2 to 5.7 TB/s) and decoded in 61 to 65 (6.2 to 6.6); one unit a lane and as many workgroups as that takes, so that their
// number hides the latency of the one load that a lane waits for.
#include "checkpoint8.hpp"

namespace tf24 {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads)
checkpoint_encode(const T* __restrict__ x, int64_t ld, int cols, UnitRows by, uint32_t total, uint8_t* __restrict__ values, uint8_t* __restrict__ scales) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= total) return;                                        // (a multiple of 4: whole blocks)
  const uint32_t row = row_of_unit(by, u), col = (u - row * by.units) * kKeptUnit;
  float v[8];
  load_up_to_8(x + (int64_t)row * ld + col, min(max(cols - (int)col, 0), 8), v);
  const Kept8 k = keep_8<T>(v);
  *reinterpret_cast<uint2*>(values + (uint64_t)u * 8) = k.values;
  if ((u & 3) == 0) scales[u >> 2] = (uint8_t)k.scale;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
checkpoint_decode(const uint8_t* __restrict__ values, const uint8_t* __restrict__ scales, int cols, UnitRows by, uint32_t total, T* __restrict__ out, int64_t ld) {
  const uint32_t u = blockIdx.x * kThreads + threadIdx.x;
  if (u >= total) return;
  const uint32_t row = row_of_unit(by, u), col = (u - row * by.units) * kKeptUnit;
  const int n = min(cols - (int)col, 8);
  if (n <= 0) return;
  float v[8];
  kept_to_float(*reinterpret_cast<const uint2*>(values + (uint64_t)u * 8), scales[u >> 2], v);
  store_up_to_8(out + (int64_t)row * ld + col, n, v);
}

int check_matrix(const char* fn, int dtype, int64_t ld, int64_t rows, int64_t cols) {
  if (dtype != TF24_F32 && dtype != TF24_F16 && dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (rows < 0 || cols < 1 || cols > (int64_t)1 << 30) return fail(TF24_ERR_SHAPE, "%s: shape (%lld, %lld) is not supported", fn, (long long)rows, (long long)cols);
  if (too_many_units(rows, cols)) return fail(TF24_ERR_SHAPE, "%s: matrix too large (%lld x %lld)", fn, (long long)rows, (long long)cols);
  if (ld < 0) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  return TF24_OK;
}

}  // namespace
}  // namespace tf24

extern "C" int64_t tf24_checkpoint_blocks(int64_t cols) { return cols < 0 ? 0 : tf24::kept_blocks(cols); }

extern "C" int tf24_checkpoint_encode(const void* x, int dtype, int64_t ld, int64_t rows, int64_t cols, void* values, void* scales, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_checkpoint_encode";
  if (int rc = check_matrix(fn, dtype, ld, rows, cols)) return rc;
  if (!rows) return TF24_OK;
  if (!x || !values || !scales) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, dtype_size(dtype), {x})) return rc;
  if (int rc = check_aligned(fn, 16, {values})) return rc;
  const UnitRows by = unit_rows(cols);
  const uint32_t total = (uint32_t)rows * by.units;
  const dim3 grid((total + kThreads - 1) / kThreads), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TF24_F32) hipLaunchKernelGGL(checkpoint_encode<float>, grid, block, 0, s, (const float*)x, ld, (int)cols, by, total, (uint8_t*)values, (uint8_t*)scales);
  else if (dtype == TF24_F16) hipLaunchKernelGGL(checkpoint_encode<f16_t>, grid, block, 0, s, (const f16_t*)x, ld, (int)cols, by, total, (uint8_t*)values, (uint8_t*)scales);
  else hipLaunchKernelGGL(checkpoint_encode<bf16_t>, grid, block, 0, s, (const bf16_t*)x, ld, (int)cols, by, total, (uint8_t*)values, (uint8_t*)scales);
  return check_launch(fn);
}

extern "C" int tf24_checkpoint_decode(const void* values, const void* scales, int64_t rows, int64_t cols, void* out, int dtype, int64_t ld, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_checkpoint_decode";
  if (int rc = check_matrix(fn, dtype, ld, rows, cols)) return rc;
  if (rows > 1 && ld < cols) return fail(TF24_ERR_STRIDE, "%s: leading dimension %lld < %lld", fn, (long long)ld, (long long)cols);
  if (!rows) return TF24_OK;
  if (!out || !values || !scales) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, dtype_size(dtype), {out})) return rc;
  if (int rc = check_aligned(fn, 16, {values})) return rc;
  const UnitRows by = unit_rows(cols);
  const uint32_t total = (uint32_t)rows * by.units;
  const dim3 grid((total + kThreads - 1) / kThreads), block(kThreads);
  hipStream_t s = (hipStream_t)stream;
  const uint8_t *v = (const uint8_t*)values, *c = (const uint8_t*)scales;
  if (dtype == TF24_F32) hipLaunchKernelGGL(checkpoint_decode<float>, grid, block, 0, s, v, c, (int)cols, by, total, (float*)out, ld);
  else if (dtype == TF24_F16) hipLaunchKernelGGL(checkpoint_decode<f16_t>, grid, block, 0, s, v, c, (int)cols, by, total, (f16_t*)out, ld);
  else hipLaunchKernelGGL(checkpoint_decode<bf16_t>, grid, block, 0, s, v, c, (int)cols, by, total, (bf16_t*)out, ld);
  return check_launch(fn);
}
