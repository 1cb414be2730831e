// Launches of the vocabulary head's products (head_tiles.hpp).
#include "linear_loss.hpp"
#include "head_tiles.hpp"
#include <algorithm>

namespace tf24 {
namespace {

template <typename T, typename OutT, int KIND, bool SMOOTH>
void launch(const HeadProduct& p, const HeadResult& r, hipStream_t s) {
  const int64_t units = (int64_t)p.tiles_i * p.tiles_j * p.splits;
  const int64_t per_xcd = (units + 7) / 8, slots = std::max(1, compute_units() / 8);
  hipLaunchKernelGGL((head_product<T, OutT, KIND, SMOOTH>), dim3((unsigned)(std::min(per_xcd, slots) * 8)), dim3(kThreads), 0, s, p, r);
}

template <typename T>
void launch_kind(int kind, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, hipStream_t s) {
  if (kind == HEAD_STATS) smooth ? launch<T, T, HEAD_STATS, true>(p, r, s) : launch<T, T, HEAD_STATS, false>(p, r, s);
  else if (kind == HEAD_SLOPE) smooth ? launch<T, T, HEAD_SLOPE, true>(p, r, s) : launch<T, T, HEAD_SLOPE, false>(p, r, s);
  else if (kind == HEAD_INPUT) launch<T, T, HEAD_INPUT, false>(p, r, s);
  else wide ? launch<T, float, HEAD_WEIGHT, false>(p, r, s) : launch<T, T, HEAD_WEIGHT, false>(p, r, s);
}

}  // namespace

int launch_head_product(int kind, int dtype, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, void* stream) {
  (dtype == TF24_F16 ? launch_kind<f16_t> : launch_kind<bf16_t>)(kind, smooth, wide, p, r, (hipStream_t)stream);
  return check_launch("tf24_linear_loss");
}

}  // namespace tf24
