// Launches of the vocabulary head's products (head_tiles.hpp).
#include "linear_loss.hpp"
#include "head_tiles.hpp"
#include <algorithm>

namespace tf24 {
namespace {

template <typename T, typename OutT, int KIND, bool SMOOTH>
void launch(const HeadProduct& p, const HeadResult& r, hipStream_t s) {
  const int64_t per_xcd = ((int64_t)p.tiles_i * p.tiles_j + 7) / 8, slots = std::max(1, compute_units() / 8);
  const unsigned groups = KIND <= HEAD_SLOPE ? (unsigned)(std::min(per_xcd, slots) * 8) : (unsigned)p.groups;
  hipLaunchKernelGGL((head_product<T, OutT, KIND, SMOOTH>), dim3(groups), dim3(kThreads), 0, s, p, r);
}

template <typename T>
void launch_kind(int kind, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, hipStream_t s) {
  if (kind == HEAD_STATS) smooth ? launch<T, T, HEAD_STATS, true>(p, r, s) : launch<T, T, HEAD_STATS, false>(p, r, s);
  else if (kind == HEAD_SLOPE) smooth ? launch<T, T, HEAD_SLOPE, true>(p, r, s) : launch<T, T, HEAD_SLOPE, false>(p, r, s);
  else if (kind == HEAD_INPUT) smooth ? launch<T, T, HEAD_INPUT, true>(p, r, s) : launch<T, T, HEAD_INPUT, false>(p, r, s);
  else if (wide) smooth ? launch<T, float, HEAD_WEIGHT, true>(p, r, s) : launch<T, float, HEAD_WEIGHT, false>(p, r, s);
  else smooth ? launch<T, T, HEAD_WEIGHT, true>(p, r, s) : launch<T, T, HEAD_WEIGHT, false>(p, r, s);
}

// What the pieces of the rest of a product's tiles add up to: block (tile of the rest, some of the fragments of one row).  Bound by memory: 144 tiles of 5 pieces, 189
// MB, 52 us (4 TB/s with the result); 79 of 3 20.
template <typename T, typename OutT, int KIND>
__global__ void __launch_bounds__(kThreads)
join_pieces(const HeadProduct p, const HeadResult r) {
  const int count = *p.count, tiles_j = KIND == HEAD_WEIGHT ? p.tiles_j : token_tiles(count);
  const Share share = share_out(p.tiles_i * tiles_j, KIND == HEAD_WEIGHT ? token_stages(count) : p.stages, p.groups, p.most);
  if (share.pieces == 1 || (int)blockIdx.x >= share.rest) return;
  const int tile = share.whole + (int)blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ti = blockIdx.y % F, each = F / (gridDim.y / F), tj0 = blockIdx.y / F * each;
  const int group = tile / (kRaster * tiles_j), in_group = tile - group * (kRaster * tiles_j), gh = min(kRaster, p.tiles_i - group * kRaster);
  const int64_t i = (int64_t)(group * kRaster + in_group % gh) * kTile + (wave >> 1) * kSlab + ti * 16 + (lane >> 4) * 4;
  const int64_t j0 = (int64_t)(in_group / gh) * kTile + (wave & 1) * kSlab + (lane & 15), rows = KIND == HEAD_INPUT ? (int64_t)count : r.rows_j;
  const float scale = *r.out_scale;
  const bool aligned = r.cols_out % 4 == 0 && (uintptr_t)r.out % (4 * sizeof(OutT)) == 0;
#pragma unroll 2
  for (int tj = tj0; tj < tj0 + each; tj++) {
    const int64_t at = (int64_t)(ti * F + tj) * (kThreads * 4) + tid * 4, j = j0 + tj * 16;
    float4v v = {0, 0, 0, 0};
    if (r.add) v = *reinterpret_cast<const float4v*>(r.sum + (int64_t)tile * (kTile * kTile) + at);
    for (int s0 = 0; s0 < share.pieces; s0 += 4) {               // four independent loads in flight
      float4v part[4];
#pragma unroll
      for (int u = 0; u < 4; u++)
        part[u] = *reinterpret_cast<const float4v*>(r.partial + ((int64_t)min(s0 + u, share.pieces - 1) * share.rest + blockIdx.x) * (kTile * kTile) + at);
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (s0 + u < share.pieces) v += part[u];
    }
    if (!r.last) {
      *reinterpret_cast<float4v*>(r.sum + (int64_t)tile * (kTile * kTile) + at) = v;
      continue;
    }
    if (j >= rows) continue;
    if (r.common) {                                              // (filled up to whole tiles)
      const float times = KIND == HEAD_INPUT ? r.level_rest[j] : 1.0f;
      const float4v common = *reinterpret_cast<const float4v*>(r.common + i);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = __builtin_fmaf(-times, common[e], v[e]);
    }
    OutT* out = (OutT*)r.out + (KIND == HEAD_INPUT ? (int64_t)r.row_of[j] : j) * r.cols_out + i;
    OutT o[4];
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = from_float<OutT>(scaled(v[e], scale));
    if (aligned) {
      if (i < r.cols_out) *reinterpret_cast<Pack<OutT, 4>*>(out) = *reinterpret_cast<Pack<OutT, 4>*>(o);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (i + e < r.cols_out) out[e] = o[e];
    }
  }
}

template <typename T>
void join_kind(int kind, bool wide, const HeadProduct& p, const HeadResult& r, int rest, hipStream_t s) {
  // workgroups for every compute unit (12 tiles of 21 pieces, 1024 tokens, 50304 x 768: 17 us, with 8 to a tile 22 more), and few that find nothing to do (as many as
  // 255 tiles: 5 us, with 32 to a tile 26)
  const dim3 grid((unsigned)rest, rest < 64 ? 4 * F : F);
  if (kind == HEAD_INPUT) hipLaunchKernelGGL((join_pieces<T, T, HEAD_INPUT>), grid, dim3(kThreads), 0, s, p, r);
  else if (wide) hipLaunchKernelGGL((join_pieces<T, float, HEAD_WEIGHT>), grid, dim3(kThreads), 0, s, p, r);
  else hipLaunchKernelGGL((join_pieces<T, T, HEAD_WEIGHT>), grid, dim3(kThreads), 0, s, p, r);
}

}  // namespace

int launch_head_product(int kind, int dtype, bool smooth, bool wide, const HeadProduct& p, const HeadResult& r, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  (dtype == TF24_F16 ? launch_kind<f16_t> : launch_kind<bf16_t>)(kind, smooth, wide, p, r, s);
  // (of a gradient of x fewer tiles may count than there are at most, and the rest be another number of them: whatever number there may be)
  if (kind >= HEAD_INPUT && p.most > 0)
    (dtype == TF24_F16 ? join_kind<f16_t> : join_kind<bf16_t>)(kind, wide, p, r, kind == HEAD_INPUT ? std::min(p.groups - 1, p.tiles_i * p.tiles_j) : p.tiles_i * p.tiles_j % p.groups, s);
  return check_launch("tf24_linear_loss");
}

}  // namespace tf24
