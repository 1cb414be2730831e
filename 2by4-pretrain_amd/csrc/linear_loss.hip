// The loss of a vocabulary head, logits z = x W^T + b of `words` words, without keeping them:
//
//   cross entropy   lse - (1 - s) z[target] - s mean(z) + c lse^2             u = z, lse = log sum exp u
//   distillation    sum_k q_k (log q_k - u[i_k] + lse)                        u = z / temperature, q the teacher's probabilities of its listed words
//
// Forward: one product whose tiles leave a maximum and a sum of exponentials per token and 128 words behind, and the logits of the listed
// words; a small kernel joins them.  Backward: the product once more, P = dloss/dz in 16 bits for a piece of the vocabulary at a time (at most
// 2 GiB of it), the listed words put right in it, then  dx += P W  and  dW = P^T x.  The product that is formed again is a quarter of the
// arithmetic of a training step; kept, the logits would be the largest tensor of it.
//
// Tokens that do not count (their target is to be ignored, or no word of the teacher's is listed) are left out from the start: the others are
// brought together, and the products run over those alone, whose number stays on the device.  Nothing of a token that does not count is read.
//
// P is rounded to the operands' type as the operand of a matrix instruction: relative to each of its elements, which is what a
// 16-bit gradient of the logits is rounded to as well.  It is formed in units of the largest gradient of a token's loss (float16: of 2^-14 of it), which come
// back behind the products, so that the small probabilities of a large batch do not vanish in float16.
// All sums are float32 (the loss over tokens: float64), in an order that the sizes, the number of tokens that count and that of compute units decide.
//
// Bound by the matrix units and, in long products, by the power that they may draw (zeros for operands: 22.4 ms instead of 26.5).  Both passes in bf16, floor at the
// 1.52 PFLOP/s of a large library product (three products) and measured (cards differ by 4 %; two figures that are compared are of one card): 12288 tokens, 50304 x 768 1.87
// and 3.46 to 3.67 ms; 8192 tokens, 128000 x 4096 16.9 and 25.8 to 27.0 ms, four products at 1.27 to 1.33 PFLOP/s.  Everything but the four products: 0.14 and 0.15 ms.  The kernels' own figures stand beside them (us; head_tiles.hpp has
// the products').
#include "linear_loss.hpp"
#include "head_tiles.hpp"
#include <algorithm>
#include <cmath>

namespace tf24 {
namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kMaxEntries = 1024;
constexpr int64_t kMostBlocks = 1 << 16;                         // of entries, one to a thread: 2^22 x 1024 threads are more than one launch has
constexpr int64_t kSlopeBytes = (int64_t)2 << 30;                // (8192 tokens, 128000 x 4096, both passes: 26.53 ms, with 512 MB 26.63)
constexpr int kMostPieces = 1024;                                // tiles' pieces of a product: 256 MB

// ---------------------------------------------------------------- which tokens count
// A token's place among those that count, and back; the target of each, -2 one that no word has.  One workgroup, so that places follow the tokens' order without a
// second launch: 3 for 1024 tokens, 11 for 12288 (bound by the two passes' loads that wait for each other).
__global__ void __launch_bounds__(1024)
count_tokens(const int64_t* __restrict__ targets, int64_t ignore, const int* __restrict__ flags, int tokens, int filled, int64_t words, int* __restrict__ count,
             int* __restrict__ row_of, int* __restrict__ place_of, int* __restrict__ target, float* __restrict__ loss) {
  __shared__ int sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, each = (tokens + 1023) / 1024 * 64;
  const int begin = min(wave * each, tokens), end = min(begin + each, tokens);
  auto counts = [&](int t) { return t < end && (targets ? targets[t] != ignore : flags[t] != 0); };
  int own = 0;
  for (int t0 = begin; t0 < end; t0 += 256) {                    // four loads in flight
    bool yes[4];
#pragma unroll
    for (int u = 0; u < 4; u++) yes[u] = counts(t0 + u * 64 + lane);
#pragma unroll
    for (int u = 0; u < 4; u++) own += __popcll(__ballot(yes[u]));
  }
  if (lane == 0) sums[wave] = own;
  __syncthreads();
  int at = 0, total = 0;
  for (int w = 0; w < 16; w++) {
    if (w < wave) at += sums[w];
    total += sums[w];
  }
  for (int t0 = begin; t0 < end; t0 += 256) {
    bool yes[4];
    int64_t wanted[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int t = t0 + u * 64 + lane;
      wanted[u] = targets && t < end ? targets[t] : -1;
      yes[u] = counts(t);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int t = t0 + u * 64 + lane;
      const uint64_t mask = __ballot(yes[u]);
      const int place = at + __popcll(mask & ((1ull << lane) - 1));
      at += __popcll(mask);
      if (t < end) {
        place_of[t] = yes[u] ? place : -1;
        if (yes[u]) {
          row_of[place] = t;
          if (targets) target[place] = wanted[u] >= 0 && wanted[u] < words ? (int)wanted[u] : -2;
        } else if (loss) loss[t] = 0.0f;
      }
    }
  }
  for (int c = total + tid; c < filled; c += 1024) {
    row_of[c] = -1;
    if (targets) target[c] = -1;
  }
  if (tid == 0) *count = total;
}

// ---------------------------------------------------------------- the teacher's entries
// A token counts if one of its entries is used (its word is not negative) and has a logit above -infinity (or NaN).  A wave per token: 5 for 8192 tokens of 64.
template <typename L>
__global__ void __launch_bounds__(256)
flag_tokens(const int64_t* __restrict__ indices, int64_t ld_indices, const L* __restrict__ logits, int64_t ld_logits, int tokens, int entries, int* __restrict__ flags) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= tokens) return;
  bool any = false;
  for (int k = lane; k < entries; k += 64) any = any || (indices[t * ld_indices + k] >= 0 && to_float(logits[t * ld_logits + k]) != -__builtin_inff());
  any = __any(any);
  if (lane == 0) flags[t] = any;
}

// The entries of a token in ascending order of their words (one word listed twice: in the order of the list), the logarithm of the teacher's
// probability of each, their sum, and where in the list the entries of a slab of words begin.  A workgroup of one wave per token, which sorts them in LDS (a bitonic
// network): 25 for 8192 tokens of 64 entries as for 4096 of 128, bound by the network's steps that wait for each other.
template <typename L>
__global__ void __launch_bounds__(64)
list_entries(const int64_t* __restrict__ indices, int64_t ld_indices, const L* __restrict__ logits, int64_t ld_logits, const float* __restrict__ teacher_lse,
             float inv_temperature, int entries, int padded, int64_t words, const int* __restrict__ count, const int* __restrict__ row_of,
             int* __restrict__ entry_words, float* __restrict__ logq, float* __restrict__ mass, uint32_t* __restrict__ slab_entries, int64_t filled, int slab_words) {
  __shared__ uint64_t key[kMaxEntries];
  __shared__ float value[kMaxEntries];
  const int c = blockIdx.x, lane = threadIdx.x;
  if (c >= *count) return;
  const int64_t row = row_of[c];
  float top = -__builtin_inff();
  bool bad = false;
  for (int k = lane; k < padded; k += 64) {
    uint64_t at = ~0ull;
    if (k < entries) {
      const int64_t w = indices[row * ld_indices + k];
      const float v = to_float(logits[row * ld_logits + k]) * inv_temperature;
      value[k] = v;
      if (w >= words) bad = true;
      else if (w >= 0) {
        at = (uint64_t)w << 32 | (uint32_t)k;
        top = fmaxf(top, v);
      }
    }
    key[k] = at;
  }
  __syncthreads();
  for (int size = 2; size <= padded; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      for (int n = lane; n < padded / 2; n += 64) {
        const int i = (n / step) * step * 2 + n % step, j = i + step;
        const uint64_t a = key[i], b = key[j];
        if ((a > b) == ((i & size) == 0)) { key[i] = b; key[j] = a; }
      }
      __syncthreads();
    }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  bad = __any(bad);
  const float from = top == -__builtin_inff() ? 0.0f : top;
  float lse;
  if (teacher_lse) lse = teacher_lse[row];
  else {
    float s = 0.0f;
    for (int k = lane; k < entries; k += 64)
      if (key[k] != ~0ull) s += expf(value[(uint32_t)key[k]] - from);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
    lse = from + logf(s);
  }
  float q = 0.0f;
  for (int k = lane; k < entries; k += 64) {
    const uint64_t at = key[k];
    const int64_t to = (int64_t)c * entries + k;
    const int w = at == ~0ull ? -1 : (int)(at >> 32);
    entry_words[to] = w;
    if (w < 0) continue;
    const float l = value[(uint32_t)at] - lse;
    logq[to] = l;
    q += expf(l);
    const int slab = w / slab_words;
    if (k == 0 || (int)(key[k - 1] >> 32) / slab_words != slab) {     // the first of its slab
      int low = k, high = entries;                               // low: one of them, high: the first behind them
      while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (key[mid] != ~0ull && (int)(key[mid] >> 32) / slab_words == slab) low = mid;
        else high = mid;
      }
      slab_entries[(int64_t)slab * filled + c] = (uint32_t)k | (uint32_t)(high - k) << 11;
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) q += __shfl_xor(q, d);
  if (lane == 0) mass[c] = bad ? __builtin_nanf("") : q;
}

// ---------------------------------------------------------------- operands as the products read them
// Rows of `cols` 16-bit elements, filled up with zeros to `ld_out` (a multiple of 8): row c of the result is row row_of[c] of the source (null: row c).
// Behind the last of *count, up to a whole stage, the first one stands once more (none: zeros).  P is 0 times an exponential there, which is 0 where the logits are numbers or
// -inf: those of a row of zeros are NaN where a weight is -inf, those of a token that counts are not, or all that it gives is NaN.  Bound by memory: 25 for 8192 x 4096
// (5.4 TB/s); the weight of 50257 x 1601, whose rows are not aligned, 52 (6.2 TB/s, some of it from the caches).
__global__ void __launch_bounds__(256)
pack_rows(const uint16_t* __restrict__ in, int64_t ld, int64_t rows, int64_t cols, const int* __restrict__ count, const int* __restrict__ row_of,
          uint16_t* __restrict__ out, int64_t ld_out) {
  const int64_t units = ld_out / 8;
  const int n = count ? *count : 0;
  if (count) rows = (int64_t)token_stages(n) * kUnitK;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < rows * units; u += (int64_t)gridDim.x * 256) {
    const int64_t c = u / units, col = (u - c * units) * 8, row = row_of ? row_of[c < n ? c : 0] : c;
    int4v v = {0, 0, 0, 0};
    if (row >= 0 && col < cols) {
      const uint16_t* at = in + row * ld + col;
      if (col + 8 <= cols) v = load8(at);
      else {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (col + e < cols) v[e >> 1] |= (int)((uint32_t)at[e] << (e & 1) * 16);
      }
    }
    *reinterpret_cast<int4v*>(out + c * ld_out + col) = v;
  }
}

// bias in units of log 2, -inf behind the last word; and zeros where the teacher's entries will be listed
__global__ void __launch_bounds__(256)
prepare_words(const void* __restrict__ bias, int dtype, int64_t words, int64_t filled, float scale, float* __restrict__ out, uint32_t* __restrict__ clear, int64_t cleared) {
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = first; out && i < filled; i += step) {
    float v = -__builtin_inff();
    if (i < words) v = (dtype == TF24_F32 ? ((const float*)bias)[i] : dtype == TF24_F16 ? to_float(((const f16_t*)bias)[i]) : to_float(((const bf16_t*)bias)[i])) * scale;
    out[i] = v;
  }
  for (int64_t i = first; i < cleared; i += step) reinterpret_cast<uint4*>(clear)[i] = uint4{0, 0, 0, 0};
}

// ---------------------------------------------------------------- losses of the tokens
struct LossTerms { float smoothing, z_loss; int64_t words; int slabs, entries; };

// 2^by tokens of a workgroup, the slabs of each shared out to 256 / 2^by threads.  Bound by memory and, with few tokens, by the launch: 15 for 12288 tokens of 394
// slabs (2.6 TB/s), 40 for 8192 tokens of 1000.
__global__ void __launch_bounds__(256)
token_losses(const float2* __restrict__ stats, const float* __restrict__ sums, int64_t filled, LossTerms how, const int* __restrict__ count, const int* __restrict__ row_of,
             const int* __restrict__ target, const float* __restrict__ picked, const int* __restrict__ entry_words, const float* __restrict__ logq,
             const float* __restrict__ mass, float* __restrict__ lse2, float* __restrict__ by_place, float* __restrict__ by_token, int by) {
  __shared__ float ms[256], ss[256], zs[256];
  const int tid = threadIdx.x, per = 1 << by, share = tid >> by, shares = 256 >> by;
  const int64_t c = (int64_t)blockIdx.x * per + (tid & (per - 1));
  const int n = *count;
  const bool counts = c < n;
  if ((int64_t)blockIdx.x * per >= n) return;
  float m = -__builtin_inff(), s = 0.0f, z = 0.0f;
  auto join = [](float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2), from = top == -__builtin_inff() ? 0.0f : top;
    s = s * exp2f(m - from) + s2 * exp2f(m2 - from);
    m = top;
  };
  if (counts)
    for (int i = share; i < how.slabs; i += shares) {
      const float2 v = stats[(int64_t)i * filled + c];
      join(m, s, v.x, v.y);
      if (sums) z += sums[(int64_t)i * filled + c];
    }
  ms[tid] = m; ss[tid] = s; zs[tid] = z;
  __syncthreads();
  for (int d = shares / 2; d > 0; d /= 2) {
    if (share < d) {
      const int other = tid + (d << by);
      join(ms[tid], ss[tid], ms[other], ss[other]);
      zs[tid] += zs[other];
    }
    __syncthreads();
  }
  const float lse = ms[tid & (per - 1)] + log2f(ss[tid & (per - 1)]);
  const float sum = zs[tid & (per - 1)];
  __syncthreads();
  float loss = 0.0f;
  if (entry_words && counts) {
    for (int k = share; k < how.entries; k += shares) {
      const int64_t at = c * how.entries + k;
      if (entry_words[at] < 0) break;                            // (used ones first)
      const float l = logq[at], q = expf(l);
      if (q != 0.0f) loss += q * (l - (picked[at] - lse) * kLn2);
    }
  }
  zs[tid] = loss;
  __syncthreads();
  for (int d = shares / 2; d > 0; d /= 2) {
    if (share < d) zs[tid] += zs[tid + (d << by)];
    __syncthreads();
  }
  if (share) return;
  if (!counts) return;
  lse2[c] = lse;
  if (entry_words) loss = mass[c] != mass[c] ? mass[c] : zs[tid];
  else {
    const float y = target[c] < 0 ? __builtin_nanf("") : picked[c], natural = lse * kLn2;
    loss = (1.0f - how.smoothing) * ((lse - y) * kLn2) + how.z_loss * natural * natural;
    if (how.smoothing != 0.0f) loss += how.smoothing * ((lse - sum / (float)how.words) * kLn2);
  }
  by_place[c] = loss;
  if (by_token) by_token[row_of[c]] = loss;
}

// One workgroup, in a fixed order: 5 for 12288 tokens
__global__ void __launch_bounds__(1024)
total_loss(const float* __restrict__ by_place, const int* __restrict__ count, bool mean, float* __restrict__ loss) {
  __shared__ double sums[1024];
  const int tid = threadIdx.x, n = *count;
  double v = 0.0;
  for (int c = tid; c < n; c += 1024) v += (double)by_place[c];
  sums[tid] = v;
  __syncthreads();
  for (int d = 512; d > 0; d /= 2) {
    if (tid < d) sums[tid] += sums[tid + d];
    __syncthreads();
  }
  if (tid == 0) *loss = (float)(mean ? sums[0] / (double)max(n, 1) : sums[0]);
}

// ---------------------------------------------------------------- gradient of the logits
// Per token that counts: P = factor exp2(y - lse2) - level everywhere, less `pull` times the listed probabilities, all of it in units of the largest gradient of
// a token's loss: of a mean P is 1 - p at the target, which rounding to 8 bits moves by 2^-9 where 4/3 of it (1 / 12288 less its power of
// two) is moved by 2^-8.
// The level, g smoothing / words, is nearly all of the gradient of a word that is far less probable.  Rounded in P it would be off in the same way for all of those words and
// all tokens (by 0.39 % of it at worst in bfloat16), which no sum averages out.  So P has the nearest number of 16 bits in its place, and what is left of it comes to the results
// in float32: dx is P W less the rest times the sum of W's rows, dW P^T x less the sum of x's rows times their rests, db the sum of P less that of the rests.  (Without a
// level in P a word whose probability is near it would be off by more: by a step of p, not one of the difference.)  W is read once more for it: both passes of 2000 tokens against
// 50257 x 1280 1172 and 1204, of one token against 50304 x 768 156 and 176.
struct SlopeTerms { const float* grad; int reduction; LossTerms how; float inv_temperature; int to_exponent; };
__device__ __forceinline__ float upstream_of(const SlopeTerms& t, int row, int n) {
  const float g = t.reduction == TF24_REDUCE_NONE ? t.grad[row] : t.reduction == TF24_REDUCE_MEAN ? t.grad[0] / (float)n : t.grad[0];
  return g * t.inv_temperature;
}
__device__ __forceinline__ float widened_by(const SlopeTerms& t, const float* mass, const float* lse2, int c) {
  return mass ? mass[c] : 1.0f + 2.0f * t.how.z_loss * (lse2[c] * kLn2);
}

// largest * 2^exponent, kept among float32's normal numbers: P is multiplied by the unit in the end, and nothing may become 0 times infinity on the way
__device__ __forceinline__ float unit_of(float largest, int exponent) { return fminf(fmaxf(ldexpf(largest, exponent), 0x1p-126f), 0x1p127f); }

// The unit, where tokens differ: from the largest gradient of a token's loss, and the largest factor of one relative to it (what is not finite is that anyhow).
// 9 for 8192 tokens: two passes of one workgroup
__global__ void __launch_bounds__(1024)
slope_unit(SlopeTerms terms, const int* __restrict__ count, const int* __restrict__ row_of, const float* __restrict__ mass, const float* __restrict__ lse2,
           float* __restrict__ out_scale) {
  __shared__ float largest[1024];
  const int tid = threadIdx.x, n = *count;
  auto most = [&](float v) {
    largest[tid] = v;
    __syncthreads();
    for (int d = 512; d > 0; d /= 2) {
      if (tid < d) largest[tid] = fmaxf(largest[tid], largest[tid + d]);
      __syncthreads();
    }
    const float top = largest[0];
    __syncthreads();
    return top;
  };
  auto finite = [](float v) { return v < __builtin_inff() ? v : 0.0f; };
  float v = 0.0f;
  for (int c = tid; c < n; c += 1024) v = fmaxf(v, finite(fabsf(upstream_of(terms, row_of[c], n))));
  float unit = most(v);
  if (unit == 0.0f) unit = 1.0f;
  v = 0.0f;
  for (int c = tid; c < n; c += 1024) v = fmaxf(v, finite(fabsf(upstream_of(terms, row_of[c], n) / unit * widened_by(terms, mass, lse2, c))));
  v = most(v);
  if (tid == 0) *out_scale = unit_of(unit, (v > 1.0f ? ilogbf(v) + 1 : 0) - terms.to_exponent);
}

// The terms of 256 tokens; `alike`: all have the same gradient and a factor of one, which is the unit.  Tokens behind the last get a factor of zero, and rows of dx
// that do not count are zero.  5 for 12288 tokens, 12 with 3000 rows of 1280 columns to clear.
template <typename T>
__global__ void __launch_bounds__(256)
slope_terms(SlopeTerms terms, bool alike, const int* __restrict__ count, const int* __restrict__ row_of, const int* __restrict__ target,
            const float* __restrict__ mass, const float* __restrict__ lse2, float2* __restrict__ coef, float* __restrict__ level, float* __restrict__ level_rest,
            float* __restrict__ pull, float* __restrict__ out_scale, T* __restrict__ dx, int64_t width, const int* __restrict__ place_of, int64_t tokens) {
  const int n = *count, c = blockIdx.x * 256 + threadIdx.x;
  float unit;
  if (alike) {
    unit = n ? fabsf(upstream_of(terms, 0, n)) : 0.0f;
    unit = unit_of(unit > 0.0f && unit < __builtin_inff() ? unit : 1.0f, -terms.to_exponent);
    if (c == 0) *out_scale = unit;
  } else unit = *out_scale;
  float2 v = {__builtin_inff(), 0.0f};
  float l = 0.0f, p = 0.0f;
  if (c < n) {
    const float g = upstream_of(terms, row_of[c], n) / unit;
    v = float2{lse2[c], g * widened_by(terms, mass, lse2, c)};
    if (target && target[c] < 0) v.y = __builtin_nanf("");
    l = g * (terms.how.smoothing / (float)terms.how.words);
    p = g * (1.0f - terms.how.smoothing);
  }
  coef[c] = v; pull[c] = p;                                      // (tokens are filled up to whole workgroups)
  if (level) {
    level[c] = to_float(from_float<T>(l));
    level_rest[c] = l - level[c];                                // (exact)
  }
  if (!dx) return;
  const int64_t row0 = (int64_t)blockIdx.x * 256 + (threadIdx.x & ~63);
  const int lane = threadIdx.x & 63;
  for (uint64_t left = __ballot(row0 + lane < tokens && place_of[min(row0 + lane, tokens - 1)] < 0); left; left &= left - 1) {
    T* at = dx + (row0 + __builtin_ctzll(left)) * width;
    if (width % 8 == 0 && (uintptr_t)dx % 16 == 0)
      for (int64_t i = lane * 8; i < width; i += 512) *reinterpret_cast<uint4*>(at + i) = uint4{0, 0, 0, 0};
    else
      for (int64_t i = lane; i < width; i += 64) at[i] = T{0};
  }
}

// The listed words of a piece of the vocabulary in P: one thread per token, or per entry of one; of a word listed twice the first does both.
// `rest` (null: no gradient of the bias is wanted): by word, what rounding takes from them, in units of 2^-32.  They are most of the bias's gradient, whose sum over
// tokens is of rounded values otherwise; as whole numbers they can be added in any order.  Where no token counts, P of the stage of rows that the gradient of the weight
// reads all the same is cleared: what the products made of rows of zeros is NaN where the weight or the bias is not finite.  Bound by single accesses to P: 5 for 12288
// targets, 17 for 8192 x 64 entries.
template <typename T>
__global__ void __launch_bounds__(256)
pull_listed(const int* __restrict__ count, const int* __restrict__ listed, const float* __restrict__ picked, const float* __restrict__ logq, int entries,
            const float2* __restrict__ coef, const float* __restrict__ level, const float* __restrict__ pull, int64_t first_word, int64_t words, T* __restrict__ slope,
            int64_t ld, unsigned long long* __restrict__ rest) {
  const int64_t listed_here = (int64_t)*count * entries;
  if (!listed_here)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < kUnitK * ld / 8; i += (int64_t)gridDim.x * 256) reinterpret_cast<uint4*>(slope)[i] = uint4{0, 0, 0, 0};
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < listed_here; at += (int64_t)gridDim.x * 256) {
    const int w = listed[at];
    if (w < first_word || w >= first_word + words) continue;
    const int64_t c = at / entries;
    float q = 1.0f;
    if (logq) {
      const int k = (int)(at - c * entries);
      if (k && listed[at - 1] == w) continue;
      q = expf(logq[at]);
      for (int j = 1; k + j < entries && listed[at + j] == w; j++) q += expf(logq[at + j]);
    }
    float v = coef[c].y * exp2f(picked[at] - coef[c].x) - pull[c] * q;
    if (level) v -= level[c];
    const T rounded = from_float<T>(v);
    slope[c * ld + (w - first_word)] = rounded;
    if (rest) {
      const float off = v - to_float(rounded);
      if (fabsf(off) < 65536.0f) atomicAdd(rest + (w - first_word), (unsigned long long)(long long)(off * 4294967296.0f));     // (not of what is infinite or NaN)
    }
  }
}
__global__ void __launch_bounds__(256) clear_rest(unsigned long long* __restrict__ rest, int64_t words) {
  for (int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x; w < words; w += (int64_t)gridDim.x * 256) rest[w] = 0;
}

// Sums of the columns of one or two operands (blockIdx.z), in as many pieces of their rows (*count of them, or `rows`) as the grid is high: of P, for db; with smoothing of W,
// and of x with each row times the rest of its level.  Bound by memory: P of 2000 tokens and 50257 words 30 (6.7 TB/s, much of it still in the caches), the weight of 50257 x
// 1280 and 2000 rows of x 20 (6.7 TB/s, from the caches as well).
struct ColumnSums { const void* in; int64_t ld; const int* count; int64_t rows; const float* times; float *pieces, *out; };
constexpr int kBiasPieces = 16, kOperandPieces = 64;
template <typename T>
__global__ void __launch_bounds__(256)
sum_columns(const ColumnSums one, const ColumnSums other, int64_t cols) {
  __shared__ float part[8][256];
  const ColumnSums& which = blockIdx.z ? other : one;
  const T* in = (const T*)which.in;
  const float* times = which.times;
  const int64_t ld = which.ld;
  const int n = which.count ? *which.count : (int)which.rows, tid = threadIdx.x, chunk = tid & 31, group = tid >> 5;
  const int64_t col = (int64_t)blockIdx.x * 256 + chunk * 8;
  const int begin = (int)((int64_t)blockIdx.y * n / gridDim.y), end = (int)((int64_t)(blockIdx.y + 1) * n / gridDim.y);
  float v[8] = {};
  if (col < cols)
#pragma unroll 4
    for (int c = begin + group; c < end; c += 8) {
      Pack<T, 8> p;
      p.load(in + c * ld + col);
      const float by = times ? times[c] : 1.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(to_float(p.v[e]), by, v[e]);
    }
#pragma unroll
  for (int e = 0; e < 8; e++) part[group][chunk * 8 + e] = v[e];
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int g = 0; g < 8; g++) s += part[g][tid];
  if ((int64_t)blockIdx.x * 256 + tid < cols) which.pieces[blockIdx.y * cols + (int64_t)blockIdx.x * 256 + tid] = s;
}
__global__ void __launch_bounds__(64) join_columns(const ColumnSums one, const ColumnSums other, int64_t cols) {
  const ColumnSums& which = blockIdx.y ? other : one;
  const int64_t col = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (col >= cols) return;
  float s = 0.0f;
#pragma unroll 16
  for (int p = 0; p < kOperandPieces; p++) s += which.pieces[p * cols + col];
  which.out[col] = s;
}
// db, over the pieces; `level_rests`: what the rests of all tokens' levels add up to, or null.  5 for 50257 words
__global__ void __launch_bounds__(256)
join_bias(const float* __restrict__ sums, int64_t ld, int64_t words, const unsigned long long* __restrict__ rest, const float* __restrict__ level_rests, const float* __restrict__ scale,
          void* __restrict__ out, int dtype) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= words) return;
  float v = (float)((double)(long long)rest[w] * 0x1p-32);
  for (int p = 0; p < kBiasPieces; p++) v += sums[p * ld + w];
  if (level_rests) v -= *level_rests;
  v = scaled(v, *scale);
  if (dtype == TF24_F32) ((float*)out)[w] = v;
  else if (dtype == TF24_F16) ((f16_t*)out)[w] = from_float<f16_t>(v);
  else ((bf16_t*)out)[w] = from_float<bf16_t>(v);
}

// ---------------------------------------------------------------- buffers
int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Carve {                                                   // parts of a buffer, or (no buffer) how long it has to be
  uint8_t* base;
  int64_t used = 0;
  template <typename P>
  void operator()(P*& p, int64_t bytes) {
    p = base ? (P*)(base + used) : nullptr;
    used += up(bytes, 256);
  }
};

// what the forward pass leaves for the backward pass
struct State {
  int *count, *row_of, *place_of, *listed;
  float *lse2, *picked, *logq = nullptr, *mass = nullptr;
  int64_t bytes;
};
State state_of(void* base, int64_t tokens, int64_t entries) {
  State s;
  Carve part{(uint8_t*)base};
  const int64_t filled = up(tokens, kTile), many = filled * std::max<int64_t>(entries, 1);
  part(s.count, 4);
  part(s.row_of, filled * 4 + kOverread);
  part(s.place_of, filled * 4);
  part(s.lse2, filled * 4);
  part(s.listed, many * 4 + kOverread);
  part(s.picked, many * 4);
  if (entries) {
    part(s.logq, many * 4);
    part(s.mass, filled * 4);
  }
  s.bytes = part.used;
  return s;
}

struct Sizes {
  int64_t tokens, width, words, entries;                         // entries: of a token, 0: a target
  int64_t filled, k, slabs, words_filled;
  bool pack_weight, smooth, few;
};
Sizes sizes_of(int64_t tokens, int64_t width, int64_t words, int64_t entries, bool smooth, const void* w, int64_t ldw) {
  Sizes z{tokens, width, words, entries, up(tokens, kTile), up(width, kUnitK), 0, up(words, kTile), false, smooth, false};
  // rows of whole stages, 16-byte aligned, within reach of 32-bit offsets in a tile
  z.pack_weight = width % kUnitK || ldw % 8 || ldw > (1 << 22) || (uintptr_t)w % 16;
  // The kernel for few tokens and the tiles, forward pass in us: 50304 x 768 1 token 25 and 40, 64 tokens 37 and 41; 128000 x 4096 16 tokens 195 and 266, 64 266
  // and 269; 50304 x 2048 16 tokens 49 and 63, 64 72 and 64.  Where tiles need a copy of the weight first: 50257 x 1601 32 tokens 56 and 119, 64 72 and 119.  One
  // limit for both kinds of rows: results do not depend on strides and alignment.
  z.few = tokens <= kFewTokens;
  z.slabs = z.few ? (words + kFewSlab - 1) / kFewSlab : z.words_filled / kSlab;
  return z;
}

struct Forward {
  uint16_t *x = nullptr, *w = nullptr;
  float *bias = nullptr, *sums = nullptr, *losses;
  float2* stats;
  int* flags = nullptr;
  uint32_t* slab_entries = nullptr;
  int64_t bytes;
};
Forward forward_of(void* base, const Sizes& z) {
  Forward f;
  Carve part{(uint8_t*)base};
  if (!z.few) {
    part(f.x, z.filled * z.k * 2);
    if (z.pack_weight) part(f.w, z.words * z.k * 2);
    part(f.bias, z.words_filled * 4 + kOverread);
  }
  part(f.stats, z.slabs * z.filled * 8);
  if (z.smooth) part(f.sums, z.slabs * z.filled * 4);
  part(f.losses, z.filled * 4);
  if (z.entries) {
    part(f.flags, z.filled * 4);
    part(f.slab_entries, z.slabs * z.filled * 4 + kOverread);
  }
  f.bytes = part.used;
  return f;
}

int64_t tiles_of(int64_t size) { return (size + kTile - 1) / kTile; }

struct Backward {
  uint16_t *x, *w = nullptr;
  float *bias, *pull, *out_scale, *partial = nullptr, *sum_x = nullptr, *bias_sums = nullptr;
  float *level = nullptr, *level_rest = nullptr, *level_rests = nullptr, *column_sums = nullptr, *sum_of_w = nullptr, *sum_of_x = nullptr;     // with smoothing
  float2* coef;
  unsigned long long* bias_rest = nullptr;
  uint8_t* slope;
  int64_t ld, pieces, bytes;                                     // words of a piece of the vocabulary, pieces
  int groups, most_x = 0, most_w = 0;                            // workgroups of the products with a long k; pieces of their tiles
};
Backward backward_of(void* base, const Sizes& z, bool input, bool weight, bool bias) {
  Backward b;
  Carve part{(uint8_t*)base};
  b.groups = std::max(1, compute_units() / 8) * 8;
  const int64_t blocks = z.words_filled / kTile, at_once = std::max<int64_t>(1, kSlopeBytes / (z.filled * 2 * kTile));
  b.pieces = (blocks + at_once - 1) / at_once;
  b.ld = (blocks + b.pieces - 1) / b.pieces * kTile;
  b.pieces = (z.words_filled + b.ld - 1) / b.ld;
  const int64_t width_tiles = tiles_of(z.k);
  auto most = [&](int64_t rest, int64_t stages) { return (int)std::min<int64_t>(kMostPieces, rest * stages); };
  if (input) b.most_x = most(std::min<int64_t>(width_tiles * tiles_of(z.tokens), b.groups - 1), b.ld / kUnitK);     // (fewer tokens may count: another rest)
  if (weight) {
    const int64_t other = z.words_filled - (b.pieces - 1) * b.ld;                                  // the last piece
    b.most_w = most(std::max(width_tiles * (b.ld / kTile) % b.groups, width_tiles * (other / kTile) % b.groups), z.filled / kUnitK);
  }
  part(b.x, z.filled * z.k * 2);
  if (z.pack_weight) part(b.w, z.words * z.k * 2);
  part(b.bias, z.words_filled * 4 + kOverread);
  part(b.coef, z.filled * 8 + kOverread);
  if (z.smooth) {
    part(b.level, z.filled * 4 + kOverread);
    part(b.level_rest, z.filled * 4 + kOverread);
    part(b.level_rests, 4);
    part(b.column_sums, 2 * kOperandPieces * z.k * 4);
    part(b.sum_of_w, width_tiles * kTile * 4 + kOverread);
    part(b.sum_of_x, width_tiles * kTile * 4 + kOverread);
  }
  part(b.pull, z.filled * 4);
  part(b.out_scale, 4);
  part(b.slope, z.filled * b.ld * 2);
  part(b.partial, (int64_t)std::max(b.most_x, b.most_w) * kTile * kTile * 4);
  if (input && b.pieces > 1) part(b.sum_x, width_tiles * z.filled * kTile * 4);
  if (bias) {
    part(b.bias_sums, kBiasPieces * b.ld * 4);
    part(b.bias_rest, b.ld * 8);
  }
  b.bytes = part.used;
  return b;
}

unsigned blocks_for(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, 4096)); }

int check_head(const char* fn, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int dtype, int64_t tokens, int64_t width,
               int64_t words, int64_t entries, float smoothing, float z_loss, float inv_temperature, int reduction) {
  if (dtype != TF24_F16 && dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (bias && bias_dtype != TF24_F32 && bias_dtype != TF24_F16 && bias_dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d of the bias", fn, bias_dtype);
  if (tokens < 1 || tokens > (1 << 22) || width < 1 || width > (1 << 16) || words < 1 || words > (1 << 22))
    return fail(TF24_ERR_SHAPE, "%s: %lld tokens of %lld columns against %lld words: 1 to 2^22, 2^16 and 2^22 are supported", fn, (long long)tokens, (long long)width,
                (long long)words);
  if (tiles_of(tokens) * tiles_of(words) > (1 << 26))
    return fail(TF24_ERR_SHAPE, "%s: %lld tokens against %lld words are more than one launch takes", fn, (long long)tokens, (long long)words);
  if (entries < 0 || entries > kMaxEntries) return fail(TF24_ERR_SHAPE, "%s: %lld entries of a token, at most %d are supported", fn, (long long)entries, kMaxEntries);
  if (ldx < 0 || ldw < 0) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  if (!(smoothing >= 0.0f && smoothing <= 1.0f) || !std::isfinite(z_loss) || !(inv_temperature > 0.0f) || !std::isfinite(inv_temperature))
    return fail(TF24_ERR_ARG, "%s: smoothing %g, z_loss %g or 1 / temperature %g is out of range", fn, smoothing, z_loss, inv_temperature);
  if (entries && (smoothing != 0.0f || z_loss != 0.0f)) return fail(TF24_ERR_ARG, "%s: smoothing and z_loss go with targets", fn);
  if (reduction != TF24_REDUCE_MEAN && reduction != TF24_REDUCE_SUM && reduction != TF24_REDUCE_NONE) return fail(TF24_ERR_ARG, "%s: bad reduction %d", fn, reduction);
  if (!x || !w) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, 2, {x, w})) return rc;
  return bias ? check_aligned(fn, dtype_size(bias_dtype), {bias}) : TF24_OK;
}

void pack(const void* in, int64_t ld, int64_t rows, int64_t cols, const int* count, const int* row_of, uint16_t* out, int64_t ld_out, hipStream_t s) {
  hipLaunchKernelGGL(pack_rows, dim3(blocks_for(rows * (ld_out / 8))), dim3(256), 0, s, (const uint16_t*)in, ld, rows, cols, count, row_of,
                     out, ld_out);
}

}  // namespace
}  // namespace tf24

extern "C" int64_t tf24_linear_loss_state_bytes(int64_t tokens, int64_t entries) {
  if (tokens < 1 || tokens > (1 << 22) || entries < 0 || entries > tf24::kMaxEntries) return 0;
  return tf24::state_of(nullptr, tokens, entries).bytes;
}

extern "C" int64_t tf24_linear_loss_forward_workspace_bytes(int64_t tokens, int64_t width, int64_t words, int64_t entries, int smooth, const void* w, int64_t ldw) {
  using namespace tf24;
  if (tokens < 1 || width < 1 || words < 1 || entries < 0) return 0;
  return forward_of(nullptr, sizes_of(tokens, width, words, entries, smooth != 0, w, ldw)).bytes;
}

extern "C" int64_t tf24_linear_loss_backward_workspace_bytes(int64_t tokens, int64_t width, int64_t words, int64_t entries, int smooth, const void* w, int64_t ldw, int input,
                                                             int weight, int bias) {
  using namespace tf24;
  if (tokens < 1 || width < 1 || words < 1 || entries < 0) return 0;
  return backward_of(nullptr, sizes_of(tokens, width, words, entries, smooth != 0, w, ldw), input != 0, weight != 0, bias != 0).bytes;
}

extern "C" int tf24_linear_loss_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int dtype, int64_t tokens, int64_t width,
                                        int64_t words, const int64_t* targets, int64_t ignore, const int64_t* indices, int64_t ld_indices, const void* teacher_logits,
                                        int64_t ld_teacher, int teacher_dtype, const float* teacher_lse, int64_t entries, float smoothing, float z_loss,
                                        float inv_temperature, int reduction, float* loss, void* state, int64_t state_bytes, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  using namespace tf24;
  const char* fn = "tf24_linear_loss_forward";
  if (int rc = check_head(fn, x, ldx, w, ldw, bias, bias_dtype, dtype, tokens, width, words, entries, smoothing, z_loss, inv_temperature, reduction)) return rc;
  if (entries ? !indices || !teacher_logits || targets : !targets || indices) return fail(TF24_ERR_ARG, "%s: either targets, or entries of a teacher", fn);
  if (entries && teacher_dtype != TF24_F32 && teacher_dtype != TF24_F16 && teacher_dtype != TF24_BF16)
    return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d of the teacher's logits", fn, teacher_dtype);
  if (entries && (ld_indices < 0 || ld_teacher < 0)) return fail(TF24_ERR_STRIDE, "%s: negative leading dimension", fn);
  if (!loss || !state || !workspace) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (int rc = check_aligned(fn, 16, {state, workspace})) return rc;
  if (int rc = check_aligned(fn, 8, {targets, indices})) return rc;
  if (int rc = check_aligned(fn, 4, {loss, teacher_lse})) return rc;
  if (entries) {
    if (int rc = check_aligned(fn, dtype_size(teacher_dtype), {teacher_logits})) return rc;
  }
  const Sizes z = sizes_of(tokens, width, words, entries, smoothing != 0.0f, w, ldw);
  const State st = state_of(state, tokens, entries);
  const Forward f = forward_of(workspace, z);
  if (state_bytes < st.bytes || workspace_bytes < f.bytes)
    return fail(TF24_ERR_ARG, "%s: %lld and %lld bytes of state and workspace, %lld and %lld are needed", fn, (long long)state_bytes, (long long)workspace_bytes,
                (long long)st.bytes, (long long)f.bytes);
  hipStream_t s = (hipStream_t)stream;
  const float scale = kLog2e * inv_temperature;
  auto teacher = [&](auto go) {
    if (teacher_dtype == TF24_F32) go((const float*)teacher_logits);
    else if (teacher_dtype == TF24_F16) go((const f16_t*)teacher_logits);
    else go((const bf16_t*)teacher_logits);
  };
  if (entries)
    teacher([&](auto* logits) {
      hipLaunchKernelGGL(flag_tokens, dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, s, indices, ld_indices, logits, ld_teacher, (int)tokens, (int)entries, f.flags);
    });
  if (!z.few || entries)
    hipLaunchKernelGGL(count_tokens, dim3(1), dim3(1024), 0, s, targets, ignore, f.flags, (int)tokens, (int)z.filled, words, st.count, st.row_of, st.place_of, st.listed,
                       reduction == TF24_REDUCE_NONE ? loss : nullptr);
  const bool with_bias = bias && !z.few;
  const int64_t cleared = entries ? z.slabs * z.filled / 4 : 0;     // (filled is a multiple of 4)
  if (with_bias || entries)
    hipLaunchKernelGGL(prepare_words, dim3(blocks_for(std::max(with_bias ? z.words_filled : 0, cleared))), dim3(256), 0, s, bias, bias_dtype, words, z.words_filled, scale,
                       with_bias ? f.bias : nullptr, f.slab_entries, cleared);
  if (entries) {
    int padded = 2;
    while (padded < entries) padded *= 2;
    teacher([&](auto* logits) {
      hipLaunchKernelGGL(list_entries, dim3((unsigned)tokens), dim3(64), 0, s, indices, ld_indices, logits, ld_teacher, teacher_lse, inv_temperature, (int)entries, padded,
                         words, st.count, st.row_of, st.listed, st.logq, st.mass, f.slab_entries, z.filled, z.few ? kFewSlab : kSlab);
    });
  }
  HeadResult r{};
  r.scale = scale; r.bias = f.bias && bias ? f.bias : nullptr; r.tokens_ld = z.filled; r.words = words;
  r.stats = f.stats; r.sums = f.sums; r.picked = st.picked;
  if (entries) { r.slab_entries = f.slab_entries; r.entry_words = st.listed; r.entries = (int)entries; }
  else r.target = st.listed;
  if (z.few) {
    const FewTokens which{(int)tokens, (int)z.filled, targets, ignore, st.count, st.row_of, st.place_of, st.listed, reduction == TF24_REDUCE_NONE ? loss : nullptr};
    if (int rc = launch_few_tokens(dtype, z.smooth, which, x, ldx, w, ldw, width, bias, bias_dtype, r, stream)) return rc;
  } else {
    pack(x, ldx, z.filled, width, st.count, st.row_of, f.x, z.k, s);
    if (f.w) pack(w, ldw, words, width, nullptr, nullptr, f.w, z.k, s);
    HeadProduct p{};
    p.a = (const uint8_t*)(f.w ? f.w : w); p.lda = (f.w ? z.k : ldw) * 2;
    p.b = (const uint8_t*)f.x; p.ldb = z.k * 2;
    p.count = st.count;
    p.rows_i = words;
    p.stages = (int)(z.k / kUnitK); p.tiles_i = (int)tiles_of(words); p.tiles_j = (int)tiles_of(tokens);
    if (int rc = launch_head_product(HEAD_STATS, dtype, z.smooth, false, p, r, stream)) return rc;
  }
  // workgroups for every compute unit, then loads of whole lines (1, 4 and 16 tokens of a workgroup, us for 50304 words: 64 tokens 6, 10 and 22; 1024 tokens 9, 7
  // and 22; 8192 tokens 32, 20 and 14)
  const int by = tokens <= 64 ? 0 : tokens <= 4096 ? 2 : 4;
  hipLaunchKernelGGL(token_losses, dim3((unsigned)((tokens + (1 << by) - 1) >> by)), dim3(256), 0, s, f.stats, f.sums, z.filled, LossTerms{smoothing, z_loss, words, (int)z.slabs, (int)entries},
                     st.count, st.row_of, st.listed, st.picked, entries ? st.listed : nullptr, st.logq, st.mass, st.lse2, f.losses,
                     reduction == TF24_REDUCE_NONE ? loss : nullptr, by);
  if (reduction != TF24_REDUCE_NONE) hipLaunchKernelGGL(total_loss, dim3(1), dim3(1024), 0, s, f.losses, st.count, reduction == TF24_REDUCE_MEAN, loss);
  return check_launch(fn);
}

extern "C" int tf24_linear_loss_backward(const float* grad_loss, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_dtype, int dtype,
                                         int64_t tokens, int64_t width, int64_t words, int64_t entries, float smoothing, float z_loss, float inv_temperature,
                                         int reduction, const void* state, int64_t state_bytes, void* dx, void* dw, int dw_dtype, void* dbias, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_linear_loss_backward";
  if (int rc = check_head(fn, x, ldx, w, ldw, bias, bias_dtype, dtype, tokens, width, words, entries, smoothing, z_loss, inv_temperature, reduction)) return rc;
  if (dw && dw_dtype != dtype && dw_dtype != TF24_F32) return fail(TF24_ERR_DTYPE, "%s: a weight gradient of dtype %d from dtype %d", fn, dw_dtype, dtype);
  if (!grad_loss || !state || !workspace) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (dbias && !bias) return fail(TF24_ERR_ARG, "%s: the gradient of a bias that is none", fn);
  if (int rc = check_aligned(fn, 16, {state, workspace})) return rc;
  if (int rc = check_aligned(fn, 4, {grad_loss})) return rc;
  if (int rc = check_aligned(fn, 2, {dx})) return rc;
  if (dw) {
    if (int rc = check_aligned(fn, dtype_size(dw_dtype), {dw})) return rc;
  }
  if (dbias) {
    if (int rc = check_aligned(fn, dtype_size(bias_dtype), {dbias})) return rc;
  }
  const Sizes z = sizes_of(tokens, width, words, entries, smoothing != 0.0f, w, ldw);
  const State st = state_of(const_cast<void*>(state), tokens, entries);
  const Backward b = backward_of(workspace, z, dx != nullptr, dw != nullptr, dbias != nullptr);
  if (state_bytes < st.bytes || workspace_bytes < b.bytes)
    return fail(TF24_ERR_ARG, "%s: %lld and %lld bytes of state and workspace, %lld and %lld are needed", fn, (long long)state_bytes, (long long)workspace_bytes,
                (long long)st.bytes, (long long)b.bytes);
  if (!dx && !dw && !dbias) return TF24_OK;
  hipStream_t s = (hipStream_t)stream;
  const float scale = kLog2e * inv_temperature;
  const LossTerms how{smoothing, z_loss, words, (int)z.slabs, (int)entries};
  const SlopeTerms terms{grad_loss, reduction, how, inv_temperature, dtype == TF24_F16 ? 14 : 0};
  const bool alike = reduction != TF24_REDUCE_NONE && z_loss == 0.0f && !entries;
  if (!alike) hipLaunchKernelGGL(slope_unit, dim3(1), dim3(1024), 0, s, terms, st.count, st.row_of, st.mass, st.lse2, b.out_scale);
  auto set_terms = [&](auto* out) {
    hipLaunchKernelGGL(slope_terms, dim3((unsigned)(z.filled / 256)), dim3(256), 0, s, terms, alike, st.count, st.row_of, entries ? nullptr : st.listed, st.mass, st.lse2, b.coef,
                       b.level, b.level_rest, b.pull, b.out_scale, out, width, st.place_of, tokens);
  };
  if (dtype == TF24_F16) set_terms((f16_t*)dx);
  else set_terms((bf16_t*)dx);
  const bool with_bias = bias != nullptr;
  if (with_bias)
    hipLaunchKernelGGL(prepare_words, dim3(blocks_for(z.words_filled)), dim3(256), 0, s, bias, bias_dtype, words, z.words_filled, scale, b.bias, (uint32_t*)nullptr,
                       (int64_t)0);
  pack(x, ldx, z.filled, width, st.count, st.row_of, b.x, z.k, s);
  if (b.w) pack(w, ldw, words, width, nullptr, nullptr, b.w, z.k, s);
  const uint8_t* w_at = (const uint8_t*)(b.w ? b.w : w);
  const int64_t w_ld = (b.w ? z.k : ldw) * 2;
  auto sum_up = [&](const ColumnSums& one, const ColumnSums* other, int64_t cols, int pieces) {
    const dim3 grid((unsigned)((cols + 255) / 256), pieces, other ? 2 : 1);
    if (dtype == TF24_F16) hipLaunchKernelGGL(sum_columns<f16_t>, grid, dim3(256), 0, s, one, other ? *other : one, cols);
    else hipLaunchKernelGGL(sum_columns<bf16_t>, grid, dim3(256), 0, s, one, other ? *other : one, cols);
  };
  if (z.smooth && (dx || dw)) {
    const ColumnSums of_w{w_at, w_ld / 2, nullptr, words, nullptr, b.column_sums, b.sum_of_w};
    const ColumnSums of_x{b.x, z.k, st.count, 0, b.level_rest, b.column_sums + kOperandPieces * z.k, b.sum_of_x};
    const ColumnSums& one = dx ? of_w : of_x;
    sum_up(one, dx && dw ? &of_x : nullptr, z.k, kOperandPieces);
    hipLaunchKernelGGL(join_columns, dim3((unsigned)(z.k / 64), dx && dw ? 2 : 1), dim3(64), 0, s, one, of_x, z.k);
  }
  if (z.smooth && dbias) hipLaunchKernelGGL(total_loss, dim3(1), dim3(1024), 0, s, b.level_rest, st.count, false, b.level_rests);
  for (int64_t piece = 0; piece < b.pieces; piece++) {
    const int64_t first = piece * b.ld, here = std::min(b.ld, words - first);
    HeadProduct p{};
    p.a = w_at + first * w_ld; p.lda = w_ld;
    p.b = (const uint8_t*)b.x; p.ldb = z.k * 2;
    p.count = st.count;
    p.rows_i = here;
    p.stages = (int)(z.k / kUnitK); p.tiles_i = (int)tiles_of(here); p.tiles_j = (int)tiles_of(tokens);
    HeadResult r{};
    r.scale = scale; r.bias = with_bias ? b.bias + first : nullptr; r.tokens_ld = z.filled;
    r.coef = b.coef; r.level = b.level; r.slope = b.slope; r.ld_slope = b.ld; r.words = here;
    if (int rc = launch_head_product(HEAD_SLOPE, dtype, z.smooth, false, p, r, stream)) return rc;
    const int64_t many = std::max<int64_t>(entries, 1);
    if (dbias) hipLaunchKernelGGL(clear_rest, dim3(blocks_for(here)), dim3(256), 0, s, b.bias_rest, here);
    auto put_right = [&](auto* slope) {
      hipLaunchKernelGGL(pull_listed, dim3((unsigned)std::min<int64_t>((tokens * many + 255) / 256, kMostBlocks)), dim3(256), 0, s, st.count, st.listed, st.picked, st.logq, (int)many, b.coef,
                         b.level, b.pull, first, here, slope, b.ld, b.bias_rest);
    };
    if (dtype == TF24_F16) put_right((f16_t*)b.slope);
    else put_right((bf16_t*)b.slope);
    HeadProduct q{};
    q.b = b.slope; q.ldb = b.ld * 2;
    q.count = st.count;
    q.rows_i = z.k; q.tiles_i = (int)tiles_of(z.k);
    q.groups = b.groups;
    HeadResult o{};
    o.partial = b.partial; o.out_scale = b.out_scale; o.cols_out = width;
    if (dx) {
      q.a = w_at + first * w_ld; q.lda = w_ld; q.rows_k = here;
      q.stages = (int)((here + kUnitK - 1) / kUnitK); q.tiles_j = (int)tiles_of(tokens); q.most = b.most_x;
      o.out = dx; o.row_of = st.row_of; o.sum = b.sum_x; o.add = piece > 0; o.last = piece == b.pieces - 1;
      o.common = b.sum_of_w; o.level_rest = b.level_rest;
      if (int rc = launch_head_product(HEAD_INPUT, dtype, z.smooth, false, q, o, stream)) return rc;
    }
    if (dw) {
      q.a = (const uint8_t*)b.x; q.lda = z.k * 2;
      q.stages = (int)((tokens + kUnitK - 1) / kUnitK); q.tiles_j = (int)tiles_of(here); q.most = b.most_w;
      if (share_out(q.tiles_i * q.tiles_j, q.stages, q.groups, q.most).pieces == 1) q.most = 0;    // no pieces, whatever number of tokens counts
      o.out = (uint8_t*)dw + first * width * dtype_size(dw_dtype); o.sum = nullptr; o.add = false; o.last = true; o.rows_j = here;
      o.common = b.sum_of_x;
      if (int rc = launch_head_product(HEAD_WEIGHT, dtype, z.smooth, dw_dtype == TF24_F32, q, o, stream)) return rc;
    }
    if (dbias) {
      sum_up(ColumnSums{b.slope, b.ld, st.count, 0, nullptr, b.bias_sums, nullptr}, nullptr, b.ld, kBiasPieces);
      hipLaunchKernelGGL(join_bias, dim3((unsigned)((here + 255) / 256)), dim3(256), 0, s, b.bias_sums, b.ld, here, b.bias_rest, b.level_rests, b.out_scale,
                         (void*)((uint8_t*)dbias + first * dtype_size(bias_dtype)), bias_dtype);
    }
  }
  return check_launch(fn);
}
