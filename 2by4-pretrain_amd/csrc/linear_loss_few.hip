// The logits of few tokens (up to 64) against a whole vocabulary, and what linear_loss.hip wants of them: per token and slab of 64 words a maximum and a sum of
// exponentials, and the logits of the listed words.
//
// Bound by memory: the weight is read once, straight into registers, and as it lies, whatever its rows' alignment (a copy of it in whole aligned stages, as the
// tiles want it, costs three times the reading).  A workgroup takes 64 words; its four waves share the width out among them, 32 columns a step, so that
// 16 waves and more of a compute unit have loads in flight, and add up their products through the LDS.  The tokens' rows come from the caches.
// One token, 50304 x 768 bf16 (77 MB): 18 us, 4.3 TB/s; 16 tokens, 128000 x 4096 (1 GB): 185 us, 5.7 TB/s; 37 tokens, 50257 x 1601 float16, every other row in the middle of a
// dword: 62 us, 2.6 TB/s, bound by the loads' passes over lines that 16 bytes from any address cross.
#include "linear_loss.hpp"
#include "head_tiles.hpp"

namespace tf24 {
namespace {

constexpr int kWords = 64;                                       // of a workgroup

// the columns of a row that are left of eight
__device__ __forceinline__ int4v load_up_to(const uint16_t* p, int64_t left) {
  int4v v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (e < left) v[e >> 1] |= (int)((uint32_t)p[e] << (e & 1) * 16);
  return v;
}

// A lane's eight columns of a step of a row, from dword to dword (loads that cross dwords take several times as long: 133 us for 37 tokens against 50257 x 1601).
// Where rows start in the middle of a dword, the columns are moved down by half of one, and the last comes from the dword that follows: the first
// of the lane 16 further on, or (the last quarter) of the next step.
struct __attribute__((packed, aligned(4))) Dwords { int4v v; };
struct Row {
  const uint32_t* at;                                            // the dword of the lane's first column
  uint32_t shift;                                                // 16: its second half
  __device__ __forceinline__ explicit Row(const uint16_t* p) : at((const uint32_t*)((uintptr_t)p & ~(uintptr_t)3)), shift(((uintptr_t)p & 2) * 8) {}
  __device__ __forceinline__ int4v load(int step) const { return reinterpret_cast<const Dwords*>(at + step * 16)->v; }
  // in the lanes of the first quarter the dword that follows the steps before `step`, where their last column lies in it (else, as in the other lanes, whatever
  // they have read already: there may be nothing behind it)
  __device__ __forceinline__ uint32_t follower(int step, bool first_quarter) const { return at[(first_quarter && shift ? step : step - 1) * 16]; }
  __device__ __forceinline__ int4v moved(int4v v, uint32_t next_first, bool first_quarter, int from_lane) const {
    const uint32_t behind = (uint32_t)__builtin_amdgcn_ds_bpermute(from_lane * 4, (int)(first_quarter ? next_first : (uint32_t)v[0]));
    int4v o;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = (int)__builtin_amdgcn_alignbit(e < 3 ? (uint32_t)v[e + 1] : behind, (uint32_t)v[e], shift);
    return o;
  }
};

// N: fragments of 16 tokens.  HALVES: rows may start in the middle of a dword.
// kSteps: steps whose loads are in flight at once.  Two, and registers for two workgroups of a compute unit at least, against four: 16 tokens, 128000 x 4096 196 us
// (so without the bound on registers; with it 225) and 238, 48 tokens 236 and 266.  Where the loads are to be moved, which takes registers of its own, four and
// no bound against two of each: 37 tokens, 50257 x 1601 68 and 70, 64 tokens 79 and 96.
template <typename T, int N, bool SMOOTH, bool HALVES>
__global__ void __launch_bounds__(256, HALVES || N == 1 ? 1 : 2)
few_tokens(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ w, int64_t ldw, int64_t width, const FewTokens which,
           const void* __restrict__ bias, int bias_dtype, const HeadResult r) {
  constexpr int STRIDE = kWords + 4;                             // floats of a token: 16 tokens start 16 bytes apart
  constexpr int kSteps = HALVES ? 4 : 2;
  // The waves' parts of a sum: of all four where the LDS holds them beside those of other workgroups, else of two, to which the others add theirs (64 tokens, 50257 x
  // 1601 102 us with four parts, 79 with two; 48 tokens, 50304 x 768 34 and 31; 32 tokens, 50257 x 1601 63 and 70).
  constexpr int PARTS = N <= 2 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) float part[PARTS][16 * N][STRIDE];
  __shared__ int rows[kFewTokens], wanted[kFewTokens];           // of the tokens that count, and their targets
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lq = lane >> 4;
  const int64_t word0 = (int64_t)blockIdx.x * kWords;
  int n;
  if (which.targets) {
    // every workgroup finds out for itself which tokens count; the first one writes it down
    const int64_t target = lane < which.tokens ? which.targets[lane] : which.ignore;
    const bool yes = lane < which.tokens && target != which.ignore;
    const uint64_t mask = __ballot(yes);
    const int place = __popcll(mask & ((1ull << lane) - 1)), word = target >= 0 && target < r.words ? (int)target : -2;
    n = __popcll(mask);
    if (wave == 0 && yes) { rows[place] = lane; wanted[place] = word; }
    if (blockIdx.x == 0 && wave == 0) {
      if (lane < which.tokens) which.place_of[lane] = yes ? place : -1;
      if (yes) { which.row_of[place] = lane; which.listed[place] = word; }
      if (lane >= n) { which.row_of[lane] = -1; which.listed[lane] = -1; }
      for (int c = 64 + lane; c < which.filled; c += 64) { which.row_of[c] = -1; which.listed[c] = -1; }
      if (which.loss && lane < which.tokens && !yes) which.loss[lane] = 0.0f;
      if (lane == 0) *which.count = n;
    }
  } else {
    n = *which.count;
    if (wave == 0 && lane < n) rows[lane] = which.row_of[lane];
  }
  if (!n) return;
  __syncthreads();
  auto weight_row = [&](int f) { return w + min(word0 + f * 16 + l16, r.words - 1) * ldw + lq * 8; };
  auto token_row = [&](int t) { return x + (int64_t)rows[t * 16 + l16 < n ? t * 16 + l16 : 0] * ldx + lq * 8; };    // (columns of tokens behind the last are not used)
  const Row a[4] = {Row(weight_row(0)), Row(weight_row(1)), Row(weight_row(2)), Row(weight_row(3))};
  const Row b[4] = {Row(token_row(0)), Row(token_row(N > 1 ? 1 : 0)), Row(token_row(N > 2 ? 2 : 0)), Row(token_row(N > 3 ? 3 : 0))};
  const int steps = (int)(width / 32), begin = wave * steps / 4, end = (wave + 1) * steps / 4;
  float4v acc[4][N];
#pragma unroll
  for (int f = 0; f < 4; f++)
#pragma unroll
    for (int t = 0; t < N; t++) acc[f][t] = float4v{0, 0, 0, 0};
  const bool first_quarter = lq == 0;
  const int from_lane = (lane + 16) & 63;
  auto some = [&](auto many, int s) {                            // so many steps
    constexpr int U = decltype(many)::value;
    int4v av[U][4], bv[U][N];
    uint32_t af[4], bf[N];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int f = 0; f < 4; f++) av[u][f] = a[f].load(s + u);
#pragma unroll
      for (int t = 0; t < N; t++) bv[u][t] = b[t].load(s + u);
    }
    if constexpr (HALVES) {
#pragma unroll
      for (int f = 0; f < 4; f++) af[f] = a[f].follower(s + U, first_quarter);
#pragma unroll
      for (int t = 0; t < N; t++) bf[t] = b[t].follower(s + U, first_quarter);
#pragma unroll
      for (int u = 0; u < U; u++) {
#pragma unroll
        for (int f = 0; f < 4; f++) av[u][f] = a[f].moved(av[u][f], u + 1 < U ? (uint32_t)av[u + 1 < U ? u + 1 : u][f][0] : af[f], first_quarter, from_lane);
#pragma unroll
        for (int t = 0; t < N; t++) bv[u][t] = b[t].moved(bv[u][t], u + 1 < U ? (uint32_t)bv[u + 1 < U ? u + 1 : u][t][0] : bf[t], first_quarter, from_lane);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int f = 0; f < 4; f++)
#pragma unroll
        for (int t = 0; t < N; t++) acc[f][t] = mma(T{}, av[u][f], bv[u][t], acc[f][t]);
  };
  int s = begin;
  for (; s + kSteps <= end; s += kSteps) some(std::integral_constant<int, kSteps>{}, s);
  if (kSteps > 2 && s + 2 <= end) { some(std::integral_constant<int, 2>{}, s); s += 2; }
  if (s < end) some(std::integral_constant<int, 1>{}, s);
  if (wave == 3 && width % 32) {                                 // the columns behind the last whole step
    const int64_t left = width - steps * 32 - lq * 8;
    int4v av[4], bv[N];
#pragma unroll
    for (int f = 0; f < 4; f++) av[f] = load_up_to(weight_row(f) + steps * 32, left);
#pragma unroll
    for (int t = 0; t < N; t++) bv[t] = load_up_to(token_row(t) + steps * 32, left);
#pragma unroll
    for (int f = 0; f < 4; f++)
#pragma unroll
      for (int t = 0; t < N; t++) acc[f][t] = mma(T{}, av[f], bv[t], acc[f][t]);
  }

#pragma unroll
  for (int turn = 4 / PARTS - 1; turn >= 0; turn--) {            // (the last waves first)
    if (wave / PARTS == turn) {
#pragma unroll
      for (int f = 0; f < 4; f++)
#pragma unroll
        for (int t = 0; t < N; t++) {
          float4v* at = reinterpret_cast<float4v*>(&part[wave % PARTS][t * 16 + l16][f * 16 + lq * 4]);
          *at = PARTS == 4 || turn ? acc[f][t] : acc[f][t] + *at;
        }
    }
    __syncthreads();
  }
  // four threads a token, 16 words each
  const int token = tid >> 2, quarter = tid & 3;
  if (token >= n || token >= 16 * N) return;                     // (whole groups of four)
  float y[16], m = -__builtin_inff(), sum = 0.0f, total = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int c = quarter * 16 + e;
    const int64_t word = word0 + c;
    float z = part[0][token][c] + part[1][token][c];
    if constexpr (PARTS == 4) z += part[2][token][c] + part[3][token][c];
    float add = 0.0f;
    if (word >= r.words) add = -__builtin_inff();
    else if (bias) add = (bias_dtype == TF24_F32 ? ((const float*)bias)[word] : bias_dtype == TF24_F16 ? to_float(((const f16_t*)bias)[word]) : to_float(((const bf16_t*)bias)[word])) * r.scale;
    y[e] = __builtin_fmaf(z, r.scale, add);
    m = fmaxf(m, y[e]);
    if constexpr (SMOOTH) total += word < r.words ? y[e] : 0.0f;
  }
  m = fmaxf(m, __shfl_xor(m, 1));
  m = fmaxf(m, __shfl_xor(m, 2));
  const float from = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    sum += __builtin_amdgcn_exp2f(y[e] - from);
    part[0][token][quarter * 16 + e] = y[e];
  }
  sum += __shfl_xor(sum, 1);
  sum += __shfl_xor(sum, 2);
  if constexpr (SMOOTH) {
    total += __shfl_xor(total, 1);
    total += __shfl_xor(total, 2);
  }
  const int64_t at = (int64_t)blockIdx.x * r.tokens_ld + token;
  if (quarter == 0) {
    r.stats[at] = float2{m, sum};
    if constexpr (SMOOTH) r.sums[at] = total;
  }
  wave_lds_fence();
  if (which.targets) {
    const int64_t c = wanted[token] - word0;
    if (quarter == 0 && c >= 0 && c < kWords) r.picked[token] = part[0][token][c];
  } else {
    const uint32_t listed = r.slab_entries[at];
    const int first = (int)(listed & 0x7ff), many = (int)(listed >> 11 & 0x7ff);
    for (int k = quarter; k < many; k += 4) {
      const int64_t entry = (int64_t)token * r.entries + first + k;
      r.picked[entry] = part[0][token][r.entry_words[entry] - word0];
    }
  }
}

}  // namespace

int launch_few_tokens(int dtype, bool smooth, const FewTokens& which, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t width, const void* bias,
                      int bias_dtype, const HeadResult& r, void* stream) {
  auto go = [&](auto type, auto n) {
    using T = decltype(type);
    auto launch = [&](auto smoothed, auto halves) {
      hipLaunchKernelGGL((few_tokens<T, decltype(n)::value, decltype(smoothed)::value, decltype(halves)::value>), dim3((unsigned)((r.words + kWords - 1) / kWords)), dim3(256), 0, (hipStream_t)stream,
                         (const uint16_t*)x, ldx, (const uint16_t*)w, ldw, width, which, bias, bias_dtype, r);
    };
    const bool halves = ldw % 2 || ldx % 2 || (uintptr_t)w % 4 || (uintptr_t)x % 4;
    if (smooth && halves) launch(std::true_type{}, std::true_type{});
    else if (smooth) launch(std::true_type{}, std::false_type{});
    else if (halves) launch(std::false_type{}, std::true_type{});
    else launch(std::false_type{}, std::false_type{});
  };
  auto sized = [&](auto type) {
    if (which.tokens <= 16) go(type, std::integral_constant<int, 1>{});
    else if (which.tokens <= 32) go(type, std::integral_constant<int, 2>{});
    else if (which.tokens <= 48) go(type, std::integral_constant<int, 3>{});
    else go(type, std::integral_constant<int, 4>{});
  };
  if (dtype == TF24_F16) sized(f16_t{}); else sized(bf16_t{});
  return check_launch("tf24_linear_loss");
}

}  // namespace tf24
