// The logits of few tokens (up to 64) against a whole vocabulary, and what linear_loss.hip wants of them: per token and slab of 64 words a maximum and a sum of
// exponentials, and the logits of the listed words.
//
// Bound by memory: the weight is read once, straight into registers, and as it lies, whatever its rows' alignment (a copy of it in whole aligned stages, as the
// tiles want it, costs three times the reading).  A workgroup takes 64 words; its four waves share the width out among them, 32 columns a step, so that
// 16 waves and more of a compute unit have loads in flight, and add up their products through the LDS.  The tokens' rows come from the caches.
// One token, 50304 x 768 bf16 (77 MB): 18 us, 4.3 TB/s; 16 tokens, 128000 x 4096 (1 GB): 185 us, 5.7 TB/s; 37 tokens, 50257 x 1601 float16, every other row in the middle of a
// dword: 58 us, 2.8 TB/s, bound by what moves the tokens' and the weight's columns into place (one token: 43 us).
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

// A step's 64 bytes of a row, 16 to each of the four lanes that share it.  What a load costs is the blocks of 64 bytes that it touches: rows that do not start at one
// are loaded block by block, each once (16 bytes from wherever they start: 16 tokens, 50257 x 1601 62 us for 50, 37 tokens x 4097 195 for 151; two whole pieces of
// 16 bytes for each: 139), and a step is put together from two of them: dword j of a lane's 16 bytes is dword j + `turn` of a
// block that lies `quarters` (or one more) lanes further on, in the same block or in the next.  In the end halves of dwords are moved.
template <bool MOVED>
struct Row {
  const uint8_t* at;                                             // the lane's 16 bytes of the first block
  uint32_t turn, half;
  int quarters, last;                                            // last: block that the row's part has something in
  __device__ __forceinline__ Row(const uint16_t* p, int lq, int end) {
    const uint32_t off = MOVED ? (uint32_t)(uintptr_t)p & 63 : 0;
    at = (const uint8_t*)p - off + lq * 16;
    turn = off >> 2 & 3; half = (off & 2) * 8; quarters = (int)(off >> 4);
    last = off ? end : end - 1;
  }
  __device__ __forceinline__ int4v load(int step) const { return *reinterpret_cast<const int4v*>(at + step * 64); }
  __device__ __forceinline__ int4v block(int step) const { return load(min(step, last)); }
  __device__ __forceinline__ int4v turned(int4v v) const {
    const int4v t = {turn & 2 ? v[2] : v[0], turn & 2 ? v[3] : v[1], turn & 2 ? v[0] : v[2], turn & 2 ? v[1] : v[3]};
    return int4v{turn & 1 ? t[1] : t[0], turn & 1 ? t[2] : t[1], turn & 1 ? t[3] : t[2], turn & 1 ? t[0] : t[3]};
  }
  __device__ __forceinline__ int4v joined(int4v now, int4v next, int lq, int l16) const {      // both turned
    uint32_t d[5];
#pragma unroll
    for (int j = 0; j < 5; j++) {
      const int on = quarters + (j + (int)turn >= 4 ? 1 : 0);
      d[j] = (uint32_t)__builtin_amdgcn_ds_bpermute((((lq + on) & 3) * 16 + l16) * 4, lq >= on ? now[j & 3] : next[j & 3]);
    }
    int4v o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (int)__builtin_amdgcn_alignbit(d[i + 1], d[i], half);
    return o;
  }
};

// N: fragments of 16 tokens.  MOVED: rows do not all start at 16 bytes (where they do, but not at 64, the moving costs more than it saves: 16 tokens, 50304 x 776 31
// us, moved 38).
// kSteps: steps whose loads are in flight at once.  Two, and registers for two workgroups of a compute unit at least, against four: 16 tokens, 128000 x 4096 196 us
// (so without the bound on registers; with it 225) and 238, 48 tokens 236 and 266.  Where steps are moved, which takes registers of its own, one against two: 37
// tokens, 50257 x 1601 62 and 81, 64 tokens 72 and 93, and with the bound 68 and 63, 73 and 92.
template <typename T, int N, bool SMOOTH, bool MOVED>
__global__ void __launch_bounds__(256, MOVED || N == 1 ? 1 : 2)
few_tokens(const uint16_t* __restrict__ x, int64_t ldx, const uint16_t* __restrict__ w, int64_t ldw, int64_t width, const FewTokens which,
           const void* __restrict__ bias, int bias_dtype, const HeadResult r) {
  constexpr int STRIDE = kWords + 4;                             // floats of a token: 16 tokens start 16 bytes apart
  constexpr int kSteps = MOVED ? 1 : 2;
  // the parts of a sum that two waves have, to which the others add theirs (parts of all four: fewer workgroups; 48 tokens, 50304 x 768 33 us for 31)
  __shared__ __attribute__((aligned(16))) float part[2][16 * N][STRIDE];
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
  const int steps = (int)(width / 32), begin = wave * steps / 4, end = (wave + 1) * steps / 4;
  auto weight_row = [&](int f) { return w + min(word0 + f * 16 + l16, r.words - 1) * ldw; };
  auto token_row = [&](int t) { return x + (int64_t)rows[t * 16 + l16 < n ? t * 16 + l16 : 0] * ldx; };    // (columns of tokens behind the last are not used)
  const Row<MOVED> a[4] = {Row<MOVED>(weight_row(0), lq, end), Row<MOVED>(weight_row(1), lq, end), Row<MOVED>(weight_row(2), lq, end), Row<MOVED>(weight_row(3), lq, end)};
  const Row<MOVED> b[4] = {Row<MOVED>(token_row(0), lq, end), Row<MOVED>(token_row(N > 1 ? 1 : 0), lq, end), Row<MOVED>(token_row(N > 2 ? 2 : 0), lq, end), Row<MOVED>(token_row(N > 3 ? 3 : 0), lq, end)};
  float4v acc[4][N];
#pragma unroll
  for (int f = 0; f < 4; f++)
#pragma unroll
    for (int t = 0; t < N; t++) acc[f][t] = float4v{0, 0, 0, 0};
  int4v a0[4], b0[N];                                            // MOVED: the blocks that the steps from here on begin in
  if (MOVED && begin < end) {
#pragma unroll
    for (int f = 0; f < 4; f++) a0[f] = a[f].turned(a[f].load(begin));
#pragma unroll
    for (int t = 0; t < N; t++) b0[t] = b[t].turned(b[t].load(begin));
  }
  auto some = [&](auto many, int s) {                            // so many steps
    constexpr int U = decltype(many)::value;
    int4v av[U][4], bv[U][N];
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
      for (int f = 0; f < 4; f++) av[u][f] = MOVED ? a[f].block(s + u + 1) : a[f].load(s + u);
#pragma unroll
      for (int t = 0; t < N; t++) bv[u][t] = MOVED ? b[t].block(s + u + 1) : b[t].load(s + u);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if constexpr (MOVED) {
        auto move = [&](const Row<MOVED>& row, int4v& before, int4v& v) {
          const int4v next = row.turned(v);
          v = row.joined(before, next, lq, l16);
          before = next;
        };
#pragma unroll
        for (int f = 0; f < 4; f++) move(a[f], a0[f], av[u][f]);
#pragma unroll
        for (int t = 0; t < N; t++) move(b[t], b0[t], bv[u][t]);
      }
#pragma unroll
      for (int f = 0; f < 4; f++)
#pragma unroll
        for (int t = 0; t < N; t++) acc[f][t] = mma(T{}, av[u][f], bv[u][t], acc[f][t]);
    }
  };
  int s = begin;
  for (; s + kSteps <= end; s += kSteps) some(std::integral_constant<int, kSteps>{}, s);
  if (kSteps > 1 && s < end) some(std::integral_constant<int, 1>{}, s);
  if (wave == 3 && width % 32) {                                 // the columns behind the last whole step
    const int64_t left = width - steps * 32 - lq * 8;
    int4v av[4], bv[N];
#pragma unroll
    for (int f = 0; f < 4; f++) av[f] = load_up_to(weight_row(f) + steps * 32 + lq * 8, left);
#pragma unroll
    for (int t = 0; t < N; t++) bv[t] = load_up_to(token_row(t) + steps * 32 + lq * 8, left);
#pragma unroll
    for (int f = 0; f < 4; f++)
#pragma unroll
      for (int t = 0; t < N; t++) acc[f][t] = mma(T{}, av[f], bv[t], acc[f][t]);
  }

#pragma unroll
  for (int first = 2; first >= 0; first -= 2) {
    if (wave - first == 0 || wave - first == 1) {
#pragma unroll
      for (int f = 0; f < 4; f++)
#pragma unroll
        for (int t = 0; t < N; t++) {
          float4v* at = reinterpret_cast<float4v*>(&part[wave - first][t * 16 + l16][f * 16 + lq * 4]);
          *at = first ? acc[f][t] : acc[f][t] + *at;
        }
    }
    __syncthreads();
  }
  // four threads a token, 16 words each
  const int token = tid >> 2, quarter = tid & 3;
  if (token >= n) return;                                        // (whole groups of four; n is 16 * N at most)
  float y[16], m = -__builtin_inff(), sum = 0.0f, total = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int c = quarter * 16 + e;
    const int64_t word = word0 + c;
    const float z = part[0][token][c] + part[1][token][c];
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
    auto launch = [&](auto smoothed, auto moved) {
      hipLaunchKernelGGL((few_tokens<T, decltype(n)::value, decltype(smoothed)::value, decltype(moved)::value>), dim3((unsigned)((r.words + kWords - 1) / kWords)), dim3(256), 0, (hipStream_t)stream,
                         (const uint16_t*)x, ldx, (const uint16_t*)w, ldw, width, which, bias, bias_dtype, r);
    };
    const bool moved = ldw % 8 || ldx % 8 || (uintptr_t)w % 16 || (uintptr_t)x % 16;
    if (smooth && moved) launch(std::true_type{}, std::true_type{});
    else if (smooth) launch(std::true_type{}, std::false_type{});
    else if (moved) launch(std::false_type{}, std::true_type{});
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
