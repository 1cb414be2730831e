// Tiles of the products of a vocabulary head with its loss (linear_loss.hip), 16-bit operands, float32 accumulation:
//
//     C[j, i] = sum_k A(i, k) * B(j, k)
//
//   HEAD_STATS  i: words, j: tokens, k: width      A = W, B = x     per token and slab of 96 words: maximum and sum of exponentials of the logits
//   HEAD_SLOPE  the same product once more, and from it the gradient of the logits, 16-bit, token by token
//   HEAD_INPUT  i: width, j: tokens, k: words      A = W (k is its slow axis), B = the gradient of the logits
//   HEAD_WEIGHT i: width, j: words,  k: tokens     A = x, B = the gradient of the logits (k is the slow axis of both)
//
// A workgroup of four waves (2 x 2, one per SIMD) computes 192(i) x 192(j) tiles, wave tile 96 x 96 = 6 x 6 V_MFMA_F32_16X16X32 with 144 accumulators.
// 64 elements of k of both operands are a stage of 48 KB, three of which rotate through the LDS: while one is multiplied the copies of
// the two behind it are in flight, memory to LDS directly.  A workgroup walks its units (a tile, or a piece of its k) as ONE sequence of stages, so
// that the copies of the next unit run under the end of this one and under what is done with its accumulators.
// The number of tokens that count lies in device memory: no call waits for it.
#pragma once
#include "lds_copies.hpp"
#include <type_traits>

namespace tf24 {
namespace {

constexpr int kTile = 192, kThreads = 256, kWaves = 4, kFrags = 6, kSlab = kTile / 2;
constexpr int kStageK = 64, kRowBytes = kStageK * 2, kStridedRowBytes = kTile * 2;
constexpr int kOperand = kTile * kRowBytes, kStage = 2 * kOperand;          // [A | B]
constexpr int kCopies = kOperand / 1024 / kWaves;                           // 1 KB copies per wave and operand of a stage
constexpr int kRaster = 8;                                                  // tiles along i of a group
constexpr int kSlice = kOperand / kWaves;                                   // a wave's part of a stage's operand: where its own copies go

enum { HEAD_STATS, HEAD_SLOPE, HEAD_INPUT, HEAD_WEIGHT };

}  // namespace

struct HeadProduct {
  const uint8_t *a, *b;
  int64_t lda, ldb;                  // bytes; B's rows (and, k slow, columns) are filled up to whole tiles
  const int* count;                  // tokens that count
  int64_t rows_i, rows_k;            // rows of A; HEAD_INPUT: words, A has none beyond (B holds zeros there)
  int stages, tiles_i, tiles_j, splits;    // upper bounds where the tokens that count decide
};

// What becomes of a tile
struct HeadResult {
  // logits: y = acc * scale + bias (in units of log 2)
  float scale;
  const float* bias;                 // [words, filled up with -inf to whole tiles] or null: none, and whole tiles
  int64_t tokens_ld;                 // tokens, filled up to whole tiles
  // HEAD_STATS
  float2* stats;                     // [slab][token] maximum, sum
  float* sums;                       // SMOOTH: [slab][token] sum of y
  const int* target;                 // [token], or null: the teacher's entries
  float* picked;                     // y of the target [token], of the entries [token][entries]
  const uint32_t* slab_entries;      // [slab][token] first entry of the slab | entries << 11 | column of the first << 22
  const int* entry_words;            // [token][entries] ascending
  int entries;
  // HEAD_SLOPE
  const float2* coef;                // [token] log-sum-exp, factor
  const float* level;                // SMOOTH: [token] what is subtracted everywhere
  void* slope;
  int64_t ld_slope;
  int64_t words;                     // of this piece of the vocabulary
  // HEAD_INPUT, HEAD_WEIGHT
  float* partial;                    // [split][j][ld_out] or null
  const float* out_scale;            // one number
  void* out;                         // [j][ld_out]
  int64_t rows_j, cols_out, ld_out;  // rows and columns that are stored
};

namespace {

// tokens in stages, of a product summed over tokens, and pieces that it is cut into
__device__ __forceinline__ int token_stages(int count) { return max(1, (count + kStageK - 1) / kStageK); }
__device__ __forceinline__ int token_tiles(int count) { return max(1, (count + kTile - 1) / kTile); }

// v * scale as the float32 that it is (one instruction would take it to float16 unrounded, and the float32 result of the same sum another value)
__device__ __forceinline__ float scaled(float v, float scale) {
  v *= scale;
  asm volatile("" : "+v"(v));
  return v;
}

typedef short short8v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float4v mma(f16_t, int4v a, int4v b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float4v mma(bf16_t, int4v a, int4v b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// op over the four lanes l, l + 16, l + 32, l + 48, in each of them: swaps of rows of lanes, where a shuffle would wait for the LDS
template <typename Op>
__device__ __forceinline__ float over_quarters(float v, Op op) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  const uint32_t half = __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(half, half, false, false);
  return op(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

template <typename T, typename OutT, int KIND, bool SMOOTH>
__global__ void __launch_bounds__(kThreads)
head_product(const HeadProduct p, const HeadResult r) {
  constexpr bool A_SLOW = KIND >= HEAD_INPUT, B_SLOW = KIND == HEAD_WEIGHT, LOGITS = KIND <= HEAD_SLOPE;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[3 * kStage];
  const int count = __builtin_amdgcn_readfirstlane(*p.count);
  const int tiles_i = p.tiles_i, tiles_j = B_SLOW ? p.tiles_j : token_tiles(count);
  const int stages_all = B_SLOW ? token_stages(count) : p.stages, splits = min(p.splits, stages_all);
  const int ntiles = tiles_i * tiles_j, nunits = ntiles * splits;
  // workgroup ids are dealt to the 8 XCDs round-robin: each XCD takes a run of units in a raster of groups of kRaster rows of tiles,
  // its workgroup number s the s-th of them and every `slots`-th after it
  const int per_xcd = (nunits + 7) / 8, slots = (int)(gridDim.x >> 3);
  const int xcd = (int)(blockIdx.x & 7), xcd_end = min((xcd + 1) * per_xcd, nunits);
  const int first_unit = xcd * per_xcd + (int)(blockIdx.x >> 3);
  if (first_unit >= xcd_end) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1, l16 = lane & 15, lq = lane >> 4;

  // a unit, its place among those of its piece of k, and (few instructions, which nothing covers) the way to the workgroup's next one
  struct Unit { int number, split, group, in_group; int64_t i0, j0; int begin, stages; };
  auto locate = [&](Unit& u) {
    const int gh = min(kRaster, tiles_i - u.group * kRaster);
    int col = (unsigned)u.in_group / kRaster;
    if (gh != kRaster) col = __builtin_amdgcn_readfirstlane((unsigned)u.in_group / (unsigned)gh);
    u.i0 = (int64_t)(u.group * kRaster + (u.in_group - col * gh)) * kTile;
    u.j0 = (int64_t)col * kTile;
  };
  auto unit_at = [&](int number) {
    Unit u;
    u.number = number;
    u.split = __builtin_amdgcn_readfirstlane((unsigned)number / (unsigned)ntiles);
    const int tile = number - u.split * ntiles;
    u.group = __builtin_amdgcn_readfirstlane((unsigned)tile / (unsigned)(kRaster * tiles_j));
    u.in_group = tile - u.group * (kRaster * tiles_j);
    u.begin = __builtin_amdgcn_readfirstlane((unsigned)(u.split * stages_all) / (unsigned)splits);
    u.stages = __builtin_amdgcn_readfirstlane((unsigned)((u.split + 1) * stages_all) / (unsigned)splits) - u.begin;
    locate(u);
    return u;
  };
  auto advance = [&](Unit& u) {
    u.in_group += slots;
    u.number += slots;
    if (u.in_group < min(kRaster, tiles_i - u.group * kRaster) * tiles_j) locate(u);
    else u = unit_at(u.number);
  };
  Unit now = unit_at(first_unit);
  const int units_here = (xcd_end - first_unit + slots - 1) / slots;

  // ---- copies: number q of a wave brings 1 KB of an operand's stage, 8 rows of 128 bytes with their 16-byte chunks XOR-swizzled by row,
  // or (k slow) 1 KB of 64 rows of 384, swizzled for the transposing reads below.  Rows and columns past A's last re-read it.
  auto slow_swizzle = [](uint32_t krow) { return (((krow >> 1) & 1) << 2) | (((krow >> 3) & 1) << 1); };
  uint32_t oa[kCopies], ob[kCopies];
  auto offset_of = [&](bool slow, int q, uint32_t ld, uint32_t last, uint32_t last_k) {     // last: of the tile's 192 (k slow: its last whole chunk of eight)
    if (slow) {
      const uint32_t piece = (uint32_t)((wave * kCopies + q) * 64 + lane), krow = piece / (kTile / 8);
      return min(krow, last_k) * ld + min(((piece % (kTile / 8)) ^ slow_swizzle(krow)) * 8, last) * 2;
    }
    const uint32_t row = (uint32_t)((wave * kCopies + q) * 8 + (lane >> 3)), chunk = (uint32_t)(lane & 7) ^ ((row >> 1) & 7);
    return min(row, last) * ld + chunk * 16;
  };
  const uint8_t *a_at, *b_at;
  const int64_t a_step = A_SLOW ? kStageK * p.lda : kRowBytes, b_step = B_SLOW ? kStageK * p.ldb : kRowBytes;
  Unit next = now;                                               // whose stages are being copied
  int next_left = 0, units_left = units_here;                    // of its stages, of the units
  int64_t next_k = 0;
  auto point_a = [&]() {
    asm volatile("");                                            // (rarely come by: not to be worked out ahead)
    const uint32_t last = (uint32_t)min((int64_t)kTile, p.rows_i - next.i0) - (A_SLOW ? 8 : 1);
    const uint32_t last_k = KIND == HEAD_INPUT ? (uint32_t)min((int64_t)kStageK, p.rows_k - next_k) - 1 : kStageK - 1;
#pragma unroll
    for (int q = 0; q < kCopies; q++) oa[q] = offset_of(A_SLOW, q, (uint32_t)p.lda, last, last_k);
  };
  bool whole = false;                                            // the offsets in A are those of any tile that lies in it
  auto point_at = [&]() {
    next_k = (int64_t)next.begin * kStageK; next_left = next.stages;
    a_at = p.a + (A_SLOW ? next.i0 * 2 : next.i0 * p.lda) + next.begin * a_step;
    b_at = p.b + (B_SLOW ? next.j0 * 2 : next.j0 * p.ldb) + next.begin * b_step;
    const bool inside = next.i0 + kTile <= p.rows_i && (KIND != HEAD_INPUT || next_k + kStageK <= p.rows_k);
    if (!(inside && whole)) point_a();
    whole = inside;
  };
#pragma unroll
  for (int q = 0; q < kCopies; q++) ob[q] = offset_of(B_SLOW, q, (uint32_t)p.ldb, kTile, kStageK - 1);
  point_at();
  const uint32_t smem_at = lds_offset(smem);
  auto copy_one = [&](int q, uint32_t buf) {                     // the wave's copies of B, then those of A
    if (q < kCopies) g2l16(b_at, ob[q], smem_at + buf + kOperand + (uint32_t)(wave * kCopies + q) * 1024);
    else g2l16(a_at, oa[q - kCopies], smem_at + buf + (uint32_t)(wave * kCopies + q - kCopies) * 1024);
  };
  auto copied = [&]() {                                          // to the next stage, of this unit or of the next
    if (!units_left) return;
    if (--next_left) {
      a_at += a_step; b_at += b_step;
      if constexpr (KIND == HEAD_INPUT) {
        next_k += kStageK;
        if (next_k + kStageK > p.rows_k) { point_a(); whole = false; }       // the last words
      }
    } else if (--units_left) {
      advance(next);
      point_at();
    }
  };
  auto copy_stage = [&](uint32_t buf) {
#pragma unroll
    for (int q = 0; q < 2 * kCopies; q++) copy_one(q, buf);
    copied();
  };

  float4v acc[kFrags][kFrags];

  // ---- fragments of a step (32 elements of k): lane l takes row l % 16, elements 8 * (l / 16) .. + 7.  k slow: in a group of 16 lanes,
  // lane i receives the halfwords i % 4 of the source lanes 4e + i / 4 (e = 0..3), so source lane s addresses k-row s / 4 (of
  // four), columns 4 * (s % 4).. of the group's 16; two such reads make eight elements of k.
  uint32_t a_off[A_SLOW ? kFrags : 2], b_off[B_SLOW ? kFrags : 2];
  auto fragment_offsets = [&](auto is_slow, uint32_t* off, int half) {
    if constexpr (decltype(is_slow)::value) {
      const uint32_t krow = lq * 8 + (l16 >> 2);
#pragma unroll
      for (int f = 0; f < kFrags; f++) {
        const uint32_t col = (uint32_t)(half * kSlab + f * 16) + (l16 & 3) * 4;
        off[f] = krow * kStridedRowBytes + (((col >> 3) ^ slow_swizzle(krow)) * 16) + ((col >> 2) & 1) * 8;
      }
    } else {
#pragma unroll
      for (int step = 0; step < 2; step++) off[step] = (uint32_t)(half * kSlab + l16) * kRowBytes + (uint32_t)((step * 4 + lq) ^ ((l16 >> 1) & 7)) * 16;
    }
  };
  fragment_offsets(std::bool_constant<A_SLOW>{}, a_off, wi);
  fragment_offsets(std::bool_constant<B_SLOW>{}, b_off, wj);
  int4v af[2][kFrags], bf[2][kFrags];                            // [register set][fragment]
  short4v aq[2][kFrags][2], bq[2][kFrags][2];                    // k slow: the halves of a fragment
  constexpr int A_READS = A_SLOW ? 2 * kFrags : kFrags, B_READS = B_SLOW ? 2 * kFrags : kFrags, READS = A_READS + B_READS, MMAS = kFrags * kFrags;
  auto read_slow = [&](const uint8_t* base, uint32_t off, int q, int step) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(lds_ptr_t)(base + off + (step * 32 + (q & 1) * 4) * kStridedRowBytes));
  };
  auto read_a = [&](int set, int q, uint32_t buf, int step) {
    if constexpr (A_SLOW) aq[set][q >> 1][q & 1] = read_slow(smem + buf, a_off[q >> 1], q, step);
    else af[set][q] = *reinterpret_cast<const int4v*>(smem + buf + a_off[step] + q * 16 * kRowBytes);
  };
  auto read_b = [&](int set, int q, uint32_t buf, int step) {
    if constexpr (B_SLOW) bq[set][q >> 1][q & 1] = read_slow(smem + buf + kOperand, b_off[q >> 1], q, step);
    else bf[set][q] = *reinterpret_cast<const int4v*>(smem + buf + kOperand + b_off[step] + q * 16 * kRowBytes);
  };
  // the reads of a step in the order the next step's instructions need them: A's first fragment, B's, A's others
  auto read_one = [&](int set, int n, uint32_t buf, int step) {
    constexpr int FIRST = A_READS / kFrags;
    if (n >= FIRST && n < FIRST + B_READS) read_b(set, n - FIRST, buf, step);
    else read_a(set, n < FIRST ? n : n - B_READS, buf, step);
  };
  auto fragment = [&](auto is_slow, int4v& whole, short4v (&halves)[2]) {
    if constexpr (decltype(is_slow)::value) return __builtin_bit_cast(int4v, __builtin_shufflevector(halves[0], halves[1], 0, 1, 2, 3, 4, 5, 6, 7));
    else return whole;
  };
  // The instructions of a step from one register set; behind them, one by one, the next step's reads into the other set and N copies
  // of a stage.
  auto mma_step = [&](int set, auto copies, uint32_t dst, uint32_t src, int rstep) {
    constexpr int N = decltype(copies)::value;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < MMAS; n++) {
      const int ti = n / kFrags, tj = n % kFrags;
      acc[ti][tj] = mma(T{}, fragment(std::bool_constant<A_SLOW>{}, af[set][ti], aq[set][ti]), fragment(std::bool_constant<B_SLOW>{}, bf[set][tj], bq[set][tj]), acc[ti][tj]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = n * READS / MMAS; q < (n + 1) * READS / MMAS; q++) read_one(set ^ 1, q, src, rstep);
#pragma unroll
      for (int q = 0; q < N; q++)
        if (q * MMAS / (N ? N : 1) == n) copy_one(q, dst);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using C0 = std::integral_constant<int, 0>;
  using CA = std::integral_constant<int, 2 * kCopies>;

  // ---- what is done with a unit's accumulators.  The buffer `fre` is nobody's then; a wave keeps to the two slices of it that its own next copies go to.
  float bias_at[2] = {0, 0};
  float2 coef[kFrags];
  float level[kFrags];
  int target[kFrags];
  uint32_t listed[kFrags];
  auto token_of = [&](int tj) { return now.j0 + wj * kSlab + tj * 16 + l16; };
  auto fetch = [&]() {
    if constexpr (LOGITS) {
      if (r.bias) {
#pragma unroll
        for (int q = 0; q < 2; q++) bias_at[q] = r.bias[now.i0 + wi * kSlab + min(q * 64 + lane, kSlab - 1)];
      }
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) {
        if constexpr (KIND == HEAD_STATS) {
          if (r.target) target[tj] = r.target[token_of(tj)];
          else listed[tj] = r.slab_entries[(now.i0 / kSlab + wi) * r.tokens_ld + token_of(tj)];
        } else {
          coef[tj] = r.coef[token_of(tj)];
          if constexpr (SMOOTH) level[tj] = r.level[token_of(tj)];
        }
      }
    }
  };
  auto chunk_at = [](int row, int ch) { return row * 192 + (ch ^ ((row >> 2) & 3)) * 16; };
  auto finish = [&](uint32_t fre) {
    // (numbers of their own: what is worked out from them, addresses above all, would be kept in registers through the loop over the stages otherwise)
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int l16 = lane & 15, lq = lane >> 4;
    auto token_of = [&](int tj) { return now.j0 + wj * kSlab + tj * 16 + l16; };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // the copies in flight: from here on stores count as well
    uint8_t* slice = smem + fre + wave * kSlice;
    float* bias_lds = reinterpret_cast<float*>(smem + fre + kOperand + wave * kSlice);
    if constexpr (LOGITS) {
#pragma unroll
      for (int q = 0; q < 2; q++)
        if (q * 64 + lane < kSlab) bias_lds[q * 64 + lane] = bias_at[q];
      wave_lds_fence();
    }
    auto bias_of = [&](int ti) { return *reinterpret_cast<const float4v*>(bias_lds + ti * 16 + lq * 4); };
    if constexpr (KIND == HEAD_STATS) {
      const int64_t slab = now.i0 / kSlab + wi;
      const int base = (int)(slab * kSlab);
      // (the accumulators are read once: vector instructions reach them through copies alone)
      float4v y[kFrags][kFrags];
      float m[kFrags], t[kFrags], s[kFrags], sum[kFrags];
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) { m[tj] = -__builtin_inff(); s[tj] = 0.0f; sum[tj] = 0.0f; }
#pragma unroll
      for (int ti = 0; ti < kFrags; ti++) {
        const float4v add = bias_of(ti);
#pragma unroll
        for (int tj = 0; tj < kFrags; tj++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            y[ti][tj][e] = __builtin_fmaf(acc[ti][tj][e], r.scale, add[e]);
            if constexpr (SMOOTH) sum[tj] += base + ti * 16 + lq * 4 + e < r.words ? y[ti][tj][e] : 0.0f;
          }
          m[tj] = fmaxf(fmaxf(m[tj], y[ti][tj][0]), y[ti][tj][1]);
          m[tj] = fmaxf(fmaxf(m[tj], y[ti][tj][2]), y[ti][tj][3]);
        }
      }
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) {
        m[tj] = over_quarters(m[tj], [](float a, float b) { return fmaxf(a, b); });
        t[tj] = m[tj] == -__builtin_inff() ? 0.0f : m[tj];
      }
#pragma unroll
      for (int ti = 0; ti < kFrags; ti++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
          for (int tj = 0; tj < kFrags; tj++) s[tj] += __builtin_amdgcn_exp2f(y[ti][tj][e] - t[tj]);
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) {
        s[tj] = over_quarters(s[tj], [](float a, float b) { return a + b; });
        if constexpr (SMOOTH) sum[tj] = over_quarters(sum[tj], [](float a, float b) { return a + b; });
        const int64_t token = token_of(tj);
        if (lq == 0) {
          r.stats[slab * r.tokens_ld + token] = float2{m[tj], s[tj]};
          if constexpr (SMOOTH) r.sums[slab * r.tokens_ld + token] = sum[tj];
        }
      }
      if (r.target) {
#pragma unroll
        for (int tj = 0; tj < kFrags; tj++) {
          const int at = target[tj] - base;
          if (__any(at >= 0 && at < kSlab)) {
#pragma unroll
            for (int ti = 0; ti < kFrags; ti++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (at == ti * 16 + lq * 4 + e) r.picked[token_of(tj)] = y[ti][tj][e];
          }
        }
      } else {
        // the teacher's entries of these 96 words, four of a token at a time, from the token's row in LDS
#pragma unroll
        for (int tj = 0; tj < kFrags; tj++) {
          const int many = (int)(listed[tj] >> 11 & 0x7ff), first = (int)(listed[tj] & 0x7ff);
          if (__any(many > 0)) {
            wave_lds_fence();
#pragma unroll
            for (int ti = 0; ti < kFrags; ti++)
              *reinterpret_cast<float4v*>(slice + l16 * 384 + ((ti * 4 + lq) ^ ((l16 >> 1) & 7)) * 16) = y[ti][tj];
            wave_lds_fence();
            for (int n = lq; n < many; n += 4) {
              const int64_t entry = token_of(tj) * r.entries + first + n;
              const int at = n ? r.entry_words[entry] - base : (int)(listed[tj] >> 22);
              r.picked[entry] = *reinterpret_cast<const float*>(slice + l16 * 384 + ((at >> 2) ^ ((l16 >> 1) & 7)) * 16 + (at & 3) * 4);
            }
          }
        }
      }
    } else if constexpr (KIND == HEAD_SLOPE) {
      // 32(j) x 96(i) pieces through the slice (rows of 192 bytes, chunks XOR-swizzled with the row), whole rows of them stored
#pragma unroll
      for (int tp = 0; tp < kFrags / 2; tp++) {
        if (tp > 0) wave_lds_fence();
#pragma unroll
        for (int ti = 0; ti < kFrags; ti++) {
          const float4v add = bias_of(ti);
#pragma unroll
          for (int t2 = 0; t2 < 2; t2++) {
            const int tj = tp * 2 + t2;
            T o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float v = coef[tj].y * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[ti][tj][e], r.scale, add[e]) - coef[tj].x);
              if constexpr (SMOOTH) v = now.i0 + wi * kSlab + ti * 16 + lq * 4 + e < r.words ? v - level[tj] : 0.0f;
              o[e] = from_float<T>(v);
            }
            *reinterpret_cast<Pack<T, 4>*>(slice + chunk_at(t2 * 16 + l16, ti * 2 + (lq >> 1)) + (lq & 1) * 8) = *reinterpret_cast<Pack<T, 4>*>(o);
          }
        }
        wave_lds_fence();
#pragma unroll
        for (int it = 0; it < 6; it++) {
          const uint32_t piece = it * 64 + lane;
          const int jl = piece / 12, ch = piece % 12;
          const int4v v = *reinterpret_cast<const int4v*>(slice + chunk_at(jl, ch));
          *reinterpret_cast<int4v*>((T*)r.slope + (now.j0 + wj * kSlab + tp * 32 + jl) * r.ld_slope + now.i0 + wi * kSlab + ch * 8) = v;
        }
      }
    } else if (r.partial) {
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) {
        const int64_t row = now.j0 + wj * kSlab + tj * 16 + l16;
        float* at = r.partial + ((int64_t)now.split * r.rows_j + row) * r.ld_out;
        if (row < r.rows_j) {
#pragma unroll
          for (int ti = 0; ti < kFrags; ti++) {
            const int64_t col = now.i0 + wi * kSlab + ti * 16 + lq * 4;
            if (col < r.ld_out) *reinterpret_cast<float4v*>(at + col) = acc[ti][tj];
          }
        }
      }
    } else {
      const float scale = *r.out_scale;
      if constexpr (std::is_same<OutT, float>::value) {
        const bool whole = r.ld_out % 4 == 0 && ((uintptr_t)r.out & 15) == 0;
#pragma unroll
        for (int tj = 0; tj < kFrags; tj++) {
          const int64_t row = now.j0 + wj * kSlab + tj * 16 + l16;
#pragma unroll
          for (int ti = 0; ti < kFrags; ti++) {
            const int64_t col = now.i0 + wi * kSlab + ti * 16 + lq * 4;
            float* at = (float*)r.out + row * r.ld_out + col;
            const float4v v = acc[ti][tj] * scale;
            if (row < r.rows_j) {
              if (whole && col + 4 <= r.cols_out) *reinterpret_cast<float4v*>(at) = v;
              else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                  if (col + e < r.cols_out) at[e] = v[e];
              }
            }
          }
        }
      } else {
        const bool whole = r.ld_out % 8 == 0 && ((uintptr_t)r.out & 15) == 0;
#pragma unroll
        for (int tp = 0; tp < kFrags / 2; tp++) {
          if (tp > 0) wave_lds_fence();
#pragma unroll
          for (int ti = 0; ti < kFrags; ti++)
#pragma unroll
            for (int t2 = 0; t2 < 2; t2++) {
              T o[4];
#pragma unroll
              for (int e = 0; e < 4; e++) o[e] = from_float<T>(scaled(acc[ti][tp * 2 + t2][e], scale));
              *reinterpret_cast<Pack<T, 4>*>(slice + chunk_at(t2 * 16 + l16, ti * 2 + (lq >> 1)) + (lq & 1) * 8) = *reinterpret_cast<Pack<T, 4>*>(o);
            }
          wave_lds_fence();
#pragma unroll
          for (int it = 0; it < 6; it++) {
            const uint32_t piece = it * 64 + lane;
            const int jl = piece / 12, ch = piece % 12;
            const int64_t col = now.i0 + wi * kSlab + ch * 8, row = now.j0 + wj * kSlab + tp * 32 + jl;
            const int4v v = *reinterpret_cast<const int4v*>(slice + chunk_at(jl, ch));
            if (row < r.rows_j && col < r.cols_out) {
              T* at = (T*)r.out + row * r.ld_out + col;
              if (whole && col + 8 <= r.cols_out) __builtin_nontemporal_store(v, reinterpret_cast<int4v*>(at));
              else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                  if (col + e < r.cols_out) at[e] = T{(uint16_t)((uint32_t)v[e >> 1] >> (e & 1) * 16)};
              }
            }
          }
        }
      }
    }
    wave_lds_fence();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the next copies go over what was read
  };

  // ---- the sequence of stages.  Behind its end the copies go on from the last place (two stages that nobody reads): nothing in the loop
  // depends on where the sequence ends.
  uint32_t cur = 0, nxt = kStage, fre = 2 * kStage;              // buffers of this stage, the next and the one behind (= the one before)
  copy_stage(cur);
  copy_stage(nxt);
  wait_copies_and_barrier<2 * kCopies, true>();
#pragma unroll
  for (int n = 0; n < READS; n++) read_one(0, n, cur, 0);
  bool landed = false;                                           // the next stage has arrived already
  for (int units = units_here;;) {
    fetch();
#pragma unroll
    for (int ti = 0; ti < kFrags; ti++)
#pragma unroll
      for (int tj = 0; tj < kFrags; tj++) acc[ti][tj] = float4v{0, 0, 0, 0};
    int left = now.stages;
    do {
      mma_step(0, CA{}, fre, cur, 1);                            // with the copies of the stage behind the next one
      copied();
      if (landed) wait_reads_and_barrier();
      else wait_copies_and_barrier<2 * kCopies, true>();
      landed = false;
      const uint32_t t = cur; cur = nxt; nxt = fre; fre = t;
      mma_step(1, C0{}, 0, cur, 0);
    } while (--left);
    finish(fre);
    if (!--units) break;
    landed = true;
    advance(now);
  }
}

}  // namespace
}  // namespace tf24
