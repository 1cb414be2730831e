// Tiles of the products of a vocabulary head with its loss (linear_loss.hip), 16-bit operands, float32 accumulation:
//
//     C[j, i] = sum_k A(i, k) * B(j, k)
//
//   HEAD_STATS  i: words, j: tokens, k: width      A = W, B = x     per token and slab of words (half a tile): maximum and sum of exponentials of the logits
//   HEAD_SLOPE  the same product once more, and from it the gradient of the logits, 16-bit, token by token
//   HEAD_INPUT  i: width, j: tokens, k: words      A = W (k is its slow axis), B = the gradient of the logits
//   HEAD_WEIGHT i: width, j: words,  k: tokens     A = x, B = the gradient of the logits (k is the slow axis of both)
//
// A workgroup of four waves (2 x 2, one per SIMD) computes 256 x 256 tiles, a wave a quarter of it: 8 x 8 V_MFMA_F32_16X16X32 with 256
// accumulators.  32 elements of k of both operands are a stage of 32 KB, four of which rotate through the LDS: while one is
// multiplied, from registers, its successor is read and the copies of the ones behind are in flight, memory to LDS directly.  A workgroup walks its units (a
// tile, or a piece of its k) as ONE sequence of stages, so that the copies of the next unit run under the end of this one and under what is done
// with its accumulators; for that there is an LDS area apart, to which what a tile needs of its tokens and words is copied as well.
// The number of tokens that count lies in device memory: no call waits for it.
//
// Bound by the matrix units and the power they draw: at 8192 tokens, 128000 x 4096 bf16 they are busy for 74, 69, 64 and 70 % of the cycles of the four products at
// 1.93 GHz (6.4, 6.7, 6.7 and 6.3 ms; 1.34, 1.28, 1.28 and 1.36 PFLOP/s; a library's product of the same sizes with nothing of a loss in it 5.9, 6.3 for dx, 7.4 for dW).
// Short ones by what stands between the tiles, a quarter of STATS and SLOPE at a width of 768: 12288 tokens, 50304 x 768 0.94, 0.93, 0.82 + 0.05 and 0.70 + 0.02 ms
// (1.01 to 1.35 PFLOP/s; the library 0.85, 1.33 for dx, 0.99 for dW).
// Registers: the accumulators leave 256 of a lane's 512.  The compiler keeps 4 to 9 more in memory for STATS and SLOPE (20 to 40 bytes a lane), 57 to 65 for INPUT and WEIGHT (172 to
// 200): none in the loop over the stages, all where a unit begins and ends.  A reload there waits for the copies ahead of it, which is part of what stands between the tiles.
// 256 x 256 tiles against 192 x 192, both passes: 8192 tokens, 128000 x 4096 26.5 and 30.6 ms; 8192 tokens, 50304 x 1024 2.93 and 3.33; 1024 tokens, 50304 x 768 0.42
// and 0.39 (788 tiles are 3.1 rounds on 256 compute units).  Two buffers of 64 elements of k against four
// of 32: the forward pass of the first 6.9 and 6.4 ms.
#pragma once
#include "lds_copies.hpp"
#include <algorithm>
#include <type_traits>

namespace tf24 {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int F = 8, kTile = 32 * F, kSlab = kTile / 2;                      // fragments of 16 along a side of a wave's quarter, a tile's side, the quarter's
constexpr int kUnitK = 64, kStageK = 32;                                    // k is a multiple of kUnitK: two stages
constexpr int kRowBytes = kStageK * 2, kSlowRowBytes = kTile * 2, kOperand = kTile * kRowBytes, kStage = 2 * kOperand, kRing = 4;
constexpr int kCopies = kOperand / 1024 / kWaves;                           // 1 KB copies per wave and operand of a stage
constexpr int kOverread = 1024;                                             // what is copied for a tile's tokens or words is 1 KB of each kind
constexpr int kRaster = 8;                                                  // tiles along i of a group
// a wave's own LDS: 4 KB of results (8 of logits), then 1 KB each of what the tile's columns bring and what its rows do
constexpr int kLds = 160 * 1024, kScratch = (kLds - kRing * kStage) / kWaves, kColumnsAt = 4096, kTokensAt = 5120, kLevelAt = 6144;
static_assert(kCopies * 1024 * kWaves == kOperand && kScratch >= kLevelAt + 1024 && kScratch >= 16 * kSlab * 4, "a stage's copies divide among the waves");

// 16-byte chunks of a row of 64 bytes are XOR-swizzled for reads of 16 bytes a lane, which go by lanes 0-3, 12-15, 20-23 and 24-27, then the
// other 16 of the first 32, and so on: each such group touches every bank once ((row >> 2) & 3, which suits 16 lanes in a row, took twice the cycles)
__device__ __forceinline__ uint32_t swizzle(uint32_t row) { return (0u - (row >> 2)) & 3; }
// those of a k-row so that transposing reads do
__device__ __forceinline__ uint32_t slow_swizzle(uint32_t krow) { return ((krow & 3) << 2) | (((krow >> 3) & 1) << 1); }

enum { HEAD_STATS, HEAD_SLOPE, HEAD_INPUT, HEAD_WEIGHT };

}  // namespace

struct HeadProduct {
  const uint8_t *a, *b;
  int64_t lda, ldb;                  // bytes; B's rows (and, k slow, columns) are filled up to whole tiles
  const int* count;                  // tokens that count
  int64_t rows_i, rows_k;            // rows of A; HEAD_INPUT: words, A has none beyond (B holds zeros there)
  int stages, tiles_i, tiles_j;      // stages of kUnitK; upper bounds where the tokens that count decide
  int groups, most;                  // HEAD_INPUT, HEAD_WEIGHT: workgroups, and tiles' pieces that there is room for
};

// What becomes of a tile
struct HeadResult {
  // logits: y = acc * scale + bias (in units of log 2)
  float scale;
  const float* bias;                 // [words, filled up with -inf to whole tiles] or null: none
  int64_t tokens_ld;                 // tokens, filled up to whole tiles
  int64_t words;                     // of the vocabulary, or this piece of it
  // HEAD_STATS
  float2* stats;                     // [slab][token] maximum, sum
  float* sums;                       // SMOOTH: [slab][token] sum of y
  const int* target;                 // [token], or null: the teacher's entries
  float* picked;                     // y of the target [token], of the entries [token][entries]
  const uint32_t* slab_entries;      // [slab][token] first entry of the slab | entries << 11
  const int* entry_words;            // [token][entries] ascending
  int entries;
  // HEAD_SLOPE
  const float2* coef;                // [token] log-sum-exp, factor
  const float* level;                // SMOOTH: [token] what is subtracted everywhere, a number of 16 bits
  void* slope;
  int64_t ld_slope;
  // HEAD_INPUT, HEAD_WEIGHT
  const float* common;               // SMOOTH: [column, filled up to whole tiles with anything] what is subtracted from every row
  const float* level_rest;           // INPUT, SMOOTH: so many times [token]
  float* partial;                    // [piece][tile of the rest][kTile^2], as the accumulators lie
  float* sum;                        // [tile][kTile^2]: what the pieces of the vocabulary before this one gave (add), and where it goes on (not last)
  bool add, last;
  const float* out_scale;            // one number
  void* out;                         // [row][cols_out]: row row_of[j], or j
  const int* row_of;
  int64_t rows_j, cols_out;          // WEIGHT: rows; columns that are stored
};

namespace {

// eight 16-bit elements from anywhere (one load of 16 bytes, whatever the alignment)
struct __attribute__((packed, aligned(2))) Unaligned8 { int4v v; };
__device__ __forceinline__ int4v load8(const uint16_t* p) { return reinterpret_cast<const Unaligned8*>(p)->v; }

__device__ __forceinline__ int token_stages(int count) { return max(1, (count + kUnitK - 1) / kUnitK); }
__device__ __forceinline__ int token_tiles(int count) { return max(1, (count + kTile - 1) / kTile); }

// How the tiles of a product with a long k go to `groups` workgroups: as many as fill whole rounds each in one piece, the rest cut along k into as many pieces as
// cost least, in stages of kUnitK: rounds x stages of a piece, and for each piece of a tile 0.09 of one (256 KB written and read again), 4 for the pass that joins
// them.  With pieces and without, both passes: 1024 tokens, 50304 x 768 (12 and 591 tiles) 0.42 and 1.36 ms; 12288 tokens 3.53 and 3.89 ms; 8192 tokens, 128000 x 4096
// 26.5 and 26.8.
struct Share { int whole, rest, pieces; };
__host__ __device__ inline Share share_out(int tiles, int stages, int groups, int most) {
  Share s{tiles / groups * groups, tiles % groups, 1};
  int least = stages * 256;
  for (int rounds = 1; rounds <= 4 && s.rest; rounds++) {        // (of the numbers of pieces that fit into so many rounds the largest)
    const int p = min(min(rounds * groups / s.rest, stages), most / s.rest);
    const int cost = p > 1 ? (rounds * ((stages + p - 1) / p) + 4) * 256 + s.rest * p * 23 : least;
    if (cost < least) { least = cost; s.pieces = p; }
  }
  return s;
}

// v * scale as the float32 that it is (one instruction would take it to float16 unrounded, and the float32 result of the same sum another value)
__device__ __forceinline__ float scaled(float v, float scale) {
  v *= scale;
  asm volatile("" : "+v"(v));
  return v;
}

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
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kLds];
  const int count = __builtin_amdgcn_readfirstlane(*p.count);
  const int tiles_i = p.tiles_i, tiles_j = B_SLOW ? p.tiles_j : token_tiles(count), ntiles = tiles_i * tiles_j;
  const int stages_all = B_SLOW ? token_stages(count) : p.stages;
  // units: whole tiles (LOGITS: none, all of them are the rest, in one piece), then the pieces of the rest
  const Share share = LOGITS ? Share{0, ntiles, 1} : share_out(ntiles, stages_all, p.groups, p.most);
  const int whole = __builtin_amdgcn_readfirstlane(share.whole), rest = __builtin_amdgcn_readfirstlane(share.rest), pieces = __builtin_amdgcn_readfirstlane(share.pieces);
  // workgroup ids are dealt to the 8 XCDs round-robin: each XCD takes a run of either kind of units, in a raster of groups of kRaster rows of tiles,
  // its workgroup number s the s-th of them and every `slots`-th after it
  const int slots = (int)(gridDim.x >> 3), xcd = (int)(blockIdx.x & 7), slot = (int)(blockIdx.x >> 3);
  const int rounds = LOGITS ? 0 : __builtin_amdgcn_readfirstlane((unsigned)whole / (unsigned)(8 * slots));
  const int run = (rest * pieces + 7) / 8, first = xcd * run + slot, end = min((xcd + 1) * run, rest * pieces);
  const int units_here = rounds + (first < end ? (end - first + slots - 1) / slots : 0);
  if (!units_here) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave >> 1, wj = wave & 1, l16 = lane & 15, lq = lane >> 4;

  // The workgroup's m-th unit, its place in its group, and (few instructions, which nothing covers) the way to the next one
  struct Unit { int m, tile, piece, group, in_group; int64_t i0, j0; int begin, stages; };
  auto locate = [&](Unit& u) {
    const int gh = min(kRaster, tiles_i - u.group * kRaster);
    int col = (unsigned)u.in_group / kRaster;
    if (gh != kRaster) col = __builtin_amdgcn_readfirstlane((unsigned)u.in_group / (unsigned)gh);
    int row = u.in_group - col * gh;
    // (a workgroup's tiles go round the rows: most of the words that a teacher lists are the frequent ones, in the first row of tiles; 12288 tokens of 64 entries,
    // forward pass 1.045 ms, as they come 1.076)
    if (LOGITS && gh == kRaster) row = (row + col) % kRaster;
    u.i0 = (int64_t)(u.group * kRaster + row) * kTile;
    u.j0 = (int64_t)col * kTile;
  };
  auto unit_at = [&](int m) {
    Unit u;
    u.m = m; u.piece = 0; u.begin = 0; u.stages = stages_all;
    if (m < rounds) u.tile = xcd * (whole >> 3) + slot + m * slots;
    else {
      const int number = first + (m - rounds) * slots;
      u.tile = whole + number;
      if (!LOGITS && pieces > 1) {
        u.piece = __builtin_amdgcn_readfirstlane((unsigned)number / (unsigned)rest);
        u.tile = whole + number - u.piece * rest;
        u.begin = __builtin_amdgcn_readfirstlane((unsigned)(u.piece * stages_all) / (unsigned)pieces);
        u.stages = __builtin_amdgcn_readfirstlane((unsigned)((u.piece + 1) * stages_all) / (unsigned)pieces) - u.begin;
      }
    }
    u.group = __builtin_amdgcn_readfirstlane((unsigned)u.tile / (unsigned)(kRaster * tiles_j));
    u.in_group = u.tile - u.group * (kRaster * tiles_j);
    locate(u);
    return u;
  };
  auto advance = [&](Unit& u) {
    if (LOGITS && u.in_group + slots < min(kRaster, tiles_i - u.group * kRaster) * tiles_j) {
      u.m++;
      u.in_group += slots;
      locate(u);
    } else u = unit_at(u.m + 1);
  };
  Unit now = unit_at(0);

  // ---- copies: number q of a wave brings 1 KB of an operand's stage, 16 rows of 64 bytes with their 16-byte chunks XOR-swizzled by row,
  // or (k slow) 1 KB of 32 rows of the tile's columns, swizzled for the transposing reads below.  Rows and columns past A's last re-read it.
  uint32_t oa[kCopies], ob[kCopies];
  auto offset_of = [&](bool slow, int q, uint32_t ld, uint32_t last, uint32_t last_k) {     // last: of the tile's (k slow: its last whole chunk of eight)
    if (slow) {
      const uint32_t piece = (uint32_t)((wave * kCopies + q) * 64 + lane), krow = piece / (kTile / 8);
      return min(krow, last_k) * ld + min(((piece % (kTile / 8)) ^ slow_swizzle(krow)) * 8, last) * 2;
    }
    const uint32_t row = (uint32_t)((wave * kCopies + q) * 16 + (lane >> 2)), chunk = (uint32_t)(lane & 3) ^ swizzle(row);
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
  bool inner = false;                                            // the offsets in A are those of any tile that lies in it
  auto point_at = [&]() {
    next_k = (int64_t)next.begin * kUnitK; next_left = next.stages * 2;
    a_at = p.a + (A_SLOW ? next.i0 * 2 : next.i0 * p.lda) + next.begin * 2 * a_step;
    b_at = p.b + (B_SLOW ? next.j0 * 2 : next.j0 * p.ldb) + next.begin * 2 * b_step;
    const bool inside = next.i0 + kTile <= p.rows_i && (KIND != HEAD_INPUT || next_k + kStageK <= p.rows_k);
    if (!(inside && inner)) point_a();
    inner = inside;
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
      b_at += b_step;
      if constexpr (KIND == HEAD_INPUT) {
        next_k += kStageK;
        if (next_k < p.rows_k) {                                 // (behind the last word B holds zeros, whatever they meet)
          a_at += a_step;
          if (next_k + kStageK > p.rows_k) { point_a(); inner = false; }     // the last words
        }
      } else a_at += a_step;
    } else if (--units_left) {
      advance(next);
      point_at();
    }
  };

  // ---- fragments of a stage: lane l takes row l % 16, elements 8 * (l / 16) .. + 7.  k slow: in a group of 16 lanes,
  // lane i receives the halfwords i % 4 of the source lanes 4e + i / 4 (e = 0..3), so source lane s addresses k-row s / 4 (of
  // four), columns 4 * (s % 4).. of the group's 16; two such reads make eight elements of k.
  uint32_t a_off[A_SLOW ? F : 1], b_off[B_SLOW ? F : 1];
  auto fragment_offsets = [&](auto is_slow, uint32_t* off, int half) {
    if constexpr (decltype(is_slow)::value) {
      const uint32_t krow = lq * 8 + (l16 >> 2);
#pragma unroll
      for (int f = 0; f < F; f++) {
        const uint32_t col = (uint32_t)(half * kSlab + f * 16) + (l16 & 3) * 4;
        off[f] = krow * kSlowRowBytes + (((col >> 3) ^ slow_swizzle(krow)) * 16) + ((col >> 2) & 1) * 8;
      }
    } else {
      off[0] = (uint32_t)(half * kSlab + l16) * kRowBytes + ((uint32_t)lq ^ swizzle(l16)) * 16;
    }
  };
  fragment_offsets(std::bool_constant<A_SLOW>{}, a_off, wi);
  fragment_offsets(std::bool_constant<B_SLOW>{}, b_off, wj);
  int4v af[2][F], bf[2][F];                                      // [register set][fragment]
  short4v aq[2][F][2], bq[2][F][2];                              // k slow: the halves of a fragment
  constexpr int A_READS = A_SLOW ? 2 * F : F, B_READS = B_SLOW ? 2 * F : F, READS = A_READS + B_READS, MMAS = F * F;
  auto read_slow = [&](const uint8_t* base, uint32_t off, int q) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(lds_ptr_t)(base + off + (q & 1) * 4 * kSlowRowBytes));
  };
  auto read_a = [&](int set, int q, uint32_t buf) {
    if constexpr (A_SLOW) aq[set][q >> 1][q & 1] = read_slow(smem + buf, a_off[q >> 1], q);
    else af[set][q] = *reinterpret_cast<const int4v*>(smem + buf + a_off[0] + q * 16 * kRowBytes);
  };
  auto read_b = [&](int set, int q, uint32_t buf) {
    if constexpr (B_SLOW) bq[set][q >> 1][q & 1] = read_slow(smem + buf + kOperand, b_off[q >> 1], q);
    else bf[set][q] = *reinterpret_cast<const int4v*>(smem + buf + kOperand + b_off[0] + q * 16 * kRowBytes);
  };
  // the reads of a stage in the order its instructions need them: A's first fragment, B's, A's others
  auto read_one = [&](int set, int n, uint32_t buf) {
    constexpr int FIRST = A_READS / F;
    if (n >= FIRST && n < FIRST + B_READS) read_b(set, n - FIRST, buf);
    else read_a(set, n < FIRST ? n : n - B_READS, buf);
  };
  auto fragment = [&](auto is_slow, int4v& whole_one, short4v (&halves)[2]) {
    if constexpr (decltype(is_slow)::value) return __builtin_bit_cast(int4v, __builtin_shufflevector(halves[0], halves[1], 0, 1, 2, 3, 4, 5, 6, 7));
    else return whole_one;
  };
  float4v acc[F][F];
  // The instructions of a stage from one register set; behind them, one by one, the next stage's reads into the other set and the copies of the stage that
  // takes this one's buffer.
  auto mma_stage = [&](auto which, auto is_first, uint32_t dst, uint32_t src) __attribute__((always_inline)) {
    constexpr int set = decltype(which)::value;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < MMAS; n++) {
      const int ti = n / F, tj = n % F;
      acc[ti][tj] = mma(T{}, fragment(std::bool_constant<A_SLOW>{}, af[set][ti], aq[set][ti]), fragment(std::bool_constant<B_SLOW>{}, bf[set][tj], bq[set][tj]), decltype(is_first)::value ? float4v{0, 0, 0, 0} : acc[ti][tj]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = n * READS / MMAS; q < (n + 1) * READS / MMAS; q++) read_one(set ^ 1, q, src);
      if (n * 2 * kCopies % MMAS < 2 * kCopies) copy_one(n * 2 * kCopies / MMAS, dst);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- what is done with a unit's accumulators, in the wave's own part of the LDS
  constexpr uint32_t scratch_at = kRing * kStage;
  auto fetch = [&]() {                                           // what the tile needs of its words and tokens
    const uint32_t to = smem_at + scratch_at + wave * kScratch, off = (uint32_t)lane * 16;
    const int64_t token = now.j0 + wj * kSlab;
    if constexpr (KIND == HEAD_INPUT) g2l16((const uint8_t*)(r.row_of + token), off, to + kTokensAt);
    if constexpr (LOGITS) {
      if (r.bias) g2l16((const uint8_t*)(r.bias + now.i0 + wi * kSlab), off, to + kColumnsAt);
      if constexpr (KIND == HEAD_STATS) {
        const uint8_t* from = r.target ? (const uint8_t*)(r.target + token) : (const uint8_t*)(r.slab_entries + (now.i0 / kSlab + wi) * r.tokens_ld + token);
        g2l16(from, off, to + kTokensAt);
      } else {
        g2l16((const uint8_t*)(r.coef + token), off, to + kTokensAt);
        if constexpr (SMOOTH) g2l16((const uint8_t*)(r.level + token), off, to + kLevelAt);
      }
    } else if constexpr (SMOOTH) {
      g2l16((const uint8_t*)(r.common + now.i0 + wi * kSlab), off, to + kColumnsAt);
      if constexpr (KIND == HEAD_INPUT) g2l16((const uint8_t*)(r.level_rest + token), off, to + kLevelAt);
    }
  };
  constexpr int ROW16 = kSlab * 2, CHUNKS = kSlab / 8;             // 16-bit results go out by 16 rows, through the wave's 4 KB
  auto chunk_at = [](int row, int ch) { return row * ROW16 + (ch ^ row) * 16; };
  auto pieces_of = [&](const Unit& u) { return u.m < rounds ? 1 : pieces; };
  auto finish = [&]() __attribute__((always_inline)) {
    // (numbers of their own: what is worked out from them, addresses above all, would be kept in registers through the loop over the stages otherwise)
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int l16 = lane & 15, lq = lane >> 4;
    uint8_t* slice = smem + scratch_at + wave * kScratch;
    // what was fetched is older than the copies that the loop's last wait left in flight, if there were enough of them
    if (KIND != HEAD_WEIGHT && now.stages < 4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    float4v add[F];
    if constexpr (LOGITS) {
#pragma unroll
      for (int ti = 0; ti < F; ti++) {
        if (r.bias) add[ti] = *reinterpret_cast<const float4v*>(slice + kColumnsAt + (ti * 16 + lq * 4) * 4);
        else {
#pragma unroll
          for (int e = 0; e < 4; e++) add[ti][e] = now.i0 + wi * kSlab + ti * 16 + lq * 4 + e < r.words ? 0.0f : -__builtin_inff();
        }
      }
    }
    if constexpr (KIND == HEAD_STATS) {
      const int64_t slab = now.i0 / kSlab + wi;
      const int base = (int)(slab * kSlab);
      int brought_all[F];                                        // (from here on all of the wave's LDS is for the logits of listed words)
#pragma unroll
      for (int tj = 0; tj < F; tj++) brought_all[tj] = *reinterpret_cast<const int*>(slice + kTokensAt + (tj * 16 + l16) * 4);
      constexpr int G = F / 2;                          // columns of fragments at a time, as far as registers go
#pragma unroll
      for (int t0 = 0; t0 < F; t0 += G) {
        // (the accumulators are read once: vector instructions reach them through copies alone)
        float4v y[F][G];
        float m[G], from[G], s[G], sum[G];
        constexpr int AHEAD = 2;
        int brought[G], word[G][AHEAD] = {};
#pragma unroll
        for (int tj = 0; tj < G; tj++) { m[tj] = -__builtin_inff(); s[tj] = 0.0f; sum[tj] = 0.0f; }
#pragma unroll
        for (int ti = 0; ti < F; ti++)
#pragma unroll
          for (int tj = 0; tj < G; tj++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              y[ti][tj][e] = __builtin_fmaf(acc[ti][t0 + tj][e], r.scale, add[ti][e]);
              if constexpr (SMOOTH) sum[tj] += base + ti * 16 + lq * 4 + e < r.words ? y[ti][tj][e] : 0.0f;
            }
            m[tj] = fmaxf(fmaxf(m[tj], y[ti][tj][0]), y[ti][tj][1]);
            m[tj] = fmaxf(fmaxf(m[tj], y[ti][tj][2]), y[ti][tj][3]);
          }
#pragma unroll
        for (int tj = 0; tj < G; tj++) brought[tj] = brought_all[t0 + tj];
        if (!r.target) {                                         // the first entries' words, ahead of their use
#pragma unroll
          for (int tj = 0; tj < G; tj++) {
            const int many = brought[tj] >> 11 & 0x7ff;
            const int64_t entry = (now.j0 + wj * kSlab + (t0 + tj) * 16 + l16) * r.entries + (brought[tj] & 0x7ff);
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
              if (lq + 4 * u < many) word[tj][u] = r.entry_words[entry + lq + 4 * u];
          }
        }
#pragma unroll
        for (int tj = 0; tj < G; tj++) {
          m[tj] = over_quarters(m[tj], [](float a, float b) { return fmaxf(a, b); });
          from[tj] = m[tj] == -__builtin_inff() ? 0.0f : m[tj];
        }
#pragma unroll
        for (int ti = 0; ti < F; ti++)
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int tj = 0; tj < G; tj++) s[tj] += __builtin_amdgcn_exp2f(y[ti][tj][e] - from[tj]);
#pragma unroll
        for (int tj = 0; tj < G; tj++) {
          const int64_t token = now.j0 + wj * kSlab + (t0 + tj) * 16 + l16;
          s[tj] = over_quarters(s[tj], [](float a, float b) { return a + b; });
          if constexpr (SMOOTH) sum[tj] = over_quarters(sum[tj], [](float a, float b) { return a + b; });
          if (lq == 0) {
            r.stats[slab * r.tokens_ld + token] = float2{m[tj], s[tj]};
            if constexpr (SMOOTH) r.sums[slab * r.tokens_ld + token] = sum[tj];
          }
          if (r.target) {
            const int at = brought[tj] - base;
            if (__any(at >= 0 && at < kSlab)) {
#pragma unroll
              for (int ti = 0; ti < F; ti++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                  if (at == ti * 16 + lq * 4 + e) r.picked[token] = y[ti][tj][e];
            }
          } else {
            // the teacher's entries of these words, four of a token at a time, from the token's row in LDS
            const int many = brought[tj] >> 11 & 0x7ff;
            const int64_t entry = token * r.entries + (brought[tj] & 0x7ff);
            if (__any(many > 0)) {
              uint8_t* row = slice + l16 * (kSlab * 4);
              auto pick = [&](int n, int word) {
                const int at = word - base;
                r.picked[entry + n] = *reinterpret_cast<const float*>(row + ((at >> 2) ^ (l16 & 7)) * 16 + (at & 3) * 4);
              };
              wave_lds_fence();
#pragma unroll
              for (int ti = 0; ti < F; ti++) *reinterpret_cast<float4v*>(row + ((ti * 4 + lq) ^ (l16 & 7)) * 16) = y[ti][tj];
              wave_lds_fence();
#pragma unroll
              for (int u = 0; u < AHEAD; u++)
                if (lq + 4 * u < many) pick(lq + 4 * u, word[tj][u]);
              for (int n0 = lq + 4 * AHEAD; n0 < many; n0 += 16) {           // (four loads in flight)
                int more[4];
#pragma unroll
                for (int u = 0; u < 4; u++) more[u] = r.entry_words[entry + min(n0 + 4 * u, many - 1)];
#pragma unroll
                for (int u = 0; u < 4; u++)
                  if (n0 + 4 * u < many) pick(n0 + 4 * u, more[u]);
              }
            }
          }
        }
      }
    } else {
      // float32 as the accumulators lie, 16 bytes a lane
      auto slots_of = [&](float* base, int64_t tile) { return base + tile * (kTile * kTile) + (wave * 64 + lane) * 4; };
      if constexpr (!LOGITS) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the copies in flight: from here on stores count as well
        if (r.add && pieces_of(now) == 1) {
          const float* from = slots_of(r.sum, now.tile);
#pragma unroll
          for (int ti = 0; ti < F; ti++)
#pragma unroll
            for (int tj = 0; tj < F; tj++) acc[ti][tj] += *reinterpret_cast<const float4v*>(from + (ti * F + tj) * (kThreads * 4));
        }
        if (pieces_of(now) > 1 || !r.last) {
          float* to = pieces_of(now) > 1 ? slots_of(r.partial, (int64_t)now.piece * rest + now.tile - whole) : slots_of(r.sum, now.tile);
#pragma unroll
          for (int ti = 0; ti < F; ti++)
#pragma unroll
            for (int tj = 0; tj < F; tj++) *reinterpret_cast<float4v*>(to + (ti * F + tj) * (kThreads * 4)) = acc[ti][tj];
          wave_lds_fence();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          return;
        }
        if constexpr (SMOOTH) {
          float times[F];
#pragma unroll
          for (int tj = 0; tj < F; tj++) times[tj] = KIND == HEAD_INPUT ? *reinterpret_cast<const float*>(slice + kLevelAt + (tj * 16 + l16) * 4) : 1.0f;
#pragma unroll
          for (int ti = 0; ti < F; ti++) {
            const float4v common = *reinterpret_cast<const float4v*>(slice + kColumnsAt + (ti * 16 + lq * 4) * 4);
#pragma unroll
            for (int tj = 0; tj < F; tj++)
#pragma unroll
              for (int e = 0; e < 4; e++) acc[ti][tj][e] = __builtin_fmaf(-times[tj], common[e], acc[ti][tj][e]);
          }
        }
      }
      const int64_t rows = KIND == HEAD_INPUT ? (int64_t)count : r.rows_j, cols = r.cols_out;
      const float scale = LOGITS ? 1.0f : *r.out_scale;
      if constexpr (!LOGITS && std::is_same<OutT, float>::value) {
        const bool aligned = cols % 4 == 0 && ((uintptr_t)r.out & 15) == 0;
#pragma unroll
        for (int tj = 0; tj < F; tj++) {
          const int64_t row = now.j0 + wj * kSlab + tj * 16 + l16;
          float* at = (float*)r.out + row * cols + now.i0 + wi * kSlab + lq * 4;
          if (row < rows) {
#pragma unroll
            for (int ti = 0; ti < F; ti++) {
              const int64_t col = now.i0 + wi * kSlab + ti * 16 + lq * 4;
              const float4v v = acc[ti][tj] * scale;
              if (aligned && col < cols) *reinterpret_cast<float4v*>(at + ti * 16) = v;
              else if (!aligned) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                  if (col + e < cols) at[ti * 16 + e] = v[e];
              }
            }
          }
        }
      } else {
        // 16(j) x 128(i) pieces through the slice, chunks XOR-swizzled with the row, whole rows of them stored
        const bool aligned = LOGITS || (cols % 8 == 0 && ((uintptr_t)r.out & 15) == 0);
        T* out = (T*)(LOGITS ? r.slope : r.out);
        const int64_t ld = LOGITS ? r.ld_slope : cols;
#pragma unroll
        for (int tj = 0; tj < F; tj++) {
          float2 coef = {0, 0};
          float level = 0.0f;
          if constexpr (LOGITS) coef = *reinterpret_cast<const float2*>(slice + kTokensAt + (tj * 16 + l16) * 8);
          if constexpr (LOGITS && SMOOTH) level = *reinterpret_cast<const float*>(slice + kLevelAt + (tj * 16 + l16) * 4);
          if (tj > 0) wave_lds_fence();                          // behind the reads of the piece before
#pragma unroll
          for (int ti = 0; ti < F; ti++) {
            T o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float v;
              if constexpr (LOGITS) {
                v = coef.y * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[ti][tj][e], r.scale, add[ti][e]) - coef.x);
                if constexpr (SMOOTH) v = now.i0 + wi * kSlab + ti * 16 + lq * 4 + e < r.words ? v - level : 0.0f;
              } else v = scaled(acc[ti][tj][e], scale);
              o[e] = from_float<T>(v);
            }
            *reinterpret_cast<Pack<T, 4>*>(slice + chunk_at(l16, ti * 2 + (lq >> 1)) + (lq & 1) * 8) = *reinterpret_cast<Pack<T, 4>*>(o);
          }
          if (LOGITS && tj == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the copies in flight, as above
          wave_lds_fence();
#pragma unroll
          for (int it = 0; it < CHUNKS / 4; it++) {
            const uint32_t piece = it * 64 + lane;
            const int jl = piece / CHUNKS, ch = piece % CHUNKS;
            const int64_t row = now.j0 + wj * kSlab + tj * 16 + jl, col = now.i0 + wi * kSlab + ch * 8;
            const int4v v = *reinterpret_cast<const int4v*>(slice + chunk_at(jl, ch));
            if constexpr (LOGITS) *reinterpret_cast<int4v*>(out + row * ld + col) = v;
            else if (row < rows && col < cols) {
              const int64_t to = KIND == HEAD_INPUT ? (int64_t)*reinterpret_cast<const int*>(slice + kTokensAt + (tj * 16 + jl) * 4) : row;
              T* at = out + to * ld + col;
              if (aligned) __builtin_nontemporal_store(v, reinterpret_cast<int4v*>(at));
              else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                  if (col + e < cols) at[e] = T{(uint16_t)((uint32_t)v[e >> 1] >> (e & 1) * 16)};
              }
            }
          }
        }
      }
    }
    wave_lds_fence();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the next copies go over what was read
  };

  // ---- the sequence of stages.  Behind its end the copies go on from the last place (stages that nobody reads): nothing in the loop depends on where
  // the sequence ends.
#pragma unroll
  for (int b = 0; b < kRing; b++) {
#pragma unroll
    for (int q = 0; q < 2 * kCopies; q++) copy_one(q, b * kStage);
    copied();
  }
  wait_copies_and_barrier<(kRing - 1) * 2 * kCopies, true>();
#pragma unroll
  for (int n = 0; n < READS; n++) read_one(0, n, 0);
  uint32_t cur = 0;                                              // buffer of the stage that is multiplied
  int landed = 0;                                                // so many stages behind the next one have arrived already
  // The next stage has arrived when the copies of those behind it are all that is in flight; and everyone has read this one.  (Loads complete in order: stores
  // between them can only make this wait longer, and where there are many, all copies were waited for ahead of the first.)
  auto arrive = [&]() {
    if (KIND != HEAD_STATS && landed > 0) { wait_reads_and_barrier(); landed--; }
    else wait_copies_and_barrier<(kRing - 2) * 2 * kCopies, true>();
  };
  auto stage = [&](auto set, auto is_first) __attribute__((always_inline)) {
    const uint32_t nxt = cur + kStage == kRing * kStage ? 0u : cur + kStage;
    arrive();
    mma_stage(set, is_first, cur, nxt);
    copied();
    cur = nxt;
  };
  for (int units = units_here;;) {
    fetch();
    // (the first stage adds to zero, and not to accumulators that were cleared: those the compiler would move about in the loop)
    stage(std::integral_constant<int, 0>{}, std::true_type{});
    stage(std::integral_constant<int, 1>{}, std::false_type{});
    for (int left = now.stages - 1; left > 0; left--) {
      stage(std::integral_constant<int, 0>{}, std::false_type{});
      stage(std::integral_constant<int, 1>{}, std::false_type{});
    }
    finish();
    if (!--units) break;
    landed = kRing - 1;
    advance(now);
    // (once more: kept through finish() the first fragments of the next unit would be in the way of what that needs)
#pragma unroll
    for (int n = 0; n < READS; n++) read_one(0, n, cur);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace
}  // namespace tf24
