// Weight and bias gradient of a linear layer whose input was kept in 8 bits (checkpoint8.hpp):
//
//     dW[i, j] = sum_t G[t, i] * X[t, j]        db[i] = sum_t G[t, i]
//
// G [tokens, m] 16-bit as it lies, X [tokens, n] as blocks of e4m3 and their scales.  Two ways, by expected time (takes_decoded):
//
// - X is decoded to 16 bits in the workspace and multiplied by the kernels of tf24_grad_weight: large products, of which the pass over X is a few
//   percent (total, product with the sum of its pieces, decoding: 12288 tokens, 4096 x 1024 106, 98, 7 us; 8192 tokens, 11008 x 4096 594, 576, 16).
// - One kernel that widens X (exactly: 4 bits of mantissa) on its way through the registers into LDS; products that are small, where the
//   launch of a pass more shows, and those that its smaller tiles divide better (1003 tokens, 2304 x 768: 15.2 us, 23.8 the other way; 4096 tokens, 2048 x
//   2048 46 and 51).  Its loads and its writes to LDS are issued by the waves that multiply, in whose place: a stage of a tile takes 0.55 to
//   0.65 us (1.0 PFLOP/s), on one card 0.65, without the writes 0.49, without the loads 0.55.  Tiles of 192 x 192 come to the same rate (8192 tokens,
//   4096 x 4096 275 us, without writes 206, without loads 232), and writes in both halves of a stage are no better than all in one.
//
// The kernel.  The summed axis is the slow one of both operands: eight consecutive tokens of a column, which a lane of a matrix instruction takes,
// come from transposing LDS reads (DS_READ_B64_TR_B16) of rows of a tile's columns.  A block of four waves (2 x 2) multiplies a tile of 128 x 128 over a
// piece of the token axis with V_MFMA_F32_16X16X32.  64 tokens are a stage; two stage buffers rotate in LDS, and the global loads of two more
// stages are in flight in registers.  One barrier a stage, between its halves; the fragments of a half are read while the half before is multiplied.
// Tokens past the last one are read as zeros by the buffer loads' own bounds (both operands: a zero times whatever lies there would not do).
// 16-byte chunks of a row are XOR-swizzled by token, so that the four tokens x 64 bytes that 32 lanes read touch every bank once.
// Few tiles and a long token axis: the axis is cut into pieces, whose float32 partial tiles a second kernel adds in piece order.
#include "checkpoint8.hpp"
#include "lds_copies.hpp"

namespace tf24 {
namespace {

typedef short short8v __attribute__((ext_vector_type(8)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kMaxPieces = 16;

struct KeptTile {
  static constexpr int F = 4;                                      // fragments of 16 rows and of 16 columns per wave
  static constexpr int TILE = 32 * F, THREADS = 256, TOKENS = 64;
  static constexpr int ROW = TILE * 2, OPERAND = TOKENS * ROW, STAGE = 2 * OPERAND;
  static constexpr int G_CHUNKS = TILE / 8, G_LOADS = TOKENS * G_CHUNKS / THREADS;      // 16 bytes each: 8 columns of G, 16 of X
  static constexpr int X_CHUNKS = TILE / 16, X_LOADS = TOKENS * X_CHUNKS / THREADS;
  static constexpr int MMA = F * F, READS = 4 * F, SUMS = F / 2;   // of a half stage; row fragments whose column sums a wave forms
  static_assert(G_LOADS * THREADS == TOKENS * G_CHUNKS && X_LOADS * THREADS == TOKENS * X_CHUNKS && F % 2 == 0 && 2 * STAGE <= 160 * 1024, "a stage divides among the threads");
  static __device__ __forceinline__ uint32_t swizzle(uint32_t token) { return ((token & 3) << 2) | (((token >> 3) & 1) << 1); }
  // rows of fragment f of a wave: the two waves that share rows hold them rotated, so that the first SUMS fragments of each are its own
  static __device__ __forceinline__ int fragment_row(int wave, int f) { return (wave >> 1) * (16 * F) + ((f + (wave & 1) * SUMS) % F) * 16; }
};

template <typename T>
__device__ __forceinline__ float4v mma(short8v a, short8v b, float4v c) {
  if constexpr (std::is_same<T, f16_t>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// two kept values (of the lower or the upper half of a word) in T
template <typename T, bool UPPER>
__device__ __forceinline__ uint32_t widen2(uint32_t w, float scale) {
  if constexpr (std::is_same<T, f16_t>::value) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, UPPER));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, UPPER));
}

// `bytes` of memory from `base` on; loads past them give zeros and touch nothing
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const uint8_t* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00027000);
}

struct KeptArgs {
  const uint8_t *g, *values, *scales;
  int ldg;                                          // bytes
  int64_t m, n;
  int tokens, blocks;                               // blocks of 32 columns in a row of X
  int tiles_i, tiles_j, pieces;
  float *partial, *sums;                            // [pieces][tiles][TILE * TILE], [pieces][tiles_i * TILE]
};

template <typename T, typename OutT, bool SUMS>
__global__ void __launch_bounds__(KeptTile::THREADS)
grad_weight_kept(const KeptArgs a, OutT* __restrict__ dw, OutT* __restrict__ db) {
  using C = KeptTile;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * C::STAGE];
  // workgroup ids are dealt to the 8 XCDs round-robin: each XCD takes a run of units, which share operand columns in its L2
  const int tiles = a.tiles_i * a.tiles_j, units = tiles * a.pieces, per_xcd = (units + 7) / 8;
  const int unit = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3);
  if (unit >= min(((int)(blockIdx.x & 7) + 1) * per_xcd, units)) return;
  // (quotients come out of the vector registers)
  const int piece = __builtin_amdgcn_readfirstlane(unit / tiles), tile = unit - piece * tiles;
  const int tile_i = __builtin_amdgcn_readfirstlane(tile / a.tiles_j), tile_j = tile - tile_i * a.tiles_j;
  const int64_t i0 = (int64_t)tile_i * C::TILE, j0 = (int64_t)tile_j * C::TILE;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 15, lblock = lane >> 4;
  // stages go by twos (the last one of all may be empty: zeros)
  const int pairs_all = (a.tokens + 2 * C::TOKENS - 1) / (2 * C::TOKENS);
  const int first_pair = __builtin_amdgcn_readfirstlane(piece * pairs_all / a.pieces);
  const int pairs = __builtin_amdgcn_readfirstlane((piece + 1) * pairs_all / a.pieces) - first_pair;
  const int64_t first = (int64_t)first_pair * 2 * C::TOKENS;

  // ---- global loads: number q of a thread
  const int x_row = a.blocks * kKeptBlock;
  // (a lane's 16 columns of X are two chunks of LDS: four lanes write the lower one first, the next four the upper one, so that eight of them
  // touch 128 different bytes of banks either time)
  const uint32_t upper_first = (tid >> 2) & 1;
  uint32_t g_from[C::G_LOADS], g_to[C::G_LOADS], x_from[C::X_LOADS], s_from[C::X_LOADS], x_to[C::X_LOADS];
#pragma unroll
  for (int q = 0; q < C::G_LOADS; q++) {
    const uint32_t at = q * C::THREADS + tid, token = at / C::G_CHUNKS, chunk = at % C::G_CHUNKS;
    g_from[q] = token * a.ldg + chunk * 16;
    g_to[q] = token * C::ROW + ((chunk ^ C::swizzle(token)) * 16);
  }
#pragma unroll
  for (int q = 0; q < C::X_LOADS; q++) {
    const uint32_t at = q * C::THREADS + tid, token = at / C::X_CHUNKS, chunk = at % C::X_CHUNKS;
    x_from[q] = token * x_row + chunk * 16;
    s_from[q] = token * a.blocks + chunk / 2;
    x_to[q] = C::OPERAND + token * C::ROW + (((2 * chunk) ^ C::swizzle(token)) * 16) + upper_first * 16;
  }
  struct Loads { uint4v g[C::G_LOADS], x[C::X_LOADS]; uint8_t s[C::X_LOADS]; };
  Loads regs[2];
  // the rows of the stage to load next, as far as there are any
  int rows_left = a.tokens - (int)first, rows = 0;
  const uint8_t* g_at = a.g + first * a.ldg + i0 * 2;
  const uint8_t* x_at = a.values + first * x_row + j0;
  const uint8_t* s_at = a.scales + first * a.blocks + j0 / kKeptBlock;
  const int g_end = (int)(a.m - i0) * 2, x_end = x_row - (int)j0, s_end = a.blocks - (int)(j0 / kKeptBlock);
  __amdgpu_buffer_rsrc_t g_window, x_window, s_window;
  auto open_x = [&] {
    rows = min(rows_left, C::TOKENS) - 1;
    x_window = window(x_at, rows < 0 ? 0 : rows * x_row + x_end);
    s_window = window(s_at, rows < 0 ? 0 : rows * a.blocks + s_end);
    x_at += (int64_t)C::TOKENS * x_row;
    s_at += (int64_t)C::TOKENS * a.blocks;
    rows_left -= C::TOKENS;
  };
  auto open_g = [&] {                                             // of the same stage, behind open_x
    g_window = window(g_at, rows < 0 ? 0 : rows * a.ldg + g_end);
    g_at += (int64_t)C::TOKENS * a.ldg;
  };
  auto load_x = [&](Loads& r, int k) {                            // all scales, then all values
    if (k < C::X_LOADS) r.s[k] = __builtin_amdgcn_raw_buffer_load_b8(s_window, s_from[k], 0, 0);
    else r.x[k - C::X_LOADS] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(x_window, x_from[k - C::X_LOADS], 0, 0));
  };
  auto load_g = [&](Loads& r, int k) { r.g[k] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(g_window, g_from[k], 0, 0)); };
  auto store_x = [&](const Loads& r, int k, uint32_t buf) {
    const float scale = __builtin_bit_cast(float, (uint32_t)r.s[k] << 23);
    const uint4v w = r.x[k];
    const uint32_t w0 = upper_first ? w[2] : w[0], w1 = upper_first ? w[3] : w[1], w2 = upper_first ? w[0] : w[2], w3 = upper_first ? w[1] : w[3];
    *reinterpret_cast<uint4v*>(smem + buf + x_to[k]) = uint4v{widen2<T, false>(w0, scale), widen2<T, true>(w0, scale), widen2<T, false>(w1, scale), widen2<T, true>(w1, scale)};
    *reinterpret_cast<uint4v*>(smem + buf + (x_to[k] ^ 16)) = uint4v{widen2<T, false>(w2, scale), widen2<T, true>(w2, scale), widen2<T, false>(w3, scale), widen2<T, true>(w3, scale)};
  };
  auto store_g = [&](const Loads& r, int k, uint32_t buf) { *reinterpret_cast<uint4v*>(smem + buf + g_to[k]) = r.g[k]; };
  auto load_stage = [&](Loads& r) {
    open_x();
    open_g();
#pragma unroll
    for (int k = 0; k < 2 * C::X_LOADS; k++) load_x(r, k);
#pragma unroll
    for (int k = 0; k < C::G_LOADS; k++) load_g(r, k);
  };

  // ---- fragments: in a group of 16 lanes, lane i receives the halfwords i % 4 of the source lanes 4e + i / 4 (e = 0..3).
  // Source lane s addresses token t0 + s / 4, columns 4 * (s % 4).. of the group's 16, so lane i gets tokens t0..t0+3 of
  // column i; the lanes of block b take tokens 8b .. 8b + 7 of an instruction's 32 (t0 = 8b, 8b + 4).
  const uint32_t token0 = (uint32_t)(lblock * 8 + (lrow >> 2));
  uint32_t a_off[C::F], b_off[C::F];
#pragma unroll
  for (int f = 0; f < C::F; f++) {
    const uint32_t ca = (uint32_t)(C::fragment_row(wave, f) + (lrow & 3) * 4), cb = (uint32_t)(((wave & 1) * C::F + f) * 16 + (lrow & 3) * 4);
    a_off[f] = token0 * C::ROW + (((ca >> 3) ^ C::swizzle(token0)) * 16) + ((ca >> 2) & 1) * 8;
    b_off[f] = C::OPERAND + token0 * C::ROW + (((cb >> 3) ^ C::swizzle(token0)) * 16) + ((cb >> 2) & 1) * 8;
  }
  float4v acc[C::F][C::F];
#pragma unroll
  for (int i = 0; i < C::F; i++)
#pragma unroll
    for (int j = 0; j < C::F; j++) acc[i][j] = float4v{0, 0, 0, 0};
  float colsum[C::SUMS] = {};
  short4v af[2][C::F][2], bf[2][C::F][2];
  // in the order in which the next half's instructions need them: G's fragment 0, X's, G's others
  auto read_one = [&](int set, int q, uint32_t buf, int half) {
    const uint8_t* base = smem + buf + half * (32 * C::ROW) + (q & 1) * (4 * C::ROW);
    const int f = q >> 1;
    if (f >= 1 && f <= C::F) bf[set][f - 1][q & 1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(lds_ptr_t)(base + b_off[f - 1]));
    else af[set][f ? f - C::F : 0][q & 1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_ptr)(lds_ptr_t)(base + a_off[f ? f - C::F : 0]));
  };
  constexpr int READ_SLOTS = C::MMA * 2 / 3;                      // (all of them are back by the barrier)
  constexpr int PER_MMA = (8 * C::SUMS + C::MMA - 1) / C::MMA;
  // The instructions of a half from one register set; among them the reads of the next half into the other set and, `work` saying which, the
  // stage's stores to LDS or global loads.
  auto half_stage = [&](int set, uint32_t src, int next_half, auto&& work) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < C::MMA; i++) {
      const int ti = i / C::F, tj = i % C::F;
      const short8v x = __builtin_shufflevector(af[set][ti][0], af[set][ti][1], 0, 1, 2, 3, 4, 5, 6, 7);
      const short8v y = __builtin_shufflevector(bf[set][tj][0], bf[set][tj][1], 0, 1, 2, 3, 4, 5, 6, 7);
      acc[ti][tj] = mma<T>(x, y, acc[ti][tj]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = i * C::READS / READ_SLOTS; q < min((i + 1) * C::READS / READ_SLOTS, C::READS); q++) read_one(set ^ 1, q, src, next_half);
      work(i);
      if constexpr (SUMS) {
#pragma unroll
        for (int e = i * PER_MMA; e < (i + 1) * PER_MMA && e < 8 * C::SUMS; e++) {
          colsum[e >> 3] += to_float(T{(uint16_t)af[set][e >> 3][(e >> 2) & 1][e & 3]});
          asm volatile("" : "+v"(colsum[e >> 3]));               // (kept here: moved together they would run after the last instruction)
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // The halves of stage s, in buffer P.  Buffer P is free from the barrier in the middle on, the other one holds stage s + 1 up to there: the first
  // half stores G of stage s + 1 and loads X of stage s + 3 (into the registers that held X of stage s + 1), the second half stores X of stage
  // s + 2 and loads G of stage s + 3.  Half of the writes to LDS in either half: all of them in the first one kept it busier than the matrix cores.
  auto first_half = [&](auto parity) {
    constexpr int P = decltype(parity)::value;
    half_stage(0, P * C::STAGE, 1, [&](int i) {
      if (i == 0) open_x();
#pragma unroll
      for (int k = 0; k < C::G_LOADS; k++)
        if (i == k * (C::MMA / 2) / C::G_LOADS + 1) store_g(regs[1 - P], k, (1 - P) * C::STAGE);
#pragma unroll
      for (int k = 0; k < 2 * C::X_LOADS; k++)
        if (i == C::MMA / 4 + k * (C::MMA * 3 / 4) / (2 * C::X_LOADS)) load_x(regs[1 - P], k);
    });
  };
  auto second_half = [&](auto parity) {
    constexpr int P = decltype(parity)::value;
    wait_reads_and_barrier();
    half_stage(1, (1 - P) * C::STAGE, 0, [&](int i) {
      if (i == 0) open_g();
#pragma unroll
      for (int k = 0; k < C::X_LOADS; k++)
        if (i == k * (C::MMA / 2) / C::X_LOADS + 1) store_x(regs[P], k, P * C::STAGE);
#pragma unroll
      for (int k = 0; k < C::G_LOADS; k++)
        if (i == C::MMA / 4 + k * (C::MMA * 3 / 4) / C::G_LOADS) load_g(regs[1 - P], k);
    });
  };
  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};

  load_stage(regs[0]);
  load_stage(regs[1]);
#pragma unroll
  for (int k = 0; k < C::X_LOADS; k++) store_x(regs[0], k, 0);
#pragma unroll
  for (int k = 0; k < C::G_LOADS; k++) store_g(regs[0], k, 0);
  load_stage(regs[0]);
#pragma unroll
  for (int k = 0; k < C::X_LOADS; k++) store_x(regs[1], k, C::STAGE);
  wait_reads_and_barrier();
#pragma unroll
  for (int q = 0; q < C::READS; q++) read_one(0, q, 0, 0);
  // (the loop begins in the middle of a stage: with the zeros of the accumulators at its head the compiler moves them all in every round)
  first_half(even);
  for (int pair = 1; pair < pairs; pair++) {
    second_half(even);
    first_half(odd);
    second_half(odd);
    first_half(even);
  }
  second_half(even);
  first_half(odd);
  second_half(odd);

  if (SUMS && tile_j == 0) {
#pragma unroll
    for (int h = 0; h < C::SUMS; h++) {
      float v = colsum[h];
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      const int64_t row = i0 + C::fragment_row(wave, h) + lrow;
      if (lblock == 0) {
        if (a.pieces > 1) a.sums[(int64_t)piece * a.tiles_i * C::TILE + row] = v;
        else if (row < a.m) db[row] = from_float<OutT>(v);
      }
    }
  }
  if (a.pieces > 1) {
    float* out = a.partial + (int64_t)unit * (C::TILE * C::TILE) + tid * 4;
#pragma unroll
    for (int s = 0; s < C::MMA; s++) *reinterpret_cast<float4v*>(out + s * (C::THREADS * 4)) = acc[s / C::F][s % C::F];
    return;
  }
#pragma unroll
  for (int s = 0; s < C::MMA; s++) {
    const int64_t row = i0 + C::fragment_row(wave, s / C::F) + lblock * 4, col = j0 + ((wave & 1) * C::F + s % C::F) * 16 + lrow;
    if (row < a.m && col < a.n) {
#pragma unroll
      for (int r = 0; r < 4; r++) dw[(row + r) * a.n + col] = from_float<OutT>(acc[s / C::F][s % C::F][r]);
    }
  }
}

// dW and db from the pieces: block (tile, fragment), and with blockIdx.x one past the tiles the column sums
template <typename OutT>
__global__ void __launch_bounds__(KeptTile::THREADS)
grad_weight_kept_reduce(const KeptArgs a, OutT* __restrict__ dw, OutT* __restrict__ db) {
  using C = KeptTile;
  const int tiles = a.tiles_i * a.tiles_j, tid = threadIdx.x;
  if ((int)blockIdx.x == tiles) {
    for (int64_t i = (int64_t)blockIdx.y * C::THREADS + tid; i < a.m; i += (int64_t)gridDim.y * C::THREADS) {
      float v = 0.0f;
      for (int p = 0; p < a.pieces; p++) v += a.sums[(int64_t)p * a.tiles_i * C::TILE + i];
      db[i] = from_float<OutT>(v);
    }
    return;
  }
  const int tile_i = (int)blockIdx.x / a.tiles_j, tile_j = (int)blockIdx.x % a.tiles_j, lane = tid & 63, wave = tid >> 6, s = (int)blockIdx.y;
  const int64_t row = (int64_t)tile_i * C::TILE + C::fragment_row(wave, s / C::F) + (lane >> 4) * 4;
  const int64_t col = (int64_t)tile_j * C::TILE + ((wave & 1) * C::F + s % C::F) * 16 + (lane & 15);
  if (row >= a.m || col >= a.n) return;
  const float* from = a.partial + (int64_t)blockIdx.x * (C::TILE * C::TILE) + s * (C::THREADS * 4) + tid * 4;
  const int64_t piece = (int64_t)tiles * (C::TILE * C::TILE);
  float4v v = {0, 0, 0, 0};
  for (int p0 = 0; p0 < a.pieces; p0 += 8) {                       // eight independent loads in flight
    float4v part[8];
#pragma unroll
    for (int u = 0; u < 8; u++) part[u] = *reinterpret_cast<const float4v*>(from + (int64_t)min(p0 + u, a.pieces - 1) * piece);
#pragma unroll
    for (int u = 0; u < 8; u++)
      if (p0 + u < a.pieces) v += part[u];
  }
#pragma unroll
  for (int r = 0; r < 4; r++) dw[(row + r) * a.n + col] = from_float<OutT>(v[r]);
}

// The number of pieces with the least estimated time: 4 us, 0.535 us a stage in each round of the compute units, and for the partial tiles 3 us and
// 0.35 us a MB.  (Fitted to 120 products of 33 to 12288 tokens and 256 x 2048 to 11008 x 4096 outputs.)
struct Cut { int pieces; double us; };
Cut cut(int64_t tokens, int64_t m, int64_t n, int64_t workspace_bytes) {
  const int64_t tiles_i = (m + KeptTile::TILE - 1) / KeptTile::TILE, tiles = tiles_i * ((n + KeptTile::TILE - 1) / KeptTile::TILE);
  const int64_t pairs = (tokens + 2 * KeptTile::TOKENS - 1) / (2 * KeptTile::TOKENS), bytes = (tiles + tiles_i) * KeptTile::TILE * KeptTile::TILE * 4;
  Cut best{1, 4.0 + (double)(2 * pairs * ((tiles + 255) / 256)) * 0.535};
  for (int64_t p = 2; p <= kMaxPieces && p <= pairs && p * tiles <= 1024 && p * bytes <= workspace_bytes; p++) {
    const double us = 7.0 + (double)((pairs + p - 1) / p * 2 * ((p * tiles + 255) / 256)) * 0.535 + (double)(p * tiles) * (KeptTile::TILE * KeptTile::TILE * 4e-6 * 0.35);
    if (us < best.us) best = {(int)p, us};
  }
  return best;
}
int64_t pieces_bytes(int64_t tokens, int64_t m, int64_t n) {
  const int pieces = cut(tokens, m, n, (int64_t)1 << 40).pieces;
  const int64_t tiles_i = (m + KeptTile::TILE - 1) / KeptTile::TILE;
  return pieces > 1 ? pieces * (tiles_i * ((n + KeptTile::TILE - 1) / KeptTile::TILE) + tiles_i) * KeptTile::TILE * KeptTile::TILE * 4 : 0;
}
// Decoded to the workspace first: 7.5 us for the launch and what the products' estimate leaves out, 0.41 us for a million elements.  (The kernel's
// estimate on the same 120 products: the way taken is 2 % slower than the better one in the mean; 12288 tokens, 1024 x 4096 126 for 121.)
bool takes_decoded(int64_t tokens, int64_t m, int64_t n) {
  if (n % 8 || too_many_units(tokens, n)) return false;
  return 7.5 + dense_weight_grad_us(tokens, m, n) + (double)(tokens * n) * 0.41e-6 < cut(tokens, m, n, (int64_t)1 << 40).us;
}
int64_t decoded_bytes(int64_t tokens, int64_t n) { return (tokens * n * 2 + 255) / 256 * 256; }

template <typename T, typename OutT>
int launch(KeptArgs a, void* dw, void* db, void* workspace, int64_t workspace_bytes, hipStream_t s) {
  using C = KeptTile;
  a.tiles_i = (int)((a.m + C::TILE - 1) / C::TILE);
  a.tiles_j = (int)((a.n + C::TILE - 1) / C::TILE);
  a.pieces = cut(a.tokens, a.m, a.n, workspace ? workspace_bytes : 0).pieces;
  a.partial = (float*)workspace;
  a.sums = a.pieces > 1 ? a.partial + (int64_t)a.pieces * a.tiles_i * a.tiles_j * C::TILE * C::TILE : nullptr;
  const int per_xcd = (a.tiles_i * a.tiles_j * a.pieces + 7) / 8;
  auto* kernel = db ? grad_weight_kept<T, OutT, true> : grad_weight_kept<T, OutT, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(per_xcd * 8)), dim3(C::THREADS), 0, s, a, (OutT*)dw, (OutT*)db);
  if (a.pieces > 1)
    hipLaunchKernelGGL(grad_weight_kept_reduce<OutT>, dim3((unsigned)(a.tiles_i * a.tiles_j + (db ? 1 : 0)), C::MMA), dim3(C::THREADS), 0, s, a, (OutT*)dw, (OutT*)db);
  return check_launch("tf24_checkpoint_weight_grad");
}

}  // namespace
}  // namespace tf24

extern "C" int64_t tf24_checkpoint_weight_grad_workspace_bytes(int64_t tokens, int64_t m, int64_t n) {
  using namespace tf24;
  if (tokens <= 0 || m <= 0 || n <= 0) return 0;
  return takes_decoded(tokens, m, n) ? decoded_bytes(tokens, n) + dense_weight_grad_workspace_bytes(tokens, m, n) : pieces_bytes(tokens, m, n);
}

extern "C" int tf24_checkpoint_weight_grad(const void* g, int64_t ldg, int dtype, const void* values, const void* scales, int64_t tokens, int64_t m, int64_t n, void* dw,
                                           void* db, int out_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace tf24;
  const char* fn = "tf24_checkpoint_weight_grad";
  if (dtype != TF24_F16 && dtype != TF24_BF16) return fail(TF24_ERR_DTYPE, "%s: unsupported dtype %d", fn, dtype);
  if (out_dtype != dtype && out_dtype != TF24_F32) return fail(TF24_ERR_DTYPE, "%s: unsupported output dtype %d", fn, out_dtype);
  if (tokens < 1 || tokens > 0x7fffffffLL - 256) return fail(TF24_ERR_SHAPE, "%s: bad number of tokens %lld", fn, (long long)tokens);
  if (m < 8 || m % 8 || n < 1 || m > (1 << 20) || n > (1 << 20))
    return fail(TF24_ERR_SHAPE, "%s: %lld outputs must be a positive multiple of 8 and %lld inputs positive, at most %d", fn, (long long)m, (long long)n, 1 << 20);
  // a stage's tokens are addressed by 32-bit lane offsets
  if (ldg < m || ldg % 8 || ldg > (1 << 23)) return fail(TF24_ERR_STRIDE, "%s: leading dimension %lld must cover the rows, be a multiple of 8 and at most %d", fn, (long long)ldg, 1 << 23);
  if (!g || !values || !scales || !dw) return fail(TF24_ERR_ARG, "%s: null pointer", fn);
  if (workspace_bytes < 0) return fail(TF24_ERR_ARG, "%s: negative workspace size", fn);
  if (int rc = check_aligned(fn, 16, {g, values, workspace})) return rc;
  if (int rc = check_aligned(fn, dtype_size(out_dtype), {dw, db})) return rc;
  const bool wide = out_dtype == TF24_F32;
  if (workspace && takes_decoded(tokens, m, n) && workspace_bytes >= decoded_bytes(tokens, n) + dense_weight_grad_workspace_bytes(tokens, m, n)) {
    if (int rc = tf24_checkpoint_decode(values, scales, tokens, n, workspace, dtype, n, stream)) return rc;
    const int64_t at = decoded_bytes(tokens, n);
    return dense_weight_grad(fn, wide ? GRAD_SUMS : GRAD_AS_OPERANDS, g, ldg, workspace, n, dtype, tokens, m, n, dw, db, (uint8_t*)workspace + at, workspace_bytes - at, stream);
  }
  KeptArgs a{};
  a.blocks = (int)kept_blocks(n);
  a.g = (const uint8_t*)g, a.values = (const uint8_t*)values, a.scales = (const uint8_t*)scales;
  a.ldg = (int)ldg * 2, a.m = m, a.n = n, a.tokens = (int)tokens;
  auto* go = dtype == TF24_F16 ? (wide ? launch<f16_t, float> : launch<f16_t, f16_t>) : (wide ? launch<bf16_t, float> : launch<bf16_t, bf16_t>);
  return go(a, dw, db, workspace, workspace_bytes, (hipStream_t)stream);
}
