// Tiled matrix products on MFMA shared by the language-model kernels:
//   C(m, n) = sum_k A(m, k) * B(n, k)
// with either operand stored k-fast ([rows][k], the layout of a weight matrix
// and its input) or k-slow ([k][rows], what the gradient products meet), so
// that no operand is ever transposed in memory.
//
// LDS image of a panel of R rows x one K tile (128 bytes of k: 64 16-bit or 128
// 8-bit elements):
//   k-fast: [R][128 bytes]; 16-byte chunk c of row r is kept at c ^ (r & 7), so
//     the sixteen rows of an MFMA operand read lie in different banks.
//   k-slow: [64][R * 2 bytes]; the 32-byte unit u (sixteen rows of the operand)
//     of k is kept at u ^ f(k), f(k) = (k & 3) | ((k >> 3 & 1) << 2).  Operands
//     come out through ds_read_b64_tr_b16: sixteen lanes read a 4 (k) x 16 (rows)
//     block and each receives the four k of its own row; the eight segments of
//     half a wave (two k groups x four k) then start in eight different units.
// MFMA 16x16x32 (16-bit) / 16x16x64 (8-bit): lane l supplies row l % 16 and the
// 16 bytes of k at l / 16.  B goes in as the first operand and A as the second:
// lane l then holds C[m = l % 16][n = 4 * (l / 16) + e], four consecutive n.
#pragma once
#include "common.h"
#include "op_args.h"
#include "pieces.h"

#include <type_traits>

namespace hcamd {

enum Layout { kKFast = 0, kKSlow = 1 };

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;
typedef const __attribute__((address_space(1))) u32x4_u *global_u32x4_ptr;

template <class E> struct MmaType {
  using acc = f32x4;
  static constexpr int kBK = 64;     // elements of k in a tile
  static constexpr int kChunk = 8;   // elements in 16 bytes
};
template <> struct MmaType<int8_t> {
  using acc = i32x4;
  static constexpr int kBK = 128;
  static constexpr int kChunk = 16;
};

template <class E>
__device__ __forceinline__ typename MmaType<E>::acc mma16(u32x4 b, u32x4 a, typename MmaType<E>::acc c) {
  if constexpr (std::is_same<E, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c,
                                                   0, 0, 0);
  else if constexpr (std::is_same<E, _Float16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0, 0,
                                                 0);
}

// Consecutive workgroup ids go to different XCDs, each with an L2 of its own:
// every XCD gets a contiguous range of tiles, walked in bands of four tile rows.
__device__ __forceinline__ void tile_of(int wg, int tiles_m, int tiles_n, int &tm, int &tn) {
  constexpr int kXcds = 8, kBand = 4;
  const int n = tiles_m * tiles_n, q = n / kXcds, r = n % kXcds, x = wg % kXcds;
  wg = x * q + min(x, r) + wg / kXcds;
  const int band = kBand * tiles_n;
  const int first = (wg / band) * kBand;
  const int rows = min(tiles_m - first, kBand);
  const int in = wg % band;
  // (quotients come out of the vector unit; the tile is the same for every lane)
  tm = __builtin_amdgcn_readfirstlane(first + in % rows);
  tn = __builtin_amdgcn_readfirstlane(in / rows);
}

// the k tiles [kt0, kt1) of a split
__device__ __forceinline__ void split_of(int all, int split, int splits, int &kt0, int &kt1) {
  const int each = all / splits, more = all % splits;
  kt0 = __builtin_amdgcn_readfirstlane(split * each + min(split, more));
  kt1 = __builtin_amdgcn_readfirstlane(kt0 + each + (split < more ? 1 : 0));
}

__device__ __forceinline__ int slow_swizzle(int k) { return (k & 3) | ((k >> 3 & 1) << 2); }

// byte offset of row `row`'s 16 bytes of k at chunk `chunk` in a k-fast panel
__device__ __forceinline__ int fast_offset(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) * 16); }

// the operand registers of the 16 rows from `row0` (a multiple of 16) for the
// k half `h` of the tile
template <Layout L, int R>
__device__ __forceinline__ u32x4 read_operand(const unsigned char *panel, int row0, int h, int lane) {
  if constexpr (L == kKFast) {
    return *reinterpret_cast<const u32x4 *>(panel + fast_offset(row0 + lane % 16, 4 * h + lane / 16));
  } else {
    const int i = lane % 16, k = 32 * h + 8 * (lane / 16) + i / 4;
    const unsigned char *p = panel + k * (R * 2) + (((row0 / 16) ^ slow_swizzle(k)) * 32) + (i % 4) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + 4 * R * 2));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
}

// Where a workgroup's tile lies: it covers rows m0 .. and columns n0 .., and owns those
// from m_lo and n_lo on (an edge tile of the pipelined kernel begins inside its
// neighbour, whose part it computes again and does not store).
struct Tile {
  int m0, n0, m_lo, n_lo, tn;
};

// ---------------------------------------------------------------------------
// General kernel body: any sizes, leading dimensions and alignment.  128 x 128
// tile, four waves of 64 x 64, panels through registers in unaligned 16-byte pieces, two
// LDS stages, one barrier per k tile.  Panels of k-fast operands are requested two k tiles
// ahead, others one (the gradient of the weights over 100 tokens has two k tiles in all:
// 4001 x 9001 bf16 87 us one ahead, 147 us two ahead).  Every piece is one load
// whatever it crosses: one that reaches past the end of its row is fetched that much
// earlier and shifted into place on its way to LDS, rows and k past the end are those of
// the last one, and what lies past K is stored as zeros.  So a k-fast operand has a
// piece of k at least, or rows padded with zeros to one, and a k-slow operand likewise
// (their padding may hold anything).  No load stands in a branch: the compiler would
// wait there for all of them.
// Bound by the path through registers and LDS (a tile moves 32 KiB into LDS and 64 KiB out
// of it for 512 cycles of MFMA): 4000 x 11000 x 4088 bf16 both projections 0.82 PFLOP/s
// forward where the pipelined kernel reaches 1.2; small products by the latency of their
// k tiles, 0.8 us each.
// GATED: the N panel holds 32 rows of b[0], then the same 32 of b[1], alternating, so that
// a wave's blocks j and j + 2 are the two projections of the same outputs.
// ---------------------------------------------------------------------------
template <class E, Layout LA, Layout LB, bool GATED, int BM, class Init, class Epilogue>
__device__ __forceinline__ void mma_general(const MmaArgs &g, int wg, int split, unsigned char *lds, Init &&init,
                                            Epilogue &&epilogue) {
  using T = MmaType<E>;
  constexpr int BN = 128, BNO = GATED ? BN / 2 : BN;
  constexpr int kPanel = BM * 128, kStage = kPanel + BN * 128, kA = BM / 32, kMI = BM / 32, kChunk = T::kChunk;
  static_assert(BM == 128 || LA == kKFast, "a k-slow panel is 128 wide");
  static_assert(sizeof(E) == 2 || (LA == kKFast && LB == kKFast), "transposed reads are for 16-bit elements");
  int tm, tn;
  tile_of(wg, (g.M + BM - 1) / BM, (g.N + BNO - 1) / BNO, tm, tn);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int wave_m = wave / 2 * (BM / 2), wave_n = wave % 2 * 64;
  const int tiles_k = (g.K + T::kBK - 1) / T::kBK, all = tiles_k * g.segments;
  int kt0, kt1;
  split_of(all, split, g.splits, kt0, kt1);

  // This thread's four pieces of a panel.  k-fast: chunk tid % 8 of rows tid / 8 + 32 i;
  // k-slow: columns tid % 16 * 8 .. + 7 of k tid / 16 + 16 i.
  // (a k-slow operand's last tile begins 128 rows before its end, where it has as many)
  const Tile tile = {LA == kKSlow && g.M >= BM ? min(tm * BM, g.M - BM) : tm * BM,
                     LB == kKSlow && g.N >= BN ? min(tn * BNO, g.N - BN) : tn * BNO, tm * BM, tn * BNO, tn};
  const int chunk = tid % 8 * kChunk, last_chunk = max(g.K - kChunk, 0), column = tid % 16 * 8, slow_k = tid / 16;
  // columns that a narrow k-slow operand's pieces are fetched early by
  const int early_a = LA == kKSlow ? max(tile.m0 + column - max(g.M - 8, 0), 0) : 0;
  const int early_b = LB == kKSlow ? max(tile.n0 + column - max(g.N - 8, 0), 0) : 0;
  const bool narrow = (LA == kKSlow && g.M < BM) || (LB == kKSlow && g.N < BN);
  constexpr int kAhead = LA == kKFast && LB == kKFast ? 2 : 1;
  u32x4 ra[kAhead][kA], rb[kAhead][4];
  const E *pa[kA], *pb[4]; // k-fast: the rows; k-slow: the pieces at k tile 0
  size_t lda = 0, ldb = 0;
  int segment = -1;
  auto aim = [&](int seg) {
    lda = seg ? g.lda[1] : g.lda[0], ldb = seg ? g.ldb[1] : g.ldb[0];
    const E *a = static_cast<const E *>(seg ? g.a[1] : g.a[0]), *b = static_cast<const E *>(seg ? g.b[1] : g.b[0]);
#pragma unroll
    for (int i = 0; i < kA; ++i) {
      if constexpr (LA == kKFast)
        pa[i] = a + (size_t)min(tile.m0 + tid / 8 + 32 * i, g.M - 1) * lda;
      else
        pa[i] = a + (size_t)(slow_k + 16 * i) * lda + (tile.m0 + column - early_a);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (GATED) {
        const int r = tid / 8 + 32 * i, n = min(tile.n0 + i / 2 * 32 + r % 32, g.N - 1);
        pb[i] = static_cast<const E *>(i % 2 ? g.b[1] : g.b[0]) + (size_t)n * (i % 2 ? g.ldb[1] : g.ldb[0]);
      } else if constexpr (LB == kKFast) {
        pb[i] = b + (size_t)min(tile.n0 + tid / 8 + 32 * i, g.N - 1) * ldb;
      } else {
        pb[i] = b + (size_t)(slow_k + 16 * i) * ldb + (tile.n0 + column - early_b);
      }
    }
    segment = seg;
  };
  auto begin_of = [&](int kt) { return (kt >= tiles_k ? kt - tiles_k : kt) * T::kBK; };
  auto load = [&](int kt, auto set) {
    constexpr int S = decltype(set)::value;
    if ((kt >= tiles_k ? 1 : 0) != segment)
      aim(kt >= tiles_k ? 1 : 0);
    const int k0 = begin_of(kt), at = min(k0 + chunk, last_chunk);
    size_t qa[kA], qb[4];
#pragma unroll
    for (int i = 0; i < kA; ++i)
      qa[i] = LA == kKFast ? (size_t)at : k0 * lda;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qb[i] = LB == kKFast ? (size_t)at : k0 * ldb;
    if ((LA == kKSlow || LB == kKSlow) && k0 + T::kBK > g.K) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t past = max(k0 + slow_k + 16 * i - (g.K - 1), 0);
        if constexpr (LA == kKSlow)
          qa[i] -= past * lda;
        if constexpr (LB == kKSlow)
          qb[i] -= past * ldb;
      }
    }
#pragma unroll
    for (int i = 0; i < kA; ++i)
      ra[S][i] = *(global_u32x4_ptr)(pa[i] + qa[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      rb[S][i] = *(global_u32x4_ptr)(pb[i] + qb[i]);
  };
  // what was fetched early moves into place, what lies past K becomes zero
  auto place = [&](Layout l, u32x4 v, int k0, int i, int early) {
    const int by = l == kKFast ? max(k0 + chunk - last_chunk, 0) : early;
    const bool none = l == kKFast ? by >= kChunk : k0 + slow_k + 16 * i >= g.K;
    v = shift_down(v, min(by, kChunk - 1) * (int)sizeof(E));
    return none ? u32x4{0u, 0u, 0u, 0u} : v;
  };
  auto offset = [&](Layout l, int id) {
    if (l == kKFast)
      return fast_offset(id / 8, id % 8);
    const int k = id / 16, pos = id % 16;
    return k * 256 + (((pos / 2) ^ slow_swizzle(k)) * 32) + pos % 2 * 16;
  };
  auto store = [&](int kt, int buf, auto set) {
    constexpr int S = decltype(set)::value;
    const int k0 = begin_of(kt);
    if (narrow || k0 + T::kBK > g.K) {
#pragma unroll
      for (int i = 0; i < kA; ++i)
        ra[S][i] = place(LA, ra[S][i], k0, i, early_a);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        rb[S][i] = place(LB, rb[S][i], k0, i, early_b);
    }
#pragma unroll
    for (int i = 0; i < kA; ++i)
      *reinterpret_cast<u32x4 *>(lds + buf * kStage + offset(LA, tid + i * 256)) = ra[S][i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<u32x4 *>(lds + buf * kStage + kPanel + offset(LB, tid + i * 256)) = rb[S][i];
  };

  typename T::acc acc[kMI][4] = {};
  init(acc, tile, wave_m, wave_n, lane);
  using Set0 = std::integral_constant<int, 0>;
  using Set1 = std::integral_constant<int, kAhead - 1>;
  // tile kt lies in stage `buf`, its registers (set `own`) are free, tile kt + 1 is in set
  // `next` (past the last tile: the last one again, which nothing reads)
  auto tile_step = [&](int kt, int buf, auto own, auto next) {
    if constexpr (kAhead == 2)
      load(min(kt + 2, kt1 - 1), own);
    else if (kt + 1 < kt1)
      load(kt + 1, own);
    const unsigned char *pa = lds + buf * kStage, *pb = pa + kPanel;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fa[kMI], fb[4];
#pragma unroll
      for (int i = 0; i < kMI; ++i)
        fa[i] = read_operand<LA, BM>(pa, wave_m + i * 16, h, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        fb[j] = read_operand<LB, BN>(pb, wave_n + j * 16, h, lane);
#pragma unroll
      for (int i = 0; i < kMI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = mma16<E>(fb[j], fa[i], acc[i][j]);
    }
    if (kAhead == 2 || kt + 1 < kt1)
      store(min(kt + 1, kt1 - 1), buf ^ 1, next);
    __syncthreads();
  };
  if (kt0 < kt1) {
    load(kt0, Set0{});
    if constexpr (kAhead == 2)
      load(min(kt0 + 1, kt1 - 1), Set1{});
    store(kt0, 0, Set0{});
    __syncthreads();
    int kt = kt0;
    for (; kt + 1 < kt1; kt += 2) {
      tile_step(kt, 0, Set0{}, Set1{});
      tile_step(kt + 1, 1, Set1{}, Set0{});
    }
    if (kt < kt1)
      tile_step(kt, 0, Set0{}, Set1{});
  }
  epilogue(acc, tile, wave_m, wave_n, lane, lds);
}

// ---------------------------------------------------------------------------
// Pipelined kernel body for operands that can be fetched in aligned 16-byte pieces.
//   * Panels go from global memory straight into LDS (16 bytes per lane; a wave-level
//     load fills 1 KiB of consecutive LDS, the layouts' swizzles are applied on the
//     global side).  Two stages; the loads of tile t + 2 are issued while tile t is
//     consumed.
//   * A tile is two halves of k.  While the MFMAs of one half run, the operands of
//     the next are read from LDS into a second register set, one fenced slot per
//     MFMA in hand order (the slots are worked out below).
//   * One barrier per tile, in front of its second half: there this wave's loads
//     of the next tile have landed and its reads of this tile are done.
//   * Edges: the last tile of a row or column of tiles begins BM rows (BN columns)
//     before the end; N >= BN, and M >= BM except with 128-row tiles and a k-fast A,
//     whose rows past M are fetched from row 0's group.  In the last tile of a k segment the
//     pieces past K are fetched from valid addresses and overwritten with zeros in
//     LDS by the lane that fetched them.  A k-fast operand whose K is not a multiple
//     of 8 must hold zeros up to there, a k-slow one whose rows are not must have
//     readable elements up to there (the library's own buffers).
// A load's address is a lane part, held in a register for the whole loop, plus a
// scalar part; from tile to tile only the base of the buffer descriptor moves.
// Bound by the matrix cores: they are busy 66 % of the cycles with two k-fast operands, 58 %
// with one k-slow operand, 54 % with two (whose reads are two of 8 bytes and must not
// stand behind loads into LDS); the clock gives way under the load as it does for a
// plain product.  256 x 256 tiles over 4096 x 4096 x 11264 bf16: both projections and their
// storing 601 us (1.26 PFLOP/s), dx 590 us, dW 645 us; 2000 x 4096 x 11264 int8 168 us (2.19
// POP/s).  For 2048 cycles of MFMA a tile's eight waves of 128 x 64 read 192 KiB from LDS;
// four waves of 128 x 128 would read a third less, but spill (dx 700 -> 1007 us).
// ---------------------------------------------------------------------------
constexpr int waitcnt_imm(int vmcnt, int lgkmcnt) {
  return (vmcnt & 0xf) | ((vmcnt >> 4) << 14) | (7 << 4) | ((lgkmcnt & 0xf) << 8);
}
constexpr int kNoVm = 63, kNoLgkm = 15;
typedef __attribute__((address_space(3))) void *lds_void_ptr;

template <int B> constexpr int pipelined_lds() { return 4 * B * 128; }

template <class E, Layout LA, Layout LB, bool GATED, int BM, int BN, int WM, int WN, class Init, class Epilogue>
__device__ __forceinline__ void mma_pipelined(const MmaArgs &g, int m_lo, int tn, int split, unsigned char *lds, Init &&init,
                                              Epilogue &&epilogue) {
  using T = MmaType<E>;
  constexpr int kWaves = WM * WN, kWaveM = BM / WM, kWaveN = BN / WN;
  constexpr int kMI = kWaveM / 16, kNI = kWaveN / 16, kMfma = kMI * kNI;
  constexpr int kALoads = BM / (8 * kWaves), kBLoads = BN / (8 * kWaves), kLoads = kALoads + kBLoads;
  constexpr int kReads = kMI + kNI;
  // The MFMA in front of which an operand read or a load goes.  k-fast operands: reads
  // over the first half of the MFMAs, loads evenly over all.  The compiler lets a
  // transposed read wait for every load into LDS that is under way, whatever stage it
  // fills, so k-slow operands are read before a half's loads are issued (second
  // half of a tile), and as late as there is time for them (first half), when the
  // loads of the half before have had most of a tile to land.
  constexpr int kSlow = (LA == kKSlow ? kMI : 0) + (LB == kKSlow ? kNI : 0), kQuick = kReads - kSlow;
  constexpr int kSlowSpan = kSlow == 0 ? 0 : kSlow * kMfma / 32 > kMfma / 4 ? kMfma / 4 : kMfma / 8;
  constexpr int LF = kSlow == 0 ? 1 : kSlowSpan;
  constexpr int LS = kSlow == 0 ? kMfma / kLoads : (kMfma * 3 / 4 - LF) / kLoads;
  static_assert(LF + (kLoads - 1) * LS < kMfma, "every load has its MFMA");
  // read r of a half, in the order B blocks, A blocks (as the MFMAs take them); first:
  // the half that reads the same tile's second half
  auto slot_of = [](int r, bool first) constexpr {
    const bool slow = r < kNI ? LB == kKSlow : LA == kKSlow;
    const int nth = slow ? (LB == kKSlow ? r : r - kNI) : (LB == kKSlow ? r - kNI : r);
    if (kSlow == 0)
      return nth * (kMfma / 2) / kReads;
    if (slow)
      return first ? kMfma * 9 / 16 + nth * (kMfma * 5 / 16) / kSlow : nth * kSlowSpan / kSlow;
    return (first ? 0 : kSlowSpan) + nth * (kMfma / 2) / (kQuick ? kQuick : 1);
  };
  constexpr int kPanelA = BM * 128, kStage = (BM + BN) * 128;
  constexpr int BNO = GATED ? BN / 2 : BN;
  static_assert(sizeof(E) == 2 || (LA == kKFast && LB == kKFast), "transposed reads are for 16-bit elements");

  // (k-slow rows come in aligned pieces of 8: their origin stays a multiple of 8)
  const int end_m = LA == kKSlow ? (g.M + 7) & ~7 : g.M, end_n = LB == kKSlow ? (g.N + 7) & ~7 : g.N;
  constexpr bool kFewRows = BM == 128 && LA == kKFast; // M may be less than a tile
  const Tile tile = {kFewRows ? max(min(m_lo, end_m - BM), 0) : min(m_lo, end_m - BM), min(tn * BNO, end_n - BNO), m_lo,
                     tn * BNO, tn};
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave_m = wave / WN * kWaveM, wave_n = wave % WN * kWaveN;
  const int tiles_k = (g.K + T::kBK - 1) / T::kBK, all = tiles_k * g.segments;
  int kt0, kt1;
  split_of(all, split, g.splits, kt0, kt1);
  const int steps = kt1 - kt0;
  // valid k of the last tile of a segment: elements (k-slow), 16-byte chunks (k-fast)
  const int tail_k = g.K - (tiles_k - 1) * T::kBK;
  const int tail_chunks = (tail_k + T::kChunk - 1) / T::kChunk;
  const bool has_tail = tail_k < T::kBK;
  auto is_tail = [&](int kt) { return has_tail && (kt == tiles_k - 1 || kt == all - 1); };

  // ---- global -> LDS -----------------------------------------------------------
  // The wave-level load v of a panel fills its rows (k-fast) (v * kWaves + wave) * 8 .. + 7,
  // or its k (k-slow) (v * kWaves + wave) * kPer .. + kPer - 1, kPer = 512 / R.
  const int fast_chunk = (lane % 8) ^ (lane / 8);
  // the lane parts: k-fast row * ld + chunk; k-slow k * ld + column, and the same with
  // the k of a group that K cuts clamped to its last valid one
  struct Lane {
    int off, cut;
  };
  // (k-slow: the k of consecutive loads of a wave differ by kWaves * 512 / R, 16 or 8; with
  // 8 the swizzle of every other load differs, in its third bit)
  constexpr int kParA = LA == kKSlow && kWaves * 512 / BM % 16 ? 2 : 1;
  constexpr int kParB = LB == kKSlow && kWaves * 512 / BN % 16 ? 2 : 1;
  auto lane_part = [&](Layout l, int R, int ld, bool tail, int odd) {
    Lane p;
    if (l == kKFast) {
      const int chunk = (tail && fast_chunk >= tail_chunks ? 0 : fast_chunk) * 16, left = g.M % 8;
      p.off = lane / 8 * ld + chunk;
      p.cut = (left ? min(lane / 8, left - 1) : lane / 8) * ld + chunk; // (A with few rows only)
    } else {
      const int per = 512 / R, sub = lane / (R / 8), pos = lane % (R / 8);
      const int col = ((pos / 2) ^ slow_swizzle(wave * per + sub) ^ (odd * 4)) * 16 + pos % 2 * 8;
      const int left = tail_k % per;
      p.off = sub * ld + col * 2;
      p.cut = (tail && left ? min(sub, left - 1) : sub) * ld + col * 2;
    }
    return p;
  };
  static_assert(LA == kKFast || kWaves * 512 / BM % 8 == 0, "the swizzle repeats from load to load");
  static_assert(LB == kKFast || kWaves * 512 / BN % 8 == 0, "the swizzle repeats from load to load");
  // GATED: rows of the N panel alternate in 32s between the two matrices; eight waves
  // meet one of them in all their loads, four waves the other one in every other
  constexpr int kBOps = GATED && kWaves == 4 ? 2 : 1;
  static_assert(!GATED || kParB == 1, "");
  const int my_b = GATED && kWaves == 8 ? wave / 4 : 0;
  Lane lane_a[kParA], lane_b[kBOps * kParB];
  int ld_a, ld_b[kBOps];
  __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b[kBOps];
  auto rsrc_of = [&](const void *p, size_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(static_cast<const char *>(p)) + bytes, 0, 0x7fffffff,
                                             0x00020000);
  };
  auto origin = [&](Layout l, size_t row, size_t ld, size_t kt) {
    return l == kKFast ? row * ld * sizeof(E) + kt * 128 : (kt * 64 * ld + row) * 2;
  };
  int state = -1; // segment and tail that the lane parts are set for
  auto prepare = [&](int kt) {
    const int seg = kt >= tiles_k ? 1 : 0, k = kt - seg * tiles_k;
    rsrc_a = rsrc_of(g.a[seg], origin(LA, tile.m0, g.lda[seg], k));
#pragma unroll
    for (int o = 0; o < kBOps; ++o) {
      const int w = GATED ? (kBOps == 2 ? o : my_b) : seg;
      rsrc_b[o] = rsrc_of(w ? g.b[1] : g.b[0], origin(LB, tile.n0, w ? g.ldb[1] : g.ldb[0], k));
    }
    const int want = seg * 2 + (is_tail(kt) ? 1 : 0);
    if (want != state) {
      ld_a = (int)g.lda[seg] * (int)sizeof(E);
#pragma unroll
      for (int o = 0; o < kParA; ++o)
        lane_a[o] = lane_part(LA, BM, ld_a, want & 1, o);
#pragma unroll
      for (int o = 0; o < kBOps; ++o) {
        const int w = GATED ? (kBOps == 2 ? o : my_b) : seg;
        ld_b[o] = (int)(w ? g.ldb[1] : g.ldb[0]) * (int)sizeof(E);
#pragma unroll
        for (int q = 0; q < kParB; ++q)
          lane_b[o * kParB + q] = lane_part(LB, BN, ld_b[o], want & 1, q);
      }
      state = want;
    }
  };
  auto fetch = [&](Layout l, int R, const __amdgpu_buffer_rsrc_t &rsrc, const Lane &p, int ld, int first, void *to,
                   bool few) {
    // first: the load's first row or k
    if (few) {
      const int off = first + 8 <= g.M ? p.off : p.cut;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)to, 16, off, first < g.M ? first * ld : 0, 0, 0);
    } else if (l == kKFast) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)to, 16, p.off, first * ld, 0, 0);
    } else {
      const int limit = (state & 1) ? tail_k : 64;
      const int off = first + 512 / R <= limit ? p.off : p.cut;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)to, 16, off, first < limit ? first * ld : 0, 0, 0);
    }
  };
  auto load_one = [&](int buf, int v) {
    unsigned char *base = lds + buf * kStage + wave * 1024;
    if (v < kALoads) {
      const int first = (v * kWaves + wave) * (LA == kKFast ? 8 : 512 / BM);
      fetch(LA, BM, rsrc_a, lane_a[v % kParA], ld_a, first, base + v * kWaves * 1024, kFewRows);
    } else {
      const int b = v - kALoads;
      int first = (b * kWaves + wave) * (LB == kKFast ? 8 : 512 / BN);
      if constexpr (GATED)
        first = first / 64 * 32 + first % 32;
      const int o = kBOps == 2 ? b % 2 : 0;
      fetch(LB, BN, rsrc_b[o], lane_b[o * kParB + b % kParB], ld_b[o], first, base + kPanelA + b * kWaves * 1024, false);
    }
  };
  auto zero_tail = [&](int buf) {
    unsigned char *base = lds + buf * kStage + wave * 1024 + lane * 16;
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int v = 0; v < kALoads; ++v)
      if (LA == kKFast ? fast_chunk >= tail_chunks : (v * kWaves + wave) * (512 / BM) + lane / (BM / 8) >= tail_k)
        *reinterpret_cast<u32x4 *>(base + v * kWaves * 1024) = zero;
#pragma unroll
    for (int v = 0; v < kBLoads; ++v)
      if (LB == kKFast ? fast_chunk >= tail_chunks : (v * kWaves + wave) * (512 / BN) + lane / (BN / 8) >= tail_k)
        *reinterpret_cast<u32x4 *>(base + kPanelA + v * kWaves * 1024) = zero;
  };

  // ---- LDS -> operand registers --------------------------------------------------
  // byte offsets of this lane in a panel, per block (k-slow) or common (k-fast, a block
  // is 2 KiB further)
  const int lk = 8 * (lane / 16) + lane % 16 / 4; // k-slow: k of the first read
  const int fast_lane = lane % 16 * 128;
  const int coff[2] = {((lane / 16) ^ (lane & 7)) * 16, ((4 + lane / 16) ^ (lane & 7)) * 16};
  // a k-slow block i is at block 0's address with bits 5 .. 7 xored by i (the origin of
  // a wave is a multiple of its blocks, and every other part of the address lies
  // outside those bits)
  const int slow_a = lk * (BM * 2) + (((wave_m / 16) ^ slow_swizzle(lk)) * 32) + lane % 4 * 8;
  const int slow_b = lk * (BN * 2) + (((wave_n / 16) ^ slow_swizzle(lk)) * 32) + lane % 4 * 8;
  static_assert(LA == kKFast || kMI <= 8, "blocks of a wave lie in one 256-byte group");
  auto read_slow = [&](const unsigned char *p, int four_k) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p + four_k));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return u32x4{a[0], a[1], b[0], b[1]};
  };
  u32x4 fa[2][kMI], fb[2][kNI];
  // fragment r of half h in stage buf: the B blocks first, then the A blocks, as the MFMAs take them
  auto read_one = [&](int buf, int h, auto slot, int r) {
    constexpr int S = decltype(slot)::value;
    const unsigned char *stage = lds + buf * kStage;
    if (r < kNI) {
      if constexpr (LB == kKFast)
        fb[S][r] = *reinterpret_cast<const u32x4 *>(stage + kPanelA + fast_lane + coff[h] + (wave_n + r * 16) * 128);
      else
        fb[S][r] = read_slow(stage + kPanelA + ((slow_b ^ (r * 32)) + h * 32 * (BN * 2)), 4 * BN * 2);
    } else {
      const int i = r - kNI;
      if constexpr (LA == kKFast)
        fa[S][i] = *reinterpret_cast<const u32x4 *>(stage + fast_lane + coff[h] + (wave_m + i * 16) * 128);
      else
        fa[S][i] = read_slow(stage + ((slow_a ^ (i * 32)) + h * 32 * (BM * 2)), 4 * BM * 2);
    }
  };

  typename T::acc acc[kMI][kNI] = {};
  init(acc, tile, wave_m, wave_n, lane);
  using Slot0 = std::integral_constant<int, 0>;
  using Slot1 = std::integral_constant<int, 1>;
  // MFMAs in a serpentine over the blocks: consecutive ones share an operand (four
  // waves: row by row, the serpentine costs them)
  auto half_step = [&](auto use, auto fill, int buf, int h, bool do_read, bool do_load, int load_buf) {
    constexpr int Uu = decltype(use)::value;
#pragma unroll
    for (int slot = 0; slot < kMfma; ++slot) {
      const int i = slot / kNI, j = kWaves == 8 && i % 2 ? kNI - 1 - slot % kNI : slot % kNI;
      if (do_read) {
#pragma unroll
        for (int r = 0; r < kReads; ++r)
          if (slot_of(r, h == 1) == slot)
            read_one(buf, h, fill, r);
      }
      if (do_load && slot >= LF && (slot - LF) % LS == 0 && (slot - LF) / LS < kLoads)
        load_one(load_buf, (slot - LF) / LS);
      acc[i][j] = mma16<E>(fb[Uu][j], fa[Uu][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto tile_step = [&](int t, auto load_next2, auto read_next) {
    constexpr bool LOAD = decltype(load_next2)::value, READ = decltype(read_next)::value;
    const int buf = t & 1;
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0));
    __builtin_amdgcn_sched_barrier(0);
    half_step(Slot0{}, Slot1{}, buf, 1, true, false, 0);
    if constexpr (LOAD)
      prepare(kt0 + t + 2);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    if constexpr (READ) {
      if (is_tail(kt0 + t + 1)) {
        zero_tail(buf ^ 1);
        __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0));
      }
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    half_step(Slot1{}, Slot0{}, buf ^ 1, 0, READ, LOAD, buf);
  };

  if (steps > 0) {
    prepare(kt0);
#pragma unroll
    for (int v = 0; v < kLoads; ++v)
      load_one(0, v);
    if (steps > 1) {
      prepare(kt0 + 1);
#pragma unroll
      for (int v = 0; v < kLoads; ++v)
        load_one(1, v);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(kLoads, kNoLgkm));
    } else {
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, kNoLgkm));
    }
    if (is_tail(kt0)) {
      zero_tail(0);
      __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0));
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < kReads; ++r)
      read_one(0, 0, Slot0{}, r);
    int t = 0;
    for (; t < steps - 2; ++t)
      tile_step(t, std::true_type{}, std::true_type{});
    if (steps > 1)
      tile_step(t++, std::false_type{}, std::true_type{});
    tile_step(t, std::false_type{}, std::false_type{});
  }
  // the epilogue may use the stages: every wave has read its last operands
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0));
  __builtin_amdgcn_s_barrier();
  epilogue(acc, tile, wave_m, wave_n, lane, lds);
}

// The tiles of a launch: 128 x 128, or 256 x 256 of which those from half_from on are
// worked as two halves of 128 rows.  A last round of tiles that fills at most half the
// card then takes half as long (4096 x 11264 outputs of the gated block: 5.5 rounds
// instead of 6).  `tile` counts the launch's workgroups from this product's first.
template <class E, Layout LA, Layout LB, bool GATED, int B, class Init, class Epilogue>
__device__ __forceinline__ void mma_tiles(const MmaArgs &g, int tile, int split, int half_from, unsigned char *lds, Init &&init,
                                          Epilogue &&epilogue) {
  constexpr int BNO = GATED ? B / 2 : B;
  const int tiles_m = (g.M + B - 1) / B, tiles_n = (g.N + BNO - 1) / BNO;
  int tm, tn;
  if constexpr (B == 128) {
    tile_of(tile, tiles_m, tiles_n, tm, tn);
    mma_pipelined<E, LA, LB, GATED, 128, 128, 2, 2>(g, tm * 128, tn, split, lds, init, epilogue);
  } else {
    if (tile < half_from) {
      tile_of(tile, tiles_m, tiles_n, tm, tn);
      mma_pipelined<E, LA, LB, GATED, 256, 256, 2, 4>(g, tm * 256, tn, split, lds, init, epilogue);
    } else {
      tile_of(half_from + (tile - half_from) / 2, tiles_m, tiles_n, tm, tn);
      const int m_lo = tm * 256 + (tile - half_from) % 2 * 128;
      if (m_lo < g.M)
        mma_pipelined<E, LA, LB, GATED, 128, 256, 2, 4>(g, m_lo, tn, split, lds, init, epilogue);
    }
  }
}

// ---------------------------------------------------------------------------
// Few tokens (which of them: the launcher's estimate): M <= 16 * MB rows of A against NB blocks of sixteen rows of B, for
// products that are one pass over B.  Eight waves share the k of the tile; each reads B and A straight into
// MFMA operand registers (sixteen rows, 64 consecutive bytes of a row per four lanes;
// which k a lane holds does not matter as long as both operands agree), the next block
// of k is requested before the present one is multiplied, and the eight partial sums
// meet in LDS.  Any size and alignment: rows past the end are read from the last one and
// not stored, pieces that cross K go element by element.
//   row_of(j): this lane's row lane % 16 of block j
// Bound by the weights' bytes: 5.3 TB/s over 2 x 11264 x 4096 bf16 for one token.
// ODD: rows that do not all begin at a multiple of 4 bytes.  Loads of 16 bytes run at full
// speed from such addresses only, so a piece is fetched from the 4-byte word its first
// element lies in and shifted into place.  The word behind it is the first one of the
// row's next piece, which another lane holds; the last lanes of a block load it, and it
// holds an element of their piece.  (One token, 60000 x 2231 bf16: 113 us as the rows lie, 74 us
// so; 11264 x 4095 both projections 3.8 TB/s.)
// The result lies in LDS as float or int [NB][MB][256], element (m, n) of a block at
// ((n / 4) * 16 + m) * 4 + n % 4.
// ---------------------------------------------------------------------------
template <int MB, int NB> constexpr int skinny_lds() { return 8 * NB * MB * 1024; }

template <class E, int MB, int NB, int U, bool ODD, class R>
__device__ __forceinline__ void mma_skinny(const MmaArgs &g, R &&row_of, unsigned char *lds) {
  using T = MmaType<E>;
  constexpr int kStep = 4 * T::kChunk, kBlock = U * kStep;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = lane % 16, k_lane = lane / 16 * T::kChunk;
  const E *pb[NB], *pa[MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
    pb[j] = row_of(j) + k_lane;
#pragma unroll
  for (int i = 0; i < MB; ++i)
    pa[i] = static_cast<const E *>(g.a[0]) + (size_t)min(i * 16 + row, g.M - 1) * g.lda[0] + k_lane;
  typename T::acc acc[NB][MB] = {};
  uint32_t sb[NB], sa[MB]; // bits to shift by
  if constexpr (ODD) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
      sb[j] = (uint32_t)(reinterpret_cast<uintptr_t>(pb[j]) & 3) * 8;
#pragma unroll
    for (int i = 0; i < MB; ++i)
      sa[i] = (uint32_t)(reinterpret_cast<uintptr_t>(pa[i]) & 3) * 8;
  }
  u32x4 fb[NB][U], fa[MB][U];
  uint32_t eb[NB], ea[MB]; // ODD: the words behind the last pieces
  auto fetch = [&](const E *p, uint32_t bits, u32x4 &v, uint32_t &last, bool is_last) {
    if constexpr (ODD) {
      typedef u32x4 u32x4_w __attribute__((aligned(4)));
      const uint32_t *w = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
      v = *reinterpret_cast<const u32x4_w *>(w);
      if (is_last) {
        last = 0;
        if (bits && lane >= 48)
          last = w[4];
      }
    } else {
      v = *reinterpret_cast<const u32x4_u *>(p);
    }
  };
  // the word behind a piece is the first one of the next piece of its row, which the lane 16
  // further holds, or lane - 48 in the next u
  auto place = [&](const u32x4 (&f)[U], int u, uint32_t last, uint32_t bits) {
    const u32x4 &v = f[u];
    if constexpr (!ODD)
      return v;
    const uint32_t give = u + 1 < U && lane < 16 ? f[u + 1 < U ? u + 1 : u][0] : v[0];
    const uint32_t got = (uint32_t)__builtin_amdgcn_ds_bpermute((lane + 16) % kWave * 4, (int)give);
    const uint32_t extra = u + 1 == U && lane >= 48 ? last : got;
    return u32x4{__builtin_amdgcn_alignbit(v[1], v[0], bits), __builtin_amdgcn_alignbit(v[2], v[1], bits),
                 __builtin_amdgcn_alignbit(v[3], v[2], bits), __builtin_amdgcn_alignbit(extra, v[3], bits)};
  };
  auto request = [&](int block) {
    const int k = block * kBlock;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
        fetch(pb[j] + k + u * kStep, sb[j], fb[j][u], eb[j], u == U - 1);
#pragma unroll
      for (int i = 0; i < MB; ++i)
        fetch(pa[i] + k + u * kStep, sa[i], fa[i][u], ea[i], u == U - 1);
    }
  };
  auto multiply = [&](const u32x4 (&b)[NB][U], const u32x4 (&a)[MB][U]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[j][i] = mma16<E>(b[j][u], a[i][u], acc[j][i]);
  };
  const int blocks = g.K / kBlock;
  if (wave < blocks)
    request(wave);
  for (int block = wave; block < blocks; block += 8) {
    u32x4 b[NB][U], a[MB][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
        b[j][u] = place(fb[j], u, eb[j], sb[j]);
#pragma unroll
      for (int i = 0; i < MB; ++i)
        a[i][u] = place(fa[i], u, ea[i], sa[i]);
    }
    if (block + 8 < blocks)
      request(block + 8);
    multiply(b, a);
  }
  if (wave == blocks % 8 && g.K % kBlock) { // what is left of k
    const int k = blocks * kBlock;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int valid = g.K - (k + u * kStep + k_lane);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        fb[j][u] = load_chunk(pb[j] + k + u * kStep, valid, g.K - valid);
#pragma unroll
      for (int i = 0; i < MB; ++i)
        fa[i][u] = load_chunk(pa[i] + k + u * kStep, valid, g.K - valid);
    }
    multiply(fb, fa);
  }
  using V = typename T::acc;
  V *cells = reinterpret_cast<V *>(lds); // [8][NB][MB][64]
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i)
      cells[((wave * NB + j) * MB + i) * kWave + lane] = acc[j][i];
  __syncthreads();
  // the eight waves' sums, added in their order, four elements a thread
  for (int c = threadIdx.x; c < NB * MB * kWave; c += 512) {
    V sum = cells[c];
#pragma unroll
    for (int w = 1; w < 8; ++w)
      sum += cells[w * (NB * MB * kWave) + c];
    cells[c] = sum; // (only this thread reads or writes this cell here)
  }
  __syncthreads();
}

// ---- stores ------------------------------------------------------------------
// The part of the result a workgroup stores: rows [m_lo, m_hi), columns [n_lo, n_hi).
struct Window {
  int m_lo, m_hi, n_lo, n_hi;
};

// four consecutive columns n .. n + 3 of one row, as far as they are in [lo, hi)
template <class O> __device__ __forceinline__ void store4(O *row, int n, int lo, int hi, f32x4 v) {
  typedef O ox4 __attribute__((ext_vector_type(4)));
  typedef ox4 ox4_u __attribute__((aligned(1)));
  ox4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = (O)v[e];
  if (n >= lo && n + 4 <= hi) {
    *reinterpret_cast<ox4_u *>(row + n) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e >= lo && n + e < hi)
        row[n + e] = o[e];
  }
}

// A wave's block of MI * 16 x NJ * 16 16-bit values through LDS (a region of the
// wave's own, MI * NJ * 512 bytes), so that whole row segments are written with
// 16-byte stores.  Chunk c of row r lies at c ^ (r & mask).  value(i, j): the lane's
// four consecutive columns of block (i, j).
template <class O, int MI, int NJ, class F>
__device__ __forceinline__ void store_block(unsigned char *mine, O *out, size_t ld, int m0, int n0, const Window &w,
                                            int lane, F &&value) {
  typedef O ox4 __attribute__((ext_vector_type(4)));
  constexpr int kRow = NJ * 32, kChunks = NJ * 2, kRows = kWave / kChunks;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const f32x4 v = value(i, j);
      ox4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = (O)v[e];
      const int r = i * 16 + lane % 16, c = 2 * j + lane / 32;
      *reinterpret_cast<ox4 *>(mine + r * kRow + ((c ^ (r & (kChunks - 1))) * 16) + lane / 16 % 2 * 8) = o;
    }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0));
#pragma unroll 4
  for (int r0 = 0; r0 < MI * 16; r0 += kRows) {
    const int r = r0 + lane / kChunks, c = lane % kChunks;
    const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + r * kRow + ((c ^ (r & (kChunks - 1))) * 16));
    const int m = m0 + r, n = n0 + c * 8;
    if (m < w.m_lo || m >= w.m_hi)
      continue;
    O *dst = out + (size_t)m * ld + n;
    if (n >= w.n_lo && n + 8 <= w.n_hi) {
      *reinterpret_cast<u32x4_u *>(dst) = v;
    } else {
      typedef O ox8 __attribute__((ext_vector_type(8)));
      const ox8 o = __builtin_bit_cast(ox8, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e >= w.n_lo && n + e < w.n_hi)
          dst[e] = o[e];
    }
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(kNoVm, 0)); // the region may be used again
}

// a wave's block straight from registers
template <class O, int MI, int NJ, class F>
__device__ __forceinline__ void store_direct(O *out, size_t ld, int m0, int n0, const Window &w, int lane, F &&value) {
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + i * 16 + lane % 16;
    if (m < w.m_lo || m >= w.m_hi)
      continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      store4<O>(out + (size_t)m * ld, n0 + j * 16 + lane / 16 * 4, w.n_lo, w.n_hi, value(i, j));
  }
}

// v * by as fp32 values, before they are rounded to a type: folded into the conversion the
// product would be rounded once in some kernels and twice in others.
__device__ __forceinline__ f32x4 times(f32x4 v, float by) {
  v *= by;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = v[e];
    asm volatile("" : "+v"(x));
    v[e] = x;
  }
  return v;
}

// C to `out` (element type) or `partial` (fp32; its rows are padded to a multiple of 8
// and the pipelined kernels' tiles begin at multiples of 8, so four columns are stored
// or not as a whole)
template <class E, int MI, int NI, bool LDS>
__device__ __forceinline__ void store_tile(const StoreArgs &s, f32x4 (&acc)[MI][NI], const Tile &t, int m0, int n0,
                                           int lane, int split, unsigned char *mine) {
  if (s.partial && !LDS) {
    store_direct<float, MI, NI>(s.partial + (size_t)split * s.mma.M * s.ldp, s.ldp, m0, n0,
                                Window{t.m_lo, s.mma.M, t.n_lo, s.mma.N}, lane, [&](int i, int j) { return acc[i][j]; });
    return;
  }
  if (s.partial) {
    float *base = s.partial + (size_t)split * s.mma.M * s.ldp + n0 + lane / 16 * 4;
    const int left = s.mma.N - n0 - lane / 16 * 4, skip = t.n_lo - n0 - lane / 16 * 4;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + i * 16 + lane % 16;
      if (m < t.m_lo || m >= s.mma.M)
        continue;
#pragma unroll
      for (int j = 0; j < NI; ++j)
        if (j * 16 < left && j * 16 >= skip)
          *reinterpret_cast<f32x4 *>(base + (size_t)m * s.ldp + j * 16) = acc[i][j];
    }
    return;
  }
  const Window w = {t.m_lo, s.mma.M, t.n_lo, s.mma.N};
  const float by = s.undo ? *s.undo : 1.0f;
  auto value = [&](int i, int j) { return times(acc[i][j], by); };
  if constexpr (LDS)
    store_block<E, MI, NI>(mine, static_cast<E *>(s.out), s.ldo, m0, n0, w, lane, value);
  else
    store_direct<E, MI, NI>(static_cast<E *>(s.out), s.ldo, m0, n0, w, lane, value);
}
// what the sums begin with: zero, or the partial sums of the calls before
template <int MI, int NI>
__device__ __forceinline__ void begin_tile(const StoreArgs &s, f32x4 (&acc)[MI][NI], int m0, int n0, int lane, int split) {
  if (!s.accumulate)
    return;
  typedef f32x4 f32x4_u __attribute__((aligned(4)));
  const float *base = s.partial + (size_t)split * s.mma.M * s.ldp;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const float *row = base + (size_t)min(m0 + i * 16 + lane % 16, s.mma.M - 1) * s.ldp;
#pragma unroll
    for (int j = 0; j < NI; ++j) // (columns past the padded row are not stored)
      acc[i][j] = *reinterpret_cast<const f32x4_u *>(row + min(n0 + j * 16 + lane / 16 * 4, (int)s.ldp - 4));
  }
}
struct FromZero {
  template <class A> __device__ __forceinline__ void operator()(A &, const Tile &, int, int, int) const {}
};

} // namespace hcamd
