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

#include <type_traits>

namespace hcamd {

enum Layout { kKFast = 0, kKSlow = 1 };

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_u __attribute__((aligned(1)));
typedef __attribute__((address_space(3))) s16x4 *lds_s16x4_ptr;

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
  tm = first + in % rows;
  tn = in / rows;
}

// 16 bytes of which the first `valid` elements exist; the rest reads as zero.
template <class E> __device__ __forceinline__ u32x4 load_chunk(const E *p, int valid) {
  constexpr int n = 16 / (int)sizeof(E);
  if (valid >= n)
    return *reinterpret_cast<const u32x4_u *>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
  if (valid <= 0)
    return v;
  if constexpr (sizeof(E) == 2) {
    const uint16_t *s = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e < valid)
        v[e / 2] |= (uint32_t)s[e] << (16 * (e % 2));
  } else {
    const uint8_t *s = reinterpret_cast<const uint8_t *>(p);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e < valid)
        v[e / 4] |= (uint32_t)s[e] << (8 * (e % 4));
  }
  return v;
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

// ---------------------------------------------------------------------------
// General kernel body: any sizes, leading dimensions and alignment.  128 x 128
// tile, four waves of 64 x 64, panels through registers (unaligned 16-byte
// loads, element loads where a chunk crosses an edge), two LDS stages, one
// barrier per K tile.  GATED: the N panel holds 32 rows of b[0], then the same 32
// of b[1], alternating, so that a wave's blocks j and j + 2 are the two
// projections of the same outputs.
// ---------------------------------------------------------------------------
template <class E, Layout LA, Layout LB, bool GATED, class Epilogue>
__device__ __forceinline__ void mma_general(const MmaArgs &g, unsigned char *lds, Epilogue &&epilogue) {
  using T = MmaType<E>;
  constexpr int BM = 128, BN = 128, BNO = GATED ? BN / 2 : BN;
  constexpr int kPanel = 128 * 128, kStage = 2 * kPanel;
  static_assert(sizeof(E) == 2 || (LA == kKFast && LB == kKFast), "transposed reads are for 16-bit elements");
  int tm, tn;
  tile_of(blockIdx.x, (g.M + BM - 1) / BM, (g.N + BNO - 1) / BNO, tm, tn);
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int wave_m = wave / 2 * 64, wave_n = wave % 2 * 64;
  const int tiles_k = (g.K + T::kBK - 1) / T::kBK, all = tiles_k * g.segments;
  const int split = blockIdx.y;
  const int kt0 = (int)((int64_t)all * split / g.splits), kt1 = (int)((int64_t)all * (split + 1) / g.splits);

  u32x4 ra[4], rb[4];
  auto load = [&](int kt) {
    const int seg = kt >= tiles_k ? 1 : 0;
    const int k0 = (kt - seg * tiles_k) * T::kBK;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int id = tid + i * 256;
      if constexpr (LA == kKFast) {
        const int m = tm * BM + id / 8, k = k0 + id % 8 * T::kChunk;
        const E *p = static_cast<const E *>(g.a[seg]) + (size_t)m * g.lda[seg] + k;
        ra[i] = load_chunk(p, m < g.M ? g.K - k : 0);
      } else {
        const int k = k0 + id / 16, m = tm * BM + id % 16 * 8;
        const E *p = static_cast<const E *>(g.a[seg]) + (size_t)k * g.lda[seg] + m;
        ra[i] = load_chunk(p, k < g.K ? g.M - m : 0);
      }
      if constexpr (LB == kKFast) {
        const int r = id / 8, k = k0 + id % 8 * T::kChunk;
        const int which = GATED ? r / 32 % 2 : seg;
        const int n = GATED ? tn * BNO + r / 64 * 32 + r % 32 : tn * BN + r;
        const E *p = static_cast<const E *>(g.b[which]) + (size_t)n * g.ldb[which] + k;
        rb[i] = load_chunk(p, n < g.N ? g.K - k : 0);
      } else {
        const int k = k0 + id / 16, n = tn * BN + id % 16 * 8;
        const E *p = static_cast<const E *>(g.b[seg]) + (size_t)k * g.ldb[seg] + n;
        rb[i] = load_chunk(p, k < g.K ? g.N - n : 0);
      }
    }
  };
  auto offset = [&](Layout l, int id) {
    if (l == kKFast)
      return fast_offset(id / 8, id % 8);
    const int k = id / 16, pos = id % 16;
    return k * 256 + (((pos / 2) ^ slow_swizzle(k)) * 32) + pos % 2 * 16;
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<u32x4 *>(lds + buf * kStage + offset(LA, tid + i * 256)) = ra[i];
      *reinterpret_cast<u32x4 *>(lds + buf * kStage + kPanel + offset(LB, tid + i * 256)) = rb[i];
    }
  };

  typename T::acc acc[4][4] = {};
  if (kt0 < kt1) {
    load(kt0);
    store(0);
    __syncthreads();
    for (int kt = kt0; kt < kt1; ++kt) {
      const int buf = (kt - kt0) & 1;
      if (kt + 1 < kt1)
        load(kt + 1);
      const unsigned char *pa = lds + buf * kStage, *pb = pa + kPanel;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fa[i] = read_operand<LA, 128>(pa, wave_m + i * 16, h, lane);
          fb[i] = read_operand<LB, 128>(pb, wave_n + i * 16, h, lane);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = mma16<E>(fb[j], fa[i], acc[i][j]);
      }
      if (kt + 1 < kt1)
        store(buf ^ 1);
      __syncthreads();
    }
  }
  epilogue(acc, tm * BM, wave_m, tn, wave_n, lane, lds);
}

// ---- stores ------------------------------------------------------------------
// four consecutive columns n .. n + 3 of one row, as far as they exist
template <class E>
__device__ __forceinline__ void store4(E *row, int n, int N, bool vec, f32x4 v) {
  typedef E ex4 __attribute__((ext_vector_type(4)));
  if (vec && n + 3 < N) {
    ex4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = (E)v[e];
    *reinterpret_cast<ex4 *>(row + n) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N)
        row[n + e] = (E)v[e];
  }
}
template <class E> __device__ __forceinline__ bool can_store4(const void *p, size_t ld) {
  return ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(E)) == 0;
}

// C to `out` (element type) or `partial` (fp32)
template <class E, int MI, int NI, int BN>
__device__ __forceinline__ void store_tile(const StoreArgs &s, f32x4 (&acc)[MI][NI], int m0, int n0, int lane) {
  const int M = s.mma.M, N = s.mma.N;
  if (s.partial) {
    const bool vec = can_store4<float>(s.partial, s.ldp);
    float *base = s.partial + (size_t)blockIdx.y * M * s.ldp;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + i * 16 + lane % 16;
      if (m >= M)
        continue;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int n = n0 + j * 16 + lane / 16 * 4;
        float *row = base + (size_t)m * s.ldp;
        f32x4 v = acc[i][j];
        if (s.accumulate) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N)
              v[e] += row[n + e];
        }
        store4<float>(row, n, N, vec, v);
      }
    }
    return;
  }
  const float by = s.undo ? *s.undo : 1.0f;
  const bool vec = can_store4<E>(s.out, s.ldo);
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + i * 16 + lane % 16;
    if (m >= M)
      continue;
#pragma unroll
    for (int j = 0; j < NI; ++j)
      store4<E>(static_cast<E *>(s.out) + (size_t)m * s.ldo, n0 + j * 16 + lane / 16 * 4, N, vec, acc[i][j] * by);
  }
}

} // namespace hcamd
