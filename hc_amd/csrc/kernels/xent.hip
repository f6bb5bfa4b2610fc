// Softmax cross entropy of the product z = x W' against target columns, and its
// gradients, without the logits ever being stored.  x [T,D], W [V,D].
//
// Forward: the product's tiles end in per-row statistics (maximum, sum of
// exp(z - maximum)) and the target's logit; a second kernel joins the tiles of a
// row: lse = log sum exp z, loss = lse - z[target].
// Backward, vocabulary piece by piece: the product again with
// p = (exp(z - lse) - onehot) * grad_loss as its epilogue, then
//   dx += p W   (fp32 partial sums, folded once at the end)    dW = p' x
// p is rounded to the element type because it is a matrix operand.
//
// A target below 0 takes its row out: loss 0, no gradient.  A target of V or more
// is an error of the caller's: loss NaN, no gradient.
#include "mma.h"

using namespace hcamd;

namespace {

__device__ __forceinline__ int64_t target_of(const void *targets, int is64, size_t row) {
  return is64 ? static_cast<const int64_t *>(targets)[row] : (int64_t)static_cast<const int32_t *>(targets)[row];
}

__device__ __forceinline__ bool takes_part(const void *targets, int is64, size_t row, uint32_t vocab) {
  const int64_t t = target_of(targets, is64, row);
  return t >= 0 && t < (int64_t)vocab;
}

// The products dominate: 4096 x 4096 x 131072 bf16 forward 3.2 ms (1.37 PFLOP/s), backward a
// piece of 16384 rows p 453 us, dx 452 us, dW 478 us.

// What is subtracted before the exponentials: the largest value, or 0 where that is infinite.  The terms
// of a row of -infinities are then 0, +infinity gives an infinite sum (its difference with itself
// would be NaN), and a NaN, which no maximum takes, makes the sum NaN.
__device__ __forceinline__ float subtracted(float most) { return __builtin_fabsf(most) == INFINITY ? 0.0f : most; }

// per-row statistics of a tile: lanes l, l + 16, l + 32, l + 48 hold one row's
// columns; WN waves share the row and meet in LDS
template <int MI, int NI, int WN, int BM, int BN>
__device__ __forceinline__ void tile_stats(const XentArgs &a, f32x4 (&acc)[MI][NI], const Tile &t, int wave_m,
                                           int wave_n, int lane, float *lds) {
  const int M = a.mma.M, N = a.mma.N;
  const int wn = wave_n / (NI * 16);
  float *slot_m = lds, *slot_s = lds + WN * BM; // [WN][BM] each
  const int n0 = t.n0 + wave_n + lane / 16 * 4;
  const bool whole = t.n0 >= t.n_lo && t.n0 + BN <= N;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int in_tile = wave_m + i * 16 + lane % 16, m = t.m0 + in_tile;
    if (m >= t.m_lo && m < M) {
      const int64_t at = target_of(a.targets, a.target_i64, m) - a.v0 - n0;
      if (at >= 0 && at < NI * 16) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at == j * 16 + e && n0 + j * 16 + e >= t.n_lo && n0 + j * 16 + e < N)
              a.zt[m] = acc[i][j][e];
      }
    }
    if (!whole) { // columns past the last, or a neighbour's, take no part
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n0 + j * 16 + e < t.n_lo || n0 + j * 16 + e >= N)
            acc[i][j][e] = -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        most = fmaxf(most, acc[i][j][e]);
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const float from = subtracted(most);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sum += __expf(acc[i][j][e] - from);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16) {
      slot_m[wn * BM + in_tile] = most;
      slot_s[wn * BM + in_tile] = sum;
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < BM; r += blockDim.x) {
    const int m = t.m0 + r;
    if (m < t.m_lo || m >= M)
      continue;
    float most = slot_m[r];
#pragma unroll
    for (int w = 1; w < WN; ++w)
      most = fmaxf(most, slot_m[w * BM + r]);
    const float from = subtracted(most);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WN; ++w)
      sum += slot_s[w * BM + r] * __expf(slot_m[w * BM + r] - from);
    float *cell = a.stats + ((size_t)m * a.tiles + a.tile0 + t.tn) * 2;
    cell[0] = most;
    cell[1] = sum;
  }
}

template <class E, int BM> __device__ __forceinline__ void stats_general(const XentArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * (BM + 128) * 128];
  mma_general<E, kKFast, kKFast, false, BM>(
      a.mma, blockIdx.x, 0, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *l) {
        // (the main loop ends with a barrier: its stages are free)
        tile_stats<BM / 32, 4, 2, BM, 128>(a, acc, t, wave_m, wave_n, lane, reinterpret_cast<float *>(l));
      });
}

template <class E, int B> __device__ __forceinline__ void stats_tile(const XentArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[pipelined_lds<B>()];
  mma_tiles<E, kKFast, kKFast, false, B>(
      a.mma, blockIdx.x, 0, a.mma.half_from, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *l) {
        constexpr int MI = sizeof(acc) / sizeof(acc[0]), NI = sizeof(acc[0]) / sizeof(acc[0][0]);
        constexpr int WN = B / (NI * 16), BM = MI * 16 * 2;
        tile_stats<MI, NI, WN, BM, B>(a, acc, t, wave_m, wave_n, lane, reinterpret_cast<float *>(l));
      });
}

// Few tokens: one pass over the weight, NB * 16 of its rows a workgroup.  NB 4, U 2: 57 us
// for one token and 62 us for 32 over 32000 x 4096 bf16 with the joining (4.6 and 4.3
// TB/s); NB 2, U 4: 65 and 85 us (x is read once per workgroup).  Beyond 32 tokens NB 2: LDS.
template <class E, int MB, int NB, int U, bool ODD> __device__ __forceinline__ void stats_few(const XentArgs &a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[skinny_lds<MB, NB>()];
  const int n0 = blockIdx.x * (NB * 16), left = a.mma.N - n0;
  mma_skinny<E, MB, NB, U, ODD>(
      a.mma,
      [&](int j) {
        const int n = min(n0 + j * 16 + (int)threadIdx.x % 16, a.mma.N - 1);
        return static_cast<const E *>(a.mma.b[0]) + (size_t)n * a.mma.ldb[0];
      },
      lds);
  const float *cells = reinterpret_cast<const float *>(lds);
  for (int c = threadIdx.x; c < MB * 256; c += 512) {
    const int n = c % 16, m = c / 16; // sixteen lanes share a row, a column of each block
    const int at = m / 16 * 256 + ((n / 4) * 16 + m % 16) * 4 + n % 4;
    float z[NB], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      z[j] = n + j * 16 < left ? cells[j * MB * 256 + at] : -INFINITY;
      most = fmaxf(most, z[j]);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      most = fmaxf(most, __shfl_xor(most, o));
    const float from = subtracted(most);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; ++j)
      sum += __expf(z[j] - from);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      sum += __shfl_xor(sum, o);
    if (m >= a.mma.M)
      continue;
    const int64_t t = target_of(a.targets, a.target_i64, m) - a.v0 - n0;
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (t == n + j * 16 && n + j * 16 < left)
        a.zt[m] = z[j];
    if (n == 0) {
      float *cell = a.stats + ((size_t)m * a.tiles + a.tile0 + blockIdx.x) * 2;
      cell[0] = most;
      cell[1] = sum;
    }
  }
}

// p of a tile; the columns up to the next multiple of 8 become zeros (the products
// that read p take it in pieces of 8)
template <class E, int MI, int NI, bool LDS>
__device__ __forceinline__ void tile_p(const XentArgs &a, f32x4 (&acc)[MI][NI], const Tile &tile, int m0, int n0,
                                       int lane, unsigned char *mine) {
  const int M = a.mma.M, N = a.mma.N, padded = (N + 7) & ~7;
  const float factor = *a.factor;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = min(m0 + i * 16 + lane % 16, M - 1);
    const int64_t t = target_of(a.targets, a.target_i64, m);
    const bool live = t >= 0 && t < a.vocab;
    // the target's column counted from this lane's first, -1 for none
    const int64_t from = t - a.v0 - (n0 + lane / 16 * 4);
    const int hot = live && from >= 0 && from < NI * 16 ? (int)from : -1;
    const float g = live ? a.grad_loss[m] * factor : 0.0f, lse = a.lse[m];
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __expf(acc[i][j][e] - lse) - (hot == j * 16 + e ? 1.0f : 0.0f);
        // a row without a target: 0, whatever its logits are
        acc[i][j][e] = live ? p * g : 0.0f;
      }
  }
  const Window w = {tile.m_lo, M, tile.n_lo, N};
  // the padding is written by the lanes of the tile that holds the last column
  if (n0 < N && n0 + NI * 16 >= N && N < padded) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int m = m0 + i * 16 + lane % 16;
      if (m >= tile.m_lo && m < M)
        for (int n = N + lane / 16; n < padded; n += 4)
          static_cast<E *>(a.p)[(size_t)m * a.ldp + n] = (E)0.0f;
    }
  }
  auto value = [&](int i, int j) { return acc[i][j]; };
  if constexpr (LDS)
    store_block<E, MI, NI>(mine, static_cast<E *>(a.p), a.ldp, m0, n0, w, lane, value);
  else
    store_direct<E, MI, NI>(static_cast<E *>(a.p), a.ldp, m0, n0, w, lane, value);
}

template <class E, int BM> __device__ __forceinline__ void p_general(const XentArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * (BM + 128) * 128];
  mma_general<E, kKFast, kKFast, false, BM>(
      a.mma, blockIdx.x, 0, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *) {
        tile_p<E, BM / 32, 4, false>(a, acc, t, t.m0 + wave_m, t.n0 + wave_n, lane, nullptr);
      });
}
template <class E, int B> __device__ __forceinline__ void p_tile(const XentArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[pipelined_lds<B>()];
  mma_tiles<E, kKFast, kKFast, false, B>(
      a.mma, blockIdx.x, 0, a.mma.half_from, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *l) {
        constexpr int MI = sizeof(acc) / sizeof(acc[0]), NI = sizeof(acc[0]) / sizeof(acc[0][0]);
        tile_p<E, MI, NI, true>(a, acc, t, t.m0 + wave_m, t.n0 + wave_n, lane,
                                l + threadIdx.x / kWave * (MI * NI * 512));
      });
}

// Few tokens, as in the forward pass: one pass over the piece's rows of the weight, which
// the tiles feed from too few workgroups (8 tokens, 32000 x 4096 bf16: 90 us in tiles).
template <class E, int MB, int NB, int U, bool ODD> __device__ __forceinline__ void p_few(const XentArgs &a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[skinny_lds<MB, NB>()];
  const int n0 = blockIdx.x * (NB * 16), N = a.mma.N;
  mma_skinny<E, MB, NB, U, ODD>(
      a.mma,
      [&](int j) {
        const int n = min(n0 + j * 16 + (int)threadIdx.x % 16, N - 1);
        return static_cast<const E *>(a.mma.b[0]) + (size_t)n * a.mma.ldb[0];
      },
      lds);
  const f32x4 *cells = reinterpret_cast<const f32x4 *>(lds);
  const float factor = *a.factor;
  for (int c = threadIdx.x; c < MB * 16 * NB * 4; c += 512) { // four columns of a row
    const int m = c / (NB * 4), quad = c % (NB * 4), n = n0 + quad * 4;
    if (m >= a.mma.M || n >= N)
      continue;
    const int64_t t = target_of(a.targets, a.target_i64, m);
    const bool live = t >= 0 && t < a.vocab;
    f32x4 v = cells[(quad / 4 * MB + m / 16) * 64 + quad % 4 * 16 + m % 16];
    const float g = live ? a.grad_loss[m] * factor : 0.0f, lse = a.lse[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = __expf(v[e] - lse) - (t == a.v0 + n + e ? 1.0f : 0.0f);
      v[e] = live && n + e < N ? p * g : 0.0f;
    }
    const int padded = (N + 7) & ~7;
    E *row = static_cast<E *>(a.p) + (size_t)m * a.ldp;
    store4(row, n, 0, padded, v);
    if (n + 4 >= N && n + 4 < padded)
      store4(row, n + 4, 0, padded, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
  }
}

// one wave per row joins the tiles' statistics
__device__ __forceinline__ void rows_join(const XentRowsArgs &a) {
  const int lane = threadIdx.x % kWave;
  const size_t row = (size_t)blockIdx.x * (blockDim.x / kWave) + threadIdx.x / kWave;
  if (row >= a.rows)
    return;
  const f32x2 *cells = reinterpret_cast<const f32x2 *>(a.stats) + row * a.tiles;
  float most = -INFINITY;
  for (uint32_t t = lane; t < a.tiles; t += kWave)
    most = fmaxf(most, cells[t][0]);
  most = wave_reduce<MaxOp>(most);
  const float from = subtracted(most);
  float sum = 0.0f;
  for (uint32_t t = lane; t < a.tiles; t += kWave)
    sum += cells[t][1] * __expf(cells[t][0] - from);
  sum = wave_reduce<SumOp>(sum);
  if (lane == 0) {
    const float lse = most + logf(sum);
    const int64_t t = target_of(a.targets, a.target_i64, row);
    a.lse[row] = lse;
    a.loss[row] = t < 0 ? 0.0f : t >= a.vocab ? __builtin_nanf("") : lse - a.zt[row];
  }
}

// What p is multiplied by before it is rounded, factor[0], and what undoes it in the
// products, factor[1]: the largest |grad_loss| becomes 1 (bf16) or 2^15 (fp16).  With
// the usual grad_loss, one value for every live row, the -1 at a target is then
// represented exactly, where -grad_loss itself would carry one and the same rounding
// error into every row's largest entry (gradients that differ from row to row are rounded
// there, each by itself); and fp16 keeps the small p of a large
// vocabulary above its subnormals.  The first workgroup.
__device__ __forceinline__ void p_factor(const XentPrepareArgs &a) {
  __shared__ float slots[16];
  float most = 0.0f;
  for (uint32_t r = threadIdx.x; r < a.rows; r += blockDim.x)
    if (takes_part(a.targets, a.target_i64, r, a.vocab))
      most = fmaxf(most, fabsf(a.grad_loss[r]));
  most = group_reduce<MaxOp, 16>(most, slots);
  if (threadIdx.x == 0) {
    const bool usable = most > 0x1p-100f && most < 0x1p100f;
    a.factor[0] = usable ? a.top / most : 1.0f;
    a.factor[1] = usable ? most / a.top : 1.0f;
  }
}

// x as the weight's gradient takes it: rows that take no part are zeros, so that
// whatever stands in them (padding, NaN) meets no zero of p in a product; rows are
// padded to pieces of 8.  The other workgroups.
template <class E> __device__ __forceinline__ void live_rows(const XentPrepareArgs &a) {
  const uint32_t pieces = (a.cols + 7) / 8;
  const uint64_t total = (uint64_t)a.rows * pieces;
  for (uint64_t id = (uint64_t)(blockIdx.x - 1) * blockDim.x + threadIdx.x; id < total;
       id += (uint64_t)(gridDim.x - 1) * blockDim.x) {
    const uint32_t r = (uint32_t)(id / pieces), c = (uint32_t)(id % pieces) * 8;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (takes_part(a.targets, a.target_i64, r, a.vocab))
      v = load_chunk(static_cast<const E *>(a.x) + (size_t)r * a.ldx + c, (int)a.cols - (int)c, (int)c);
    *reinterpret_cast<u32x4 *>(static_cast<E *>(a.live_x) + (size_t)r * a.ldl + c) = v;
  }
}

} // namespace

#define HCAMD_XENT(SUFFIX, E)                                                                             \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_stats_##SUFFIX##_general(XentArgs a) {     \
    stats_general<E, 128>(a);  \
  }  \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_stats_##SUFFIX##_half(XentArgs a) {  \
    stats_general<E, 64>(a);  \
  }  \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_p_##SUFFIX##_general(XentArgs a) {         \
    p_general<E, 128>(a);  \
  }  \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_p_##SUFFIX##_half(XentArgs a) {  \
    p_general<E, 64>(a);  \
  }  \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_stats_##SUFFIX##_t256(XentArgs a) {        \
    stats_tile<E, 256>(a);                                                                          \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_stats_##SUFFIX##_t128(XentArgs a) {        \
    stats_tile<E, 128>(a);                                                                          \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_p_##SUFFIX##_t256(XentArgs a) {            \
    p_tile<E, 256>(a);                                                                              \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_xent_p_##SUFFIX##_t128(XentArgs a) {            \
    p_tile<E, 128>(a);                                                                              \
  }
HCAMD_XENT(bf16, __bf16)
HCAMD_XENT(f16, _Float16)
#define HCAMD_XENT_FEW(SUFFIX, E, ROWS, NB, U)                                                            \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_stats_##SUFFIX##_s##ROWS(XentArgs a) {     \
    stats_few<E, ROWS / 16, NB, U, false>(a);                                                             \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_stats_##SUFFIX##_s##ROWS##odd(XentArgs a) { \
    stats_few<E, ROWS / 16, NB, U, true>(a);                                                              \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_p_##SUFFIX##_s##ROWS(XentArgs a) {         \
    p_few<E, ROWS / 16, NB, U, false>(a);                                                                 \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_xent_p_##SUFFIX##_s##ROWS##odd(XentArgs a) {    \
    p_few<E, ROWS / 16, NB, U, true>(a);                                                                  \
  }
HCAMD_XENT_FEW(bf16, __bf16, 16, 4, 2)
HCAMD_XENT_FEW(bf16, __bf16, 32, 4, 2)
HCAMD_XENT_FEW(bf16, __bf16, 64, 2, 2)
HCAMD_XENT_FEW(bf16, __bf16, 128, 2, 1)
HCAMD_XENT_FEW(f16, _Float16, 16, 4, 2)
HCAMD_XENT_FEW(f16, _Float16, 32, 4, 2)
HCAMD_XENT_FEW(f16, _Float16, 64, 2, 2)
HCAMD_XENT_FEW(f16, _Float16, 128, 2, 1)
extern "C" __global__ __launch_bounds__(256) void hcamd_xent_rows(XentRowsArgs a) { rows_join(a); }
// (live rows are a copy of 16-bit values: one kernel for both types)
extern "C" __global__ __launch_bounds__(1024) void hcamd_xent_prepare(XentPrepareArgs a) {
  if (blockIdx.x == 0)
    p_factor(a);
  else
    live_rows<uint16_t>(a);
}
