// h = x + residual (rounded to the element type: what the residual stream keeps
// is what is normalised), y = h * rstd * weight, rstd = 1 / sqrt(mean(h^2) + eps),
// over the rows of a matrix.  y is stored in the element type, or in 8 bits with a
// scale per row: v = h * weight, most = max |v|, q = rint(127 v / most), scale =
// rstd * most / 127.  rstd is a common factor of a row and cancels in q.
//
// q is decided in 64 bits where 32 could round to the other neighbour: 127 v / most
// has at most one rounding there, so ties are ties and go to the even number, and q
// does not depend on the order of any sum.
//
// Backward: with a = grad_out * weight and n = h * rstd,
//   grad_in = grad_summed + rstd * (a - n * mean(a n)),  grad_weight = sum over rows of grad_out n.
#include "common.h"
#include "op_args.h"
#include "pieces.h"

using namespace hcamd;

namespace {


__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v = fmax(v, __shfl_xor(v, o));
  return v;
}

__device__ __forceinline__ int8_t quantise64(float h, float w, double most) {
  return (int8_t)__builtin_rint(127.0 * ((double)h * (double)w) / most);
}
// 127 v / most, rounded half to even.  The fp32 quotient h * w * per is off by less
// than 127 * 4 * 2^-24 < 2^-15: only one that close to a half asks for 64 bits (and a
// NaN, which `per` is for rows outside fp32's comfortable range).
__device__ __forceinline__ int8_t quantise(float h, float w, float per, double most) {
  const float t = h * w * per;
  const float q = __builtin_rintf(t);
  return !(__builtin_fabsf(t - q) <= 0.5f - 0x1p-14f) ? quantise64(h, w, most) : (int8_t)q;
}

// rstd * most / 127; NaN for a row that is not finite, 0 for one of zeros (whose rstd is
// infinite where eps is 0)
__device__ __forceinline__ float scale_of(double most, float rstd) {
  return !(most < (double)INFINITY) ? __builtin_nanf("") : most > 0.0 ? (float)(most * rstd / 127.0) : 0.0f;
}

template <class T, class W> struct Row {
  const T *x, *r;
  const W *w;
  __device__ __forceinline__ float h(uint32_t c) const {
    float v = (float)x[c];
    if (r)
      v = (float)(T)(v + (float)r[c]);
    return v;
  }
  __device__ __forceinline__ float weight(uint32_t c) const { return w ? (float)w[c] : 1.0f; }
};

// One workgroup per row, element by element, the row read twice: rows of more
// than 16384 columns, which registers do not hold.  (summed and out may be x or residual: a thread reads an
// element before it writes it, and no other thread touches it.)
template <class T, class W, bool I8> __device__ __forceinline__ void norm_general(const NormArgs &a) {
  __shared__ float slots[4];
  __shared__ double slots64[4];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const Row<T, W> in = {static_cast<const T *>(a.x) + row * a.ldx,
                          a.residual ? static_cast<const T *>(a.residual) + row * a.ldr : nullptr,
                          static_cast<const W *>(a.weight)};
    float sum = 0.0f;
    double most = 0.0;
    bool bad = false;
    for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
      const float h = in.h(c);
      sum = __builtin_fmaf(h, h, sum);
      if constexpr (I8) {
        const double v = __builtin_fabs((double)h * (double)in.weight(c));
        bad |= !(v < (double)INFINITY);
        most = fmax(most, v);
      }
    }
    sum = group_reduce<SumOp, 4>(sum, slots);
    const float rstd = 1.0f / __builtin_sqrtf(sum / (float)a.cols + a.eps);
    if constexpr (I8) {
      if (bad)
        most = (double)INFINITY;
      most = wave_max64(most);
      if (lane == 0)
        slots64[wave] = most;
      __syncthreads();
      most = fmax(fmax(slots64[0], slots64[1]), fmax(slots64[2], slots64[3]));
    }
    // a row with a value that is not finite has no 8-bit form: q 0, scale NaN
    const bool usable = most > 0.0 && most < (double)INFINITY;
    const float per = most > 0x1p-60 && most < 0x1p60 ? 127.0f / (float)most : __builtin_nanf("");
    for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
      const float h = in.h(c), w = in.weight(c);
      if (a.summed)
        static_cast<T *>(a.summed)[row * a.lds + c] = (T)h;
      if constexpr (I8)
        static_cast<int8_t *>(a.out)[row * a.ldo + c] = usable ? quantise(h, w, per, most) : (int8_t)0;
      else
        static_cast<T *>(a.out)[row * a.ldo + c] = (T)(h * rstd * w);
    }
    if (threadIdx.x == 0) {
      if (a.rstd)
        a.rstd[row] = rstd;
      if constexpr (I8)
        a.scale[row] = scale_of(most, rstd);
    }
    __syncthreads(); // the slots are used again
  }
}

// grad_in: one workgroup per row; grad_in may be grad_out or grad_summed
template <class T, class W> __device__ __forceinline__ void back_general(const NormBackArgs &a) {
  __shared__ float slots[4];
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *dy = static_cast<const T *>(a.grad_out) + row * a.ldg;
    const T *h = static_cast<const T *>(a.summed) + row * a.ldh;
    const T *ds = a.grad_summed ? static_cast<const T *>(a.grad_summed) + row * a.ldgs : nullptr;
    const W *w = static_cast<const W *>(a.weight);
    const float rstd = a.rstd[row];
    float dot = 0.0f;
    for (uint32_t c = threadIdx.x; c < a.cols; c += 256)
      dot += (float)dy[c] * (w ? (float)w[c] : 1.0f) * ((float)h[c] * rstd);
    dot = group_reduce<SumOp, 4>(dot, slots) / (float)a.cols;
    for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
      const float n = (float)h[c] * rstd;
      float v = rstd * ((float)dy[c] * (w ? (float)w[c] : 1.0f) - n * dot);
      if (ds)
        v += (float)ds[c];
      static_cast<T *>(a.grad_in)[row * a.ldgi + c] = (T)v;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Rows in registers: TPR lanes share a row, lane t holds its 16-byte pieces t, t + TPR,
// ... (VPT of them), so a row is read once and every wave-level access covers
// consecutive bytes.  A workgroup of T lanes walks groups of T / TPR rows; the weight
// stays in registers, the pieces of the next rows are requested before the sums of the
// present ones are joined.
// Bound by memory: 8192 x 4096 bf16 forward with sum 46 us (5.8 TB/s), backward 47 us (5.7
// TB/s); 16384 x 4096 fp16 to 8 bits 94 us (5.0 TB/s; the rounding's arithmetic shows).  Rows
// that begin at odd addresses go in unaligned pieces: 16384 x 4095 bf16 forward 133 us (4.0
// TB/s), to 8 bits 120 us, backward 114 us.  Four rows: 4 us, the latency of a launch.
// ---------------------------------------------------------------------------
template <class T> constexpr int kPiece = 16 / (int)sizeof(T);
template <class T> using Piece __attribute__((ext_vector_type(kPiece<T>))) = T;

template <class T, int TPR, int VPT>
__device__ __forceinline__ void load_pieces(u32x4 (&v)[VPT], const T *row, uint32_t cols, int t) {
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (j * TPR + t) * kPiece<T>;
    v[j] = load_chunk(row + c, (int)cols - c, c);
  }
}
// the weight's values for those pieces (1 where there is none; 0 past the row)
template <class T, int TPR, int VPT>
__device__ __forceinline__ void load_weight(float (&w)[VPT][kPiece<T>], const void *weight, int is_f32, uint32_t cols,
                                            int t) {
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e) {
      const uint32_t c = (uint32_t)(j * TPR + t) * kPiece<T> + e;
      w[j][e] = c >= cols ? 0.0f
                : !weight ? 1.0f
                : is_f32  ? static_cast<const float *>(weight)[c]
                          : (float)static_cast<const T *>(weight)[c];
    }
}
template <class Op, int TPR> __device__ __forceinline__ typename Op::T row_reduce(typename Op::T v, typename Op::T *slots) {
  return group_reduce<Op, TPR / kWave>(v, slots + threadIdx.x / TPR * (TPR / kWave));
}

template <class T, int TPR, int VPT, int kThreads, bool I8>
__device__ __forceinline__ void norm_rows(const NormArgs &a) {
  constexpr int N = kPiece<T>, kRows = kThreads / TPR, kWaves = kThreads / kWave;
  __shared__ float slots[2][kWaves];
  __shared__ double slots64[2][kWaves];
  const int t = threadIdx.x % TPR;
  const uint32_t rg = threadIdx.x / TPR, cols = a.cols;
  const T *x = static_cast<const T *>(a.x), *r = static_cast<const T *>(a.residual);
  float w[VPT][N];
  load_weight<T, TPR, VPT>(w, a.weight, a.weight_f32, cols, t);
  u32x4 px[VPT], pr[VPT];
  uint32_t row = blockIdx.x * kRows + rg;
  auto request = [&](uint32_t q) {
    const size_t from = q < a.rows ? q : 0; // (every lane takes part in the joining)
    load_pieces<T, TPR, VPT>(px, x + from * a.ldx, cols, t);
    if (r)
      load_pieces<T, TPR, VPT>(pr, r + from * a.ldr, cols, t);
  };
  request(row);
  // rows of a workgroup advance together
  for (uint32_t first = blockIdx.x * kRows, it = 0; first < a.rows; first += gridDim.x * kRows, row += gridDim.x * kRows, ++it) {
    const bool mine = row < a.rows;
    float h[VPT][N];
    float sum = 0.0f;
    double most = 0.0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const Piece<T> vx = __builtin_bit_cast(Piece<T>, px[j]);
      Piece<T> vh = vx;
      if (r) {
        const Piece<T> vr = __builtin_bit_cast(Piece<T>, pr[j]);
#pragma unroll
        for (int e = 0; e < N; ++e)
          vh[e] = (T)((float)vx[e] + (float)vr[e]);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        h[j][e] = (float)vh[e];
        sum = __builtin_fmaf(h[j][e], h[j][e], sum);
        if constexpr (I8) {
          // (elements past the row are zeros times a weight of 0)
          const double v = __builtin_fabs((double)h[j][e] * (double)w[j][e]);
          bad |= !(v < (double)INFINITY);
          most = fmax(most, v);
        }
      }
      if (a.summed && mine) {
        const int c = (j * TPR + t) * N;
        store_chunk(static_cast<T *>(a.summed) + (size_t)row * a.lds + c, __builtin_bit_cast(u32x4, vh), (int)cols - c);
      }
    }
    // (in place the next row may be written only by its own lanes: it is another row)
    if (first + gridDim.x * kRows < a.rows)
      request(row + gridDim.x * kRows);
    if constexpr (I8) {
      if (bad)
        most = (double)INFINITY;
      most = wave_max64(most);
      if (TPR > kWave && threadIdx.x % kWave == 0)
        slots64[it & 1][threadIdx.x / kWave] = most;
    }
    // (one barrier, inside: the slots alternate from row to row)
    sum = row_reduce<SumOp, TPR>(sum, slots[it & 1]);
    const float rstd = 1.0f / __builtin_sqrtf(sum / (float)cols + a.eps);
    if constexpr (I8 && TPR > kWave) {
      const double *s = slots64[it & 1] + rg * (TPR / kWave);
      most = s[0];
#pragma unroll
      for (int k = 1; k < TPR / kWave; ++k)
        most = fmax(most, s[k]);
    }
    if (!mine)
      continue;
    if (t == 0) {
      if (a.rstd)
        a.rstd[row] = rstd;
      if constexpr (I8)
        a.scale[row] = scale_of(most, rstd);
    }
    const bool usable = most > 0.0 && most < (double)INFINITY;
    const float per = most > 0x1p-60 && most < 0x1p60 ? 127.0f / (float)most : __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * TPR + t) * N, valid = (int)cols - c;
      if (valid <= 0)
        continue;
      if constexpr (I8) {
        uint32_t o[N / 4];
        bool near_half = false;
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
          o[k] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = h[j][4 * k + e] * w[j][4 * k + e] * per, q = __builtin_rintf(v);
            near_half |= !(__builtin_fabsf(v - q) <= 0.5f - 0x1p-14f);
            o[k] |= (uint32_t)(uint8_t)(int)q << (8 * e);
          }
        }
        // one piece in 2^10: 64 bits decide
        if (near_half || !usable) {
#pragma unroll
          for (int k = 0; k < N / 4; ++k) {
            o[k] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[k] |= (uint32_t)(uint8_t)(usable ? quantise64(h[j][4 * k + e], w[j][4 * k + e], most) : 0) << (8 * e);
          }
        }
        int8_t *out = static_cast<int8_t *>(a.out) + (size_t)row * a.ldo + c;
        if (valid >= N) {
          if constexpr (N == 8)
            *reinterpret_cast<u32x2_u *>(out) = u32x2{o[0], o[1]};
          else
            __builtin_memcpy(out, o, 4);
        } else {
          store_chunk(out, u32x4{o[0], N == 8 ? o[N / 4 - 1] : 0u, 0u, 0u}, valid);
        }
      } else {
        Piece<T> o;
#pragma unroll
        for (int e = 0; e < N; ++e)
          o[e] = (T)(h[j][e] * rstd * w[j][e]);
        store_chunk(static_cast<T *>(a.out) + (size_t)row * a.ldo + c, __builtin_bit_cast(u32x4, o), valid);
      }
    }
  }
}

// The backward pass in the same way; a lane's columns are the same in every row, so it
// keeps their part of grad_weight in registers, one line of `partial` per workgroup.
template <class T, int TPR, int VPT, int kThreads>
__device__ __forceinline__ void back_rows(const NormBackArgs &a) {
  // (1024 lanes have 128 registers each: no room for the next row's pieces, and the longest rows
  // keep a few values in scratch memory: 12 registers' worth in 16 bits, 25 in fp32, 28 in fp32
  // to 8 bits forward.  4096 x 16384 fp32 195 us forward (5.5 TB/s), 206 us to 8 bits, 237 us backward
  // (4.5 TB/s); rows of 20000 columns, read twice instead, take 1.9, 2.4 and 1.9 times as long a column.)
  constexpr bool kAhead = kThreads < 1024;
  constexpr int N = kPiece<T>, kRows = kThreads / TPR, kWaves = kThreads / kWave;
  __shared__ float slots[2][kWaves];
  __shared__ float joined[kRows > 1 ? kRows : 1][kRows > 1 ? TPR * VPT * N : 1];
  const int t = threadIdx.x % TPR;
  const uint32_t rg = threadIdx.x / TPR, cols = a.cols;
  const T *dy = static_cast<const T *>(a.grad_out), *hs = static_cast<const T *>(a.summed);
  const T *ds = static_cast<const T *>(a.grad_summed);
  float w[VPT][N], dw[VPT][N] = {};
  load_weight<T, TPR, VPT>(w, a.weight, a.weight_f32, cols, t);
  u32x4 pg[VPT], ph[VPT], ps[VPT];
  float next_rstd = 0.0f;
  uint32_t row = blockIdx.x * kRows + rg;
  auto request = [&](uint32_t q) {
    const size_t from = q < a.rows ? q : 0;
    load_pieces<T, TPR, VPT>(pg, dy + from * a.ldg, cols, t);
    load_pieces<T, TPR, VPT>(ph, hs + from * a.ldh, cols, t);
    if (ds)
      load_pieces<T, TPR, VPT>(ps, ds + from * a.ldgs, cols, t);
    next_rstd = a.rstd[from];
  };
  if (kAhead)
    request(row);
  for (uint32_t first = blockIdx.x * kRows, it = 0; first < a.rows; first += gridDim.x * kRows, row += gridDim.x * kRows, ++it) {
    const bool mine = row < a.rows;
    if (!kAhead)
      request(row);
    const float rstd = next_rstd;
    float g[VPT][N], n[VPT][N], s[VPT][N];
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const Piece<T> vg = __builtin_bit_cast(Piece<T>, pg[j]), vh = __builtin_bit_cast(Piece<T>, ph[j]);
      const Piece<T> vs = __builtin_bit_cast(Piece<T>, ps[j]);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        g[j][e] = (float)vg[e];
        n[j][e] = (float)vh[e] * rstd;
        s[j][e] = ds ? (float)vs[e] : 0.0f;
        if (mine)
          dw[j][e] = __builtin_fmaf(g[j][e], n[j][e], dw[j][e]);
        dot = __builtin_fmaf(g[j][e] * w[j][e], n[j][e], dot);
      }
    }
    if (kAhead && first + gridDim.x * kRows < a.rows)
      request(row + gridDim.x * kRows);
    dot = row_reduce<SumOp, TPR>(dot, slots[it & 1]) / (float)cols;
    if (!mine)
      continue;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (j * TPR + t) * N, valid = (int)cols - c;
      if (valid <= 0)
        continue;
      Piece<T> o;
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = (T)(s[j][e] + rstd * (g[j][e] * w[j][e] - n[j][e] * dot));
      store_chunk(static_cast<T *>(a.grad_in) + (size_t)row * a.ldgi + c, __builtin_bit_cast(u32x4, o), valid);
    }
  }
  if (!a.grad_weight)
    return;
  if constexpr (kRows > 1) { // the rows' groups, added in their order
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e)
        joined[rg][(j * TPR + t) * N + e] = dw[j][e];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < cols; c += kThreads) {
      float sum = joined[0][c];
#pragma unroll
      for (int k = 1; k < kRows; ++k)
        sum += joined[k][c];
      a.partial[(size_t)blockIdx.x * cols + c] = sum;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t c = (uint32_t)(j * TPR + t) * N + e;
        if (c < cols)
          a.partial[(size_t)blockIdx.x * cols + c] = dw[j][e];
      }
  }
}

// grad_weight of a band of rows, element by element: a thread owns a column
template <class T> __device__ __forceinline__ void back_weight_general(const NormBackArgs &a) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols)
    return;
  const uint32_t first = blockIdx.y * a.band, last = min(a.rows, first + a.band);
  float sum = 0.0f;
  for (uint32_t r = first; r < last; ++r)
    sum += (float)static_cast<const T *>(a.grad_out)[r * a.ldg + c] *
           ((float)static_cast<const T *>(a.summed)[r * a.ldh + c] * a.rstd[r]);
  a.partial[(size_t)blockIdx.y * a.cols + c] = sum;
}
// The bands' lines, added in a fixed order: a lane owns a column, each of the
// workgroup's sixteen waves adds every sixteenth line, the sixteen sums meet in LDS.  (512
// lines of 4096 columns: 4.5 us.)
template <class W> __device__ __forceinline__ void fold_weight(const NormBackArgs &a) {
  __shared__ float sums[16][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t c = blockIdx.x * kWave + lane;
  float sum = 0.0f;
  if (c < a.cols) {
#pragma unroll 8
    for (uint32_t b = wave; b < a.bands; b += 16)
      sum += a.partial[(size_t)b * a.cols + c];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || c >= a.cols)
    return;
  for (int k = 1; k < 16; ++k)
    sum += sums[k][lane];
  static_cast<W *>(a.grad_weight)[c] = (W)sum;
}

} // namespace

// (the weight is fp32 or of the element type)
#define HCAMD_NORM(T, NAME)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void hcamd_rmsnorm_##NAME##_general(NormArgs a) {         \
    if (a.weight_f32)                                                                                    \
      norm_general<T, float, false>(a);                                                                  \
    else                                                                                                 \
      norm_general<T, T, false>(a);                                                                      \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void hcamd_rmsnorm_##NAME##_i8_general(NormArgs a) {      \
    if (a.weight_f32)                                                                                    \
      norm_general<T, float, true>(a);                                                                   \
    else                                                                                                 \
      norm_general<T, T, true>(a);                                                                       \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void hcamd_rmsnorm_back_##NAME##_general(NormBackArgs a) { \
    if (a.weight_f32)                                                                                    \
      back_general<T, float>(a);                                                                         \
    else                                                                                                 \
      back_general<T, T>(a);                                                                             \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void hcamd_rmsnorm_back_weight_##NAME##_general(NormBackArgs a) { \
    back_weight_general<T>(a);                                                                           \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(1024) void hcamd_rmsnorm_fold_##NAME(NormBackArgs a) { fold_weight<T>(a); }
HCAMD_NORM(float, f32)
HCAMD_NORM(_Float16, f16)
HCAMD_NORM(__bf16, bf16)

#define HCAMD_NORM_I8(T, NAME, TPR, VPT, THREADS)                                                          \
  extern "C" __global__ __launch_bounds__(THREADS) void hcamd_rmsnorm_##NAME##_i8_r##TPR##v##VPT(NormArgs a) { \
    norm_rows<T, TPR, VPT, THREADS, true>(a);                                                              \
  }
#define HCAMD_NORM_ROWS(T, NAME, TPR, VPT, THREADS)                                                        \
  extern "C" __global__ __launch_bounds__(THREADS) void hcamd_rmsnorm_##NAME##_r##TPR##v##VPT(NormArgs a) { \
    norm_rows<T, TPR, VPT, THREADS, false>(a);                                                             \
  }                                                                                                        \
  HCAMD_NORM_I8(T, NAME, TPR, VPT, THREADS)
#define HCAMD_NORM_BACK(T, NAME, TPR, VPT, THREADS)                                                        \
  extern "C" __global__ __launch_bounds__(THREADS) void hcamd_rmsnorm_back_##NAME##_r##TPR##v##VPT(NormBackArgs a) { \
    back_rows<T, TPR, VPT, THREADS>(a);                                                                    \
  }
#define HCAMD_NORM_BOTH(T, NAME, TPR, VPT, THREADS)                                                        \
  HCAMD_NORM_ROWS(T, NAME, TPR, VPT, THREADS)                                                              \
  HCAMD_NORM_BACK(T, NAME, TPR, VPT, THREADS)
#define HCAMD_NORM_SHORT(T, NAME)                                                                          \
  HCAMD_NORM_BOTH(T, NAME, 64, 1, 256)                                                                     \
  HCAMD_NORM_BOTH(T, NAME, 64, 2, 256)                                                                     \
  HCAMD_NORM_BOTH(T, NAME, 256, 1, 256)
#define HCAMD_NORM_16(T, NAME)                                                                             \
  HCAMD_NORM_SHORT(T, NAME)                                                                                \
  HCAMD_NORM_I8(T, NAME, 256, 2, 256)                                                                      \
  HCAMD_NORM_BOTH(T, NAME, 512, 1, 512)                                                                    \
  HCAMD_NORM_ROWS(T, NAME, 1024, 1, 1024)                                                                  \
  HCAMD_NORM_BACK(T, NAME, 512, 2, 512)                                                                    \
  HCAMD_NORM_BOTH(T, NAME, 1024, 2, 1024)
HCAMD_NORM_16(__bf16, bf16)
HCAMD_NORM_16(_Float16, f16)
HCAMD_NORM_SHORT(float, f32)
HCAMD_NORM_BOTH(float, f32, 256, 2, 256)
HCAMD_NORM_BOTH(float, f32, 256, 4, 256)
HCAMD_NORM_BOTH(float, f32, 512, 4, 512)
HCAMD_NORM_BOTH(float, f32, 1024, 4, 1024)
