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

using namespace hcamd;

namespace {


__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v = fmax(v, __shfl_xor(v, o));
  return v;
}

// 127 v / most, rounded half to even.  The fp32 quotient h * w * per is off by less
// than 127 * 4 * 2^-24 < 2^-15: only one that close to a half asks for 64 bits (and a
// NaN, which `per` is for rows outside fp32's comfortable range).
__device__ __forceinline__ int8_t quantise(float h, float w, float per, double most) {
  const float t = h * w * per;
  float q = __builtin_rintf(t);
  if (!(__builtin_fabsf(t - q) <= 0.5f - 0x1p-14f))
    q = (float)__builtin_rint(127.0 * ((double)h * (double)w) / most);
  return (int8_t)q;
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

// One workgroup per row, element by element, the row read twice: any alignment and
// leading dimension.  (summed and out may be x or residual: a thread reads an
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
        a.scale[row] = most < (double)INFINITY ? (float)(most * rstd / 127.0) : __builtin_nanf("");
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

// grad_weight of a band of rows: a thread owns a column
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
// the bands, added in their order
template <class W> __device__ __forceinline__ void fold_weight(const NormBackArgs &a) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols)
    return;
  float sum = 0.0f;
  for (uint32_t b = 0; b < a.bands; ++b)
    sum += a.partial[(size_t)b * a.cols + c];
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
  extern "C" __global__ __launch_bounds__(256) void hcamd_rmsnorm_fold_##NAME(NormBackArgs a) { fold_weight<T>(a); }
HCAMD_NORM(float, f32)
HCAMD_NORM(_Float16, f16)
HCAMD_NORM(__bf16, bf16)
