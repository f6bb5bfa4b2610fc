// Clipping of many tensors by their joint norm:
//   norm = sqrt(sum of squares over all tensors), out = in * min(1, max_norm / (norm + 1e-6)).
// Two launches (per 64 tensors, which travel in the kernel arguments): partial sums of
// squares per workgroup, then every workgroup adds all partial sums in their order and
// scales its share.  Sums, the norm and the factor are held in 64 bits: no overflow of large
// fp32 gradients, and the result does not depend on how the tensors are cut.
// Bound by memory: no element can be stored before the last has been read, so the tensors are
// read twice.  60 tensors of 0.8 GB: 160 us for the sums (5 TB/s), 278 us for the scaling
// (5.8 TB/s); 12 small ones 3.5 + 4 us, two launches.
#include "common.h"
#include "op_args.h"
#include "pieces.h"

using namespace hcamd;

namespace {

constexpr int kAhead = 4; // 16-byte pieces a lane requests at a time

template <class T> constexpr int kPiece = 16 / (int)sizeof(T);
template <class T> using Piece __attribute__((ext_vector_type(kPiece<T>))) = T;

__device__ __forceinline__ double group_sum64(double v, double *slots) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    v += __shfl_xor(v, o);
  if (threadIdx.x % kWave == 0)
    slots[threadIdx.x / kWave] = v;
  __syncthreads();
  return (slots[0] + slots[1]) + (slots[2] + slots[3]);
}

// the tensor a chunk belongs to
__device__ __forceinline__ uint32_t tensor_of(const ClipArgs &a, uint32_t chunk) {
  uint32_t lo = 0, hi = a.tensors;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.first_chunk[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// f(piece, first element, valid elements) for this lane's pieces of n elements (a chunk:
// positions are plain ints, and what lies past the end is a count of 0 or less)
template <class T, class F> __device__ __forceinline__ void each_piece(const T *in, int n, F &&f) {
  constexpr int N = kPiece<T>;
  for (int at = threadIdx.x * N; at < n; at += 256 * N * kAhead) {
    u32x4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      v[k] = load_chunk(in + at + k * 256 * N, n - (at + k * 256 * N), at + k * 256 * N);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      f(__builtin_bit_cast(Piece<T>, v[k]), at + k * 256 * N, n - (at + k * 256 * N));
  }
}

template <class T> __device__ __forceinline__ double chunk_squares(const void *in, uint64_t first, int n) {
  double sum = 0.0;
  each_piece(static_cast<const T *>(in) + first, n, [&](Piece<T> v, int, int) {
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e) { // (elements that do not exist are zeros)
      const double x = (double)(float)v[e];
      sum = __builtin_fma(x, x, sum);
    }
  });
  return sum;
}
template <class T>
__device__ __forceinline__ void chunk_scale(const void *in, void *out, uint64_t first, int n, float pre, float by) {
  T *to = static_cast<T *>(out) + first;
  each_piece(static_cast<const T *>(in) + first, n, [&](Piece<T> v, int at, int valid) {
#pragma unroll
    for (int e = 0; e < kPiece<T>; ++e)
      v[e] = (T)((float)v[e] * pre * by);
    store_chunk(to + at, __builtin_bit_cast(u32x4, v), valid);
  });
}
// a chunk of a tensor: its first element, and how many it has
__device__ __forceinline__ int chunk_of(const ClipArgs &a, uint32_t chunk, uint32_t t, uint64_t &first) {
  first = (uint64_t)(chunk - a.first_chunk[t]) * a.chunk;
  const uint64_t left = a.count[t] - first;
  return left < a.chunk ? (int)left : (int)a.chunk;
}

__device__ __forceinline__ void square_sums(const ClipArgs &a) {
  __shared__ double slots[4];
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < a.first_chunk[a.tensors]; chunk += gridDim.x) {
    const uint32_t t = tensor_of(a, chunk);
    uint64_t first;
    const int n = chunk_of(a, chunk, t, first);
    sum += a.type[t] == 0   ? chunk_squares<float>(a.in[t], first, n)
           : a.type[t] == 1 ? chunk_squares<_Float16>(a.in[t], first, n)
                            : chunk_squares<__bf16>(a.in[t], first, n);
  }
  sum = group_sum64(sum, slots);
  if (threadIdx.x == 0)
    a.partial[a.first_cell + blockIdx.x] = sum;
}

__device__ __forceinline__ void scale(const ClipArgs &a) {
  __shared__ double slots[4];
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < a.cells; i += 256)
    sum += a.partial[i];
  const double norm = __builtin_sqrt(group_sum64(sum, slots));
  // (a NaN norm gives a NaN factor, an infinite one 0)
  double factor = (double)a.max_norm / (norm + 1e-6);
  factor = factor > 1.0 ? 1.0 : factor;
  // a factor near or below fp32's smallest normal numbers goes in two steps, the first a power
  // of two
  const float pre = factor < 0x1p-64 ? 0x1p-64f : 1.0f, by = (float)(factor < 0x1p-64 ? factor * 0x1p64 : factor);
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *a.norm = (float)norm;
  // from the last chunk to the first: what the sums read last is still in the
  // memory-side cache
  const uint32_t chunks = a.first_chunk[a.tensors];
  for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
    const uint32_t chunk = chunks - 1 - k, t = tensor_of(a, chunk);
    uint64_t first;
    const int n = chunk_of(a, chunk, t, first);
    if (a.type[t] == 0)
      chunk_scale<float>(a.in[t], a.out[t], first, n, pre, by);
    else if (a.type[t] == 1)
      chunk_scale<_Float16>(a.in[t], a.out[t], first, n, pre, by);
    else
      chunk_scale<__bf16>(a.in[t], a.out[t], first, n, pre, by);
  }
}

} // namespace

extern "C" __global__ __launch_bounds__(256) void hcamd_clip_sums(ClipArgs a) { square_sums(a); }
extern "C" __global__ __launch_bounds__(256) void hcamd_clip_scale(ClipArgs a) { scale(a); }
