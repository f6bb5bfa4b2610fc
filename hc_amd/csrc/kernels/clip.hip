// Clipping of many tensors by their joint norm:
//   norm = sqrt(sum of squares over all tensors), out = in * min(1, max_norm / (norm + 1e-6)).
// Two launches (per 64 tensors, which travel in the kernel arguments): partial sums of
// squares per workgroup, then every workgroup adds all partial sums in their order and
// scales its share.  Sums are held in 64 bits: no overflow of large fp32 gradients, and
// the result does not depend on how the tensors are cut.
#include "common.h"
#include "op_args.h"

using namespace hcamd;

namespace {

constexpr uint32_t kChunkElems = 16384; // elements a workgroup takes at a time

__device__ __forceinline__ float load1(const void *p, int type, uint64_t i) {
  return type == 0 ? static_cast<const float *>(p)[i]
         : type == 1 ? (float)static_cast<const _Float16 *>(p)[i]
                     : (float)static_cast<const __bf16 *>(p)[i];
}
__device__ __forceinline__ void store1(void *p, int type, uint64_t i, float v) {
  if (type == 0)
    static_cast<float *>(p)[i] = v;
  else if (type == 1)
    static_cast<_Float16 *>(p)[i] = (_Float16)v;
  else
    static_cast<__bf16 *>(p)[i] = (__bf16)v;
}

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

__device__ __forceinline__ void square_sums(const ClipArgs &a) {
  __shared__ double slots[4];
  double sum = 0.0;
  for (uint32_t chunk = blockIdx.x; chunk < a.first_chunk[a.tensors]; chunk += gridDim.x) {
    const uint32_t t = tensor_of(a, chunk);
    const uint64_t first = (uint64_t)(chunk - a.first_chunk[t]) * kChunkElems;
    const uint64_t last = min(a.count[t], first + kChunkElems);
    for (uint64_t i = first + threadIdx.x; i < last; i += 256) {
      const double v = (double)load1(a.in[t], a.type[t], i);
      sum = __builtin_fma(v, v, sum);
    }
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
  const float norm = (float)__builtin_sqrt(group_sum64(sum, slots));
  // (a NaN norm gives a NaN factor, an infinite one 0)
  float factor = a.max_norm / (norm + 1e-6f);
  factor = factor > 1.0f ? 1.0f : factor;
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *a.norm = norm;
  for (uint32_t chunk = blockIdx.x; chunk < a.first_chunk[a.tensors]; chunk += gridDim.x) {
    const uint32_t t = tensor_of(a, chunk);
    const uint64_t first = (uint64_t)(chunk - a.first_chunk[t]) * kChunkElems;
    const uint64_t last = min(a.count[t], first + kChunkElems);
    for (uint64_t i = first + threadIdx.x; i < last; i += 256)
      store1(a.out[t], a.type[t], i, load1(a.in[t], a.type[t], i) * factor);
  }
}

} // namespace

extern "C" __global__ __launch_bounds__(256) void hcamd_clip_sums(ClipArgs a) { square_sums(a); }
extern "C" __global__ __launch_bounds__(256) void hcamd_clip_scale(ClipArgs a) { scale(a); }
