// The gated half of a feed-forward block, out = act(x Wg') * (x Wu'), and its
// gradients.  x [T,D], Wg and Wu [F,D] (output features first), out [T,F].
//
// Forward: one kernel.  Both weight matrices are one N panel whose rows alternate
// between them in blocks of 32, so a lane holds both projections of an output in
// its own accumulators and the activation and the product happen before anything
// is stored.  4 T D F operations.
// Backward, from the stored pre-activations g and u:
//   dg = dh u act'(g), du = dh act(g)        element by element, rounded to the
//                                            element type as matrix operands
//   dx = dg Wg + du Wu                        one product, k runs through both pairs
//   dWg = dg' x, dWu = du' x                  one launch, both operands k-slow
#include "mma.h"

using namespace hcamd;

namespace {

enum { kSilu = 0, kGelu = 1 };

// 1 / (1 + exp(-x)): exp overflows to infinity for large negative x, the
// quotient is then 0
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

constexpr float kGeluA = 0.7978845608028654f; // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// silu: x sigmoid(x); gelu (the tanh form): x (1 + tanh(a (x + b x^3))) / 2, which is
// x sigmoid(2 a (x + b x^3))
__device__ __forceinline__ float activate(int kind, float x) {
  const float t = kind == kSilu ? x : 2.0f * kGeluA * (x + kGeluB * x * x * x);
  const float s = sigmoid(t);
  // x = -inf: the limit 0, not -inf * 0
  return s == 0.0f ? 0.0f : x * s;
}
// the activation and its derivative s + x s (1 - s) t'
__device__ __forceinline__ void activate_both(int kind, float x, float &f, float &df) {
  const float t = kind == kSilu ? x : 2.0f * kGeluA * (x + kGeluB * x * x * x);
  const float dt = kind == kSilu ? 1.0f : 2.0f * kGeluA * (1.0f + 3.0f * kGeluB * x * x);
  const float s = sigmoid(t);
  const float rest = sigmoid(-t); // 1 - s without cancellation
  f = s == 0.0f ? 0.0f : x * s;
  // where either factor has vanished the product's limit is 0 (x dt may be infinite)
  const float p = s * rest;
  df = p == 0.0f ? s : s + x * dt * p;
}

template <class E, class O, int MI, int NI>
__device__ __forceinline__ void gated_store(const GatedArgs &a, typename MmaType<E>::acc (&acc)[MI][NI], int m0,
                                            int f0, int lane) {
  constexpr int H = NI / 2;
  const int M = a.mma.M, F = a.mma.N;
  const bool vo = can_store4<O>(a.out, a.ldo);
  const bool vg = a.gate && can_store4<O>(a.gate, a.ldgate), vu = a.up && can_store4<O>(a.up, a.ldup);
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + i * 16 + lane % 16;
    if (m >= M)
      continue;
    const float xs = sizeof(E) == 1 ? a.x_scale[m] : 1.0f;
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int f = f0 + j * 16 + lane / 16 * 4;
      f32x4 g, u, o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = (float)acc[i][j][e];
        u[e] = (float)acc[i][j + H][e];
        if constexpr (sizeof(E) == 1) {
          const int c = min(f + e, F - 1);
          g[e] = g[e] * xs * a.gate_scale[c];
          u[e] = u[e] * xs * a.up_scale[c];
        }
        o[e] = activate(a.activation, g[e]) * u[e];
      }
      store4<O>(static_cast<O *>(a.out) + (size_t)m * a.ldo, f, F, vo, o);
      if (a.gate)
        store4<O>(static_cast<O *>(a.gate) + (size_t)m * a.ldgate, f, F, vg, g);
      if (a.up)
        store4<O>(static_cast<O *>(a.up) + (size_t)m * a.ldup, f, F, vu, u);
    }
  }
}

template <class E> __device__ __forceinline__ void gated_general(const GatedArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * 128 * 128];
  mma_general<E, kKFast, kKFast, true>(
      a.mma, lds, [&](auto &acc, int m0, int wave_m, int tn, int wave_n, int lane, unsigned char *) {
        const int f0 = tn * 64 + wave_n / 2;
        if constexpr (sizeof(E) == 1) {
          if (a.out_f16)
            gated_store<E, _Float16>(a, acc, m0 + wave_m, f0, lane);
          else
            gated_store<E, __bf16>(a, acc, m0 + wave_m, f0, lane);
        } else {
          gated_store<E, E>(a, acc, m0 + wave_m, f0, lane);
        }
      });
}

// pre-activation gradients: a workgroup walks rows, eight elements a lane.  The
// destination is the library's own, its rows padded to a multiple of 8.
template <class E> __device__ __forceinline__ void gated_back(const GatedBackArgs &a) {
  const uint32_t chunks = (a.cols + 7) / 8;
  const uint64_t total = (uint64_t)a.rows * chunks;
  for (uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total;
       id += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t r = (uint32_t)(id / chunks), c = (uint32_t)(id % chunks) * 8;
    const int valid = (int)(a.cols - c);
    typedef E ex8 __attribute__((ext_vector_type(8)));
    const ex8 dh = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.grad_out) + (size_t)r * a.ldg + c, valid));
    const ex8 g = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.gate) + (size_t)r * a.ldgate + c, valid));
    const ex8 u = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.up) + (size_t)r * a.ldup + c, valid));
    ex8 dg, du;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float f, df;
      activate_both(a.activation, (float)g[e], f, df);
      dg[e] = (E)((float)dh[e] * (float)u[e] * df);
      du[e] = (E)((float)dh[e] * f);
    }
    *reinterpret_cast<ex8 *>(static_cast<E *>(a.dgate) + (size_t)r * a.ldd + c) = dg;
    *reinterpret_cast<ex8 *>(static_cast<E *>(a.dup) + (size_t)r * a.ldd + c) = du;
  }
}

// dx: A k-fast, B k-slow, sum over both pairs
template <class E> __device__ __forceinline__ void product_nn(const StoreArgs &s) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * 128 * 128];
  mma_general<E, kKFast, kKSlow, false>(
      s.mma, lds, [&](auto &acc, int m0, int wave_m, int tn, int wave_n, int lane, unsigned char *) {
        store_tile<E, 4, 4, 128>(s, acc, m0 + wave_m, tn * 128 + wave_n, lane);
      });
}
// dW: both operands k-slow, grid z selects the product
template <class E> __device__ __forceinline__ void product_tn(const PairStoreArgs &a) {
  const StoreArgs &s = a.p[blockIdx.z];
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * 128 * 128];
  mma_general<E, kKSlow, kKSlow, false>(
      s.mma, lds, [&](auto &acc, int m0, int wave_m, int tn, int wave_n, int lane, unsigned char *) {
        store_tile<E, 4, 4, 128>(s, acc, m0 + wave_m, tn * 128 + wave_n, lane);
      });
}

// the partial sums of the splits, added in the order of the splits
template <class E> __device__ __forceinline__ void fold(const FoldArgs &a) {
  const uint64_t total = (uint64_t)a.rows * a.cols;
  const float by = a.undo ? *a.undo : 1.0f;
  for (uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total;
       id += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t r = (uint32_t)(id / a.cols), c = (uint32_t)(id % a.cols);
    float v = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s)
      v += a.partial[((size_t)s * a.rows + r) * a.ldp + c];
    static_cast<E *>(a.out)[(size_t)r * a.ldo + c] = (E)(v * by);
  }
}

} // namespace

#define HCAMD_FFN(SUFFIX, E)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_##SUFFIX##_general(GatedArgs a) {         \
    gated_general<E>(a);                                                                                  \
  }
HCAMD_FFN(bf16, __bf16)
HCAMD_FFN(f16, _Float16)
HCAMD_FFN(i8, int8_t)
#define HCAMD_FFN_BACK(SUFFIX, E)                                                                         \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_back_##SUFFIX(GatedBackArgs a) {          \
    gated_back<E>(a);                                                                                     \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_product_nn_##SUFFIX##_general(StoreArgs a) {    \
    product_nn<E>(a);                                                                                     \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_product_tn_##SUFFIX##_general(PairStoreArgs a) { \
    product_tn<E>(a);                                                                                     \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_fold_##SUFFIX(FoldArgs a) { fold<E>(a); }
HCAMD_FFN_BACK(bf16, __bf16)
HCAMD_FFN_BACK(f16, _Float16)
