// The gated half of a feed-forward block, out = act(x Wg') * (x Wu'), and its
// gradients.  x [T,D], Wg and Wu [F,D] (output features first), out [T,F].
//
// Forward: one kernel.  Both weight matrices are one N panel whose rows alternate
// between them in blocks of 32, so a lane holds both projections of an output in
// its own accumulators and the activation and the product happen before anything
// is stored.  4 T D F operations.
// Backward, from the stored pre-activations g and u:
//   dg = dh u act'(g), du = dh act(g)        element by element, rounded to the
//                                            element type as matrix operands (fp16:
//                                            scaled by a power of two first)
//   dx = dg Wg + du Wu                        one product, k runs through both pairs
//   dWg = dg' x, dWu = du' x                  one launch, both operands k-slow
#include "mma.h"

using namespace hcamd;

namespace {

enum { kSilu = 0, kGelu = 1 };

// 1 / (1 + exp(-x)): exp overflows to infinity for large negative x, the
// reciprocal is then 0 (the hardware's exponential and reciprocal, 1 ulp each)
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

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

// gate and up are rounded to the element type: half the bytes to keep and to read again, and dg
// and du, which come from them, are rounded all the same, being matrix operands.  The gradients
// are thereby 1.8 times as far from the exact ones as a single rounding at the end would leave
// them (bf16 0.0030 of their size against 0.0017, fp16 0.00037 against 0.00021): of the added
// squares gate and up bring 56 %, dg and du 44 %.
//
// the outputs of a wave: blocks j and j + NI / 2 are the two projections of the same
// columns.  LDS: through the wave's region `mine`, else straight from registers
template <class E, class O, int MI, int NI, bool LDS>
__device__ __forceinline__ void gated_store(const GatedArgs &a, typename MmaType<E>::acc (&acc)[MI][NI],
                                            const Tile &t, int m0, int f0, int lane, unsigned char *mine) {
  constexpr int H = NI / 2;
  const int M = a.mma.M, F = a.mma.N;
  const Window w = {t.m_lo, M, t.n_lo, F};
  auto both = [&](int i, int j, f32x4 &g, f32x4 &u) {
    const float xs = sizeof(E) == 1 ? a.x_scale[min(m0 + i * 16 + lane % 16, M - 1)] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g[e] = (float)acc[i][j][e];
      u[e] = (float)acc[i][j + H][e];
      if constexpr (sizeof(E) == 1) {
        const int c = min(f0 + j * 16 + lane / 16 * 4 + e, F - 1);
        g[e] = g[e] * xs * a.gate_scale[c];
        u[e] = u[e] * xs * a.up_scale[c];
      }
    }
  };
  auto value = [&](int i, int j) {
    f32x4 g, u, o;
    both(i, j, g, u);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = activate(a.activation, g[e]) * u[e];
    return o;
  };
  auto pre_gate = [&](int i, int j) { return __builtin_convertvector(acc[i][j], f32x4); };
  auto pre_up = [&](int i, int j) { return __builtin_convertvector(acc[i][j + H], f32x4); };
  auto store = [&](void *to, size_t ld, auto &&what) {
    if constexpr (LDS)
      store_block<O, MI, H>(mine, static_cast<O *>(to), ld, m0, f0, w, lane, what);
    else
      store_direct<O, MI, H>(static_cast<O *>(to), ld, m0, f0, w, lane, what);
  };
  store(a.out, a.ldo, value);
  if constexpr (sizeof(E) == 2) {
    if (a.gate)
      store(a.gate, a.ldgate, pre_gate);
    if (a.up)
      store(a.up, a.ldup, pre_up);
  }
}

template <class E, int MI, int NI, bool LDS>
__device__ __forceinline__ void gated_epilogue(const GatedArgs &a, typename MmaType<E>::acc (&acc)[MI][NI],
                                               const Tile &t, int m0, int f0, int lane, unsigned char *mine) {
  if constexpr (sizeof(E) == 1) {
    if (a.out_f16)
      gated_store<E, _Float16, MI, NI, LDS>(a, acc, t, m0, f0, lane, mine);
    else
      gated_store<E, __bf16, MI, NI, LDS>(a, acc, t, m0, f0, lane, mine);
  } else {
    gated_store<E, E, MI, NI, LDS>(a, acc, t, m0, f0, lane, mine);
  }
}

template <class E, int BM> __device__ __forceinline__ void gated_general(const GatedArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * (BM + 128) * 128];
  mma_general<E, kKFast, kKFast, true, BM>(
      a.mma, blockIdx.x, 0, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *) {
        gated_epilogue<E, BM / 32, 4, false>(a, acc, t, t.m0 + wave_m, t.n0 + wave_n / 2, lane, nullptr);
      });
}
template <class E, int B> __device__ __forceinline__ void gated_tile(const GatedArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[pipelined_lds<B>()];
  mma_tiles<E, kKFast, kKFast, true, B>(
      a.mma, blockIdx.x, 0, a.mma.half_from, lds, FromZero{},
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *l) {
        constexpr int MI = sizeof(acc) / sizeof(acc[0]), NI = sizeof(acc[0]) / sizeof(acc[0][0]);
        gated_epilogue<E, MI, NI, true>(a, acc, t, t.m0 + wave_m, t.n0 + wave_n / 2, lane,
                                        l + threadIdx.x / kWave * (MI * NI * 256));
      });
}

// Few tokens: one pass over the weights; a workgroup holds NB * 8 outputs' rows of both
// (blocks j and j + NB / 2 belong together).  NB 2, U 4: 35 us for one token and 48 us for
// 32 over 2 x 11264 x 4096 bf16 (5.3 and 3.8 TB/s); NB 4, U 2: 47 and 54 us, half as
// many workgroups.  Beyond 32 tokens fewer pieces of k are under way (U 2, 1): registers.
template <class E, class O, int MB, int NB, int U, bool ODD>
__device__ __forceinline__ void gated_skinny(const GatedArgs &a, unsigned char *lds) {
  constexpr int H = NB / 2;
  const int f0 = blockIdx.x * (H * 16), left = a.mma.N - f0;
  mma_skinny<E, MB, NB, U, ODD>(
      a.mma,
      [&](int j) {
        const int f = min(f0 + j % H * 16 + (int)threadIdx.x % 16, a.mma.N - 1), w = j / H;
        return static_cast<const E *>(a.mma.b[w]) + (size_t)f * a.mma.ldb[w];
      },
      lds);
  typedef typename MmaType<E>::acc acc_t;
  using V = decltype(acc_t{}[0] + acc_t{}[0]);
  const V *cells = reinterpret_cast<const V *>(lds);
  for (int c = threadIdx.x; c < H * MB * 256; c += 512) {
    const int n = c % (H * 16), m = c / (H * 16); // neighbouring lanes write one token's outputs
    if (m >= a.mma.M || n >= left)
      continue;
    const int at = (n / 16 * MB + m / 16) * 256 + ((n % 16 / 4) * 16 + m % 16) * 4 + n % 4;
    float g = (float)cells[at], u = (float)cells[H * MB * 256 + at];
    if constexpr (sizeof(E) == 1) {
      g = g * a.x_scale[m] * a.gate_scale[f0 + n];
      u = u * a.x_scale[m] * a.up_scale[f0 + n];
    }
    static_cast<O *>(a.out)[(size_t)m * a.ldo + f0 + n] = (O)(activate(a.activation, g) * u);
    if (sizeof(E) == 2 && a.gate)
      static_cast<O *>(a.gate)[(size_t)m * a.ldgate + f0 + n] = (O)g;
    if (sizeof(E) == 2 && a.up)
      static_cast<O *>(a.up)[(size_t)m * a.ldup + f0 + n] = (O)u;
  }
}
template <class E, int MB, int NB, int U, bool ODD> __device__ __forceinline__ void gated_few(const GatedArgs &a) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[skinny_lds<MB, NB>()];
  if constexpr (sizeof(E) == 1) {
    if (a.out_f16)
      gated_skinny<E, _Float16, MB, NB, U, ODD>(a, lds);
    else
      gated_skinny<E, __bf16, MB, NB, U, ODD>(a, lds);
  } else {
    gated_skinny<E, E, MB, NB, U, ODD>(a, lds);
  }
}

// f(row, first column, dg, du) for this lane's eights of pre-activation gradients, in fp32
// (zeros past the end of a row)
template <class E, class F> __device__ __forceinline__ void each_gated_back(const GatedBackArgs &a, F &&f) {
  const uint32_t chunks = (a.cols + 7) / 8;
  const uint64_t total = (uint64_t)a.rows * chunks;
  for (uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total;
       id += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t r = (uint32_t)(id / chunks), c = (uint32_t)(id % chunks) * 8;
    const int valid = (int)(a.cols - c);
    typedef E ex8 __attribute__((ext_vector_type(8)));
    const ex8 dh = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.grad_out) + (size_t)r * a.ldg + c, valid, (int)c));
    const ex8 g = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.gate) + (size_t)r * a.ldgate + c, valid, (int)c));
    const ex8 u = __builtin_bit_cast(ex8, load_chunk(static_cast<const E *>(a.up) + (size_t)r * a.ldup + c, valid, (int)c));
    float dg[8], du[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float act, dact;
      activate_both(a.activation, (float)g[e], act, dact);
      dg[e] = (float)dh[e] * (float)u[e] * dact;
      du[e] = (float)dh[e] * act;
    }
    f(r, c, dg, du);
  }
}

// fp16 holds 40 binary places, of which the lowest ten lack precision, and dg and du are products of
// values that may stand anywhere in them: rounded as they are, those of a gradient of 1e-6
// would keep four bits, and those of one of 3e4 overflow and meet other terms as NaN.  So they
// are scaled by the power of two that brings the largest of them to 2^14 .. 2^15, and the
// products undo it in fp32 (exactly: a block whose dg and du are normal numbers below 2^15 has
// the results it would have unscaled).  One more launch reads the operands for that maximum (333 x 2731 4 us, 4096 x 11264 76 us).
__device__ __forceinline__ void gated_back_most(const GatedBackArgs &a) {
  __shared__ float slots[4];
  float most = 0.0f;
  each_gated_back<_Float16>(a, [&](uint32_t, uint32_t, const float *dg, const float *du) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      most = fmaxf(most, fmaxf(__builtin_fabsf(dg[e]), __builtin_fabsf(du[e]))); // (of a NaN and a number: the number)
  });
  most = group_reduce<MaxOp, 4>(most, slots);
  if (threadIdx.x == 0)
    a.most[blockIdx.x] = most;
}
// that power of two; 1 where the largest is zero or infinite (which it then stays)
__device__ __forceinline__ float gated_back_scale(const GatedBackArgs &a) {
  __shared__ float slots[4];
  float most = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.mosts; i += 256)
    most = fmaxf(most, a.most[i]);
  most = group_reduce<MaxOp, 4>(most, slots);
  const int exponent = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127; // (at most 33: products of fp16 values)
  const int by = most > 0.0f && most < INFINITY ? min(14 - exponent, 100) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0)
    *a.undo = __builtin_bit_cast(float, (uint32_t)(127 - by) << 23);
  return __builtin_bit_cast(float, (uint32_t)(127 + by) << 23);
}

// pre-activation gradients: a workgroup walks rows, eight elements a lane.  The
// destination is the library's own, its rows padded to a multiple of 8.  Bound by memory:
// 4096 x 11264 bf16 84 us (5.5 TB/s).
template <class E> __device__ __forceinline__ void gated_back(const GatedBackArgs &a) {
  float by = 1.0f;
  if constexpr (std::is_same<E, _Float16>::value)
    by = gated_back_scale(a);
  each_gated_back<E>(a, [&](uint32_t r, uint32_t c, const float *dg, const float *du) {
    typedef E ex8 __attribute__((ext_vector_type(8)));
    ex8 vg, vu;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      vg[e] = (E)(dg[e] * by);
      vu[e] = (E)(du[e] * by);
    }
    *reinterpret_cast<ex8 *>(static_cast<E *>(a.dgate) + (size_t)r * a.ldd + c) = vg;
    *reinterpret_cast<ex8 *>(static_cast<E *>(a.dup) + (size_t)r * a.ldd + c) = vu;
  });
}

// a product that is stored; `tile` counts its workgroups
template <class E, Layout LA, Layout LB>
__device__ __forceinline__ void product_general(const StoreArgs &s, int tile, int split, unsigned char *lds) {
  mma_general<E, LA, LB, false, 128>(
      s.mma, tile, split, lds,
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane) {
        begin_tile<4, 4>(s, acc, t.m0 + wave_m, t.n0 + wave_n, lane, split);
      },
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *) {
        store_tile<E, 4, 4, false>(s, acc, t, t.m0 + wave_m, t.n0 + wave_n, lane, split, nullptr);
      });
}
template <class E, Layout LA, Layout LB, int B>
__device__ __forceinline__ void product_tile(const StoreArgs &s, int tile, int split, int half_from,
                                             unsigned char *lds) {
  mma_tiles<E, LA, LB, false, B>(
      s.mma, tile, split, half_from, lds,
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane) {
        constexpr int MI = sizeof(acc) / sizeof(acc[0]), NI = sizeof(acc[0]) / sizeof(acc[0][0]);
        begin_tile<MI, NI>(s, acc, t.m0 + wave_m, t.n0 + wave_n, lane, split);
      },
      [&](auto &acc, const Tile &t, int wave_m, int wave_n, int lane, unsigned char *l) {
        constexpr int MI = sizeof(acc) / sizeof(acc[0]), NI = sizeof(acc[0]) / sizeof(acc[0][0]);
        store_tile<E, MI, NI, true>(s, acc, t, t.m0 + wave_m, t.n0 + wave_n, lane, split,
                                    l + threadIdx.x / kWave * (MI * NI * 512));
      });
}
// Up to two products: workgroups below `tiles` belong to the first; half tiles, which
// come last, to the one their tile belongs to.
struct OfPair {
  int which, tile, half_from;
};
__device__ __forceinline__ OfPair of_pair(const PairStoreArgs &a, int wg) {
  const int from = a.p[0].mma.half_from;
  const int tile = wg < from ? wg : from + (wg - from) / 2; // among the tiles of both
  const int which = tile >= a.tiles ? 1 : 0, first = which * a.tiles;
  // the product's own count, with its half tiles from half_from on
  const int half_from = max(0, min(from - first, a.tiles));
  const int own = tile - first;
  return {which, own < half_from ? own : half_from + 2 * (own - half_from) + (wg - from) % 2, half_from};
}

// The products of a backward pass with 128 x 128 tiles in one launch, dx's workgroups first:
// alone neither of them fills the card for long (333 x 1001 x 2731 fp16: 20 and 18.5 us one
// after the other).
template <class E, bool PIPELINED> __device__ __forceinline__ void products(const ProductsArgs &a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * 128 * 128];
  static_assert(pipelined_lds<128>() == sizeof(lds), "");
  const int first = a.nn_groups * a.nn.mma.splits, wg = blockIdx.x;
  if (wg < first) {
    const int split = __builtin_amdgcn_readfirstlane(wg / a.nn_groups), tile = wg - split * a.nn_groups;
    if constexpr (PIPELINED)
      product_tile<E, kKFast, kKSlow, 128>(a.nn, tile, split, 0, lds);
    else
      product_general<E, kKFast, kKSlow>(a.nn, tile, split, lds);
  } else {
    const int split = __builtin_amdgcn_readfirstlane((wg - first) / a.tn_groups);
    const OfPair o = of_pair(a.tn, wg - first - split * a.tn_groups);
    if constexpr (PIPELINED)
      product_tile<E, kKSlow, kKSlow, 128>(a.tn.p[o.which], o.tile, split, 0, lds);
    else
      product_general<E, kKSlow, kKSlow>(a.tn.p[o.which], o.tile, split, lds);
  }
}

// the partial sums of the splits, added in the order of the splits, four columns a lane
// (rows of partial sums are padded to a multiple of 8).  Bound by memory, or by its launch:
// 333 x 1001 from 8 splits 4.5 us.
template <class E> __device__ __forceinline__ void fold(const FoldArgs &a) {
  const uint32_t quads = (a.cols + 3) / 4;
  const uint64_t total = (uint64_t)a.rows * quads;
  const float by = a.undo ? *a.undo : 1.0f;
  for (uint64_t id = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total;
       id += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t r = (uint32_t)(id / quads), c = (uint32_t)(id % quads) * 4;
    const float *from = a.partial + (size_t)r * a.ldp + c;
    f32x4 v = *reinterpret_cast<const f32x4 *>(from);
#pragma unroll 4
    for (uint32_t s = 1; s < a.splits; ++s)
      v += *reinterpret_cast<const f32x4 *>(from + (size_t)s * a.rows * a.ldp);
    store4<E>(static_cast<E *>(a.out) + (size_t)r * a.ldo, (int)c, 0, (int)a.cols, times(v, by));
  }
}

// Rows of any length and alignment copied to rows the pipelined kernels can fetch: whole
// 16-byte pieces, zeros behind the last element.  One wave to a row, kAhead pieces a lane
// under way.  Bound by memory: 50021 x 1025 bf16 60 us (3.4 TB/s; fetching from 4-byte words
// instead changes nothing).
template <class E> __device__ __forceinline__ void lay_out(const LayArgs &a) {
  constexpr int n = 16 / (int)sizeof(E), kAhead = 4;
  const uint32_t lane = threadIdx.x % kWave, cols = a.cols;
  for (uint32_t r = blockIdx.x * 4 + threadIdx.x / kWave; r < a.rows; r += gridDim.x * 4) {
    const E *from = static_cast<const E *>(a.from) + (size_t)r * a.ld_from;
    E *to = static_cast<E *>(a.to) + (size_t)r * a.ld_to;
    for (uint32_t c0 = lane * n; c0 < cols; c0 += kAhead * kWave * n) {
      u32x4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t c = c0 + k * kWave * n;
        v[k] = load_chunk(from + c, (int)(cols - c), (int)c);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (c0 + k * kWave * n < cols)
          *reinterpret_cast<u32x4 *>(to + c0 + k * kWave * n) = v[k];
    }
  }
}

} // namespace

#define HCAMD_FFN(SUFFIX, E)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_##SUFFIX##_general(GatedArgs a) {         \
    gated_general<E, 128>(a);                                                                             \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_##SUFFIX##_half(GatedArgs a) {            \
    gated_general<E, 64>(a);                                                                              \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_gated_##SUFFIX##_t256(GatedArgs a) {            \
    gated_tile<E, 256>(a);                                                                          \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_##SUFFIX##_t128(GatedArgs a) {            \
    gated_tile<E, 128>(a);                                                                          \
  }
HCAMD_FFN(bf16, __bf16)
HCAMD_FFN(f16, _Float16)
HCAMD_FFN(i8, int8_t)
#define HCAMD_FFN_FEW(SUFFIX, E, ROWS, NB, U)                                                             \
  extern "C" __global__ __launch_bounds__(512) void hcamd_gated_##SUFFIX##_s##ROWS(GatedArgs a) {         \
    gated_few<E, ROWS / 16, NB, U, false>(a);                                                             \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_gated_##SUFFIX##_s##ROWS##odd(GatedArgs a) {    \
    gated_few<E, ROWS / 16, NB, U, true>(a);                                                              \
  }
#define HCAMD_FFN_FEWS(SUFFIX, E)                                                                         \
  HCAMD_FFN_FEW(SUFFIX, E, 16, 2, 4)                                                                      \
  HCAMD_FFN_FEW(SUFFIX, E, 32, 2, 4)                                                                      \
  HCAMD_FFN_FEW(SUFFIX, E, 64, 2, 2)                                                                      \
  HCAMD_FFN_FEW(SUFFIX, E, 128, 2, 1)
HCAMD_FFN_FEWS(bf16, __bf16)
HCAMD_FFN_FEWS(f16, _Float16)
HCAMD_FFN_FEWS(i8, int8_t)
#define HCAMD_FFN_BACK(SUFFIX, E)                                                                         \
  extern "C" __global__ __launch_bounds__(256) void hcamd_gated_back_##SUFFIX(GatedBackArgs a) {          \
    gated_back<E>(a);                                                                                     \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_products_##SUFFIX##_general(ProductsArgs a) {   \
    products<E, false>(a);                                                                                \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_products_##SUFFIX##_t128(ProductsArgs a) {      \
    products<E, true>(a);                                                                                 \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_product_nn_##SUFFIX##_t256(StoreArgs a) {       \
    __shared__ __attribute__((aligned(1024))) unsigned char lds[pipelined_lds<256>()];                    \
    product_tile<E, kKFast, kKSlow, 256>(a, blockIdx.x, blockIdx.y, a.mma.half_from, lds);                \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(512) void hcamd_product_tn_##SUFFIX##_t256(PairStoreArgs a) {   \
    __shared__ __attribute__((aligned(1024))) unsigned char lds[pipelined_lds<256>()];                    \
    const OfPair o = of_pair(a, blockIdx.x);                                                              \
    product_tile<E, kKSlow, kKSlow, 256>(a.p[o.which], o.tile, blockIdx.y, o.half_from, lds);             \
  }                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void hcamd_fold_##SUFFIX(FoldJobs a) { fold<E>(a.job[blockIdx.y]); }
HCAMD_FFN_BACK(bf16, __bf16)
HCAMD_FFN_BACK(f16, _Float16)
extern "C" __global__ __launch_bounds__(256) void hcamd_gated_back_most_f16(GatedBackArgs a) { gated_back_most(a); }
// (copies: one kernel for both 16-bit types)
extern "C" __global__ __launch_bounds__(256) void hcamd_lay_out_2(LayJobs a) { lay_out<uint16_t>(a.job[blockIdx.y]); }
extern "C" __global__ __launch_bounds__(256) void hcamd_lay_out_1(LayJobs a) { lay_out<uint8_t>(a.job[blockIdx.y]); }
