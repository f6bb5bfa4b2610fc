// Rows in 16-byte pieces at any alignment.  gfx950 serves 16-byte accesses at every
// address; a piece that crosses the end of its row goes element by element.
#pragma once
#include "common.h"

namespace hcamd {

typedef u32x4 u32x4_u __attribute__((aligned(1)));
typedef u32x2 u32x2_u __attribute__((aligned(1)));

// v shifted down by `bytes` (0 .. 15), zeros from above
__device__ __forceinline__ u32x4 shift_down(u32x4 v, int bytes) {
  if (bytes & 8)
    v = u32x4{v[2], v[3], 0u, 0u};
  if (bytes & 4)
    v = u32x4{v[1], v[2], v[3], 0u};
  const uint32_t bits = (bytes & 3) * 8;
  return u32x4{__builtin_amdgcn_alignbit(v[1], v[0], bits), __builtin_amdgcn_alignbit(v[2], v[1], bits),
               __builtin_amdgcn_alignbit(v[3], v[2], bits), v[3] >> bits};
}

// 16 bytes of which the first `valid` elements exist; the rest reads as zero.  With
// `before` elements of the row in front of p the last piece of a row is the row's last 16
// bytes, shifted; only rows shorter than a piece go element by element (the
// gated block of 200 x 300 x 400 in 8 bits: 16.9 us when every last piece did).
template <class E> __device__ __forceinline__ u32x4 load_chunk(const E *p, int valid, int before) {
  constexpr int n = 16 / (int)sizeof(E);
  if (valid >= n)
    return *reinterpret_cast<const u32x4_u *>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
  if (valid <= 0)
    return v;
  if (before >= n - valid)
    return shift_down(*reinterpret_cast<const u32x4_u *>(p - (n - valid)), (n - valid) * (int)sizeof(E));
  if constexpr (sizeof(E) == 2) {
    const uint16_t *s = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e < valid)
        v[e / 2] |= (uint32_t)s[e] << (16 * (e % 2));
  } else if constexpr (sizeof(E) == 4) {
    const uint32_t *s = reinterpret_cast<const uint32_t *>(p);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e < valid)
        v[e] = s[e];
  } else {
    const uint8_t *s = reinterpret_cast<const uint8_t *>(p);
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e < valid)
        v[e / 4] |= (uint32_t)s[e] << (8 * (e % 4));
  }
  return v;
}

// the first `valid` of the elements of 16 bytes: what is not whole goes in pieces of 8, 4,
// 2 and 1 bytes
template <class E> __device__ __forceinline__ void store_chunk(E *p, u32x4 v, int valid) {
  constexpr int n = 16 / (int)sizeof(E);
  if (valid >= n) {
    *reinterpret_cast<u32x4_u *>(p) = v;
    return;
  }
  if (valid <= 0)
    return;
  const int bytes = valid * (int)sizeof(E);
  char *to = reinterpret_cast<char *>(p);
  if (bytes & 8) {
    *reinterpret_cast<u32x2_u *>(to) = u32x2{v[0], v[1]};
    v = shift_down(v, 8);
    to += 8;
  }
  if (bytes & 4) {
    typedef uint32_t u32_u __attribute__((aligned(1)));
    *reinterpret_cast<u32_u *>(to) = v[0];
    v[0] = v[1];
    to += 4;
  }
  if constexpr (sizeof(E) <= 2) {
    typedef uint16_t u16_u __attribute__((aligned(1)));
    if (bytes & 2) {
      *reinterpret_cast<u16_u *>(to) = (uint16_t)v[0];
      v[0] >>= 16;
      to += 2;
    }
  }
  if constexpr (sizeof(E) == 1) {
    if (bytes & 1)
      *reinterpret_cast<uint8_t *>(to) = (uint8_t)v[0];
  }
}

} // namespace hcamd
