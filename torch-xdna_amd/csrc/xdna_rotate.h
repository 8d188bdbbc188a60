// Positions as turns, for the kernels that rotate queries and keys (gfx950 only).
//
// A pair (a, b) of dims at place pos turns by theta = pos f: (a cos - b sin, b cos + a sin). In float32 pos f loses the
// angle (100000 f is off by 0.004), so the quarter turns pos f 2 / pi are formed in float64: a fused multiply-add with
// 1.5 * 2^52 rounds them to a whole number, whose low bits name the quadrant, and a second one leaves the rest, exact
// but for the rounding of f 2 / pi, in -1/2 .. 1/2. Its sine and cosine are Taylor's series to r^9 and r^10: the terms left out are
// below 2^-28. f 2 / pi, and 2 / pi itself, are rounded to float64, so the angle is off by up to 2^-52 of itself: below float32's 2^-24 up
// to 2^28 radians, 2.5e-4 at 2^40. From 2^50 on the quadrant is lost, and there, as where f is not finite, the result means
// nothing.
#pragma once

#include "xdna_common.h"

namespace xdna {

// n / d for 0 <= n < 2^31 by a product: m = 2^32 (2^s - d) / d + 1, s = ceil(log2 d); q = (n + high(n m)) >> s
struct Divisor {
  uint32_t m, s, d;
  Divisor() = default;
  explicit Divisor(int64_t by) : m(0), s(0), d((uint32_t)by) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)((((1ull << s) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int of(int n) const { return (int)(((uint32_t)n + __umulhi((uint32_t)n, m)) >> s); }
};

constexpr double QUARTERS = 0.636619772367581343;      // 2 / pi

struct Turn {
  float cos, sin;
};

// pos, and f 2 / pi
__device__ __forceinline__ Turn turn_of(double pos, double quarters) {
  constexpr double WHOLE = 6755399441055744.0;         // 1.5 * 2^52
  const double s = __builtin_fma(pos, quarters, WHOLE);
  const uint32_t quadrant = (uint32_t)__builtin_bit_cast(uint64_t, s);
  const float r = (float)__builtin_fma(pos, quarters, -(s - WHOLE));
  const float r2 = r * r;
  // (pi / 2)^n / n!, alternating
  float sn = __builtin_fmaf(r2, 1.6044118478735982e-4f, -4.6817541353186881e-3f);
  sn = __builtin_fmaf(r2, sn, 7.9692626246167046e-2f);
  sn = __builtin_fmaf(r2, sn, -6.4596409750624625e-1f);
  sn = __builtin_fmaf(r2, sn, 1.5707963267948966f) * r;
  float cs = __builtin_fmaf(r2, -2.5202042373060605e-5f, 9.1926027483942658e-4f);
  cs = __builtin_fmaf(r2, cs, -2.0863480763352961e-2f);
  cs = __builtin_fmaf(r2, cs, 2.5366950790104802e-1f);
  cs = __builtin_fmaf(r2, cs, -1.2337005501361698f);
  cs = __builtin_fmaf(r2, cs, 1.0f);
  const bool odd = quadrant & 1;
  const float c = odd ? sn : cs, n = odd ? cs : sn;
  return {((quadrant + 1) & 2) ? -c : c, (quadrant & 2) ? -n : n};
}

// Rows of 16-bit or 32-bit floats start wherever their strides put them: eight values in one or two loads of no alignment
// but the type's.
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (DT == XDNA_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4_4 w = *reinterpret_cast<const u32x4_4*>(static_cast<const float*>(base) + at + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * h + e] = __uint_as_float(w[e]);
    }
  } else {
    const u32x4_2 w = *reinterpret_cast<const u32x4_2*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
      x[e] = DT == XDNA_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&x)[8]) {
  if constexpr (DT == XDNA_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4_4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(x[4 * h + e]);
      *reinterpret_cast<u32x4_4*>(static_cast<float*>(base) + at + 4 * h) = w;
    }
  } else {
    u32x4_2 w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = DT == XDNA_F16 ? f32x2_to_f16x2_bits(x[2 * e], x[2 * e + 1]) : f32x2_to_bf16x2_bits(x[2 * e], x[2 * e + 1]);
    *reinterpret_cast<u32x4_2*>(static_cast<uint16_t*>(base) + at) = w;
  }
}

// The first n of eight (n <= 8): all of them at once, or one by one at the end of a row. Those past n are 0.
template <int DT>
__device__ __forceinline__ void load_upto8(const void* base, int64_t at, int n, float (&x)[8]) {
  if (n == 8) return load8<DT>(base, at, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < n ? load_as_f32<DT>(base, at + e) : 0.0f;
}
template <int DT>
__device__ __forceinline__ void store_upto8(void* base, int64_t at, int n, const float (&x)[8]) {
  if (n == 8) return store8<DT>(base, at, x);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) store_from_f32<DT>(base, at + e, x[e]);
}

// A head's dims in units of up to 16 values, two runs of up to eight: eight pairs of those that turn (pair j: dims j and
// half + j, or 2 j and 2 j + 1), or sixteen of the dims behind them, which stay as they are.
struct Unit {
  int a, b, na, nb;       // first dims of the two runs and how many
  int pair;               // first pair, or -1
};
__host__ __device__ inline int units_of(int d, int half) { return (half + 7) / 8 + (d - 2 * half + 15) / 16; }

template <bool INTER>
__device__ __forceinline__ Unit unit_of(int u, int d, int half) {
  const int turning = (half + 7) / 8;
  if (u < turning) {
    const int n = min(8, half - 8 * u);
    if (INTER) return {16 * u, 16 * u + 8, min(8, 2 * n), max(0, 2 * n - 8), 8 * u};
    return {8 * u, half + 8 * u, n, n, 8 * u};
  }
  const int at = 2 * half + 16 * (u - turning);
  return {at, at + 8, min(8, d - at), max(0, min(8, d - at - 8)), -1};
}

// The pairs of a unit's two runs by cos and sin (of its eight pairs).
template <bool INTER>
__device__ __forceinline__ void turn16(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float &x = INTER ? (e < 4 ? a[2 * e] : b[2 * e - 8]) : a[e], &y = INTER ? (e < 4 ? a[2 * e + 1] : b[2 * e - 7]) : b[e];
    const float p = x, q = y;
    x = __builtin_fmaf(p, cs[e], -(q * sn[e]));
    y = __builtin_fmaf(q, cs[e], p * sn[e]);
  }
}

}  // namespace xdna
