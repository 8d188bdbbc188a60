// Products with 4-bit weights, for gfx950 (MI355X):
//
//   y[m, n] = sum over groups g of s[n, g] * (sum over k in g of (q[n, k] - z[n, g]) * x[m, k])  (+ bias[n])
//
// q: two weights a byte along K, the even one in the low nibble; a group is G consecutive k (G % 32 == 0, K % G == 0).
//
// The weights are whole numbers until their group's sum is done, so nothing is rounded before the float32 sums: the
// matrix instruction multiplies x by q - z (or by 128 + q, below), its float32 result takes the group's scale as one
// fma per output. x is the row operand (lane l: row l % 16, 8 of 32 k), the weights the column operand (lane l:
// column l % 16), so a lane of the result holds four rows of one column and needs one scale.
//
// Unpacking: nibbles i and i + 4 of a word are the halves of (w >> 4 i) & 0x000f000f, so the bits of 128 (bfloat16) or
// 1024 (float16) ORed into both halves make two floats of value 128 + q or 1024 + q in one more instruction; x takes
// the same order of k by four byte permutes per 8 values. float16 subtracts 1024 + z at once (exact, packed).
// bfloat16 has no packed add here: the sum over 128 + q stays, and (128 + z) times the group's sum of x, a product
// with a column of ones, is taken off in float32. The sums are then up to 30 times the result's own size, 2^-19 in the
// float32 sums against the output's 2^-9. Where x is not finite that difference is not what the formula says
// (inf - inf), so a lane whose sum came out not finite adds its part again, value by value. float32 x
// goes in as three bfloat16 numbers that add up to it exactly (8 bits each, cut, not rounded) and meets
// weights converted one by one, q - z.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xdna_common.h"
#include "xdna_hip.h"

namespace xdna {
namespace {

typedef __bf16 bf16x8w __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8w __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const i32x4& a, const i32x4& b, const f32x4& c) {
  if constexpr (DT == XDNA_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8w, a), __builtin_bit_cast(f16x8w, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8w, a), __builtin_bit_cast(bf16x8w, b), c, 0, 0,
                                                   0);
}

// 8 weights of one word, nibbles 0 4 1 5 2 6 3 7. bfloat16: 128 + q; float16: q - z; float32: q - z as bfloat16.
template <int DT>
__device__ __forceinline__ i32x4 unpack(uint32_t w, float z) {
  i32x4 r;
  if constexpr (DT == XDNA_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)(((w >> (4 * i)) & 0x000f000fu) | 0x43004300u);
  } else if constexpr (DT == XDNA_F16) {
    const _Float16 off = (_Float16)(-1024.0f - z);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2_t v = __builtin_bit_cast(f16x2_t, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u);
      r[i] = __builtin_bit_cast(int, v + (f16x2_t){off, off});
    }
  } else {
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;    // nibbles 0 2 4 6 and 1 3 5 7, a byte each
    auto f = [&](uint32_t v, int byte) { return (float)((v >> (8 * byte)) & 0xffu) - z; };
    r[0] = (int)f32x2_to_bf16x2_bits(f(even, 0), f(even, 2));
    r[1] = (int)f32x2_to_bf16x2_bits(f(odd, 0), f(odd, 2));
    r[2] = (int)f32x2_to_bf16x2_bits(f(even, 1), f(even, 3));
    r[3] = (int)f32x2_to_bf16x2_bits(f(odd, 1), f(odd, 3));
  }
  return r;
}

// 8 consecutive 16-bit values in the order of unpack's.
__device__ __forceinline__ i32x4 reorder(const uint4& v) {
  return i32x4{(int)__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), (int)__builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
               (int)__builtin_amdgcn_perm(v.w, v.y, 0x05040100u), (int)__builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}

// word j of the result in the lanes of quarter a: word a of v in the lanes of quarter j
__device__ __forceinline__ void transpose_quarters(uint32_t (&v)[4]) {
  const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v[0] = c[0];
  v[1] = c[1];
  v[2] = d[0];
  v[3] = d[1];
}

// One workgroup: 16 columns x 16 MT rows, the chunks of 128 k dealt out to its W waves, which meet in LDS. FL: matrix
// steps (32 k each) of a group's sum before its scale, 4 where G % 128 == 0, 2 where G % 64 == 0, else 1. A lane's
// 16-byte load holds 32 consecutive weights of its column; with FL == 4 the four quarters of a step may be any 32 of
// the chunk's 128 k, else they have to be 32 consecutive ones and the words change quarters first.
template <int DT, int SDT, int MT, int FL, int W>
__global__ __launch_bounds__(W * 64) void w4_kernel(const void* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ qw,
                                                    const void* __restrict__ scales, const uint8_t* __restrict__ zeros,
                                                    const void* __restrict__ bias, int bias_dt, void* __restrict__ y,
                                                    int64_t M, int64_t N, int K, int G) {
  constexpr int U = MT == 1 ? 4 : 2;           // chunks in flight
  constexpr int XP = DT == XDNA_F32 ? 3 : 1;   // bfloat16 parts of x
  __shared__ f32x4 red[W * MT * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quarter = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
  const int cols = (int)min<int64_t>(16, N - n0), rows = (int)min<int64_t>(16 * MT, M - m0);
  const int groups = K / G, chunks = (K + 127) >> 7;
  const uint32_t esz = DT == XDNA_F32 ? 4 : 2;
  const auto wr = make_rsrc(qw + n0 * (K / 2), (uint32_t)(cols * (K / 2)));
  const auto xr = make_rsrc(static_cast<const char*>(x) + m0 * ldx * esz, (uint32_t)(((rows - 1) * ldx + K) * esz));
  const int64_t sbase = (n0 + min(col, cols - 1)) * groups;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int c0 = wave; c0 < chunks; c0 += W * U) {
    uint4 wv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * W;
      const bool in = c < chunks && c * 128 + quarter * 32 < K;
      wv[u] = buf_load_u4(wr, in ? (uint32_t)(col * (K / 2) + c * 64 + quarter * 16) : OOB);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * W;
      if (c >= chunks) break;
      uint32_t w[4] = {wv[u].x, wv[u].y, wv[u].z, wv[u].w};
      if constexpr (FL < 4) transpose_quarters(w);
#pragma unroll
      for (int f = 0; f < 4 / FL; ++f) {
        const int k0 = c * 128 + f * FL * 32;    // uniform
        if (k0 >= K) break;
        const int g = k0 / G;
        const float s = load_as_f32<SDT>(scales, sbase + g);
        const float z = zeros ? (float)zeros[sbase + g] : 8.0f;
        f32x4 part[MT], sum[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) part[t] = sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = f * FL; j < (f + 1) * FL; ++j) {
          const int k = c * 128 + (FL == 4 ? 32 * quarter + 8 * j : 32 * j + 8 * quarter);
          const i32x4 wf = unpack<DT>(w[j], z);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int row = 16 * t + col;
            const uint32_t off = row < rows && k < K ? (uint32_t)((row * ldx + k) * esz) : OOB;
            if constexpr (DT == XDNA_F32) {
              const uint4 a = buf_load_u4(xr, off), b = buf_load_u4(xr, off == OOB ? OOB : off + 16);
              const uint32_t raw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
              uint32_t h[XP][8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const bool fin = (raw[e] & 0x7f800000u) != 0x7f800000u;
                const float v = __uint_as_float(raw[e]);
                h[0][e] = (raw[e] & 0xffff0000u) | (!fin && (raw[e] & 0x007fffffu) ? 0x00400000u : 0u);   // NaN stays NaN
                const float r1 = fin ? v - __uint_as_float(h[0][e]) : 0.0f;
                h[1][e] = __float_as_uint(r1) & 0xffff0000u;
                h[2][e] = __float_as_uint(r1 - __uint_as_float(h[1][e]));
              }
#pragma unroll
              for (int p = XP - 1; p >= 0; --p) {
                i32x4 xf;
#pragma unroll
                for (int e = 0; e < 4; ++e) xf[e] = (int)((h[p][e] >> 16) | (h[p][e + 4] & 0xffff0000u));
                part[t] = mfma16<DT>(xf, wf, part[t]);
              }
            } else {
              const i32x4 xf = reorder(buf_load_u4(xr, off));
              part[t] = mfma16<DT>(xf, wf, part[t]);
              if constexpr (DT == XDNA_BF16) {
                const i32x4 ones = i32x4{0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};
                sum[t] = mfma16<DT>(xf, ones, sum[t]);
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = part[t][r];
            if constexpr (DT == XDNA_BF16) v = __builtin_fmaf(-(128.0f + z), sum[t][r], v);
            acc[t][r] = __builtin_fmaf(s, v, acc[t][r]);
          }
      }
    }
  }
  if constexpr (DT == XDNA_BF16) {
    bool odd = false;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !(fabsf(acc[t][r]) < INFINITY);
    if (__builtin_amdgcn_ballot_w64(odd)) {      // x (or a scale) that is not finite: the wave's part again, one by one
#pragma unroll 1
      for (int e = 0; e < MT * 4; ++e) {
        const int row = 16 * (e >> 2) + 4 * quarter + (e & 3);
        if (row >= rows || col >= cols) continue;
        float v = 0.0f;
        for (int c = wave; c < chunks; c += W)
          for (int k = c * 128; k < min(K, c * 128 + 128); ++k) {
            const int64_t sg = sbase + k / G;
            const uint8_t b = qw[(n0 + col) * (K / 2) + (k >> 1)];
            const float q = (float)((k & 1) ? b >> 4 : b & 15) - (zeros ? (float)zeros[sg] : 8.0f);
            v = __builtin_fmaf(q * load_as_f32<SDT>(scales, sg), load_as_f32<DT>(x, (m0 + row) * ldx + k), v);
          }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t == (e >> 2) && r == (e & 3) && !(fabsf(acc[t][r]) < INFINITY)) acc[t][r] = v;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[(wave * MT + t) * 64 + lane] = acc[t];
  __syncthreads();
  // element i of the tile: row i / 16, column i % 16, which lane 16 (row % 16 / 4) + column holds in its element row % 4
  for (int i = threadIdx.x; i < MT * 256; i += W * 64) {
    const int row = i >> 4, cc = i & 15;
    if (row >= rows || cc >= cols) continue;
    const int at = (row >> 4) * 64 + ((row & 15) >> 2) * 16 + cc;
    float v = 0.0f;
#pragma unroll
    for (int wv = 0; wv < W; ++wv) v += red[wv * MT * 64 + at][row & 3];
    if (bias) {
      v += bias_dt == XDNA_F32    ? load_as_f32<XDNA_F32>(bias, n0 + cc)
           : bias_dt == XDNA_BF16 ? load_as_f32<XDNA_BF16>(bias, n0 + cc)
                                  : load_as_f32<XDNA_F16>(bias, n0 + cc);
    }
    store_from_f32<DT>(y, (m0 + row) * N + n0 + cc, v);
  }
}

struct W4Args {
  const void* x;
  int64_t ldx;
  const uint8_t* qw;
  const void* scales;
  const uint8_t* zeros;
  const void* bias;
  int bias_dt;
  void* y;
  int64_t M, N;
  int K, G;
  hipStream_t st;
};

template <int DT, int SDT, int MT, int FL>
int w4_go(const W4Args& a) {
  constexpr int W = 8;
  // rows of a launch: the grid's y and the threads of a launch along x
  const int64_t rows = std::min<int64_t>(65535, cdiv(a.M, 16 * MT)) * (16 * MT);
  for (int64_t m = 0; m < a.M; m += rows) {
    const int64_t n = std::min(rows, a.M - m);
    const int esz = DT == XDNA_F32 ? 4 : 2;
    w4_kernel<DT, SDT, MT, FL, W><<<dim3((unsigned)cdiv(a.N, 16), (unsigned)cdiv(n, 16 * MT)), W * 64, 0, a.st>>>(
        static_cast<const char*>(a.x) + m * a.ldx * esz, a.ldx, a.qw, a.scales, a.zeros, a.bias, a.bias_dt,
        static_cast<char*>(a.y) + m * a.N * esz, n, a.N, a.K, a.G);
  }
  return launch_status("linear_w4");
}

template <int DT, int SDT, int MT>
int w4_group(const W4Args& a) {
  if (a.G % 128 == 0) return w4_go<DT, SDT, MT, 4>(a);
  if (a.G % 64 == 0) return w4_go<DT, SDT, MT, 2>(a);
  return w4_go<DT, SDT, MT, 1>(a);
}

template <int DT, int SDT>
int w4_rows(const W4Args& a) {
  if (a.M <= 16) return w4_group<DT, SDT, 1>(a);
  if (a.M <= 32) return w4_group<DT, SDT, 2>(a);
  return w4_group<DT, SDT, 4>(a);
}

template <int DT>
int w4_scales(const W4Args& a, int sdt) {
  if (sdt == XDNA_F32) return w4_rows<DT, XDNA_F32>(a);
  if (sdt == XDNA_BF16) return w4_rows<DT, XDNA_BF16>(a);
  return w4_rows<DT, XDNA_F16>(a);
}

bool is_float(int dt) { return dt == XDNA_F32 || dt == XDNA_BF16 || dt == XDNA_F16; }

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_linear_w4(const void* x, int x_dtype, int64_t ldx, const void* qweight, const void* scales, int s_dtype,
                   const void* zeros, const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                   int64_t group, void* stream) {
  XDNA_REQUIRE(is_float(x_dtype) && is_float(s_dtype), "x_dtype and s_dtype must be F32/BF16/F16");
  XDNA_REQUIRE(!bias || is_float(bias_dtype), "bias_dtype must be F32/BF16/F16");
  XDNA_REQUIRE(M >= 0 && N >= 0 && K >= 0 && group >= 32 && group % 32 == 0 && K % group == 0,
               "group must be a multiple of 32 and K one of the group");
  if (M == 0 || N == 0) return XDNA_OK;
  const int64_t esz = x_dtype == XDNA_F32 ? 4 : 2;
  // 31-bit offsets within 64 rows of x and 16 columns of the weights, and the launch's threads along x
  XDNA_REQUIRE(K >= 1 && K <= (1ll << 22) && ldx >= K && ldx <= (1ll << 22) && N <= (1ll << 26), "sizes too large, or ldx < K");
  XDNA_REQUIRE(x && qweight && scales && y, "null pointer");
  XDNA_REQUIRE(aligned(x, 16) && ldx * esz % 16 == 0 && aligned(qweight, 16), "x rows and qweight must be 16-byte aligned");
  const W4Args a{x, ldx, static_cast<const uint8_t*>(qweight), scales, static_cast<const uint8_t*>(zeros), bias, bias_dtype,
                 y, M, N, (int)K, (int)group, as_stream(stream)};
  if (x_dtype == XDNA_F32) return w4_scales<XDNA_F32>(a, s_dtype);
  if (x_dtype == XDNA_BF16) return w4_scales<XDNA_BF16>(a, s_dtype);
  return w4_scales<XDNA_F16>(a, s_dtype);
}

}  // extern "C"
