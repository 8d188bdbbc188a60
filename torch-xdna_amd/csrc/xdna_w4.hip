// Products with 4-bit weights, for gfx950 (MI355X):
//
//   y[m, n] = sum over groups g of s[n, g] * (sum over k in g of (q[n, k] - z[n, g]) * x[m, k])  (+ bias[n])
//
// q: two weights a byte along K, the even one in the low nibble; a group is G consecutive k (G % 32 == 0, K % G == 0).
//
// The weights are whole numbers until their group's sum is done, so nothing is rounded before the float32 sums: x is
// multiplied by q - z (or by 128 + q, below), the float32 sum takes the group's scale as one fma.
//
// Unpacking: byte p of a word and of the word shifted by 4, put side by side by one byte permute, have q[2p] and q[2p
// + 1] in the low bits of their halves; masked and with the bits of 128 (bfloat16) or 1024 (float16) ORed in they are
// two floats of value 128 + q or 1024 + q. float16 subtracts 1024 + z at once (exact, packed). bfloat16 has no packed
// add here: the sum over 128 + q stays, and (128 + z) times the group's sum of x is taken off in float32. The sums
// are then up to 30 times the result's own size, 2^-19 in the float32 sums against the output's 2^-9. Where x is not
// finite that difference is not what the formula says (inf - inf), so such sums are formed again, value by value.
// float32 x meets weights converted one by one, q - z; for the matrix units it is cut into three bfloat16 numbers
// that add up to it exactly; its sums before the scale, up to 255 times |x|, may pass float32 where the result does not,
// and those that do are formed again too, the scale first.
//
// One row (a decode step), and up to four where the weights are few, are dot products on the vector units:
// w4_row_kernel. More go to the matrix units, x through LDS: w4_tile_kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "xdna_common.h"
#include "xdna_hip.h"

namespace xdna {
namespace {

typedef __bf16 bf16x8w __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8w __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_void;

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const i32x4& a, const i32x4& b, const f32x4& c) {
  if constexpr (DT == XDNA_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8w, a), __builtin_bit_cast(f16x8w, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8w, a), __builtin_bit_cast(bf16x8w, b), c, 0, 0,
                                                   0);
}

// 8 weights of one word in their order. bfloat16: 128 + q; float16: q - z; float32: q - z as bfloat16.
template <int DT>
__device__ __forceinline__ i32x4 unpack(uint32_t w, float z) {
  i32x4 r;
  const uint32_t w4 = w >> 4;
  if constexpr (DT == XDNA_F32) {
    auto f = [&](uint32_t v, int byte) { return (float)((v & 0x0f0f0f0fu) >> (8 * byte) & 0xffu) - z; };
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (int)f32x2_to_bf16x2_bits(f(w, i), f(w4, i));
  } else {
    uint32_t mask = 0x000f000fu, one = DT == XDNA_BF16 ? 0x43004300u : 0x64006400u;
    asm("" : "+v"(mask), "+s"(one));         // in registers, so that and and or are one instruction
    const _Float16 off = (_Float16)(-1024.0f - z);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // bytes 0 and 1: byte i of w and a zero; bytes 2 and 3: byte i of w4 and a zero
      const uint32_t v = __builtin_amdgcn_perm(w4, w, 0x0c000c00u | (uint32_t)((4 + i) << 16) | (uint32_t)i);
      if constexpr (DT == XDNA_BF16) {
        r[i] = (int)((v & mask) | one);
      } else {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, (v & mask) | one);
        r[i] = __builtin_bit_cast(int, h + (f16x2_t){off, off});
      }
    }
  }
  return r;
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

// A float32 x as three bfloat16 numbers (8 bits each, cut, not rounded) whose sum it is; not finite: itself and zeros.
__device__ __forceinline__ void split3(const uint32_t (&v)[8], i32x4 (&p)[3]) {
  uint32_t h[3][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool fin = (v[e] & 0x7f800000u) != 0x7f800000u;
    h[0][e] = (v[e] & 0xffff0000u) | (!fin && (v[e] & 0x007fffffu) ? 0x00400000u : 0u);   // NaN stays NaN
    const float r1 = fin ? __uint_as_float(v[e]) - __uint_as_float(h[0][e]) : 0.0f;
    h[1][e] = __float_as_uint(r1) & 0xffff0000u;
    h[2][e] = __float_as_uint(r1 - __uint_as_float(h[1][e]));
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) p[i][e] = (int)((h[i][2 * e] >> 16) | (h[i][2 * e + 1] & 0xffff0000u));
}

// The words of a load, taken apart here and not before: the compiler would otherwise copy them to registers of their
// own, and wait for the load, right where it is issued.
__device__ __forceinline__ void words(const uint4& v, uint32_t (&w)[4]) {
  i32x4 t = {(int)v.x, (int)v.y, (int)v.z, (int)v.w};
  asm volatile("" : "+v"(t));
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)t[i];
}

struct W4Args {
  const void* x;
  int64_t ldx;
  const uint8_t* qw;
  const void* scales;
  int sdt;
  const uint8_t* zeros;
  const void* bias;
  int bias_dt;
  void* y;
  float* part;          // [parts][M][N] float32 sums where K is split over workgroups
  int64_t M, N;
  int K, G;
  int per;              // rows: waves that share a set of columns; tiles: x tiles of a part of K
};

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dt) {
  return dt == XDNA_F32 ? load_as_f32<XDNA_F32>(p, i) : dt == XDNA_BF16 ? load_as_f32<XDNA_BF16>(p, i) : load_as_f32<XDNA_F16>(p, i);
}

// a scale's bits as they are loaded, and its value
template <bool S4>
__device__ __forceinline__ uint32_t scale_bits(const void* p, int64_t i) {
  if constexpr (S4) return static_cast<const uint32_t*>(p)[i];
  else return static_cast<const uint16_t*>(p)[i];
}
template <bool S4>
__device__ __forceinline__ float scale_value(uint32_t s, int dt) {
  return S4 ? __uint_as_float(s) : dt == XDNA_BF16 ? __uint_as_float(s << 16) : f16_bits_to_f32((uint16_t)s);
}

// ------------------------------------------------------------------------------ one to four rows
constexpr int W4_ROW_LDS = 32768;     // of x
constexpr int W4_ROW_GROUPS = 4096;   // scales and zero points of a workgroup
// A wave has 64 / KL columns; a lane's 16-byte load is 32 consecutive weights of one column, KL lanes side by side read
// 16 KL bytes of it. a.per waves share a set of columns, the blocks of 32 KL weights dealt out to them; lanes meet by
// shuffles, waves in LDS, both in a fixed order.
// What a CU's address unit can take bounds such a kernel as much as the memory: a load costs it 16 cycles at least,
// however little it fetches. So x, the scales and the zero points come into LDS once per workgroup, line by line, by
// pieces of PB blocks (with a lane's own loads of them 1 x 4096 -> 14336 took 24 us, so 12.5).
template <int DT, bool S4, int KL, int R>
__global__ __launch_bounds__(512) void w4_row_kernel(W4Args a) {
  constexpr int W = 8, CL = 64 / KL;                    // waves, columns of a load
  constexpr int XV = DT == XDNA_F32 ? 8 : 4;            // 16-byte chunks of a lane's 32 values
  constexpr int BCH = KL * XV;                          // chunks of a block of x
  constexpr int PB = W4_ROW_LDS / (BCH * 16 * R);
  constexpr int COLS = W * CL;                          // of a workgroup where each wave has its own
  constexpr int SB = S4 ? 4 : 2, GW = W4_ROW_GROUPS / COLS;    // groups of a column that LDS holds
  static_assert(PB >= 1, "a block fits");
  __shared__ uint4 xl[R][PB * BCH];
  __shared__ __attribute__((aligned(16))) uint8_t sl[COLS * GW * SB], zl[COLS * GW];
  __shared__ float red[W][R][CL];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kl = lane % KL, cl = lane / KL;
  const int K = a.K, G = a.G, groups = K / G, per = a.per;
  const int set = wave / per, sets = W / per;
  const int64_t wg0 = (int64_t)blockIdx.x * sets * CL, n0 = wg0 + set * CL;
  const int ki = wave % per, blocks = (K + 32 * KL - 1) / (32 * KL);
  const int rows = (int)a.M;
  constexpr uint32_t esz = DT == XDNA_F32 ? 4 : 2;
  const int cols = (int)max<int64_t>(0, min<int64_t>(CL, a.N - n0)), wcols = (int)min<int64_t>(sets * CL, a.N - wg0);
  const auto wr = make_rsrc(a.qw + (cols ? n0 : 0) * (K / 2), (uint32_t)cols * (uint32_t)(K / 2));
  auto place = [](int l, int i) { return l * XV + (i ^ (XV == 4 ? (l >> 2) & 3 : (l >> 1) & 7)); };   // banks apart
  float acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  uint4 x_[R][XV];
  float s, z;
  const uint8_t* const zeros = a.zeros ? a.zeros : static_cast<const uint8_t*>(a.scales);    // read in any case, 8 put in later
  auto fetch = [&](int b, int end, uint4& l) {
    const int k = (b * KL + kl) * 32;
    l = buf_load_u4<true>(wr, b < end && k < K ? (uint32_t)(cl * (K / 2) + k / 2) : OOB);
  };
  auto use = [&](const uint4& l) {
    const uint32_t w[4] = {l.x, l.y, l.z, l.w};
    float v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = 0.0f;
    if constexpr (DT == XDNA_F32) {
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float q = (float)(w[e >> 3] >> (4 * (e & 7)) & 15u) - z;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4 x = x_[r][e >> 2];
          const uint32_t xe[4] = {x.x, x.y, x.z, x.w};
          v[r] = __builtin_fmaf(q, __uint_as_float(xe[e & 3]), v[r]);
        }
      }
    } else {
      auto dot = [](uint32_t x, uint32_t y, float v) {
        if constexpr (DT == XDNA_F16)
          return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, x), __builtin_bit_cast(f16x2_t, y), v, false);
        else
          return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, y), v, false);
      };
      float xs[R];
#pragma unroll
      for (int r = 0; r < R; ++r) xs[r] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const i32x4 q = unpack<DT>(w[j], z);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t x[4] = {x_[r][j].x, x_[r][j].y, x_[r][j].z, x_[r][j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[r] = dot(x[e], (uint32_t)q[e], v[r]);
            if constexpr (DT == XDNA_BF16) xs[r] = dot(x[e], 0x3f803f80u, xs[r]);
          }
        }
      }
      if constexpr (DT == XDNA_BF16) {
        bool odd = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          v[r] = __builtin_fmaf(-(128.0f + z), xs[r], v[r]);
          odd |= !(fabsf(v[r]) < INFINITY);
        }
        if (__builtin_amdgcn_ballot_w64(odd)) {
          // x is not finite, or so large that the sums before the scale are not: value by value, the scale first
#pragma unroll 1
          for (int e = 0; e < 32; ++e) {
            const uint32_t we = e < 16 ? (e < 8 ? w[0] : w[1]) : (e < 24 ? w[2] : w[3]);
            const float q = ((float)(we >> (4 * (e & 7)) & 15u) - z) * s;
#pragma unroll
            for (int r = 0; r < R; ++r) {
              uint32_t x = 0;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t xv[4] = {x_[r][i >> 2].x, x_[r][i >> 2].y, x_[r][i >> 2].z, x_[r][i >> 2].w};
                x = e >> 1 == i ? xv[i & 3] : x;
              }
              acc[r] = __builtin_fmaf(q, bf16_bits_to_f32((uint16_t)((e & 1) ? x >> 16 : x)), acc[r]);
            }
          }
          return;
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = __builtin_fmaf(s, v[r], acc[r]);
  };
  // Two blocks of weights are in flight, the first two from before x and the scales are. Pieces: as many blocks as both
  // hold of x and of the scales.
  uint4 ring[2];
  const int piece = min(PB, (GW - 1) * G / (32 * KL));
  for (int p0 = 0; p0 < blocks; p0 += piece) {
    const int pend = min(p0 + piece, blocks);
    const int k0 = p0 * (32 * KL), g0 = k0 / G, gn = (min(K, pend * (32 * KL)) - 1) / G + 1 - g0;     // groups of the piece
    if (p0) __syncthreads();
    fetch(p0 + ki, pend, ring[0]);
    fetch(p0 + ki + per, pend, ring[1]);
    // chunk i of a row: values i * 16 / esz .. of the piece
    for (int i = threadIdx.x; i < PB * BCH; i += W * 64) {
      const int64_t k = (int64_t)k0 + i * (int)(16 / esz);
      if (k >= K) break;
#pragma unroll
      for (int r = 0; r < R; ++r)
        xl[r][i / BCH * BCH + place(i % BCH / XV, i % XV)] =
            *reinterpret_cast<const uint4*>(static_cast<const char*>(a.x) + (min(r, rows - 1) * a.ldx + k) * esz);
    }
    const bool whole = gn == groups;           // then the columns' groups are one run
    const int elems = wcols * gn;
    for (int i0 = threadIdx.x; i0 < elems; i0 += 4 * W * 64) {     // four loads of each at a time
      uint32_t sv[4], zv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = min(i0 + j * (W * 64), elems - 1);
        const int64_t at = whole ? wg0 * groups + i : (wg0 + i / gn) * groups + g0 + i % gn;
        sv[j] = scale_bits<S4>(a.scales, at);
        zv[j] = zeros[at];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = min(i0 + j * (W * 64), elems - 1);           // past the end: the last one again
        if constexpr (S4) reinterpret_cast<uint32_t*>(sl)[i] = sv[j];
        else reinterpret_cast<uint16_t*>(sl)[i] = (uint16_t)sv[j];
        zl[i] = a.zeros ? (uint8_t)zv[j] : 8;
      }
    }
    __syncthreads();
    auto block = [&](int b, const uint4& l) {
      const int k = min((b * KL + kl) * 32, K - 32), g = k / G - g0;
      const int i = min(set * CL + cl, wcols - 1) * gn + g;
      s = S4 ? reinterpret_cast<const float*>(sl)[i]
             : scale_value<false>(reinterpret_cast<const uint16_t*>(sl)[i], a.sdt);
      z = (float)zl[i];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < XV; ++v) {
          x_[r][v] = xl[r][(b - p0) * BCH + place(kl, v)];
          if ((b * KL + kl) * 32 >= K) x_[r][v] = make_uint4(0, 0, 0, 0);
        }
      use(l);
    };
    int b = p0 + ki;
    for (; b + 2 * per < pend; b += 2 * per) {
      block(b, ring[0]);
      fetch(b + 2 * per, pend, ring[0]);
      block(b + per, ring[1]);
      fetch(b + 3 * per, pend, ring[1]);
    }
    if (b < pend) block(b, ring[0]);
    if (b + per < pend) block(b + per, ring[1]);
  }
  if constexpr (DT == XDNA_F32) {
    // x or a scale is not finite, or a sum before its scale passes float32: the lane's values again, the scale first
    bool odd = false;
#pragma unroll
    for (int r = 0; r < R; ++r) odd |= cl < cols && !(fabsf(acc[r]) < INFINITY);
    if (__builtin_amdgcn_ballot_w64(odd)) {
      const int64_t n = wg0 + min(set * CL + cl, wcols - 1);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (cl >= cols || fabsf(acc[r]) < INFINITY) continue;
        float v = 0.0f;
        for (int p0 = 0; p0 < blocks; p0 += piece)
          for (int b = p0 + ki; b < min(p0 + piece, blocks); b += per)
            for (int k = (b * KL + kl) * 32; k < min(K, (b * KL + kl) * 32 + 32); ++k) {
              const int64_t at = n * groups + k / G;
              const uint8_t w = a.qw[n * (K / 2) + (k >> 1)];
              const float q = (float)((k & 1) ? w >> 4 : w & 15) - (a.zeros ? (float)a.zeros[at] : 8.0f);
              v = __builtin_fmaf(q * load_any(a.scales, at, a.sdt), load_as_f32<DT>(a.x, min(r, rows - 1) * a.ldx + k), v);
            }
        acc[r] = v;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float v = acc[r];
#pragma unroll
    for (int o = KL / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if (kl == 0) red[wave][r][cl] = v;
  }
  __syncthreads();
  // output i: column i % CL of set i / CL / R, row i / CL % R
  for (int i = threadIdx.x; i < sets * R * CL; i += W * 64) {
    const int cc = i % CL, r = i / CL % R, of = i / (CL * R);
    const int64_t n = wg0 + of * CL + cc;
    if (n >= a.N || r >= rows) continue;
    float v = 0.0f;
    for (int q = 0; q < per; ++q) v += red[of * per + q][r][cc];
    if (a.bias) v += load_any(a.bias, n, a.bias_dt);
    store_from_f32<DT>(a.y, r * a.N + n, v);
  }
}

// ------------------------------------------------------------------------------ more rows
// One workgroup: 16 MT rows x 16 W columns (wave w: columns 16 w .. + 15), one part of K (grid z) in tiles of 128 or
// 256 k, whose x all waves read from LDS. x is the MFMA's row operand (lane l: row l % 16, 8 of 32 k), the weights
// its column operand (lane l: column l % 16), so a lane of the result holds four rows of one column and needs one
// scale. A lane's 16-byte load of weights is 32 consecutive ones of its column; the words change quarters so that a
// step's four quarters are 32 consecutive k. Two tiles' x (DMA into LDS) and weights are on their way while a third is
// used. Scales and zero points come into LDS for WIN k at a time. FL: steps (32 k each) of a group's sum
// before its scale: 4 where G % 128 == 0, 2 where G % 64 == 0, else 1. Measured with the join: 40 x 14336 -> 4096 in
// float16 23 us (33.6 MB), 8 x 4096 -> 14336 in bfloat16 13.8 us (33 MB). Counted: 40 rows about 190 vector instructions a
// wave and 128 k against 12 MFMAs, 1 x 4096 -> 14336 about 200 a wave and 256 k against 16; vector units active 48% and 52%
// of the CUs' busy time, MFMA 11% and 15%, and waves wait 43% of theirs in both: two waves a SIMD hide neither in the other.
// KG groups of four waves share out a part's tiles (group GI the GI-th run of them), each with LDS of its own, and meet in
// LDS at the end: as good as more parts, without their join. All groups pass the same barriers, whatever tiles there are.
template <int DT, bool S4, int MT, int FL, int KG, int GI>
__device__ __forceinline__ void w4_tiles(const W4Args& a, f32x4 (&acc)[MT]) {
  constexpr int W = 4;                                  // waves
  constexpr int XP = DT == XDNA_F32 ? 3 : 1, GC = 4 / FL, D = 3;
  constexpr uint32_t esz = DT == XDNA_F32 ? 4 : 2;
  constexpr int U = DT == XDNA_F32 || MT > 2 ? 1 : 2, KT = 128 * U;     // chunks of 128 k of a tile
  constexpr int RB = KT * (int)esz, RCH = RB / 16;      // bytes and 16-byte chunks of a row
  constexpr int TILE = 16 * MT * RB, NL = TILE / 1024 / W;     // 1 KB loads of x per wave
  constexpr int LP = NL + U;                            // loads of a tile per wave
  constexpr int COLS = 16 * W, WIN = MT > 2 ? 1024 : 2048, GW = WIN / (FL * 32);     // k and groups of a window
  static_assert(NL >= 1, "every wave loads");
  // one array for each tile: the compiler then knows which loads a read has to wait for
  __shared__ __attribute__((aligned(1024))) int8_t lds0[TILE];
  __shared__ __attribute__((aligned(1024))) int8_t lds1[TILE];
  __shared__ __attribute__((aligned(1024))) int8_t lds2[TILE];
  __shared__ float sl[GW * COLS];                       // group by group, so that a wave's columns lie side by side
  __shared__ uint8_t zl[GW * COLS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W, tid = threadIdx.x % (W * 64);
  const int col = lane & 15, quarter = lane >> 4;
  const int64_t N = a.N;
  const int K = a.K, G = a.G, groups = K / G;
  const int64_t w0 = (int64_t)blockIdx.x * COLS, n0 = w0 + wave * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
  const int cols = (int)max<int64_t>(0, min<int64_t>(16, N - n0)), rows = (int)min<int64_t>(16 * MT, a.M - m0);
  const int wcols = (int)min<int64_t>(COLS, N - w0), scol = min(wave * 16 + col, wcols - 1);     // past N: the last one's scales
  // tiles tbeg .. tend - 1 are there, tbeg .. tnom - 1 are gone through
  const int part = blockIdx.z * a.per, last = min((K + KT - 1) / KT, part + a.per), share = (a.per + KG - 1) / KG;
  const int tbeg = part + GI * share, tend = min(last, tbeg + share), tnom = KG == 1 ? tend : tbeg + share;
  const auto wr = make_rsrc(a.qw + (cols ? n0 : 0) * (K / 2), (uint32_t)cols * (uint32_t)(K / 2));
  const auto xr = make_rsrc(static_cast<const char*>(a.x) + m0 * a.ldx * esz, (uint32_t)(((rows - 1) * a.ldx + K) * esz));
  const uint8_t* const zeros = a.zeros ? a.zeros : static_cast<const uint8_t*>(a.scales);    // read in any case, 8 put in later
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // load j: the rows of the tile's KB j, a row's chunk c at place c ^ (row & 15); what lies past K is zeros
  uint32_t xoff[NL];
  int xk[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int at = (wave * NL + i) * 64 + lane, row = at / RCH, k = (at % RCH ^ (row & 15)) * (int)(16 / esz);
    xk[i] = row < rows ? k : K;
    xoff[i] = (uint32_t)((row * a.ldx + k) * esz);
  }
  // k / G (uniform): k < 2^22 and G >= 32, so the product with the reciprocal is off by less than 2^-1 / G of a
  // quotient's step
  const float rg = 1.0f / (float)G;
  auto group_of = [&](int k) { return (int)(((float)min(k, K - 1) + 0.5f) * rg); };
  uint4 ring[D][U];
  // a tile past the part's end loads nothing (the bounds check), so that the loads under way are always as many
  auto fetch = [&](int tile, int slot) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int off = (int)(tile < tend && xk[i] + tile * KT < K ? xoff[i] + (uint32_t)tile * RB : OOB);
      const int at = (wave * NL + i) * 1024;
      if (slot == 0) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void)(lds0 + at), 16, off, 0, 0, 0);
      if (slot == 1) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void)(lds1 + at), 16, off, 0, 0, 0);
      if (slot == 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void)(lds2 + at), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = tile < tend && tile * KT + u * 128 + quarter * 32 < K;
      ring[slot][u] = buf_load_u4<true>(wr, in ? (uint32_t)(col * (K / 2) + tile * (KT / 2) + u * 64 + quarter * 16) : OOB);
    }
  };
  for (int win = tbeg; win < tnom; win += WIN / KT) {
    const int wend = min(tnom, win + WIN / KT), g0 = min(win * KT, K - 1) / G, gn = (min(K, wend * KT) - 1) / G + 1 - g0;
    if (win > tbeg) __syncthreads();
#pragma unroll
    for (int i = 0; i < D - 1; ++i) fetch(win + i, i);
    const int elems = wcols * gn;
    for (int i0 = tid; i0 < elems; i0 += 8 * W * 64) {     // eight loads of each at a time
      uint32_t sv[8], zv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = min(i0 + j * (W * 64), elems - 1);
        const int64_t at = (w0 + i / gn) * groups + g0 + i % gn;
        sv[j] = scale_bits<S4>(a.scales, at);
        zv[j] = zeros[at];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = min(i0 + j * (W * 64), elems - 1);           // past the end: the last one again
        sl[i % gn * COLS + i / gn] = scale_value<S4>(sv[j], a.sdt);
        zl[i % gn * COLS + i / gn] = a.zeros ? (uint8_t)zv[j] : 8;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the barrier of the first tile does the rest
    auto step = [&](auto slot, int tile, auto steady) {
      constexpr int d = decltype(slot)::value;
      if constexpr (decltype(steady)::value) {
        // this tile's loads are done, D - 2 tiles' later ones need not be
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((D - 2) * LP) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_s_barrier();                // the tile is whole; every wave is done with the one before
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (decltype(steady)::value) fetch(tile + D - 1, (d + D - 1) % D);
      __builtin_amdgcn_sched_barrier(0);
      if (KG > 1 && tile >= tend) return;          // uniform
      const int8_t* const cur = d == 0 ? lds0 : d == 1 ? lds1 : lds2;
      // x's fragments of a chunk are read one chunk ahead of their use, all at once
      constexpr int XR = DT == XDNA_F32 ? 2 : 1;
      uint4 xf[2][4][MT][XR];
      auto read_x = [&](int u) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < XR; ++r)
              xf[u & 1][j][t][r] = *reinterpret_cast<const uint4*>(
                  cur + (16 * t + col) * RB + (((16 * XR * u + XR * (4 * j + quarter) + r) ^ col) << 4));
      };
      read_x(0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t w[4];
        words(ring[d][u], w);
        transpose_quarters(w);
        if (u + 1 < U) read_x(u + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < GC; ++f) {
          const int i = (group_of(tile * KT + u * 128 + f * FL * 32) - g0) * COLS + scol;
          const float s = sl[i], z = (float)zl[i];
          f32x4 part[MT], sum[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) part[t] = sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = f * FL; j < (f + 1) * FL; ++j) {
            const i32x4 wf = unpack<DT>(w[j], z);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              i32x4 xp[XP];
              if constexpr (DT == XDNA_F32) {
                const uint4 p = xf[u & 1][j][t][0], q = xf[u & 1][j][t][XR - 1];
                const uint32_t v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
                split3(v, xp);
              } else {
                xp[0] = __builtin_bit_cast(i32x4, xf[u & 1][j][t][0]);
              }
#pragma unroll
              for (int p = XP - 1; p >= 0; --p) part[t] = mfma16<DT>(xp[p], wf, part[t]);
              if constexpr (DT == XDNA_BF16)
                sum[t] = mfma16<DT>(xp[0], i32x4{0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80}, sum[t]);
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
    };
    constexpr std::integral_constant<int, 0> s0;
    constexpr std::integral_constant<int, 1> s1;
    constexpr std::integral_constant<int, 2> s2;
    int t0 = win;
    for (; t0 + D <= wend; t0 += D) {              // no way out in between: the compiler would take loads for pending
      step(s0, t0, std::true_type{});
      step(s1, t0 + 1, std::true_type{});
      step(s2, t0 + 2, std::true_type{});
    }
    if (t0 < wend) step(s0, t0, std::false_type{});
    if (t0 + 1 < wend) step(s1, t0 + 1, std::false_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // what is still under way goes to LDS that the next window reuses
  }
  // element r of a lane's tile t: row 16 t + 4 quarter + r, column col
  bool odd = false;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd |= col < cols && 16 * t + 4 * quarter + r < rows && !(fabsf(acc[t][r]) < INFINITY);
  // x or a scale is not finite, or a sum before its scale passes float32: again, one by one, the scale first
  if (DT != XDNA_F16 && __builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
    for (int e = 0; e < MT * 4; ++e) {
      const int row = 16 * (e >> 2) + 4 * quarter + (e & 3);
      bool again = false;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) again |= t == (e >> 2) && r == (e & 3) && !(fabsf(acc[t][r]) < INFINITY);
      if (!again || row >= rows || col >= cols) continue;
      float v = 0.0f;
      for (int k = tbeg * KT; k < min(K, tend * KT); ++k) {
        const int64_t sg = (n0 + col) * groups + k / G;
        const uint8_t b = a.qw[(n0 + col) * (K / 2) + (k >> 1)];
        const float q = (float)((k & 1) ? b >> 4 : b & 15) - (a.zeros ? (float)a.zeros[sg] : 8.0f);
        v = __builtin_fmaf(q * load_any(a.scales, sg, a.sdt), load_as_f32<DT>(a.x, (m0 + row) * a.ldx + k), v);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t == (e >> 2) && r == (e & 3)) acc[t][r] = v;
    }
  }
}

template <int DT, bool S4, int MT, int FL, int KG>
__global__ __launch_bounds__(256 * KG, 2) void w4_tile_kernel(W4Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 acc[MT];
  if (KG == 1 || wave < 4) w4_tiles<DT, S4, MT, FL, KG, 0>(a, acc);
  if constexpr (KG == 2) {
    __shared__ f32x4 red[MT][4][64];
    if (wave >= 4) {
      w4_tiles<DT, S4, MT, FL, KG, 1>(a, acc);
#pragma unroll
      for (int t = 0; t < MT; ++t) red[t][wave - 4][lane] = acc[t];
    }
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const f32x4 x = red[t][wave][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[t][r] += x[r];
    }
  }
  const int col = lane & 15, quarter = lane >> 4;
  const int64_t N = a.N, n = (int64_t)blockIdx.x * 64 + wave * 16 + col, m0 = (int64_t)blockIdx.y * (16 * MT);
  if (n >= N) return;
  const float bias = a.bias && !a.part ? load_any(a.bias, n, a.bias_dt) : 0.0f;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = m0 + 16 * t + 4 * quarter + r;
      if (row >= a.M) continue;
      if (a.part) a.part[blockIdx.z * a.M * N + row * N + n] = acc[t][r];
      else store_from_f32<DT>(a.y, row * N + n, a.bias ? acc[t][r] + bias : acc[t][r]);
    }
}

// The parts of K added up in their order, the bias, and the one rounding.
template <int DT>
__global__ __launch_bounds__(256) void w4_join_kernel(const float* __restrict__ part, int parts, int64_t MN, int64_t N,
                                                      const void* __restrict__ bias, int bias_dt, void* __restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= MN) return;
  float v = 0.0f;
  for (int p0 = 0; p0 < parts; p0 += 8) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = part[min(p0 + j, parts - 1) * MN + i];      // all on their way at once
#pragma unroll
    for (int j = 0; j < 8; ++j) v += p0 + j < parts ? x[j] : 0.0f;
  }
  if (bias) v += load_any(bias, i % N, bias_dt);
  store_from_f32<DT>(y, i, v);
}

struct W4Plan {
  bool row;             // w4_row_kernel
  int kl, per;          // its lanes and waves along K
  int mt, kg, parts;    // w4_tile_kernel's row blocks of 16, groups of waves and split of K
};

// One row: the row kernel, but for 16-bit rows and 32 columns a CU (8192) or more (bfloat16, row / tiles: 1 x 4096 -> 14336
// 12.5 / 12.6 us; 1 x 512 -> 14336 5.4 / 5.7; 1 x 14336 -> 4096 12.4 / 14.1; float32 1 x 4096 -> 14336 13.3 / 38.6). Two to four
// rows: where the weights are few (3 x 1504 -> 1001 in float32 8.7 / 9.2 us, 4 x 8192 -> 512 in bfloat16 9.4 / 8.2,
// 4 x 4096 -> 4096 12.4 / 9.3). Its lanes along K: 64, so that long K makes waves enough, or 16 where the columns do (4096 ->
// 14336 in bfloat16: 12.5 with 16, 15.9 with 64; 14336 -> 4096: 19.9 / 12.4), and more waves along K below four a CU (14336 ->
// 64: one wave 8.3 us, four 5.5).
//
// Tiles of 16-bit rows: two groups of waves share out K from 512 k on, unless there are two workgroups a CU without
// (1 x 4096 -> 14336: one group 15.6 us, two 12.6, four no better; 64 x 4096 -> 14336 31.6 / 26.4), and K goes in parts on
// top until there is a workgroup a CU, none under 512 k, 16 at most (40 x 14336 -> 4096 with two groups: 3 / 4 / 8 parts
// 29.1 / 23.3 / 26.7 us, of which 4.0 the joining; 2 x 14336 -> 1000: 8 / 16 parts 11.0 / 9.6; 5 x 992 -> 2000: 7.5
// with one). float32, whose tiles take three times the work: parts alone, up to two workgroups a CU and 16 parts, none
// under 128 k (14 x 1536 -> 138: 1 / 4 / 8 / 12 parts 22.3 / 10.3 / 8.7 / 8.0 us; 8 x 4096 -> 4096 16.7 with
// 4, 15.5 with 8).
W4Plan w4_plan(int64_t M, int64_t N, int64_t K, bool f32) {
  W4Plan p{};
  const int64_t cus = device_cus();
  p.parts = 1;
  p.row = M == 1 ? f32 || N < 32 * cus : M <= 4 && N * K <= (4ll << 20);
  if (p.row) {
    p.kl = K <= 1024 || N >= 32 * cus ? 16 : 64;
    p.per = 1;
    const int64_t blocks = cdiv(K, 32 * p.kl);
    const int64_t most = std::min<int64_t>(8, W4_ROW_LDS / (p.kl * 32 * (f32 ? 4 : 2) * (M == 1 ? 1 : 4)));
    while (2 * p.per <= std::min(most, blocks) && cdiv(N, 64 / p.kl) * p.per < 4 * cus) p.per *= 2;
  } else {
    p.mt = (int)std::min<int64_t>(f32 ? 2 : 4, cdiv(M, 16));
    const int64_t wgs = cdiv(N, 64) * cdiv(M, 16 * p.mt);
    p.kg = !f32 && K >= 512 && wgs < 2 * cus ? 2 : 1;
    p.parts = (int)std::max<int64_t>(
        1, p.kg == 2 ? std::min<int64_t>({cus / wgs, K / 512, 16}) : std::min<int64_t>({2 * cus / wgs, K / 128, 16}));
  }
  return p;
}

template <int DT, bool S4, int MT, int FL, int KG>
int w4_tile_go(W4Args a, int parts, hipStream_t st) {
  // rows of a launch: the grid's y
  const int64_t rows = a.part ? a.M : std::min<int64_t>(65535, cdiv(a.M, 16 * MT)) * (16 * MT), M = a.M;
  const int esz = DT == XDNA_F32 ? 4 : 2;
  a.per = (int)cdiv(cdiv(a.K, DT == XDNA_F32 || MT > 2 ? 128 : 256), parts);
  for (int64_t m = 0; m < M; m += rows) {
    W4Args b = a;
    b.M = std::min(rows, M - m);
    b.x = static_cast<const char*>(a.x) + m * a.ldx * esz;
    b.y = static_cast<char*>(a.y) + m * a.N * esz;
    w4_tile_kernel<DT, S4, MT, FL, KG>
        <<<dim3((unsigned)cdiv(a.N, 64), (unsigned)cdiv(b.M, 16 * MT), (unsigned)parts), 256 * KG, 0, st>>>(b);
  }
  if (a.part)
    w4_join_kernel<DT><<<(unsigned)cdiv(M * a.N, 256), 256, 0, st>>>(a.part, parts, M * a.N, a.N, a.bias, a.bias_dt, a.y);
  return launch_status("linear_w4");
}

template <int DT, bool S4, int MT, int KG>
int w4_group(const W4Args& a, const W4Plan& p, hipStream_t st) {
  if (a.G % 128 == 0) return w4_tile_go<DT, S4, MT, 4, KG>(a, p.parts, st);
  if (a.G % 64 == 0) return w4_tile_go<DT, S4, MT, 2, KG>(a, p.parts, st);
  return w4_tile_go<DT, S4, MT, 1, KG>(a, p.parts, st);
}

template <int DT, bool S4, int MT>
int w4_tiles_go(const W4Args& a, const W4Plan& p, hipStream_t st) {
  if constexpr (DT != XDNA_F32) {
    if (p.kg == 2) return w4_group<DT, S4, MT, 2>(a, p, st);
  }
  return w4_group<DT, S4, MT, 1>(a, p, st);
}

template <int DT, bool S4, int KL>
int w4_row_go(W4Args a, const W4Plan& p, hipStream_t st) {
  a.per = p.per;
  const unsigned grid = (unsigned)cdiv(a.N, (64 / KL) * (8 / p.per));
  if (a.M == 1) w4_row_kernel<DT, S4, KL, 1><<<grid, 512, 0, st>>>(a);
  else w4_row_kernel<DT, S4, KL, 4><<<grid, 512, 0, st>>>(a);
  return launch_status("linear_w4");
}

template <int DT, bool S4>
int w4_go(const W4Args& a, const W4Plan& p, hipStream_t st) {
  if (p.row) return p.kl == 16 ? w4_row_go<DT, S4, 16>(a, p, st) : w4_row_go<DT, S4, 64>(a, p, st);
  if (p.mt == 1) return w4_tiles_go<DT, S4, 1>(a, p, st);
  if (DT == XDNA_F32 || p.mt == 2) return w4_tiles_go<DT, S4, 2>(a, p, st);
  if constexpr (DT != XDNA_F32) return p.mt == 3 ? w4_tiles_go<DT, S4, 3>(a, p, st) : w4_tiles_go<DT, S4, 4>(a, p, st);
  return XDNA_EUNSUPPORTED;
}

bool is_float(int dt) { return dt == XDNA_F32 || dt == XDNA_BF16 || dt == XDNA_F16; }

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int64_t xdna_linear_w4_ws_bytes(int x_dtype, int64_t M, int64_t N, int64_t K) {
  XDNA_REQUIRE(is_float(x_dtype), "x_dtype must be F32/BF16/F16");
  XDNA_REQUIRE(M >= 0 && N >= 0 && K >= 0 && K <= (1ll << 22) && N <= (1ll << 26), "bad sizes");
  if (M == 0 || N == 0 || K == 0) return 0;
  const W4Plan p = w4_plan(M, N, K, x_dtype == XDNA_F32);
  return p.parts > 1 ? p.parts * M * N * 4 : 0;
}

int xdna_linear_w4_ws(const void* x, int x_dtype, int64_t ldx, const void* qweight, const void* scales, int s_dtype,
                      const void* zeros, const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                      int64_t group, void* ws, int64_t ws_bytes, void* stream) {
  XDNA_REQUIRE(is_float(x_dtype) && is_float(s_dtype), "x_dtype and s_dtype must be F32/BF16/F16");
  XDNA_REQUIRE(!bias || is_float(bias_dtype), "bias_dtype must be F32/BF16/F16");
  XDNA_REQUIRE(M >= 0 && N >= 0 && K >= 0 && group >= 32 && group % 32 == 0 && K % group == 0,
               "group must be a multiple of 32 and K one of the group");
  if (M == 0 || N == 0) return XDNA_OK;
  const int64_t esz = x_dtype == XDNA_F32 ? 4 : 2;
  // 31-bit offsets within 64 rows of x and 64 columns of the weights, and the launch's threads along x
  XDNA_REQUIRE(K >= 1 && K <= (1ll << 22) && ldx >= K && ldx <= (1ll << 22) && N <= (1ll << 26), "sizes too large, or ldx < K");
  XDNA_REQUIRE(x && qweight && scales && y, "null pointer");
  XDNA_REQUIRE(aligned(x, 16) && ldx * esz % 16 == 0 && aligned(qweight, 16), "x rows and qweight must be 16-byte aligned");
  XDNA_REQUIRE(!ws || aligned(ws, 16), "ws must be 16-byte aligned");
  W4Plan p = w4_plan(M, N, K, x_dtype == XDNA_F32);
  const int64_t need = p.parts > 1 ? p.parts * M * N * 4 : 0;
  if (!ws || ws_bytes < need) p.parts = 1;
  const W4Args a{x, ldx, static_cast<const uint8_t*>(qweight), scales, s_dtype, static_cast<const uint8_t*>(zeros), bias,
                 bias_dtype, y, p.parts > 1 ? static_cast<float*>(ws) : nullptr, M, N, (int)K, (int)group, 0};
  const bool s4 = s_dtype == XDNA_F32;
  hipStream_t st = as_stream(stream);
  if (x_dtype == XDNA_F32) return s4 ? w4_go<XDNA_F32, true>(a, p, st) : w4_go<XDNA_F32, false>(a, p, st);
  if (x_dtype == XDNA_BF16) return s4 ? w4_go<XDNA_BF16, true>(a, p, st) : w4_go<XDNA_BF16, false>(a, p, st);
  return s4 ? w4_go<XDNA_F16, true>(a, p, st) : w4_go<XDNA_F16, false>(a, p, st);
}

int xdna_linear_w4(const void* x, int x_dtype, int64_t ldx, const void* qweight, const void* scales, int s_dtype,
                   const void* zeros, const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                   int64_t group, void* stream) {
  return xdna_linear_w4_ws(x, x_dtype, ldx, qweight, scales, s_dtype, zeros, bias, bias_dtype, y, M, N, K, group, nullptr, 0,
                           stream);
}

}  // extern "C"
