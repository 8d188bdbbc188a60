// A cache of keys and values in 8 bits, paged, for a language model that serves many texts, for gfx950 (MI355X), bfloat16 and
// float16:
//
//   cache_append      new tokens' keys (turned to their places) and values go into the cache; queries turn with them
//   attention_cache   the attention of each text's newest tokens over its cache
//
// A page has G tokens (16, 32, 64 or 128). It is int8 with a float32 scale for each head, scale = max|x| / 127 over its G x D
// values, x ~= q scale, and is written once, when its last token comes; the tokens of a text's open page lie in 16 bits in a
// ring of R >= G places (place = position % R). So no value is rounded twice, and what the cache holds does not depend on
// the calls that its tokens came in.
//
// K's pages are [G, D] and V's [D, G], as the two products of attention read them: both take 16 bytes along the dimension
// that lies dense and put nothing through LDS. MFMA 16x16x32 (srcA = X, srcB = Y): lane l supplies values 8 (l / 16) .. + 7 of
// the 32-deep step for row l % 16 of its operand and gets, in element r, row 4 (l / 16) + r of X and row l % 16 of Y. In
// what order a product's steps go through its depth is free, as long as both operands agree:
//   S = K Q^T over 64 keys, four tiles of 16: row 4 h' + r of tile t is key 16 h' + 4 t + r, so that lane l, h = l / 16, gets the
//     scores of keys 16 h .. 16 h + 15 for query row l % 16; lane h's 16 bytes of K are dims 16 (h + 4 j) .. + 15, two steps.
//   O^T = V^T P^T: those 16 scores are lane h's values of two 32-deep steps, and 16 bytes of a row of V are the same keys.
// int8 is exact in either 16-bit type. K's scale is applied to the float32 scores; V's, as a share of the largest met so far,
// goes into P before its rounding, and O is held in units of that largest one.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "xdna_common.h"
#include "xdna_hip.h"
#include "xdna_rotate.h"

namespace xdna {
namespace {

typedef __bf16 bf16x8c __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8c __attribute__((ext_vector_type(8)));

bool sixteen(int dtype) { return dtype == XDNA_BF16 || dtype == XDNA_F16; }
int log2_page(int64_t g) { return g == 16 ? 4 : g == 32 ? 5 : g == 64 ? 6 : g == 128 ? 7 : -1; }

// ------------------------------------------------------------------------------ cache_append
struct AppendArgs {
  const uint16_t *k, *v, *q;
  int64_t kt, kh, vt, vh, qt, qh;       // elements from token to token and from head to head
  int8_t *kp, *vp;
  float *ks, *vs;
  uint16_t *ktail, *vtail;
  const int32_t *table, *lens, *starts; // starts NULL: `each` tokens of every text
  int64_t ldt;
  int B, P, pages, nkv, nh, d, logg, R, each;
  int64_t T;
  const double* freqs;
  int half;
  float magnitude;
  uint16_t* qout;
  int items, qtokens;                   // pages that the new tokens can fall into, of all texts; tokens of a workgroup of q
};

// A text's part of the call: its tokens [s0, s1) go to the places len ..
struct Text {
  int64_t s0, s1;
  int len, end;             // end: len + new tokens, at most what the table has room for
};

__device__ __forceinline__ Text text_of(const AppendArgs& a, int b) {
  Text x;
  if (a.starts) {
    x.s0 = min<int64_t>(max(a.starts[b], 0), a.T);
    x.s1 = min<int64_t>(max<int64_t>(a.starts[b + 1], x.s0), a.T);
  } else {
    x.s0 = (int64_t)b * a.each;
    x.s1 = x.s0 + a.each;
  }
  const int room = a.P << a.logg;
  x.len = min(max(a.lens[b], 0), room);
  x.end = (int)min<int64_t>(x.len + (x.s1 - x.s0), room);
  return x;
}

// The work of page number i of all texts: text b's pages start at starts[b] / G + 2 b, which leaves room for as many as its
// tokens can touch, (n - 2) / G + 2. 64 texts at a time; starts that do not ascend give some text or other, in range.
__device__ __forceinline__ int text_of_item(const AppendArgs& a, int i, int& first) {
  int b = 0;
  for (int at = 0; at < a.B; at += 64) {
    const int t = at + (threadIdx.x & 63);
    const int f = t < a.B ? (int)(min<int64_t>(max(a.starts[t], 0), a.T) >> a.logg) + 2 * t : 0x7fffffff;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(f <= i));
    if (n) {
      b = at + n - 1;
      first = __builtin_amdgcn_readlane(f, n - 1);
    }
  }
  return b;
}

template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return DT == XDNA_F16 ? f32x2_to_f16x2_bits(lo, hi) : f32x2_to_bf16x2_bits(lo, hi);
}
template <int DT>
__device__ __forceinline__ float rounded(float x) {
  return DT == XDNA_F16 ? (float)(_Float16)x : bf16_bits_to_f32(f32_to_bf16_bits(x));
}

// The largest |x| of a workgroup's values (NaN if one is NaN).
__device__ __forceinline__ float group_amax(float v, float* part) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = __builtin_elementwise_maximum(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(part[0], part[1]), __builtin_elementwise_maximum(part[2], part[3]));
}

// round_half_even(x / s) as a byte; a block of zeros (s == 0) is zeros; a value that is not a number, or of a block that
// holds one or an infinity, is 0 (its scale is not finite, so the whole block reads as NaN).
__device__ __forceinline__ int quant_byte(float x, float s) {
  const float t = s > 0.0f ? rintf(x / s) : 0.0f;
  return t == t ? (int)fminf(fmaxf(t, -127.0f), 127.0f) : 0;
}

// A unit of a key: from the call (turned), or from the open page.
template <int DT, bool INTER>
__device__ __forceinline__ void key_unit(const AppendArgs& a, const Text& x, int b, int kvh, const Unit& u, int pos, float (&p)[8],
                                         float (&q)[8]) {
  if (pos < x.len) {
    const int64_t at = (((int64_t)b * a.nkv + kvh) * a.R + pos % a.R) * a.d;
    load_upto8<DT>(a.ktail, at + u.a, u.na, p);
    load_upto8<DT>(a.ktail, at + u.b, u.nb, q);
    return;
  }
  const int64_t from = (x.s0 + pos - x.len) * a.kt + kvh * a.kh;
  load_upto8<DT>(a.k, from + u.a, u.na, p);
  load_upto8<DT>(a.k, from + u.b, u.nb, q);
  if (u.pair < 0) return;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const Turn t = turn_of((double)pos, a.freqs[min(u.pair + e, a.half - 1)] * QUARTERS);
    c[e] = t.cos * a.magnitude;
    s[e] = t.sin * a.magnitude;
  }
  turn16<INTER>(p, q, c, s);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p[e] = rounded<DT>(p[e]);
    q[e] = rounded<DT>(q[e]);
  }
}

template <int DT>
__device__ __forceinline__ void key_to_tail(const AppendArgs& a, int b, int kvh, const Unit& u, int pos, const float (&p)[8],
                                            const float (&q)[8]) {
  const int64_t at = (((int64_t)b * a.nkv + kvh) * a.R + pos % a.R) * a.d;
  store_upto8<DT>(a.ktail, at + u.a, u.na, p);
  store_upto8<DT>(a.ktail, at + u.b, u.nb, q);
}

__device__ __forceinline__ void store_bytes(int8_t* to, int n, const float (&x)[8], float s) {
  int w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = quant_byte(x[e], s);
  if (n == 8) {
    typedef uint32_t u32x2_1 __attribute__((ext_vector_type(2), aligned(1)));
    u32x2_1 v;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v[h] = (w[4 * h] & 255) | (w[4 * h + 1] & 255) << 8 | (w[4 * h + 2] & 255) << 16 | (uint32_t)w[4 * h + 3] << 24;
    *reinterpret_cast<u32x2_1*>(to) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) to[e] = (int8_t)w[e];
  }
}

// A workgroup has a page of one head's keys (blockIdx.y 0) or values (1), or some tokens of all heads' queries (2, the first
// qblocks). Texts whose open page holds old tokens: only their first page's workgroup reads the ring, and writes what would
// fall on the old tokens' places after that. U: units of keys a thread has.
template <int DT, bool INTER, int U>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  __shared__ float part[4];
  const int g = 1 << a.logg;
  if (blockIdx.y == 2) {
    __shared__ float cs[256], sn[256];
    __shared__ int known[16];
    const int64_t t0 = (int64_t)blockIdx.x * a.qtokens;
    if (t0 >= a.T) return;
    const int n = (int)min<int64_t>(a.qtokens, a.T - t0);
    for (int i = threadIdx.x; i < n * max(1, a.half); i += 256) {
      const int tok = i / max(1, a.half), j = i - tok * max(1, a.half);
      const int64_t t = t0 + tok;
      int b;
      int64_t s0;
      bool mine = true;
      if (a.starts) {
        int lo = 0, hi = a.B;                     // starts[0 .. lo) <= t
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (a.starts[mid] <= t) lo = mid + 1;
          else hi = mid;
        }
        b = max(lo - 1, 0);
        s0 = a.starts[b];
        mine = lo > 0 && t < a.starts[a.B];
      } else {
        b = (int)(t / a.each);
        s0 = (int64_t)b * a.each;
      }
      if (j == 0) known[tok] = mine;
      if (a.half) {
        const Turn w = turn_of((double)(max(a.lens[b], 0) + t - s0), a.freqs[j] * QUARTERS);
        cs[i] = w.cos * a.magnitude;
        sn[i] = w.sin * a.magnitude;
      }
    }
    __syncthreads();
    const int per_head = units_of(a.d, a.half), per_token = per_head * a.nh;
    for (int i = threadIdx.x; i < n * per_token; i += 256) {
      const int tok = i / per_token, at = i - tok * per_token, head = at / per_head;
      const Unit u = unit_of<INTER>(at - head * per_head, a.d, a.half);
      const int64_t from = (t0 + tok) * a.qt + head * a.qh, to = ((t0 + tok) * a.nh + head) * a.d;
      float p[8], q[8];
      load_upto8<DT>(a.q, from + u.a, u.na, p);
      load_upto8<DT>(a.q, from + u.b, u.nb, q);
      if (u.pair >= 0) {
        float c[8], s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = tok * a.half + min(u.pair + e, a.half - 1);
          c[e] = cs[j];
          s[e] = sn[j];
        }
        turn16<INTER>(p, q, c, s);
      }
      if (!known[tok]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = q[e] = 0.0f;
      }
      store_upto8<DT>(a.qout, to + u.a, u.na, p);
      store_upto8<DT>(a.qout, to + u.b, u.nb, q);
    }
    return;
  }
  const int item = blockIdx.x / a.nkv, kvh = blockIdx.x - item * a.nkv;
  if (item >= a.items) return;
  int b, nth;
  if (a.starts) {
    int first = 0x7fffffff;
    b = __builtin_amdgcn_readfirstlane(text_of_item(a, item, first));
    nth = item - __builtin_amdgcn_readfirstlane(first);
  } else {
    const int each = ((a.each + g - 2) >> a.logg) + 1;
    b = item / each;
    nth = item - b * each;
  }
  const Text x = text_of(a, b);
  const int page0 = x.len >> a.logg, page = page0 + nth;
  if (nth < 0 || ((int64_t)page << a.logg) >= x.end) return;
  const int begin = page << a.logg, lo = max(x.len, begin), hi = min(x.end, begin + g);
  const bool whole = hi == begin + g && hi > lo;
  const int id = a.table[b * a.ldt + page];
  const bool good = id >= 0 && id < a.pages;      // no page for it: its tokens pass through the ring only
  // places of the ring that old tokens hold while the first page's workgroup reads them: written by it, afterwards
  const int later = (x.len & (g - 1)) ? (page0 << a.logg) + a.R : 0x7fffffff, oldest = x.end - a.R;
  const int64_t head = (int64_t)b * a.nkv + kvh, block = (int64_t)id * a.nkv + kvh;
  if (blockIdx.y == 0) {
    const int per_token = units_of(a.d, a.half), units = g * per_token;
    float p[U][8], q[U][8], top = 0.0f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = i * 256 + threadIdx.x, tok = at / per_token, pos = begin + tok;
      if (at >= units || pos >= hi || (pos < lo && !whole)) continue;
      const Unit u = unit_of<INTER>(at - tok * per_token, a.d, a.half);
      key_unit<DT, INTER>(a, x, b, kvh, u, pos, p[i], q[i]);
      if (pos >= lo && pos >= oldest && pos < later) key_to_tail<DT>(a, b, kvh, u, pos, p[i], q[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = __builtin_elementwise_maximum(top, fabsf(p[i][e]));
        top = __builtin_elementwise_maximum(top, fabsf(q[i][e]));
      }
    }
    if (whole) {
      const float amax = group_amax(top, part), s = __builtin_isfinite(amax) ? amax / 127.0f : __builtin_nanf("");
      if (good) {
        if (threadIdx.x == 0) a.ks[block] = s;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int at = i * 256 + threadIdx.x, tok = at / per_token;
          if (at >= units) continue;
          const Unit u = unit_of<INTER>(at - tok * per_token, a.d, a.half);
          int8_t* const to = a.kp + (block * g + tok) * a.d;
          store_bytes(to + u.a, u.na, p[i], s);
          store_bytes(to + u.b, u.nb, q[i], s);
        }
      }
    }
    if (nth == 0 && later < x.end) {
      __syncthreads();
      const int from = max(later, oldest), n = (x.end - from) * per_token;
      for (int at = threadIdx.x; at < n; at += 256) {
        const int tok = at / per_token;
        const Unit u = unit_of<INTER>(at - tok * per_token, a.d, a.half);
        float pp[8], qq[8];
        key_unit<DT, INTER>(a, x, b, kvh, u, from + tok, pp, qq);
        key_to_tail<DT>(a, b, kvh, u, from + tok, pp, qq);
      }
    }
    return;
  }
  // values: through LDS, [token][d + 2] so that a walk along the tokens of 16 dims meets every bank
  extern __shared__ uint16_t vl[];
  const int per_token = a.d / 8, units = g * per_token, ld = a.d + 2;
  auto value = [&](int pos, int u, float (&p)[8]) {
    if (pos >= x.len) return load8<DT>(a.v, (x.s0 + pos - x.len) * a.vt + kvh * a.vh + 8 * u, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = load_as_f32<DT>(a.vtail, (head * a.d + 8 * u + e) * a.R + pos % a.R);
  };
  auto to_tail = [&](int pos, int u, const float (&p)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_from_f32<DT>(a.vtail, (head * a.d + 8 * u + e) * a.R + pos % a.R, p[e]);
  };
  float top = 0.0f;
  for (int at = threadIdx.x; at < units; at += 256) {
    const int tok = at / per_token, u = at - tok * per_token, pos = begin + tok;
    if (pos >= hi || (pos < lo && !whole)) continue;
    float p[8];
    value(pos, u, p);
    if (pos >= lo && pos >= oldest && pos < later) to_tail(pos, u, p);
    if (whole) {
#pragma unroll
      for (int e = 0; e < 8; ++e) top = __builtin_elementwise_maximum(top, fabsf(p[e]));
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(vl + tok * ld + 8 * u + 2 * e) = pack16<DT>(p[2 * e], p[2 * e + 1]);
    }
  }
  if (whole) {
    const float amax = group_amax(top, part), s = __builtin_isfinite(amax) ? amax / 127.0f : __builtin_nanf("");
    if (good) {
      if (threadIdx.x == 0) a.vs[block] = s;
      const int chunks = g >> 4, tasks = a.d * chunks;
      for (int i = threadIdx.x; i < tasks; i += 256) {
        const int dim = i / chunks, c = i - dim * chunks;
        u32x4 w = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[e >> 2] |= (uint32_t)(quant_byte(load_as_f32<DT>(vl, (16 * c + e) * ld + dim), s) & 255) << (8 * (e & 3));
        *reinterpret_cast<u32x4*>(a.vp + (block * a.d + dim) * g + 16 * c) = w;
      }
    }
  }
  if (nth == 0 && later < x.end) {
    __syncthreads();
    const int from = max(later, oldest), n = (x.end - from) * per_token;
    for (int at = threadIdx.x; at < n; at += 256) {
      const int tok = at / per_token, u = at - tok * per_token;
      float p[8];
      value(from + tok, u, p);
      to_tail(from + tok, u, p);
    }
  }
}

template <int DT, bool INTER>
int append_go(const AppendArgs& a, hipStream_t st) {
  const int g = 1 << a.logg;
  const int64_t blocks = (int64_t)a.items * a.nkv, qblocks = a.q ? cdiv(a.T, a.qtokens) : 0;
  const dim3 grid((unsigned)std::max(blocks, qblocks), a.q ? 3 : 2);
  const int per = (int)cdiv((int64_t)g * units_of(a.d, a.half), 256);
  const unsigned lds = (unsigned)(g * (a.d + 2) * 2);
  if (per <= 1) append_kernel<DT, INTER, 1><<<grid, 256, lds, st>>>(a);
  else if (per <= 2) append_kernel<DT, INTER, 2><<<grid, 256, lds, st>>>(a);
  else if (per <= 3) append_kernel<DT, INTER, 3><<<grid, 256, lds, st>>>(a);
  else append_kernel<DT, INTER, 5><<<grid, 256, lds, st>>>(a);
  return launch_status("cache_append");
}

// ------------------------------------------------------------------------------ attention_cache
struct CacheArgs {
  const uint16_t* q;
  int64_t qb, qn, qh;                   // elements from text, token, head to the next
  const int8_t *kp, *vp;
  const float *ks, *vs;
  const uint16_t *ktail, *vtail;
  const int32_t *table, *lens;
  int64_t ldt;
  int B, N, nh, nkv, d, P, pages, logg, R;
  int parts, rblocks;                   // parts of a text's keys; blocks of rows of a (text, kv head)
  float c;                              // scale log2 e
  uint32_t sign;
  float *po, *pml;                      // [parts][B N nh][d] sums, [parts][B N nh][2] maxima and sums of p
  uint16_t* out;
};

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const i32x4& a, const i32x4& b, const f32x4& c) {
  if constexpr (DT == XDNA_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8c, a), __builtin_bit_cast(f16x8c, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8c, a), __builtin_bit_cast(bf16x8c, b), c, 0, 0, 0);
}

// Four int8 as two words of 16-bit floats, exactly. float16: q + 128 is the low bits of 1024 + .., and 1152 comes off again.
template <int DT>
__device__ __forceinline__ void widen(uint32_t w, int& lo, int& hi) {
  if constexpr (DT == XDNA_F16) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
    hi = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
  } else {
    lo = (int)f32x2_to_bf16x2_bits((float)(int8_t)w, (float)(int8_t)(w >> 8));
    hi = (int)f32x2_to_bf16x2_bits((float)(int8_t)(w >> 16), (float)((int32_t)w >> 24));
  }
}
template <int DT>
__device__ __forceinline__ i32x4 widen8(uint32_t a, uint32_t b) {
  i32x4 r;
  int x, y;
  widen<DT>(a, x, y);
  r[0] = x, r[1] = y;
  widen<DT>(b, x, y);
  r[2] = x, r[3] = y;
  return r;
}

// over the four lanes l % 16, + 16, + 32, + 48
__device__ __forceinline__ float quad_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// float16 p are held 2^14 times as large, so that those down to 2^-28 of the largest stay normal numbers
template <int DT>
constexpr float SHIFT = DT == XDNA_F16 ? 14.0f : 0.0f;
template <int DT>
constexpr uint32_t ALL_ONES = DT == XDNA_F16 ? 0x7c00u : 0x7f80u;

// A wave's rows: RB blocks of 16, their maxima, sums and outputs. Rows of a (text, kv head) are the pairs (new token, q head
// of the group), so that the heads that share K and V share their loads.
template <int DT, int D, int RB>
struct Rows {
  static constexpr int S = D / 32, ND = D / 16;
  i32x4 q[RB][S];
  f32x4 o[RB][ND];
  float m[RB], l[RB];
  int limit[RB];            // keys that the lane's row sees
  float unit;               // O is held in units of it

  // p of the 64 keys whose scores are here, K's scale and masks applied, as the second product's operand
  __device__ __forceinline__ void weigh(f32x4 (&sc)[4], int rb, float c, float share, bool masked, int first, int lim, i32x4 (&pf)[2]) {
    float mx = sc[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, sc[t][r]);
    mx = quad_max(mx);
    const bool grow = mx > m[rb];
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float mn = grow ? mx : m[rb];
      const float alpha = m[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[rb] - mn) * c);
      l[rb] *= alpha;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[rb][i] *= alpha;
      m[rb] = mn;
    }
    const float mc = (m[rb] == -INFINITY ? 0.0f : m[rb] * c) - SHIFT<DT>;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], c, -mc)), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r + 1], c, -mc));
        l[rb] += p0;
        l[rb] += p1;
        p0 *= share, p1 *= share;
        if (masked) {                     // a share that is not finite is not the row's unless it sees the key
          if (first + 4 * t + r >= lim) p0 = 0.0f;
          if (first + 4 * t + r + 1 >= lim) p1 = 0.0f;
        }
        pf[t >> 1][(t & 1) * 2 + r / 2] = (int)pack16<DT>(p0, p1);
      }
  }

  // units for a block of keys whose values have this scale; its share of the unit
  __device__ __forceinline__ float share_of(float vs, bool uniform) {
    float top = vs;
    if (!uniform) {
      // the largest number among the four groups of keys (fmaxf leaves out NaN)
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
    }
    if (__builtin_amdgcn_ballot_w64(top > unit)) {
      const float to = unit / top;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < ND; ++i) o[rb][i] *= to;
      unit = top;
    }
    return unit > 0.0f ? vs / unit : vs * 0.0f;
  }
};

// W waves share out the 64-key steps of a part of a text's keys for 16 RB rows and meet in LDS. Registers hold the step in
// work and nothing else: K of the wave's next step is on its way once its scores are done, V after its products.
template <int DT, int D, int RB, int W>
__global__ __launch_bounds__(W * 64, RB == 1 ? 3 : 2) void cache_kernel(CacheArgs a) {
  constexpr int S = D / 32, ND = D / 16, DC = D / 64;
  __shared__ __attribute__((aligned(16))) float ol[W][RB * ND][256];
  __shared__ float ml[2][W][RB][16];
  const int lane = threadIdx.x & 63, h = lane >> 4, i16 = lane & 15, hk = i16 >> 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = a.nh / a.nkv, nrows = a.N * grp, g = 1 << a.logg;
  int rest = blockIdx.x;
  const int rblock = rest % a.rblocks;
  rest /= a.rblocks;
  const int kvh = rest % a.nkv;
  rest /= a.nkv;
  const int b = rest % a.B, part = rest / a.B;
  const int len = min(max(a.lens[b], 0), a.P << a.logg);
  const int npages = len >> a.logg, nfull = npages << a.logg, ntail = len - nfull;
  const int steps = (nfull + 63) >> 6, all = steps + ((ntail + 63) >> 6);
  const int per = (all + a.parts - 1) / a.parts, from = min(part * per, all), to = min(from + per, all);
  const int row0 = rblock * 16 * RB, dchunks = a.d >> 4;

  Rows<DT, D, RB> w;
  w.unit = 0.0f;
  int64_t orow[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(row0 + 16 * rb + i16, nrows - 1), n = row / grp, head = kvh * grp + row - n * grp;
    orow[rb] = ((int64_t)b * a.N + n) * a.nh + head;
    w.limit[rb] = len - a.N + n + 1;
    w.m[rb] = -INFINITY;
    w.l[rb] = 0.0f;
    const uint16_t* const q = a.q + b * a.qb + n * a.qn + head * a.qh;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int at = 16 * (h + 4 * (s >> 1)) + 8 * (s & 1);
      w.q[rb][s] = i32x4{0, 0, 0, 0};
      if (at < a.d) w.q[rb][s] = *reinterpret_cast<const i32x4*>(q + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) w.q[rb][s][e] ^= (int)a.sign;
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) w.o[rb][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // the first row's tokens are the fewest that a row of this workgroup sees
  const int sure = min(nfull, __builtin_amdgcn_readfirstlane(w.limit[0]));

  // A lane's part of a step: the page of the keys that it loads K of (16 hk ..), and of those that it has scores and V of
  // (16 h ..). Pages past the last one, and what is no page, are read as a page that there is, and masked.
  const int32_t* const table = a.table + b * a.ldt;
  auto page_at = [&](int step, int quarter) {
    const int at = min((step * 64 + 16 * quarter) >> a.logg, npages - 1);
    return table[max(at, 0)];
  };
  const auto safe = [&](int id) { return id >= 0 && id < a.pages ? id : 0; };
  int idk = 0, idv = 0;
  i32x4 k[4 * DC], v[ND];
  float ksc = 0.0f, vsc = 0.0f;
  auto load_k = [&](int step) {
    const int in = (step * 64 + 16 * hk) & (g - 1);
    const int8_t* const base = a.kp + (((int64_t)safe(idk) * a.nkv + kvh) * g + in + (lane & 3)) * a.d;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < DC; ++j) k[t * DC + j] = *reinterpret_cast<const i32x4*>(base + 4 * t * a.d + 16 * min(h + 4 * j, dchunks - 1));
  };
  auto load_v = [&](int step, int id) {
    const int in = (step * 64 + 16 * h) & (g - 1);
    const int8_t* const base = a.vp + ((int64_t)safe(id) * a.nkv + kvh) * a.d * g + in;
#pragma unroll
    for (int i = 0; i < ND; ++i) v[i] = *reinterpret_cast<const i32x4*>(base + (int64_t)(16 * min(i, dchunks - 1) + i16) * g);
  };
  auto load_scales = [&](int id) {
    const int64_t at = (int64_t)safe(id) * a.nkv + kvh;
    ksc = a.ks[at];
    vsc = a.vs[at];
  };
  int step = from + wave;
  const int end = min(to, steps);
  if (step < end) {
    idk = page_at(step, hk), idv = page_at(step, h);
    load_k(step);
    load_v(step, idv);
    load_scales(idv);
  }
#pragma unroll 1
  for (; step < end; step += W) {
    const int first = step * 64 + 16 * h, next = step + W;
    const bool good = idv >= 0 && idv < a.pages;
    const bool masked = step * 64 + 64 > sure || __builtin_amdgcn_ballot_w64(!good) != 0;
    f32x4 sc[RB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sc[rb][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const i32x4 x = k[t * DC + (s >> 1)];
        const i32x4 f = widen8<DT>(x[2 * (s & 1)], x[2 * (s & 1) + 1]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[rb][t] = mfma16<DT>(f, w.q[rb][s], sc[rb][t]);
      }
    }
    const float ks = ksc, vs = good && first < nfull ? vsc : 0.0f;
    if (next < end) {
      idk = page_at(next, hk), idv = page_at(next, h);
      load_k(next);
      load_scales(idv);
    }
    const float share = w.share_of(vs, g >= 64);
    i32x4 pf[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int lim = good ? min(nfull, w.limit[rb]) : 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) sc[rb][t] *= ks;
      if (masked) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (first + 4 * t + r >= lim) sc[rb][t][r] = -INFINITY;
      }
      w.weigh(sc[rb], rb, a.c, share, masked, first, lim, pf[rb]);
    }
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const i32x4 f = widen8<DT>(v[i][2 * u], v[i][2 * u + 1]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) w.o[rb][i] = mfma16<DT>(f, pf[rb][u], w.o[rb][i]);
      }
    if (next < end) load_v(next, idv);
  }
  // the open page, in 16 bits
#pragma unroll 1
  for (; step < to; step += W) {
    const int at = (step - steps) * 64, left = ntail - at;          // keys of this step: nfull + at ..
    const int slot = nfull % a.R + at;
    const int64_t head = (int64_t)b * a.nkv + kvh;
    const uint16_t* const kt = a.ktail + (head * a.R + slot) * a.d;
    // a group of 16 places without keys is read as the first one, and masked
    const uint16_t* const vt = a.vtail + head * a.d * a.R + slot + (16 * h < left ? 16 * h : 0);
    f32x4 sc[RB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint16_t* const row = kt + (int64_t)min(16 * hk + 4 * t + (lane & 3), left - 1) * a.d;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sc[rb][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const i32x4 f = *reinterpret_cast<const i32x4*>(row + 16 * min(h + 4 * (s >> 1), dchunks - 1) + 8 * (s & 1));
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[rb][t] = mfma16<DT>(f, w.q[rb][s], sc[rb][t]);
      }
    }
    const int first = nfull + at + 16 * h;
    const float share = w.share_of(1.0f, true);
    i32x4 pf[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int lim = w.limit[rb];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (first + 4 * t + r >= lim) sc[rb][t][r] = -INFINITY;
      w.weigh(sc[rb], rb, a.c, share, true, first, lim, pf[rb]);
    }
#pragma unroll 1
    for (int i = 0; i < ND; ++i) {
      if (i >= dchunks) break;
      i32x4 f[2];
      bool odd = false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f[u] = *reinterpret_cast<const i32x4*>(vt + (int64_t)(16 * i + i16) * a.R + 8 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 16 * h + 8 * u + 2 * e;
          uint32_t x = (uint32_t)f[u][e];
          if (key >= left) x = 0;
          else if (key + 1 >= left) x &= 0xffffu;
          // what is not finite may belong to a key that some rows do not see, and 0 times it would be NaN: taken out, and
          // added below to the rows that see it
          if ((x & ALL_ONES<DT>) == ALL_ONES<DT>) x &= 0xffff0000u, odd = true;
          if ((x >> 16 & ALL_ONES<DT>) == ALL_ONES<DT>) x &= 0xffffu, odd = true;
          f[u][e] = (int)x;
        }
      }
      const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        f32x4 o = w.o[rb][0];
#pragma unroll
        for (int n = 1; n < ND; ++n)
          if (n == i) o = w.o[rb][n];
#pragma unroll
        for (int u = 0; u < 2; ++u) o = mfma16<DT>(f[u], pf[rb][u], o);
        if (any) {
#pragma unroll 1
          for (int key = 0; key < min(left, 64); ++key) {
            // lane 16 (key / 16) + i16 holds the row's p of it, in half key % 2 of word (key % 16) / 2
            uint32_t x = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e == (key & 15) >> 1) x = (uint32_t)pf[rb][e >> 2][e & 3];
            x = __shfl(x, 16 * (key >> 4) + i16, 64) >> (16 * (key & 1)) & 0xffffu;
            const float p = DT == XDNA_F16 ? f16_bits_to_f32((uint16_t)x) : bf16_bits_to_f32((uint16_t)x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint16_t y = a.vtail[(head * a.d + 16 * i + 4 * h + r) * a.R + slot + key];
              if ((y & ALL_ONES<DT>) == ALL_ONES<DT> && nfull + at + key < w.limit[rb])
                o[r] += p * (DT == XDNA_F16 ? f16_bits_to_f32(y) : bf16_bits_to_f32(y));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < ND; ++n)
          if (n == i) w.o[rb][n] = o;
      }
    }
  }

  // the waves' rows joined
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    w.l[rb] = quad_sum(w.l[rb]);
    if (h == 0) ml[0][wave][rb][i16] = w.m[rb], ml[1][wave][rb][i16] = w.l[rb];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      f32x4 o = w.o[rb][i];
      o *= w.unit;
      *reinterpret_cast<f32x4*>(&ol[wave][rb * ND + i][lane * 4]) = o;
    }
  }
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float mt = -INFINITY, lt = 0.0f, weight[W];
#pragma unroll
    for (int x = 0; x < W; ++x) mt = fmaxf(mt, ml[0][x][rb][i16]);
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float mg = ml[0][x][rb][i16], lg = ml[1][x][rb][i16];
      weight[x] = mg == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mg - mt) * a.c);
      lt += mg == -INFINITY ? lg : lg * weight[x];            // lg is 0 then, or NaN
    }
    const bool mine = row0 + 16 * rb + i16 < nrows;
#pragma unroll
    for (int n = 0; n < (ND + W - 1) / W; ++n) {
      const int i = wave + n * W;
      if (i >= dchunks) break;
      f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const f32x4 part_o = *reinterpret_cast<const f32x4*>(&ol[x][rb * ND + i][lane * 4]);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] += part_o[r] * weight[x];
      }
      if (!mine) continue;
      const int dim = 16 * i + 4 * h;
      if (a.parts == 1) {
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        *reinterpret_cast<uint2*>(a.out + orow[rb] * a.d + dim) = make_uint2(pack16<DT>(o[0] * inv, o[1] * inv), pack16<DT>(o[2] * inv, o[3] * inv));
      } else {
        const int64_t at = (int64_t)part * a.B * a.N * a.nh + orow[rb];
        *reinterpret_cast<f32x4*>(a.po + at * a.d + dim) = o;
        if (dim == 0) *reinterpret_cast<float2*>(a.pml + at * 2) = make_float2(mt, lt);
      }
    }
  }
}

// The parts of a row joined: a workgroup per row, wave w the parts w, w + 4, .., then the waves in their order; lane l dims
// 2 l, 2 l + 1.
template <int DT>
__global__ __launch_bounds__(256) void cache_join_kernel(const float* __restrict__ po, const float* __restrict__ pml, int parts,
                                                         int64_t rows, int d, float c, uint16_t* __restrict__ out) {
  __shared__ float2 ov[4][64];
  __shared__ float lv[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  float mt = -INFINITY;
  for (int i = lane; i < parts; i += 64) mt = fmaxf(mt, pml[(i * rows + row) * 2]);
  mt = wave_max(mt);
  float l = 0.0f, x = 0.0f, y = 0.0f;
  const int at = min(2 * lane, d - 2);
#pragma unroll 8
  for (int i = wave; i < parts; i += 4) {
    const float2 p = *reinterpret_cast<const float2*>(pml + (i * rows + row) * 2);
    const float2 v = *reinterpret_cast<const float2*>(po + (i * rows + row) * d + at);
    const float w = p.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((p.x - mt) * c);
    l += p.x == -INFINITY ? p.y : p.y * w;
    x += v.x * w;
    y += v.y * w;
  }
  ov[wave][lane] = make_float2(x, y);
  if (lane == 0) lv[wave] = l;
  __syncthreads();
  if (wave || 2 * lane >= d) return;
  l = lv[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    l += lv[w];
    x += ov[w][lane].x;
    y += ov[w][lane].y;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint32_t*>(out + row * d + 2 * lane) = pack16<DT>(x * inv, y * inv);
}

// A workgroup has 16 rows, or 32 where there are more. The keys of a text go to as many parts as make two workgroups a CU, none
// under 256 keys if the texts are as long as the table has room for: a part is its share of the keys that there are.
void cache_plan(CacheArgs& a) {
  const int64_t rows = (int64_t)a.N * (a.nh / a.nkv), cus = device_cus();
  a.rblocks = (int)cdiv(rows, rows <= 16 ? 16 : 32);
  const int64_t wgs = (int64_t)a.B * a.nkv * a.rblocks, room = (int64_t)a.P << a.logg;
  a.parts = (int)std::max<int64_t>(1, std::min(2 * cus / wgs, cdiv(room, 256)));
}

template <int DT, int D>
int cache_go(const CacheArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.N * (a.nh / a.nkv), grid = (int64_t)a.B * a.nkv * a.rblocks * a.parts;
  if (rows <= 16) cache_kernel<DT, D, 1, 4><<<(unsigned)grid, 256, 0, st>>>(a);
  else cache_kernel<DT, D, 2, 4><<<(unsigned)grid, 256, 0, st>>>(a);
  if (a.parts > 1) {
    const int64_t all = (int64_t)a.B * a.N * a.nh;
    cache_join_kernel<DT><<<(unsigned)all, 256, 0, st>>>(a.po, a.pml, a.parts, all, a.d, a.c, a.out);
  }
  return launch_status("attention_cache");
}

bool cache_sizes_ok(int64_t B, int64_t N, int64_t nh, int64_t nkv, int64_t d, int64_t P, int64_t pages, int64_t g, int64_t R) {
  return B >= 0 && N >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && nh < (1 << 16) && B < (1 << 22) && N < (1 << 22) &&
         B * N * nh < (1ll << 22) && d >= 16 && d <= 128 && d % 16 == 0 && log2_page(g) >= 0 && P >= 0 && P * g < (1ll << 30) &&
         pages >= 0 && pages < (1ll << 31) && R >= g && R % g == 0 && R < (1 << 16);
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_cache_append(const void* k, const void* v, int dtype, const int64_t* strides, void* kpages, void* vpages, float* kscales,
                      float* vscales, void* ktail, void* vtail, const int32_t* table, int64_t ldt, const int32_t* lens,
                      const int32_t* starts, const void* q, const double* freqs, int64_t half, float magnitude, int interleaved,
                      void* q_out, int64_t T, int64_t B, int64_t P, int64_t pages, int64_t page, int64_t R, int nh, int nkv, int d,
                      void* stream) {
  XDNA_REQUIRE(sixteen(dtype), "dtype must be BF16/F16");
  XDNA_REQUIRE(cache_sizes_ok(B, 1, nkv, nkv, d, P, pages, page, R) && T >= 0 && T < (1ll << 30), "bad sizes");
  XDNA_REQUIRE(!q || (nh >= 1 && (int64_t)nh * d < (1ll << 20)), "bad number of q heads");
  XDNA_REQUIRE(half >= 0 && 2 * half <= d, "no more dims turn than there are");
  if (T == 0 || (B == 0 && !q)) return XDNA_OK;
  XDNA_REQUIRE(B > 0, "tokens of no text");
  XDNA_REQUIRE(k && v && strides && ktail && vtail && lens && (freqs || half == 0) && (!q || q_out), "null pointer");
  XDNA_REQUIRE(P == 0 || (table && ldt >= 0), "no table");
  XDNA_REQUIRE(pages == 0 || (kpages && vpages && kscales && vscales), "null pointer");
  XDNA_REQUIRE(starts || T % B == 0, "without starts every text has as many tokens");
  XDNA_REQUIRE(aligned(kpages, 16) && aligned(vpages, 16) && aligned(ktail, 16) && aligned(vtail, 16), "the cache must be 16-byte aligned");
  for (int i = 0; i < (q ? 6 : 4); ++i) XDNA_REQUIRE(strides[i] >= 0, "strides must not be negative");
  AppendArgs a{};
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v), a.q = static_cast<const uint16_t*>(q);
  a.kt = strides[0], a.kh = strides[1], a.vt = strides[2], a.vh = strides[3];
  if (q) a.qt = strides[4], a.qh = strides[5];
  a.kp = static_cast<int8_t*>(kpages), a.vp = static_cast<int8_t*>(vpages), a.ks = kscales, a.vs = vscales;
  a.ktail = static_cast<uint16_t*>(ktail), a.vtail = static_cast<uint16_t*>(vtail);
  a.table = table, a.lens = lens, a.starts = starts, a.ldt = ldt;
  a.B = (int)B, a.P = (int)P, a.pages = (int)pages, a.nkv = nkv, a.nh = nh, a.d = d, a.logg = log2_page(page), a.R = (int)R;
  a.T = T, a.freqs = freqs, a.half = (int)half, a.magnitude = magnitude, a.qout = static_cast<uint16_t*>(q_out);
  a.each = starts ? 0 : (int)(T / B);
  const int64_t items = starts ? T / page + 2 * B : B * ((a.each + page - 2) / page + 1);
  a.qtokens = (int)std::min<int64_t>(half ? std::min<int64_t>(16, std::max<int64_t>(1, 256 / half)) : 16, std::max<int64_t>(1, T / (2 * device_cus())));
  XDNA_REQUIRE(items * nkv <= MAX_LAUNCH_THREADS / 256 && T <= MAX_LAUNCH_THREADS / 256, "too many tokens");
  a.items = (int)items;
  hipStream_t st = as_stream(stream);
  if (dtype == XDNA_BF16) return interleaved ? append_go<XDNA_BF16, true>(a, st) : append_go<XDNA_BF16, false>(a, st);
  return interleaved ? append_go<XDNA_F16, true>(a, st) : append_go<XDNA_F16, false>(a, st);
}

int64_t xdna_attention_cache_ws_bytes(int64_t B, int64_t N, int nh, int nkv, int d, int64_t P, int64_t page) {
  XDNA_REQUIRE(cache_sizes_ok(B, N, nh, nkv, d, P, 0, page, page), "bad sizes");
  if (B == 0 || N == 0) return 0;
  CacheArgs a{};
  a.B = (int)B, a.N = (int)N, a.nh = nh, a.nkv = nkv, a.d = d, a.P = (int)P, a.logg = log2_page(page);
  cache_plan(a);
  return a.parts > 1 ? (int64_t)a.parts * B * N * nh * (d + 2) * 4 : 0;
}

int xdna_attention_cache(const void* q, int dtype, const int64_t* strides, const void* kpages, const void* vpages, const float* kscales,
                         const float* vscales, const void* ktail, const void* vtail, const int32_t* table, int64_t ldt,
                         const int32_t* lens, int64_t B, int64_t N, int64_t P, int64_t pages, int64_t page, int64_t R, int nh, int nkv,
                         int d, float scale, void* out, void* ws, int64_t ws_bytes, void* stream) {
  XDNA_REQUIRE(sixteen(dtype), "dtype must be BF16/F16");
  XDNA_REQUIRE(cache_sizes_ok(B, N, nh, nkv, d, P, pages, page, R), "bad sizes (head dims: a multiple of 16, at most 128)");
  if (B == 0 || N == 0) return XDNA_OK;
  XDNA_REQUIRE(q && strides && lens && out && ktail && vtail, "null pointer");
  XDNA_REQUIRE(P == 0 || (table && ldt >= 0), "no table");
  XDNA_REQUIRE(pages > 0 ? kpages && vpages && kscales && vscales : P == 0, "a table's texts need pages");
  XDNA_REQUIRE(aligned(q, 16) && aligned(out, 16) && aligned(kpages, 16) && aligned(vpages, 16) && aligned(ktail, 16) && aligned(vtail, 16),
               "operands must be 16-byte aligned");
  for (int i = 0; i < 3; ++i) XDNA_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "strides must be multiples of 8");
  CacheArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.qb = strides[0], a.qn = strides[1], a.qh = strides[2];
  a.kp = static_cast<const int8_t*>(kpages), a.vp = static_cast<const int8_t*>(vpages), a.ks = kscales, a.vs = vscales;
  a.ktail = static_cast<const uint16_t*>(ktail), a.vtail = static_cast<const uint16_t*>(vtail);
  a.table = table, a.lens = lens, a.ldt = ldt;
  a.B = (int)B, a.N = (int)N, a.nh = nh, a.nkv = nkv, a.d = d, a.P = (int)P, a.pages = (int)pages, a.logg = log2_page(page), a.R = (int)R;
  a.c = std::max(fabsf(scale) * 1.44269504088896340736f, 1.17549435e-38f);    // above 0: an unseen key's -inf stays one
  a.sign = scale < 0.0f ? 0x80008000u : 0u;
  a.out = static_cast<uint16_t*>(out);
  cache_plan(a);
  const int64_t rows = B * N * nh, need = a.parts > 1 ? a.parts * rows * (d + 2) * 4 : 0;
  XDNA_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need), "workspace too small or misaligned");
  a.po = static_cast<float*>(ws);
  a.pml = a.po + (int64_t)a.parts * rows * d;
  hipStream_t st = as_stream(stream);
  if (dtype == XDNA_BF16) return d > 64 ? cache_go<XDNA_BF16, 128>(a, st) : cache_go<XDNA_BF16, 64>(a, st);
  return d > 64 ? cache_go<XDNA_F16, 128>(a, st) : cache_go<XDNA_F16, 64>(a, st);
}

}  // extern "C"
