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
// The products with pages run in float16, which holds int8 exactly and is the cheaper to widen to: bfloat16 rows of q are brought
// into its range by a power of two. K's scale goes into the exponent's factor, in float32; V's into the weights that P holds,
// before their rounding to float16. The open page's products run in the tensors' own type, whose range its values need. So weights
// are held in 16 bits, as the matrix units take them. Against 64 bits the outputs' error grows by that, from plain float32
// weights': float16 from 0.00021 of their norm to 0.00026 - 0.00029; bfloat16 from 0.00166 to 0.00168 - 0.0018 over pages and to 0.0021
// for texts that lie in the open page whole. The open page's weights in two halves bring those to 0.00166 and cost 6 to 8% (4 x
// 330 7.24 us for 6.83, 16 texts of 5 new tokens 25.9 for 23.8), so they are not.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "xdna_common.h"
#include "xdna_hip.h"
#include "xdna_rotate.h"

namespace xdna {
namespace {

typedef __bf16 bf16x8c __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2c __attribute__((ext_vector_type(2)));
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
  Divisor by_nkv, by_each;              // heads; pages of a text, without starts
  Divisor by_token, by_value, by_qtoken, by_head;   // units of a token of keys, of values, of all q heads, of a head
  int both;                             // the smaller of the numbers of heads' pages and of workgroups of q
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

// Eight values as bytes, round_half_even(x / s), two words. By a product with the reciprocal and a division where that is near a
// half (quant_pack, the same integers) as long as the reciprocal is a normal number. Blocks of zeros (s == 0), and those
// that hold a value that is not finite (s NaN: all of it reads as NaN), are zeros.
__device__ __forceinline__ void quant8(const float (&x)[8], float s, float r, uint32_t (&w)[2]) {
  if (s >= 0x1p-100f) return quant_pack<8>(x, s, r, w);          // s is the workgroup's
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    w[g] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = s > 0.0f ? rintf(x[4 * g + e] / s) : 0.0f;
      w[g] |= (uint32_t)((int)fminf(fmaxf(t, -127.0f), 127.0f) & 255) << (8 * e);
    }
  }
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

__device__ __forceinline__ void store_bytes(int8_t* to, int n, const float (&x)[8], float s, float r) {
  uint32_t w[2];
  quant8(x, s, r, w);
  if (n == 8) {
    typedef uint32_t u32x2_1 __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<u32x2_1*>(to) = u32x2_1{w[0], w[1]};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) to[e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
  }
}

// A workgroup has a page of one head's keys (kind 0) or values (1), or some tokens of all heads' queries (2); kinds in turn, so
// that those that compute more and those that read more share a CU. Texts whose open page holds old tokens: only their first
// page's workgroup reads the ring, and writes what would fall on the old tokens' places after that. U: units of keys a thread
// has. One pass over the tokens: a page's values stay in registers (keys) or LDS (values, which turn there) until their maximum
// is known. 16384 tokens, 16 / 8 heads of 128, with q: 235 MB, 44 us (5.3 TB/s; a large copy 4.8), vector units as busy as memory
// (turns, roundings, bytes; with a division for each byte 55 us; four heads a workgroup, the angles theirs in common, 53:
// fewer workgroups side by side). 48 new tokens 5.4 us: the launch and three round trips (lengths, tokens and frequencies,
// stores).
template <int DT, bool INTER, int U, int KINDS>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  __shared__ float part[4];
  const int g = 1 << a.logg;
  int index = blockIdx.x / KINDS, kind = blockIdx.x - index * KINDS;
  if (KINDS == 3 && index >= a.both) {          // of one sort there are no more
    const int rest = blockIdx.x - 3 * a.both;
    if (a.items * a.nkv > a.both) index = a.both + (rest >> 1), kind = rest & 1;
    else index = a.both + rest, kind = 2;
  }
  if (KINDS == 3 && kind == 2) {
    __shared__ float cs[256], sn[256];
    __shared__ int known[16];
    const int64_t t0 = (int64_t)index * a.qtokens;
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
    const int per_head = a.by_head.d, per_token = a.by_qtoken.d;
    for (int i = threadIdx.x; i < n * per_token; i += 256) {
      const int tok = a.by_qtoken.of(i), at = i - tok * per_token, head = a.by_head.of(at);
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
  const int item = a.by_nkv.of(index), kvh = index - item * a.nkv;
  if (item >= a.items) return;
  int b, nth;
  if (a.starts) {
    int first = 0x7fffffff;
    b = __builtin_amdgcn_readfirstlane(text_of_item(a, item, first));
    nth = item - __builtin_amdgcn_readfirstlane(first);
  } else {
    const int each = ((a.each + g - 2) >> a.logg) + 1;
    b = a.by_each.of(item);
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
  const bool writes_later = nth == 0 && later < x.end;
  if (kind == 0) {
    const int per_token = a.by_token.d, units = g * per_token;
    float p[U][8], q[U][8], top = 0.0f;
    Unit u[U];
    int pos[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = i * 256 + threadIdx.x, tok = a.by_token.of(at);
      pos[i] = at < units ? begin + tok : 0x7fffffff;
      u[i] = unit_of<INTER>(at - tok * per_token, a.d, a.half);
      if (pos[i] >= hi || (pos[i] < lo && !whole)) continue;
      key_unit<DT, INTER>(a, x, b, kvh, u[i], pos[i], p[i], q[i]);
      if (pos[i] >= lo && pos[i] >= oldest && pos[i] < later) key_to_tail<DT>(a, b, kvh, u[i], pos[i], p[i], q[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = __builtin_elementwise_maximum(top, fabsf(p[i][e]));
        top = __builtin_elementwise_maximum(top, fabsf(q[i][e]));
      }
    }
    if (whole) {
      const int64_t block = (int64_t)id * a.nkv + kvh;
      const float amax = group_amax(top, part), scale = __builtin_isfinite(amax) ? amax / 127.0f : __builtin_nanf(""), r = 1.0f / scale;
      if (good) {
        if (threadIdx.x == 0) a.ks[block] = scale;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (pos[i] >= hi) continue;
          int8_t* const to = a.kp + (block * g + pos[i] - begin) * a.d;
          store_bytes(to + u[i].a, u[i].na, p[i], scale, r);
          store_bytes(to + u[i].b, u[i].nb, q[i], scale, r);
        }
      }
    }
    if (writes_later) {
      __syncthreads();
      const int from = max(later, oldest), n = (x.end - from) * per_token;
      for (int at = threadIdx.x; at < n; at += 256) {
        const int tok = a.by_token.of(at);
        const Unit v = unit_of<INTER>(at - tok * per_token, a.d, a.half);
        float pp[8], qq[8];
        key_unit<DT, INTER>(a, x, b, kvh, v, from + tok, pp, qq);
        key_to_tail<DT>(a, b, kvh, v, from + tok, pp, qq);
      }
    }
    return;
  }
  // values: through LDS, [token][d + 2] so that a walk along the tokens of 16 dims meets every bank
  extern __shared__ __attribute__((aligned(16))) uint16_t vl[];
  const int per_token = a.by_value.d, units = g * per_token, ld = a.d + 2;
  const int64_t head = (int64_t)b * a.nkv + kvh, block = (int64_t)id * a.nkv + kvh;
  const auto value = [&](int pos, int u, float (&p)[8]) {
    if (pos >= x.len) return load8<DT>(a.v, (x.s0 + pos - x.len) * a.vt + kvh * a.vh + 8 * u, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = load_as_f32<DT>(a.vtail, (head * a.d + 8 * u + e) * a.R + pos % a.R);
  };
  const auto to_tail = [&](int pos, int u, const float (&p)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_from_f32<DT>(a.vtail, (head * a.d + 8 * u + e) * a.R + pos % a.R, p[e]);
  };
  float top = 0.0f;
#pragma unroll 4
  for (int at = threadIdx.x; at < units; at += 256) {
    const int tok = a.by_value.of(at), u = at - tok * per_token, pos = begin + tok;
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
    const float amax = group_amax(top, part), s = __builtin_isfinite(amax) ? amax / 127.0f : __builtin_nanf(""), r = 1.0f / s;
    if (good) {
      if (threadIdx.x == 0) a.vs[block] = s;
      // two dims of 8 tokens: a word of LDS a token, 8 bytes of either dim's row of the page
      const int logc = a.logg - 3, tasks = (a.d >> 1) << logc;
      for (int i = threadIdx.x; i < tasks; i += 256) {
        const int pair = i >> logc, c = i & ((1 << logc) - 1);
        float lo8[8], hi8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t y = *reinterpret_cast<const uint32_t*>(vl + (8 * c + e) * ld + 2 * pair);
          lo8[e] = DT == XDNA_F16 ? f16_bits_to_f32((uint16_t)y) : bf16_bits_to_f32((uint16_t)y);
          hi8[e] = DT == XDNA_F16 ? f16_bits_to_f32((uint16_t)(y >> 16)) : bf16_bits_to_f32((uint16_t)(y >> 16));
        }
        uint32_t w[2];
        int8_t* const to = a.vp + (block * a.d + 2 * pair) * g + 8 * c;
        quant8(lo8, s, r, w);
        *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        quant8(hi8, s, r, w);
        *reinterpret_cast<uint2*>(to + g) = make_uint2(w[0], w[1]);
      }
    }
  }
  if (writes_later) {
    __syncthreads();
    const int from = max(later, oldest), n = (x.end - from) * per_token;
    for (int at = threadIdx.x; at < n; at += 256) {
      const int tok = a.by_value.of(at), u = at - tok * per_token;
      float p[8];
      value(from + tok, u, p);
      to_tail(from + tok, u, p);
    }
  }
}

template <int DT, bool INTER, int KINDS>
int append_go(AppendArgs a, hipStream_t st) {
  const int units = units_of(a.d, a.half), per = (int)cdiv((int64_t)units << a.logg, 256), g = 1 << a.logg;
  const int64_t blocks = (int64_t)a.items * a.nkv, qblocks = KINDS == 3 ? cdiv(a.T, a.qtokens) : 0;
  a.both = (int)std::min(blocks, qblocks);
  a.by_nkv = Divisor(a.nkv), a.by_each = Divisor(((a.each + g - 2) >> a.logg) + 1);
  a.by_head = a.by_token = Divisor(units), a.by_value = Divisor(a.d / 8);
  if (KINDS == 3) a.by_qtoken = Divisor((int64_t)units * a.nh);
  const unsigned grid = (unsigned)(2 * blocks + qblocks), lds = (unsigned)((a.d + 2) * 2 << a.logg);
  if (per <= 1) append_kernel<DT, INTER, 1, KINDS><<<grid, 256, lds, st>>>(a);
  else if (per <= 2) append_kernel<DT, INTER, 2, KINDS><<<grid, 256, lds, st>>>(a);
  else append_kernel<DT, INTER, 5, KINDS><<<grid, 256, lds, st>>>(a);
  return launch_status("cache_append");
}

template <int DT>
int append_kinds(const AppendArgs& a, bool interleaved, hipStream_t st) {
  if (a.q) return interleaved ? append_go<DT, true, 3>(a, st) : append_go<DT, false, 3>(a, st);
  return interleaved ? append_go<DT, true, 2>(a, st) : append_go<DT, false, 2>(a, st);
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
  int parts, rblocks, items;            // parts of a text's keys; blocks of rows of a (text, kv head); parts B nkv
  Divisor by_rblocks, by_nkv, by_b, by_grp, by_parts;
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

// Eight int8 as float16, exactly: q + 128 is the low bits of 1024 + .., and 1152 comes off again. Five instructions for four of
// them; to bfloat16 it would be six.
__device__ __forceinline__ i32x4 widen8(uint32_t a, uint32_t b) {
  const f16x2_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
  const uint32_t w[2] = {a ^ 0x80808080u, b ^ 0x80808080u};
  i32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    r[2 * i] = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04010400u)) - off);
    r[2 * i + 1] = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, w[i], 0x04030402u)) - off);
  }
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

// A row's maxima follow once they are passed by more than 2^SLACK: nearly never after a row's first keys, where otherwise some
// row of sixteen finds a larger one at nearly every step, and all of O is multiplied. O's weights are held 2^SHIFT times as
// large, so that float16 takes them from 2^-22 of the maximum (normal) to 2^(SLACK + 1) times it.
constexpr float SLACK = 6.0f, SHIFT = 8.0f;
// The maximum of no scores but -inf: below every other, and a number, so that differences from it are none either.
constexpr float LOWEST = -3.40282347e+38f;
template <int DT>
constexpr uint32_t ALL_ONES = DT == XDNA_F16 ? 0x7c00u : 0x7f80u;

// A wave's rows: RB blocks of 16, their maxima, sums and outputs. Rows of a (text, kv head) are the pairs (new token, q head
// of the group), so that the heads that share K and V share their loads.
// A key's weight in O is p times its values' scale, f 2^k with f in 1 .. 2: those weights have a maximum of their own, so that
// pages whose scales lie far apart all reach float16 as near to a row's largest weight as they count.
template <int D, int RB>
struct Rows {
  static constexpr int ND = D / 16;
  f32x4 o[RB][ND];
  float l[RB], m[RB];       // sum of p, 2^m its unit
  float ko[RB];             // 2^(m + ko - SHIFT) is O's: beside a large m the sum would have no fraction

  // The weights of T tiles of 16 keys as the second product's operand, 2^(c score) f 2^k in O's unit; c with K's scale, k and f
  // the lane's. same: k is that of all 64 keys.
  template <int DT, int T>
  __device__ __forceinline__ void weigh(f32x4* sc, int rb, float c, float k, float f, bool same, int* pf) {
    float top = sc[0][0];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = __builtin_elementwise_maximum(top, sc[t][r]);
    top *= c;
    const float mx = quad_max(top), rise = mx - m[rb], riseo = same ? rise + k : quad_max(top - m[rb] + k);
    const bool grow = rise > SLACK;
    if (__builtin_amdgcn_ballot_w64(grow || riseo - SLACK > ko[rb])) {
      const float mn = grow ? mx : m[rb], kn = ko[rb] + (m[rb] - mn), kx = same ? mx - mn + k : quad_max(top - mn + k);
      l[rb] *= __builtin_amdgcn_exp2f(m[rb] - mn);                               // from LOWEST: 0
      m[rb] = mn;
      const bool growo = kx - SLACK > kn;
      const float alpha = growo ? __builtin_amdgcn_exp2f(kn - kx) : 1.0f;
#pragma unroll
      for (int i = 0; i < ND; ++i) o[rb][i] *= alpha;
      ko[rb] = growo ? kx : kn;
    }
    const float out = k + SHIFT - ko[rb];                                        // from p to the weights
    float m0 = m[rb], shift = out - m0;
    bool far = false;                                                            // too far for the weights to tell p
    if (__builtin_amdgcn_ballot_w64(fabsf(m0) > 0x1p20f || out < -64.0f)) {
      // A maximum past 2^20 is rounded by a 16th and more, past 2^28 by more than float16's range, and the products that fma takes
      // are not. There the scores are rounded first, as the maximum was, and the maximum goes off them: the largest is 0.
      if (__builtin_amdgcn_ballot_w64(fabsf(m0) > 0x1p20f)) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[t][r] = sc[t][r] * c - m0;
        c = 1.0f, m0 = 0.0f, shift = out;
      }
      far = __builtin_amdgcn_ballot_w64(out < -64.0f) != 0;
      if (far) {
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) l[rb] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], c, -m0));
      }
    }
    const float scale = far ? 0.0f : __builtin_amdgcn_exp2f(-out);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], c, shift)), p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r + 1], c, shift));
        l[rb] = __builtin_fmaf(p0, scale, l[rb]);
        l[rb] = __builtin_fmaf(p1, scale, l[rb]);
        pf[2 * t + r / 2] = (int)pack16<DT>(p0 * f, p1 * f);
      }
  }
};

// W waves share out the 64-key steps of a part of a text's keys for 16 RB rows and meet in LDS. Registers hold the step in
// work and nothing else: K of the wave's next step is on its way once its scores are done, V after its products. The last
// step is a copy of the loop's body that loads nothing: past a branch around loads the compiler waits for all of them.
// Heads are held as D dims, a multiple of 32; dims past a.d (D - 16 then) are copies of others (int8, finite; in the open page, where
// keys may not be, zeros), times zeros of q, and of no output.
// EXACT: the heads have D dims, and nothing is asked about a dim. Where rows are few beside the keys it is worth nothing (48 x 8192
// 115.5 us, without 115.2; 24 x 2000 19.4 / 19.0), for short texts and more rows it is (4 x 330 6.83 / 7.07, 64 x 600 in heads of 64
// 9.5 / 9.9; 16 x 5 new tokens in heads of 96 24.1 / 25.6; 128 x 2000 of 5 new tokens in heads of 128 72.5 / 81.7, of 64 36.3 / 37.4).
//
// What bounds it: one new token a text, the stream of K and V (48 texts of 4096 .. 8192, 604 MB: 115 us, 5.2 TB/s; texts of one
// length 5.9; a kernel that only reads reaches 6.3), the rest the unequal lengths. More rows, the vector units and the registers, which
// leave two waves a SIMD: a step of 48 rows and heads of 96 is about 1000 vector instructions, 240 of them the widening, and 72 MFMAs; 16
// texts x 5 tokens x 7 heads a kv head over 2500 .. 5000 keys 21.5 us, vector units 48%, waits 45% of the waves' time. Short texts, the
// chain of lengths, pages, keys, and about 2000 instructions of one wave (4 x 330: 6.8 us).
template <int DT, int D, int RB, int W, bool EXACT>
__global__ __launch_bounds__(W * 64, 2) void cache_kernel(CacheArgs a) {
  // a lane's bytes of K: 16 of each 64 dims, and 8 of the last 32
  constexpr int S = D / 32, ND = D / 16, DC = D / 64, REST = S - 2 * DC;
  // blocks of rows that the waves join at once: all, where two workgroups' LDS has room for them
  constexpr int JB = RB * ND <= 16 ? RB : 1;
  constexpr bool QLDS = RB > 1;                 // more rows: q in LDS, registers for O
  __shared__ __attribute__((aligned(16))) float ol[W][JB * ND][256];
  __shared__ float ml[2][W][RB][16];
  __shared__ i32x4 ql[QLDS ? RB * S : 1][64];
  __shared__ float qls[QLDS ? RB : 1][16];
  __shared__ int qlim[QLDS ? RB : 1][16];
  const int lane = threadIdx.x & 63, h = lane >> 4, i16 = lane & 15, hk = i16 >> 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = a.by_grp.d, nrows = a.N * grp, g = 1 << a.logg, d = EXACT ? D : a.d;
  // the blocks of rows of one item (part, text, kv head), which read the same keys, 8 apart: on one XCD
  const int eight = a.by_rblocks.of(blockIdx.x >> 3), rblock = (blockIdx.x >> 3) - eight * a.rblocks, item = eight * 8 + (blockIdx.x & 7);
  if (item >= a.items) return;
  const int pb = a.by_nkv.of(item), kvh = item - pb * a.nkv, part = a.by_b.of(pb), b = pb - part * a.B;
  const int len = min(max(a.lens[b], 0), a.P << a.logg);
  const int npages = len >> a.logg, nfull = npages << a.logg, ntail = len - nfull;
  const int steps = (nfull + 63) >> 6, all = steps + ((ntail + 63) >> 6);
  const int per = a.by_parts.of(all + a.parts - 1), from = min(part * per, all), to = min(from + per, all);
  const int end = min(to, steps), row0 = rblock * 16 * RB, dchunks = d >> 4;

  Rows<D, RB> w;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    w.m[rb] = LOWEST;
    w.l[rb] = w.ko[rb] = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; ++i) w.o[rb][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // keys that the lane's row of a block sees
  const auto limit_of = [&](int rb) { return len - a.N + a.by_grp.of(min(row0 + 16 * rb + i16, nrows - 1)) + 1; };
  const int limit0 = limit_of(0);
  // the lane's row of a block: its new token and q head. Found again where it is needed: held, it costs the loop registers.
  const auto row_of = [&](int rb, int& n, int& head) {
    int at = row0;
    asm volatile("" : "+s"(at));
    const int row = min(at + 16 * rb + i16, nrows - 1);
    n = a.by_grp.of(row), head = kvh * grp + row - n * grp;
  };
  const auto load_q = [&](int rb, i32x4 (&x)[S]) {
    int n, head;
    row_of(rb, n, head);
    const uint16_t* const q = a.q + b * a.qb + n * a.qn + head * a.qh;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int dim = s < 2 * DC ? 16 * (h + 4 * (s >> 1)) + 8 * (s & 1) : 64 * DC + 8 * h;
      x[s] = *reinterpret_cast<const i32x4*>(q + min(dim, d - 8));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[s][e] = dim < d ? x[s][e] ^ (int)a.sign : 0;
    }
  };
  // q for the pages, in float16: bfloat16 rows are scaled by a power of two that brings their largest value to 2^14 .. 2^15;
  // those down to 2^-32 of it stay exact (beside one that is not finite none matters). The inverse goes to the scores.
  const auto half_q = [&](i32x4 (&x)[S], float& back) {
    back = 1.0f;
    if constexpr (DT == XDNA_BF16) {
      u16x2c big = {0, 0};
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2c, (uint32_t)x[s][e] & 0x7fff7fffu));
      uint32_t top = max(big[0], big[1]);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const uint32_t e8 = max(top >> 7, 15u);
      const float by = __uint_as_float((268u - e8) << 23);
      back = __uint_as_float((e8 - 14u) << 23);
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[s][e] = (int)f32x2_to_f16x2_bits(bf16_bits_to_f32((uint16_t)x[s][e]) * by, bf16_bits_to_f32((uint16_t)((uint32_t)x[s][e] >> 16)) * by);
    }
  };
  i32x4 qf[S];
  float back = 1.0f;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
    if (!QLDS || wave == rb) load_q(rb, qf);

  // A lane's part of a step: the page of the keys that it loads K of (16 hk ..), and of those that it has scores and V of
  // (16 h ..). Pages past the last one, and what is no page, are read as a page that there is, and masked. A step's pages are
  // asked for before the K of the step before it, so that no later load has to be waited for with them.
  const int32_t* const table = a.table + b * a.ldt;
  const auto page_at = [&](int at, int quarter) { return table[min((at * 64 + 16 * quarter) >> a.logg, a.P - 1)]; };
  const auto known = [&](int id) { return id >= 0 && id < a.pages; };
  int asked_k = 0, asked_v = 0;
  i32x4 k[4 * DC + 1], v[ND];
  int2 kr[4];
  float ksc = 0.0f, vsc = 0.0f;
  // what differs from lane to lane goes into one offset, the rest is uniform
  const int klane = (lane & 3) * d + 16 * min(h, dchunks - 1), kmore = 16 * (min(h + 4, dchunks - 1) - min(h, dchunks - 1));
  const int krest = (lane & 3) * d + 64 * DC + 8 * (64 * DC + 8 * h < d ? h : h & 1);
  const auto k_base = [&](int at, int id) {
    return a.kp + ((int64_t)(known(id) ? id : 0) * a.nkv + kvh) * (g * d) + ((at * 64 + 16 * hk) & (g - 1)) * d;
  };
  const auto v_base = [&](int at, int id) {
    return a.vp + ((int64_t)(known(id) ? id : 0) * a.nkv + kvh) * (g * d) + (i16 * g + ((at * 64 + 16 * h) & (g - 1)));
  };
  const auto load_k = [&](const int8_t* base) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (DC > 0) k[t * DC] = *reinterpret_cast<const i32x4*>(base + (klane + 4 * t * d));
      if constexpr (DC > 1) k[t * DC + 1] = *reinterpret_cast<const i32x4*>(base + (klane + kmore + 4 * t * d));
      if constexpr (REST) kr[t] = *reinterpret_cast<const int2*>(base + (krest + 4 * t * d));
    }
  };
  const auto load_v = [&](const int8_t* base) {
#pragma unroll
    for (int i = 0; i < ND; ++i) v[i] = *reinterpret_cast<const i32x4*>(base + 16 * min(i, dchunks - 1) * g);
  };
  const auto load_scales = [&](int id) {
    const int64_t at = (int64_t)(known(id) ? id : 0) * a.nkv + kvh;
    ksc = a.ks[at];
    vsc = a.vs[at];
  };
  int step = (a.parts == 1 ? 0 : from) + wave;       // alone, a wave's first page is known before the length is
  bool good = false;
  if (a.P > 0) {
    const int id_k = page_at(step, hk), id_v = page_at(step, h);
    asked_k = page_at(step + W, hk), asked_v = page_at(step + W, h);
    good = known(id_v);
    if (step < end) {
      load_k(k_base(step, id_k));
      load_scales(id_v);
      load_v(v_base(step, id_v));
    }
  }
  if constexpr (QLDS) {
    if (wave < RB) {
      half_q(qf, back);
#pragma unroll
      for (int s = 0; s < S; ++s) ql[wave * S + s][lane] = qf[s];
      if (h == 0) qls[wave][i16] = back * a.c, qlim[wave][i16] = limit_of(wave);
    }
    __syncthreads();
  } else {
    half_q(qf, back);
    back *= a.c;
  }
  const auto factor = [&](int rb) { return QLDS ? qls[rb][i16] : back; };
  const auto limit = [&](int rb) { return QLDS ? qlim[rb][i16] : limit0; };
  const auto q_frag = [&](int rb, int s) {
    if constexpr (QLDS) return ql[rb * S + s][lane];
    else return qf[s];
  };
  // the first row's tokens are the fewest that a row of this workgroup sees
  const int sure = min(nfull, __builtin_amdgcn_readfirstlane(limit0));

  const auto pages = [&](auto more) {
    const int first = step * 64 + 16 * h, next = step + W;
    const bool masked = step * 64 + 64 > sure || __builtin_amdgcn_ballot_w64(!good) != 0;
    const bool mine = good;
    // T tiles of 16 keys at a time: with more rows fewer scores in registers
    constexpr int T = RB == 1 ? 4 : 2;
    const float ks = ksc, vs = vsc;
    const int e8 = (int)(__float_as_uint(vs) >> 23 & 255u) - 127;
    const float vk = (float)e8, vf = __builtin_amdgcn_ldexpf(vs, -e8);          // f of a scale that is not finite is not
    const int8_t* next_v = nullptr;
#pragma unroll
    for (int t0 = 0; t0 < 4; t0 += T) {
      i32x4 pf[RB][T / 2];
      f32x4 sc[RB][T];
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[rb][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        i32x4 q[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) q[rb] = q_frag(rb, s);
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const int tt = t0 + t;
          i32x4 f;
          if (s < 2 * DC) f = widen8(k[tt * DC + (s >> 1)][2 * (s & 1)], k[tt * DC + (s >> 1)][2 * (s & 1) + 1]);
          else f = widen8(kr[tt].x, kr[tt].y);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sc[rb][t] = mfma16<XDNA_F16>(f, q[rb], sc[rb][t]);
        }
      }
      if (t0 + T == 4) {
        if constexpr (more) {
          const int8_t* const next_k = k_base(next, asked_k);
          next_v = v_base(next, asked_v);
          const int id = asked_v;
          good = known(id);
          asked_k = page_at(next + W, hk), asked_v = page_at(next + W, h);
          load_k(next_k);
          load_scales(id);
        }
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int lim = mine ? min(nfull, limit(rb)) : 0;
        if (masked) {
#pragma unroll
          for (int t = 0; t < T; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (first + 4 * (t0 + t) + r >= lim) sc[rb][t][r] = -INFINITY;
        }
        // above 0, so that an unseen key's -inf stays one; the scales of a page that the row does not see do not matter
        float c = __builtin_elementwise_maximum(ks * factor(rb), 1.17549435e-38f);
        const bool unseen = masked && first >= lim;
        if (unseen) c = 1.0f;
        w.template weigh<XDNA_F16, T>(sc[rb], rb, c, vk, unseen ? 0.0f : vf, g >= 64, reinterpret_cast<int*>(&pf[rb][0]));
      }
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int u = 0; u < T / 2; ++u) {
          const i32x4 f = widen8(v[i][t0 + 2 * u], v[i][t0 + 2 * u + 1]);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) w.o[rb][i] = mfma16<XDNA_F16>(f, pf[rb][u], w.o[rb][i]);
        }
    }
    if constexpr (more) load_v(next_v);
  };
#pragma unroll 1
  for (; step + W < end; step += W) pages(std::true_type{});
  if (step < end) {
    pages(std::false_type{});
    step += W;
  }
  // the open page, in 16 bits
#pragma unroll 1
  for (; step < to; step += W) {
    const int at = (step - steps) * 64, left = ntail - at;          // keys of this step: nfull + at ..
    const int slot = nfull % a.R + at;
    const int64_t head = (int64_t)b * a.nkv + kvh;
    const uint16_t* const kt = a.ktail + (head * a.R + slot) * d;
    // a group of 16 places without keys is read as the first one, and masked
    const uint16_t* const vt = a.vtail + head * d * a.R + (i16 * a.R + slot + (16 * h < left ? 16 * h : 0));
    f32x4 sc[RB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sc[rb][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // a block of rows after the other, so that few registers hold q and K
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      i32x4 q[S];
      load_q(rb, q);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const int dim = s < 2 * DC ? 16 * min(h + 4 * (s >> 1), dchunks - 1) + 8 * (s & 1) : 64 * DC + 8 * (64 * DC + 8 * h < d ? h : h & 1);
          i32x4 f = *reinterpret_cast<const i32x4*>(kt + (min(16 * hk + 4 * t + (lane & 3), left - 1) * d + dim));
          // dims that the heads do not have: q is 0 there, which times an infinity of the dim read instead would be NaN
          if constexpr (!EXACT) {
            const int keep = (s < 2 * DC ? 16 * (h + 4 * (s >> 1)) : 64 * DC + 8 * h) < d ? -1 : 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] &= keep;
          }
          sc[rb][t] = mfma16<DT>(f, q[s], sc[rb][t]);
        }
      if (RB > 1) asm volatile("" ::: "memory");
    }
    // V in two halves: its 16-bit fragments of all dims are as many registers again as a step of pages has
    constexpr int HALF = ND / 2;
    i32x4 f[HALF][2];
    const auto load_half = [&](int n) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < HALF; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          f[i][u] = *reinterpret_cast<const i32x4*>(vt + 16 * min(n * HALF + i, dchunks - 1) * a.R + 8 * u);
      asm volatile("" ::: "memory");
    };
    load_half(0);
    const int first = nfull + at + 16 * h;
    i32x4 pf[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int lim = limit(rb);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (first + 4 * t + r >= lim) sc[rb][t][r] = -INFINITY;
      w.template weigh<DT, 4>(sc[rb], rb, a.c, 0.0f, 1.0f, true, reinterpret_cast<int*>(&pf[rb][0]));
    }
    // Places without keys are zeros. What is not finite may belong to a key that some rows do not see (of one new token's rows
    // every row sees every key), and 0 times it would be NaN: taken out, and added below to the rows that see it.
    uint32_t keep[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) keep[e] = (16 * h + 2 * e < left ? 0xffffu : 0u) | (16 * h + 2 * e + 1 < left ? 0xffff0000u : 0u);
    bool odd = false;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n) load_half(1);
      u16x2c big = {0, 0};
#pragma unroll
      for (int i = 0; i < HALF; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[i][u][e] &= (int)keep[4 * u + e];
          }
      if (a.N > 1) {
#pragma unroll
        for (int i = 0; i < HALF; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2c, (uint32_t)f[i][u][e] & 0x7fff7fffu));
      }
      if (a.N > 1 && __builtin_amdgcn_ballot_w64(big[0] >= ALL_ONES<DT> || big[1] >= ALL_ONES<DT>)) {
        odd = true;
#pragma unroll
        for (int i = 0; i < HALF; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t x = (uint32_t)f[i][u][e];
              if ((x & ALL_ONES<DT>) == ALL_ONES<DT>) x &= 0xffff0000u;
              if ((x >> 16 & ALL_ONES<DT>) == ALL_ONES<DT>) x &= 0xffffu;
              f[i][u][e] = (int)x;
            }
      }
#pragma unroll
      for (int i = 0; i < HALF; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) w.o[rb][n * HALF + i] = mfma16<DT>(f[i][u], pf[rb][u], w.o[rb][n * HALF + i]);
    }
    if (odd) {
#pragma unroll 1
      for (int x = 0; x < min(left, 64) * dchunks; ++x) {
        const int i = x % dchunks, key = x / dchunks;
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint16_t z = a.vtail[(head * d + 16 * i + 4 * h + r) * a.R + slot + key];
          y[r] = (z & ALL_ONES<DT>) != ALL_ONES<DT> ? 0.0f : DT == XDNA_F16 ? f16_bits_to_f32(z) : bf16_bits_to_f32(z);
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          // lane 16 (key / 16) + i16 holds the row's p of it, in half key % 2 of word (key % 16) / 2
          uint32_t z = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e == (key & 15) >> 1) z = (uint32_t)pf[rb][e >> 2][e & 3];
          z = __shfl(z, 16 * (key >> 4) + i16, 64) >> (16 * (key & 1)) & 0xffffu;
          const float p = DT == XDNA_F16 ? f16_bits_to_f32((uint16_t)z) : bf16_bits_to_f32((uint16_t)z);
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n == i && y[r] != 0.0f && nfull + at + key < limit(rb)) w.o[rb][n][r] += p * y[r];
        }
      }
    }
  }

  // The waves' rows joined, JB blocks of them at a time: all waves' at once; halves in turn took 0.4 us
  // more (4 x 330).
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const float l = quad_sum(w.l[rb]);
    if (h == 0) ml[0][wave][rb][i16] = w.m[rb] == LOWEST ? -INFINITY : w.m[rb], ml[1][wave][rb][i16] = l;
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    if (rb % JB == 0) {
      if (rb > 0) __syncthreads();                   // those before are read
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        const float unit = __builtin_amdgcn_exp2f(w.ko[rb + j] - SHIFT);               // O in p's
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const f32x4 o = w.o[rb + j][i] * unit;
          *reinterpret_cast<f32x4*>(&ol[wave][j * ND + i][lane * 4]) = o;
        }
      }
      __syncthreads();
    }
    float mt = -INFINITY, lt = 0.0f, weight[W];
#pragma unroll
    for (int x = 0; x < W; ++x) mt = fmaxf(mt, ml[0][x][rb][i16]);
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float mg = ml[0][x][rb][i16], lg = ml[1][x][rb][i16];
      weight[x] = mg == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mg - mt);     // a wave without keys: nothing
      lt += mg == -INFINITY ? lg : lg * weight[x];           // lg is 0 then, or NaN
    }
    const bool mine = row0 + 16 * rb + i16 < nrows;
    int token, qhead;
    row_of(rb, token, qhead);
    const int64_t orow = ((int64_t)b * a.N + token) * a.nh + qhead;
#pragma unroll
    for (int n = 0; n < (ND + W - 1) / W; ++n) {
      const int i = wave + n * W;
      if (i >= dchunks) break;
      f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(&ol[x][(rb % JB) * ND + i][lane * 4]);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] += y[r] * weight[x];
      }
      if (!mine) continue;
      const int dim = 16 * i + 4 * h;
      if (a.parts == 1) {
        const float inv = lt == 0.0f ? 0.0f : 1.0f / lt;
        *reinterpret_cast<uint2*>(a.out + orow * d + dim) = make_uint2(pack16<DT>(o[0] * inv, o[1] * inv), pack16<DT>(o[2] * inv, o[3] * inv));
      } else {
        const int64_t at = (int64_t)part * a.B * a.N * a.nh + orow;
        *reinterpret_cast<f32x4*>(a.po + at * d + dim) = o;
        if (dim == 0) *reinterpret_cast<float2*>(a.pml + at * 2) = make_float2(mt, lt);
      }
    }
  }
}

// The parts of a row joined: G waves have a row, wave w of them the parts w, w + G, .., U at once, then the waves in their
// order; lane l dims 2 l, 2 l + 1.
template <int DT, int G, int U>
__global__ __launch_bounds__(256) void cache_join_kernel(const float* __restrict__ po, const float* __restrict__ pml, int parts,
                                                         int64_t rows, int d, uint16_t* __restrict__ out) {
  __shared__ float2 ov[4][64], mv[4];
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % G;
  const int64_t row = (int64_t)blockIdx.x * (4 / G) + all / G;
  if (G == 1 && row >= rows) return;
  float m = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
  const int at = min(2 * lane, d - 2);
  for (int i0 = wave; i0 < parts; i0 += G * U) {
    float2 p[U], v[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t from = min(i0 + G * i, parts - 1) * rows + row;
      p[i] = *reinterpret_cast<const float2*>(pml + from * 2);
      v[i] = *reinterpret_cast<const float2*>(po + from * d + at);
    }
    float mt = m;
#pragma unroll
    for (int i = 0; i < U; ++i) mt = fmaxf(mt, p[i].x);
    const float alpha = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mt);       // without a maximum l is 0 or NaN, x and y are 0
    l *= alpha, x *= alpha, y *= alpha;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i0 + G * i < parts) {
        const float w = p[i].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(p[i].x - mt);
        l += p[i].x == -INFINITY ? p[i].y : p[i].y * w;
        x += v[i].x * w;
        y += v[i].y * w;
      }
    m = mt;
  }
  if constexpr (G > 1) {
    ov[wave][lane] = make_float2(x, y);
    if (lane == 0) mv[wave] = make_float2(m, l);
    __syncthreads();
    if (wave) return;
    float mt = -INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g) mt = fmaxf(mt, mv[g].x);
    l = x = y = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float w = mv[g].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mv[g].x - mt);
      l += mv[g].x == -INFINITY ? mv[g].y : mv[g].y * w;
      x += ov[g][lane].x * w;
      y += ov[g][lane].y * w;
    }
  }
  if (2 * lane >= d) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint32_t*>(out + row * d + 2 * lane) = pack16<DT>(x * inv, y * inv);
}

// How a call is split. A workgroup has up to 48 rows, heads over 96 dims 32: rows in one workgroup share the widening of K and V.
// 48 rows take all 256 registers for heads of 96 already, and a few words of scratch a lane (5 registers, exact dims). Measured
// there, 48 rows at most / 32: 16 texts of 5 new tokens (35 rows a kv head) over 5000 24.1 / 26.0 us, 128 over 2000 45.4 / 59.5; where
// fewer rows make more workgroups on a card that has room for them it is the other way: 4 over 3000 14.4 / 11.7, 8 of 64 new
// tokens over 5000 75.0 / 70.5.
// Up to a workgroup a CU, eight waves share out the keys, and a text's keys go to as many parts as fill the CUs, at most one for
// each 512 places of the table; with more of them four waves do, two workgroups side by side on a CU, and parts are for
// balance, at most one for each 2048 places. A part is its share of the keys that there are, so short texts in a wide table have
// parts of few keys, or of none: the host knows only how long texts can be. Measured, eight waves / four (texts x longest, 16 / 8
// heads of 128): 4 x 330 6.8 / 8.3 us, 20 x 600 8.8 / 9.8, 24 x 2000 19.5 / 20.5, 8 x 32768 81 / 84, 48 x 1000 22.6 / 19.6, 64 x 600
// 20.1 / 16.6, 48 x 8192 124 / 116 (one part 125, two 118, four 116, five 115); 1 x 131000 on 4 kv heads: 64 parts 17.0, 128 21.1. Keys
// of a part side by side and not spread over the text: 8 x 32768 80.7 against 84.
struct CachePlan {
  int blocks, rblocks, parts;
  bool eight;
  explicit CachePlan(const CacheArgs& a) {
    const int64_t rows = (int64_t)a.N * (a.nh / a.nkv), cus = device_cus(), sixteens = cdiv(rows, 16);
    rblocks = (int)cdiv(sixteens, a.d > 96 ? 2 : 3);
    blocks = (int)cdiv(sixteens, rblocks);
    const int64_t wgs = (int64_t)a.B * a.nkv * rblocks, room = (int64_t)a.P << a.logg;
    eight = wgs <= cus;
    parts = (int)std::max<int64_t>(1, eight ? std::min(cus / wgs, cdiv(room, 512)) : std::min(8 * cus / wgs, room / 2048));
  }
};

template <int DT, int D, int RB, bool EXACT>
void cache_waves(const CacheArgs& a, bool eight, hipStream_t st) {
  const unsigned grid = (unsigned)(cdiv(a.items, 8) * 8 * a.rblocks);
  if (eight) cache_kernel<DT, D, RB, 8, EXACT><<<grid, 512, 0, st>>>(a);
  else cache_kernel<DT, D, RB, 4, EXACT><<<grid, 256, 0, st>>>(a);
}

template <int DT, int D, bool EXACT>
void cache_rows(const CacheArgs& a, const CachePlan& p, hipStream_t st) {
  if (p.blocks == 1) cache_waves<DT, D, 1, EXACT>(a, p.eight, st);
  else if (p.blocks == 2) cache_waves<DT, D, 2, EXACT>(a, p.eight, st);
  else if constexpr (D <= 96) cache_waves<DT, D, 3, EXACT>(a, p.eight, st);
}

template <int DT, int D>
void cache_dims(const CacheArgs& a, const CachePlan& p, hipStream_t st) {
  if (a.d == D) cache_rows<DT, D, true>(a, p, st);
  else cache_rows<DT, D, false>(a, p, st);
}

template <int DT>
int cache_go(const CacheArgs& a, const CachePlan& p, hipStream_t st) {
  if (a.d <= 32) cache_dims<DT, 32>(a, p, st);
  else if (a.d <= 64) cache_dims<DT, 64>(a, p, st);
  else if (a.d <= 96) cache_dims<DT, 96>(a, p, st);
  else cache_dims<DT, 128>(a, p, st);
  if (a.parts > 1) {
    const int64_t all = (int64_t)a.B * a.N * a.nh;
    // a wave a row for few parts, which many rows have (2240 rows of 4 parts 4.0 us, about 2 less than with sixteen loads a wave)
    if (a.parts <= 4) cache_join_kernel<DT, 1, 4><<<(unsigned)cdiv(all, 4), 256, 0, st>>>(a.po, a.pml, a.parts, all, a.d, a.out);
    else if (a.parts <= 16) cache_join_kernel<DT, 4, 4><<<(unsigned)all, 256, 0, st>>>(a.po, a.pml, a.parts, all, a.d, a.out);
    else cache_join_kernel<DT, 4, 16><<<(unsigned)all, 256, 0, st>>>(a.po, a.pml, a.parts, all, a.d, a.out);
  }
  return launch_status("attention_cache");
}

bool cache_sizes_ok(int64_t B, int64_t N, int64_t nh, int64_t nkv, int64_t d, int64_t P, int64_t pages, int64_t g, int64_t R) {
  return B >= 0 && N >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && nh < (1 << 16) && B < (1 << 22) && N < (1 << 22) &&
         B * N * nh < (1ll << 23) && d >= 16 && d <= 128 && d % 16 == 0 && log2_page(g) >= 0 && P >= 0 && P * g < (1ll << 30) &&
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
  XDNA_REQUIRE(2 * items * nkv + T <= MAX_LAUNCH_THREADS / 256, "too many tokens");
  a.items = (int)items;
  hipStream_t st = as_stream(stream);
  return dtype == XDNA_BF16 ? append_kinds<XDNA_BF16>(a, interleaved, st) : append_kinds<XDNA_F16>(a, interleaved, st);
}

int64_t xdna_attention_cache_ws_bytes(int64_t B, int64_t N, int nh, int nkv, int d, int64_t P, int64_t page) {
  XDNA_REQUIRE(cache_sizes_ok(B, N, nh, nkv, d, P, 0, page, page), "bad sizes");
  if (B == 0 || N == 0) return 0;
  CacheArgs a{};
  a.B = (int)B, a.N = (int)N, a.nh = nh, a.nkv = nkv, a.d = d, a.P = (int)P, a.logg = log2_page(page);
  const CachePlan p(a);
  return p.parts > 1 ? (int64_t)p.parts * B * N * nh * (d + 2) * 4 : 0;
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
  const CachePlan p(a);
  a.parts = p.parts, a.rblocks = p.rblocks, a.items = (int)(p.parts * B * nkv);
  a.by_rblocks = Divisor(a.rblocks), a.by_nkv = Divisor(nkv), a.by_b = Divisor(B), a.by_grp = Divisor(nh / nkv), a.by_parts = Divisor(a.parts);
  const int64_t rows = B * N * nh, need = a.parts > 1 ? a.parts * rows * (d + 2) * 4 : 0;
  XDNA_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need), "workspace too small or misaligned");
  a.po = static_cast<float*>(ws);
  a.pml = a.po + (int64_t)a.parts * rows * d;
  hipStream_t st = as_stream(stream);
  return dtype == XDNA_BF16 ? cache_go<XDNA_BF16>(a, p, st) : cache_go<XDNA_F16>(a, p, st);
}

}  // extern "C"
