// Attention of a language model that serves prompts and their continuations, for gfx950 (MI355X), bfloat16 and float16:
//
//   attention_causal   packed prompts: token t of q head h sees the tokens start(t) .. t of its sequence
//   attention_prefix   one new token of every sequence: it sees a prefix that the batch shares, held once, and
//                      its sequence's own keys
//
//   out = sum over seen keys j of p_j v_j / sum of p_j,   p_j = 2^(c (s_j - m)),  s_j = q . k_j,  c = scale log2 e
//
// with m the running maximum of s (one pass over the keys; sums and outputs rescaled when it grows), float32
// throughout except for p, which is rounded to the inputs' type for its product with V: the matrix units take it no
// wider, and two such halves of it would be twice the products. The sum of p is that of the rounded ones. Against 64 bits the
// outputs' error grows from 0.0015 - 0.0017 of their norm with p in float32 to 0.0018 - 0.0022 in bfloat16, from 0.0002 to
// 0.00024 - 0.00028 in float16. A row that sees nothing, or only scores of -inf, is zero.
//
// A wave has 32 rows: rows of a kv head are the pairs (token, q head of its group), so the heads that share K and V
// share their loads. MFMA 32x32x16 (srcA = X, srcB = Y) gives lane l row l % 32 of Y and, in element 4 g + r, row
// 8 g + 4 (l / 32) + r of X; lane l supplies values 8 (l / 32) .. + 7 of the 16-deep step of its operand's row l % 32.
// S = K Q^T leaves in a lane 16 of 32 keys of its row, and these are, 8 at a time, what O^T = V^T P^T takes from that
// lane if step u's k slot 8 h + i stands for key 16 u + 8 (i / 4) + 4 h + i % 4. V keeps its rows of one key each:
// the transposed LDS read (16 lanes, 4 rows of 16 values: lane i gets column i) makes the V^T fragments in that
// order.
//
// Tiles of KT keys come into LDS by the DMA form of the buffer load, whose bounds check fills keys past the end, and
// dims past the head's, with zeros. A 16-byte chunk's place in its row is XORed with the row so that the lanes that
// read together cover the banks: K by the row (a fragment read takes one chunk of 16 rows), V by 64 bytes (a
// transposed read takes 64 bytes of 4 rows).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "xdna_common.h"
#include "xdna_hip.h"

namespace xdna {
namespace {

typedef float f32x16a __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8a __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8a __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2a __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_void;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

template <int DT>
__device__ __forceinline__ f32x16a mfma32(const i32x4& a, const i32x4& b, const f32x16a& c) {
  if constexpr (DT == XDNA_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8a, a), __builtin_bit_cast(f16x8a, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8a, a), __builtin_bit_cast(bf16x8a, b), c, 0, 0,
                                                   0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == XDNA_F16) return f32x2_to_f16x2_bits(lo, hi);
  else return f32x2_to_bf16x2_bits(lo, hi);
}

// the larger of a lane's value and that of lane l ^ 32 (NaN if one is), and their sum
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// float16 p are held 2^14 times as large (the sum of p too, so it cancels): p down to 2^-28 of the largest stay normal
// numbers, which a sum over 10^5 keys needs; bfloat16 has float32's range.
template <int DT>
constexpr float P_BIAS = DT == XDNA_F16 ? 14.0f : 0.0f;
template <int DT>
constexpr uint32_t EXP_ONES = DT == XDNA_F16 ? 0x7c00u : 0x7f80u;

// The keys of a workgroup: up to two runs of consecutive keys, one tile after another (no tile holds keys of both).
struct Keys {
  const char *k, *v;          // first key of the run
  const char *k2, *v2;
  int64_t kp, vp, kp2, vp2;   // bytes from key to key
  int n, n2;
};

// What a lane's row sees (keys lo .. hi of the run), and what holds for all rows of its wave, where that is known: keys
// below first or above last are seen by no row, keys from_all .. to_all by every row. Used where CAUSAL; else
// every row sees every key.
struct Seen {
  int lo, hi, first, last, from_all, to_all;
};

template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  return D == 128 ? row & 3 : (row >> 1) & 1;
}

// l + the two halves of w, as they are rounded
template <int DT>
__device__ __forceinline__ float dot_ones(uint32_t w, float l) {
  if constexpr (DT == XDNA_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), (f16x2_t){(_Float16)1.0f, (_Float16)1.0f}, l, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l, false);
}

// A value of V that is not finite may belong to a key that some rows do not see: 0 times it would be NaN. Whether a
// block of 32 keys has one (uniform), frag(u, db) its fragments;
template <int DT, int DB, class Frag>
__device__ __forceinline__ bool not_finite(Frag&& frag) {
  u16x2a big = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const i32x4 vf = frag(u, db);
#pragma unroll
      for (int e = 0; e < 4; ++e) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2a, (uint32_t)vf[e] & 0x7fff7fffu));
    }
  return __builtin_amdgcn_ballot_w64(big[0] >= EXP_ONES<DT> || big[1] >= EXP_ONES<DT>) != 0;
}

// and O += P V then: the finite values by the matrix units, the others one by one to the rows that see their key.
template <int DT, int D, class Frag, class Visible>
__device__ __forceinline__ void add_not_finite(f32x16a (&o)[D / 32], const float (&p)[16], const i32x4 (&pf)[2], const int8_t* vb,
                                               Frag&& frag, Visible&& visible) {
  const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 31;
  auto finite = [&](uint32_t w) {
    if ((w & EXP_ONES<DT>) == EXP_ONES<DT>) w &= 0xffff0000u;
    if ((w >> 16 & EXP_ONES<DT>) == EXP_ONES<DT>) w &= 0xffffu;
    return (int)w;
  };
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      i32x4 vf = frag(u, db);
#pragma unroll
      for (int e = 0; e < 4; ++e) vf[e] = finite((uint32_t)vf[e]);
      o[db] = mfma32<DT>(vf, pf[u], o[db]);
    }
#pragma unroll 1
  for (int kk = 0; kk < 32; ++kk) {
    const int want = 4 * (kk >> 3) + (kk & 3);
    float pk = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) pk = e == want ? p[e] : pk;
    pk = __shfl(pk, row + 32 * ((kk >> 2) & 1), 64);
    const bool vis = visible(kk);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint2 w = *reinterpret_cast<const uint2*>(vb + kk * 2 * D + ((db ^ v_swizzle<D>(kk)) << 6) + 16 * g + 8 * half);
        const uint16_t h[4] = {(uint16_t)w.x, (uint16_t)(w.x >> 16), (uint16_t)w.y, (uint16_t)(w.y >> 16)};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = DT == XDNA_F16 ? f16_bits_to_f32(h[r]) : bf16_bits_to_f32(h[r]);
          if (vis && (h[r] & EXP_ONES<DT>) == EXP_ONES<DT>) o[db][4 * g + r] += pk * v;
        }
        asm volatile("" ::: "memory");      // one read at a time: this path is to take no registers from the others
      }
  }
}

// Attention of 32 rows by KW waves: wave w has the tiles w, w + KW, ... of 32 keys, in LDS of its own (kl_, vl_: KW
// tiles of K, and of V, each an array, so that the compiler knows which loads a read has to wait for), and the waves
// meet there at the end (O over the tiles; ml: 2 KW x 64 maxima and sums). No barriers before
// that: K of a wave's next tile loads once its scores are done, V after its products. store(chunk, o, m, l) receives
// dims 8 (chunk % 4) + 32 (chunk / 4) + 4 (lane / 32) .. + 3 of the lane's row: the sum of p v, the maximum and the
// sum of p.
template <int DT, int D, int KW, bool CAUSAL, class Store>
__device__ __forceinline__ void attend_split(int8_t* kl_, int8_t* vl_, float* ml, const Keys& ks, int d, const i32x4 (&qf)[D / 16],
                                             const Seen& seen, float c, Store&& store) {
  constexpr int KT = 32, RB = 2 * D, KB = KT * RB, DB = D / 32, CH = D / 8, RPL = 64 / CH, NI = KB / 1024;
  const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int base = wave * KB;
  const int t1 = (int)cdiv(ks.n, KT), tiles = t1 + (int)cdiv(ks.n2, KT);
  // load j: rows j RPL + lane / CH, chunk lane % CH of the LDS row; a tile past the last loads nothing (the bounds
  // check), so that the loads under way are always as many
  auto load = [&](bool v, int tile) {
    const bool two = tile >= t1;
    const int k0 = (two ? tile - t1 : tile) * KT, left = min((two ? ks.n2 : ks.n) - k0, KT) - 1;
    const int64_t pitch = v ? (two ? ks.vp2 : ks.vp) : (two ? ks.kp2 : ks.kp);
    const char* from = (v ? (two ? ks.v2 : ks.v) : (two ? ks.k2 : ks.k)) + k0 * pitch;
    const auto r = make_rsrc(from, tile < tiles && left >= 0 ? (uint32_t)left * (uint32_t)pitch + 2u * d : 0u);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int lrow = j * RPL + lane / CH;
      const uint32_t at = (uint32_t)(((lane % CH) ^ (v ? v_swizzle<D>(lrow) * 4 : k_swizzle<D>(lrow))) * 16);
      const uint32_t off = at < 2u * d ? (uint32_t)lrow * (uint32_t)pitch + at : OOB;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void)((v ? vl_ : kl_) + (base + (j << 10))), 16, (int)off, 0, 0, 0);
    }
  };
  f32x16a o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16a{};
  float m = -INFINITY, l = 0.0f;
  // each read one index from its array: through a chain of offsets the compiler loses sight of which array it is
  const int vkey = 4 * half + ((lane & 15) >> 2);
  int voff[DB], koff[D / 16];
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    voff[db] = base + vkey * RB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3) + ((db ^ v_swizzle<D>(vkey)) << 6);
    asm volatile("" : "+v"(voff[db]));
  }
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    koff[s] = base + row * RB + (((2 * s + half) ^ k_swizzle<D>(row)) << 4);
    asm volatile("" : "+v"(koff[s]));
  }
  auto v_frag = [&](int u, int db) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vl_ + (voff[db] + u * 16 * RB)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vl_ + (voff[db] + u * 16 * RB + 8 * RB)));
    const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
    return i32x4{(int)x.x, (int)x.y, (int)y.x, (int)y.y};
  };
  load(false, wave);
  load(true, wave);
#pragma unroll 1
  for (int tile = wave; tile < tiles; tile += KW) {
    const int k0 = (tile >= t1 ? tile - t1 : tile) * KT, left = (tile >= t1 ? ks.n2 : ks.n) - k0;
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NI) : "memory");      // K is here, V need not be
    f32x16a sc = f32x16a{};
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      sc = mfma32<DT>(*reinterpret_cast<const i32x4*>(kl_ + koff[s]), qf[s], sc);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load(false, tile + KW);
    __builtin_amdgcn_sched_barrier(0);
    auto visible = [&](int k) { return CAUSAL ? k0 + k >= seen.lo && k0 + k <= seen.hi : k < left; };
    const bool part = CAUSAL ? k0 < seen.from_all || k0 + KT - 1 > seen.to_all : left < KT;      // uniform over the wave
    if (part) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!visible(8 * (e >> 2) + 4 * half + (e & 3))) sc[e] = -INFINITY;
    }
    float mx = sc[0];
#pragma unroll
    for (int e = 1; e < 15; e += 2) mx = __builtin_elementwise_maximum(mx, __builtin_elementwise_maximum(sc[e], sc[e + 1]));
    mx = pair_max(__builtin_elementwise_maximum(mx, sc[15]));
    // the running maximum follows: at few tiles a wave that is as good as not asking whether it has to
    const float mn = mx > m ? mx : m;
    const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * c);
    l = m == -INFINITY ? l : l * alpha;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] *= alpha;
    m = mn;
    const float mc = (m == -INFINITY ? 0.0f : m * c) - P_BIAS<DT>;     // -inf: only -inf scores so far, p = 0
    i32x4 pf[2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const uint32_t w = pack2<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -mc)),
                                   __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e + 1], c, -mc)));
      pf[e >> 3][(e & 7) >> 1] = (int)w;
      l = dot_ones<DT>(w, l);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NI) : "memory");                 // V is here, the next K need not be
    bool odd = false;
    if (CAUSAL && part) odd = not_finite<DT, DB>(v_frag);
    if (CAUSAL && odd) {
      float p[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -mc));
      add_not_finite<DT, D>(o, p, pf, vl_ + base, v_frag, visible);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = mfma32<DT>(v_frag(u, db), pf[u], o[db]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load(true, tile + KW);
    __builtin_amdgcn_sched_barrier(0);
  }
  l = pair_sum(l);
  // each wave leaves its m, l and O where its tiles were (half of O in K's place, half in V's); wave w then joins
  // chunks w, w + KW, ..
  constexpr int OB = 32 * D * 2, NC = 4 * DB;      // bytes of half a wave's O, chunks
  static_assert(OB == KB, "half of O takes a tile of K");
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  ml[wave * 64 + lane] = m;
  ml[(KW + wave) * 64 + lane] = l;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    *reinterpret_cast<f32x4*>(i < NC / 2 ? kl_ + (base + i * 1024 + lane * 16) : vl_ + (base + (i - NC / 2) * 1024 + lane * 16)) =
        f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
  __syncthreads();
  float mt = -INFINITY, lt = 0.0f, w[KW];
#pragma unroll
  for (int g = 0; g < KW; ++g) mt = fmaxf(mt, ml[g * 64 + lane]);
#pragma unroll
  for (int g = 0; g < KW; ++g) {
    const float mg = ml[g * 64 + lane], lg = ml[(KW + g) * 64 + lane];
    w[g] = mg == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((mg - mt) * c);     // a wave without keys: nothing
    lt += mg == -INFINITY ? lg : lg * w[g];              // lg is 0 then, or NaN
  }
#pragma unroll
  for (int i = 0; i < (NC + KW - 1) / KW; ++i) {
    const int chunk = wave + i * KW;
    if (NC % KW && chunk >= NC) break;
    const int8_t* const from = chunk < NC / 2 ? kl_ + chunk * 1024 : vl_ + (chunk - NC / 2) * 1024;
    f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < KW; ++g) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(from + g * KB + lane * 16);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += x[r] * w[g];
    }
    store(chunk, v, mt, lt);
  }
}

// Four waves of 32 rows that share every tile of 64 keys: the form for many rows. Waves without rows (idle) only
// load. Two tiles have an LDS array each (K, then V), so that the compiler knows which loads a read has to wait for:
// tile t + 1 is on its way while tile t is used. Tiles that all rows see whole take the short path (tile_all); the
// others, at the ends of a prompt's keys, go by one copy of the masked one.
//
// What bounds it: a tile is 32 MFMAs (1024 cycles; heads of 64: 512) and about 130 vector instructions, 32 exps among
// them, for a wave. Heads of 128: the card's power (1 x 16384, 16 / 8 heads: 1020 us, 1080 TFLOP/s, MFMA busy 57% at
// 1.76 GHz); heads of 64 no one unit (4096 / 1500 / 700, 12 heads: 57.5 us, 523 TFLOP/s; vector units active 52% of the CUs'
// busy time, MFMA 28%, waves waiting 29% of theirs, 1.7 of them a SIMD; 8192, 16 / 8 heads: 199 us, 690 TFLOP/s). The maximum
// follows once a tile;
// l sums the p that are rounded, two at a time by a dot product with ones. With the masked tiles in the same loop the
// compiler kept two sets of O (64 moves a tile: 1160 us).
//
// KG == 2: eight waves, each group G of four with every other tile in LDS of its own; group 1 leaves its sums there,
// and group 0 joins them.
template <int DT, int D, bool CAUSAL, int KG, int G, class Store>
__device__ __forceinline__ void attend_wide(int8_t* lds0, int8_t* lds1, const Keys& ks, int d, const i32x4 (&qf)[D / 16], const Seen& seen, bool idle, float c,
                                            Store&& store, float* ml = nullptr, const int8_t* other0 = nullptr,
                                            const int8_t* other1 = nullptr) {
  constexpr int QW = 4, KT = 64, RB = 2 * D, KB = KT * RB, DB = D / 32;
  constexpr int CH = D / 8, RPL = 64 / CH, NI = KB / 1024 / QW;
  const int lane = threadIdx.x & 63, half = lane >> 5, row = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % QW;
  const int tiles = (int)cdiv(cdiv(ks.n, KT), KG);      // of a group; tile t of group G starts at key (t KG + G) KT
  auto first_key = [](int t) { return (t * KG + G) * KT; };
  int8_t *const k0_ = lds0, *const v0_ = lds0 + KB, *const k1_ = lds1, *const v1_ = lds1 + KB;
  // this lane's share of load j: row (4 NI wave + j) RPL + lane / CH of the tile, chunk lane % CH of its LDS row. V's
  // chunk is the same for every j (a multiple of 4 rows apart).
  uint32_t ko[NI], vo[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int r = (wave * NI + j) * RPL + lane / CH;
    const uint32_t kc = (uint32_t)(((lane % CH) ^ k_swizzle<D>(r)) * 16), vc = (uint32_t)(((lane % CH) ^ (v_swizzle<D>(r) * 4)) * 16);
    ko[j] = kc < 2u * d ? (uint32_t)r * (uint32_t)ks.kp + kc : OOB;
    vo[j] = vc < 2u * d ? (uint32_t)r * (uint32_t)ks.vp + vc : OOB;
  }
  auto load = [&](int tile, int8_t* kd, int8_t* vd) {
    const int left = min(ks.n - first_key(tile), KT) - 1;     // below 0: nothing is read
    const auto kr = make_rsrc(ks.k + (int64_t)first_key(tile) * ks.kp, left < 0 ? 0u : (uint32_t)left * (uint32_t)ks.kp + 2u * d);
    const auto vr = make_rsrc(ks.v + (int64_t)first_key(tile) * ks.vp, left < 0 ? 0u : (uint32_t)left * (uint32_t)ks.vp + 2u * d);
#pragma unroll
    for (int j = 0; j < NI; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void)(kd + ((wave * NI + j) << 10)), 16, (int)ko[j], 0, 0, 0);
#pragma unroll
    for (int j = 0; j < NI; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void)(vd + ((wave * NI + j) << 10)), 16, (int)vo[j], 0, 0, 0);
  };
  f32x16a o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16a{};
  float m = -INFINITY, l = 0.0f;
  // offsets of the lane's K fragments in their block of 32 keys, and of its V fragments'; kept out of the compiler's
  // sight, which would hold a set of them for each array
  uint32_t koff[D / 16], voff[DB];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    koff[s] = row * RB + (((2 * s + half) ^ k_swizzle<D>(row)) << 4);
    asm volatile("" : "+v"(koff[s]));
  }
  const int vkey = 4 * half + ((lane & 15) >> 2);
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    voff[db] = vkey * RB + 32 * ((lane >> 4) & 1) + 8 * (lane & 3) + ((db ^ v_swizzle<D>(vkey)) << 6);
    asm volatile("" : "+v"(voff[db]));
  }
  auto v_frag = [&](const int8_t* vb, int u, int db) {
    const int8_t* at = vb + u * 16 * RB + voff[db];
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 8 * RB));
    const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
    return i32x4{(int)x.x, (int)x.y, (int)y.x, (int)y.y};
  };
  auto scores = [&](const int8_t* kb) {
    f32x16a sc = f32x16a{};
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      sc = mfma32<DT>(*reinterpret_cast<const i32x4*>(kb + koff[s]), qf[s], sc);
    return sc;
  };
  // the running maximum follows that of the new scores; p of 16 scores, packed, and their sum
  auto follow = [&](float mx) {
    mx = pair_max(mx);
    const bool grow = mx > m;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float mn = grow ? mx : m;
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
      m = mn;
    }
    return (m == -INFINITY ? 0.0f : m * c) - P_BIAS<DT>;     // -inf: only -inf scores so far, p = 0
  };
  auto max16 = [&](const f32x16a& sc) {
    float mx = sc[0];
#pragma unroll
    for (int e = 1; e < 15; e += 2)
      mx = __builtin_elementwise_maximum(mx, __builtin_elementwise_maximum(sc[e], sc[e + 1]));
    return __builtin_elementwise_maximum(mx, sc[15]);
  };
  auto weigh = [&](const f32x16a& sc, float mc, i32x4 (&pf)[2]) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const uint32_t w = pack2<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -mc)),
                                   __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e + 1], c, -mc)));
      pf[e >> 3][(e & 7) >> 1] = (int)w;
      l = dot_ones<DT>(w, l);
    }
  };
  // The reads of K run six ahead of their products, those of V's first half go out before the softmax and the second
  // half's under the first half's products: with two waves a SIMD little else hides a trip to LDS.
  auto tile_all = [&](const int8_t* kt, const int8_t* vt) {
    f32x16a sc[2];
    i32x4 pf[2][2], vf[2][2][DB];
    auto read_v = [&](int b) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int db = 0; db < DB; ++db) vf[b][u][db] = v_frag(vt + b * 32 * RB, u, db);
    };
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    sc[0] = sc[1] = f32x16a{};
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        sc[b] = mfma32<DT>(*reinterpret_cast<const i32x4*>(kt + b * 32 * RB + koff[s]), qf[s], sc[b]);
    read_v(0);
    constexpr int AHEAD = 6, KF = D / 8;                      // K's fragments
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);    // LDS reads
#pragma unroll
    for (int i = 0; i < KF - AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);      // a matrix instruction
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, (4 * DB + AHEAD - 1) / AHEAD, 0);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    const float mc = follow(__builtin_elementwise_maximum(max16(sc[0]), max16(sc[1])));
    weigh(sc[0], mc, pf[0]);
    weigh(sc[1], mc, pf[1]);
    __builtin_amdgcn_sched_barrier(0);
    read_v(1);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = mfma32<DT>(vf[b][u][db], pf[b][u], o[db]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto tile_part = [&](const int8_t* kt, const int8_t* vt, int tile) {
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
      const int first = first_key(tile) + 32 * b;
      const int8_t* const vb = vt + b * 32 * RB;
      auto visible = [&](int key) { return CAUSAL ? key >= seen.lo && key <= seen.hi : key < ks.n; };
      f32x16a sc = scores(kt + b * 32 * RB);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!visible(first + 8 * (e >> 2) + 4 * half + (e & 3))) sc[e] = -INFINITY;
      const float mc = follow(max16(sc));
      i32x4 pf[2];
      weigh(sc, mc, pf);
      bool odd = false;
      if (CAUSAL) odd = not_finite<DT, DB>([&](int u, int db) { return v_frag(vb, u, db); });
      if (CAUSAL && odd) {
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c, -mc));
        add_not_finite<DT, D>(o, p, pf, vb, [&](int u, int db) { return v_frag(vb, u, db); },
                              [&](int k) { return visible(first + k); });
      } else {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = mfma32<DT>(v_frag(vb, u, db), pf[u], o[db]);
      }
    }
  };
  auto arrive = [&](int tile, int8_t* kn, int8_t* vn) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();            // the tile is whole; every wave is done with the one before
    __builtin_amdgcn_sched_barrier(0);
    load(tile + 1, kn, vn);                  // whether there is one or not: past a branch the compiler would wait for more
    __builtin_amdgcn_sched_barrier(0);
  };
  auto masked = [&](int from, int to) {
#pragma unroll 1
    for (int t = from; t < to; ++t) {
      const bool odd = t & 1;
      arrive(t, odd ? k0_ : k1_, odd ? v0_ : v1_);
      const int k0 = first_key(t);
      if (CAUSAL && (k0 > seen.last || k0 + KT - 1 < seen.first)) continue;      // no row of this wave sees a key of it
      tile_part(odd ? k1_ : k0_, odd ? v1_ : v0_, t);
    }
  };
  // The tiles that every row of this wave sees whole are a run of them; its pairs of an even tile and the next take
  // the short path. Waves may disagree on it: each passes one barrier a tile in any case.
  if (tiles > 0) load(0, k0_, v0_);
  if (idle) {
    for (int t = 0; t < tiles; ++t) arrive(t, t & 1 ? k0_ : k1_, t & 1 ? v0_ : v1_);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (KG == 2) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }
  const int from = CAUSAL ? max(0, (int)cdiv((int)cdiv(seen.from_all, KT) - G, KG)) : 0;
  const int to = max(0, (int)cdiv((CAUSAL ? seen.to_all + 1 : ks.n) / KT - G, KG));
  const int all0 = (from + 1) & ~1, all1 = max(all0, to & ~1);
  masked(0, min(all0, tiles));
  for (int t = all0; t < all1; t += 2) {
    arrive(t, k1_, v1_);
    tile_all(k0_, v0_);
    arrive(t + 1, k0_, v0_);
    tile_all(k1_, v1_);
  }
  masked(min(all1, tiles), tiles);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the load past the end: LDS may be another's soon
  l = pair_sum(l);
  if constexpr (KG == 1) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        store(4 * db + g, f32x4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]}, m, l);
  } else if constexpr (G == 1) {
    __syncthreads();
    float* const at = reinterpret_cast<float*>((wave < 2 ? lds0 : lds1) + (wave & 1) * (128 * D));
#pragma unroll
    for (int i = 0; i < 4 * DB; ++i)
      *reinterpret_cast<f32x4*>(at + i * 256 + lane * 4) =
          f32x4{o[i / 4][4 * (i % 4)], o[i / 4][4 * (i % 4) + 1], o[i / 4][4 * (i % 4) + 2], o[i / 4][4 * (i % 4) + 3]};
    ml[wave * 64 + lane] = m;
    ml[(4 + wave) * 64 + lane] = l;
    __syncthreads();
  } else {
    __syncthreads();
    __syncthreads();
    const float* const at = reinterpret_cast<const float*>((wave < 2 ? other0 : other1) + (wave & 1) * (128 * D));
    const float m1 = ml[wave * 64 + lane], l1 = ml[(4 + wave) * 64 + lane], mt = fmaxf(m, m1);
    const float w0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mt) * c);
    const float w1 = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m1 - mt) * c);
    const float lt = (m == -INFINITY ? l : l * w0) + (m1 == -INFINITY ? l1 : l1 * w1);     // 0 or NaN where there is no maximum
#pragma unroll
    for (int i = 0; i < 4 * DB; ++i) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(at + i * 256 + lane * 4);
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = o[i / 4][4 * (i % 4) + r] * w0 + x[r] * w1;
      store(i, v, mt, lt);
    }
  }
}

// A row's q in the MFMA's order, its sign bits flipped where the scale is negative, zeros past the head's dims.
template <int D>
__device__ __forceinline__ void load_q(i32x4 (&qf)[D / 16], const uint16_t* q, int half, int d, uint32_t sign) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    qf[s] = i32x4{0, 0, 0, 0};
    if (16 * s + 8 * half < d) qf[s] = *reinterpret_cast<const i32x4*>(q + 16 * s + 8 * half);
#pragma unroll
    for (int e = 0; e < 4; ++e) qf[s][e] ^= (int)sign;
  }
}

template <int DT>
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& v, float inv) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack2<DT>(v[0] * inv, v[1] * inv), pack2<DT>(v[2] * inv, v[3] * inv));
}

// ------------------------------------------------------------------------------ packed prompts, causal
// The first token of t's sequence: the largest of the starts that is not above t, 0 if none is. Whatever the starts
// hold, the result lies in 0 .. t.
__device__ __forceinline__ int seq_start(const int32_t* __restrict__ starts, int n, int t) {
  int s = 0;
  if (n <= 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int v = starts[min(i, n - 1)];
      s = v <= t ? max(s, v) : s;
    }
  } else {
    int lo = 0, hi = n;                     // starts[0 .. lo) <= t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    s = lo ? starts[lo - 1] : 0;
  }
  return max(0, min(s, t));
}

struct CausalArgs {
  const uint16_t *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;           // elements from token to token and from head to head
  const int32_t* starts;
  int nstarts, T, nh, nkv, d;
  float c;
  uint32_t sign;
  uint16_t* out;
};

// Tiles of 32 QW rows over all tokens, whatever sequences they fall into: a tile's keys run from the first token of
// its first row's sequence to its last row's token, and each row's mask does the rest. Last tiles first: in
// a long prompt they are the longest.
// KG: groups of waves in the wide form (128 rows by attend_wide); 0: 32 rows whose keys four waves share out.
template <int DT, int D, int KG>
__global__ __launch_bounds__(KG == 2 ? 512 : 256, KG == 2 ? 1 : 2) void causal_kernel(CausalArgs a) {
  constexpr int QW = KG ? 4 : 1;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = a.nh / a.nkv, nrows = a.T * grp;
  const int kvh = blockIdx.x % a.nkv, tile = gridDim.x / a.nkv - 1 - blockIdx.x / a.nkv;
  const int row0 = tile * (32 * QW), wrow0 = min(row0 + 32 * (wave % QW), nrows - 1);
  const int tfirst = row0 / grp, tlast = (min(row0 + 32 * QW, nrows) - 1) / grp;
  const int first = __builtin_amdgcn_readfirstlane(seq_start(a.starts, a.nstarts, tfirst));
  const int last = __builtin_amdgcn_readfirstlane(seq_start(a.starts, a.nstarts, tlast));
  const int idx = min(wrow0 + (lane & 31), nrows - 1);
  const int tok = idx / grp, head = kvh * grp + idx - tok * grp;
  const int lo = first == last ? first : seq_start(a.starts, a.nstarts, tok);
  Seen seen;
  seen.lo = lo - first;
  seen.hi = tok - first;
  seen.first = __builtin_amdgcn_readfirstlane(seen.lo);           // rows and their starts ascend with the lane
  seen.to_all = __builtin_amdgcn_readfirstlane(seen.hi);
  seen.from_all = __builtin_amdgcn_readlane(seen.lo, 31);
  seen.last = __builtin_amdgcn_readlane(seen.hi, 31);
  i32x4 qf[D / 16];
  load_q<D>(qf, a.q + tok * a.qt + head * a.qh, half, a.d, a.sign);
  Keys ks;
  ks.k = reinterpret_cast<const char*>(a.k + first * a.kt + kvh * a.kh);
  ks.v = reinterpret_cast<const char*>(a.v + first * a.vt + kvh * a.vh);
  ks.kp = 2 * a.kt;
  ks.vp = 2 * a.vt;
  ks.n = tlast + 1 - first;
  ks.k2 = ks.v2 = nullptr;
  ks.kp2 = ks.vp2 = 0;
  ks.n2 = 0;
  const bool mine = row0 + 32 * (wave % QW) + (lane & 31) < nrows;
  uint16_t* const orow = a.out + ((int64_t)tok * a.nh + head) * a.d;
  auto store = [&](int chunk, const f32x4& o, float, float l) {
    const int dim = 8 * chunk + 4 * half;
    if (mine && dim < a.d) store4<DT>(orow + dim, o, l == 0.0f ? 0.0f : 1.0f / l);
  };
  const bool idle = row0 + 32 * (wave % QW) >= nrows;
  if constexpr (KG == 1) {
    __shared__ __attribute__((aligned(1024))) int8_t lds0[256 * D];
    __shared__ __attribute__((aligned(1024))) int8_t lds1[256 * D];
    attend_wide<DT, D, true, 1, 0>(lds0, lds1, ks, a.d, qf, seen, idle, a.c, store);
  } else if constexpr (KG == 2) {
    __shared__ __attribute__((aligned(1024))) int8_t lds0[256 * D];
    __shared__ __attribute__((aligned(1024))) int8_t lds1[256 * D];
    __shared__ __attribute__((aligned(1024))) int8_t lds2[256 * D];
    __shared__ __attribute__((aligned(1024))) int8_t lds3[256 * D];
    __shared__ float ml[2 * 4 * 64];
    if (wave < 4) attend_wide<DT, D, true, 2, 0>(lds0, lds1, ks, a.d, qf, seen, idle, a.c, store, ml, lds2, lds3);
    else attend_wide<DT, D, true, 2, 1>(lds2, lds3, ks, a.d, qf, seen, idle, a.c, store, ml);
  } else {
    __shared__ __attribute__((aligned(1024))) int8_t kl[4 * 64 * D];
    __shared__ __attribute__((aligned(1024))) int8_t vl[4 * 64 * D];
    __shared__ float ml[2 * 4 * 64];
    attend_split<DT, D, 4, true>(kl, vl, ml, ks, a.d, qf, seen, a.c, store);
  }
}

// 128 rows to a workgroup once that makes three for four CUs, below it 32 rows with their keys shared out (1024
// tokens, 16 / 8 heads of 128: 21.8 us shared out, 31.3 with 128 rows; 2048 tokens 49.9 / 52.6). Up to two workgroups
// a CU two groups of waves share out the keys of the 128 rows, where the sequences are long (the host knows their
// mean): a CU's workgroups all run at once then, and the longest row's chain of tiles is what takes the time (2048
// tokens 44.3 us against 52.6 with one group, 4096 97.0 / 111.6; 8192 323 / 318; forty of 100 33.6 / 24.4; 4096 /
// 1500 / 700, 12 heads of 64: 69.5 / 70.0).
template <int DT, int D>
int causal_go(const CausalArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.T * (a.nh / a.nkv), cus = device_cus();
  const int64_t wgs = cdiv(rows, 128) * a.nkv;
  const int kg = 4 * wgs < 3 * cus ? 0 : wgs <= 2 * cus && a.T >= 1024ll * (a.nstarts - 1) ? 2 : 1;
  const unsigned grid = (unsigned)(kg ? wgs : cdiv(rows, 32) * a.nkv);
  if (kg == 0) causal_kernel<DT, D, 0><<<grid, 256, 0, st>>>(a);
  else if (kg == 1) causal_kernel<DT, D, 1><<<grid, 256, 0, st>>>(a);
  else causal_kernel<DT, D, 2><<<grid, 512, 0, st>>>(a);
  return launch_status("attention_causal");
}

// ------------------------------------------------------------------------------ a shared prefix and own keys
struct PrefixArgs {
  const uint16_t *q, *kp, *vp, *kc, *vc;
  int64_t qb, qh, kpt, kph, vpt, vph, kcb, kct, kch, vcb, vct, vch;   // elements from sequence, token, head to the next
  const int32_t* lens;
  int P, S, B, nh, nkv, d;
  int np, no;                 // parts of the prefix and of the own keys; 0 and 0: one workgroup for all keys of (sequence, kv head)
  int pkeys, okeys;           // keys of a part
  int rblocks;                // blocks of rows that the prefix's workgroups take
  float c;
  uint32_t sign;
  float *po, *pml;            // [np + no][B * nh][d] sums, [np + no][B * nh][2] maxima and sums of p
  uint16_t* out;
};

// Workgroups 0 .. nkv rblocks np - 1 take a part of the prefix for the rows (sequence, q head) of a kv head, 32 at a
// time, or 128 (WIDE); the others a part of a sequence's own keys for the q heads of a kv head. np == no == 0: a
// workgroup takes all the keys of its (sequence, kv head) and writes the output itself. KW: waves that share out
// keys. Measured, with the join: 48 rows of 2 / 1 heads of 128 on 8 kv heads over 4096 shared keys and up to 700 own
// ones 26 to 28 us (86 MB, 3.2 TB/s), waves waiting 41% of their time; 24 rows of 8 / 1 heads of 64 on 4 over 100000 43 to 47 us
// (107 MB, 2.4 TB/s), vector units active 49% of the CUs' busy time, MFMA 25%, waves waiting 39% of theirs, and six waves of
// rows in blocks of four.
template <int DT, int D, bool WIDE, int KW>
__global__ __launch_bounds__(KW * 64, 2) void prefix_kernel(PrefixArgs a) {
  static_assert(!WIDE || KW == 4, "four waves in the wide form");
  constexpr int QW = WIDE ? 4 : 1;
  // K and V of the split form; a tile each of the wide one
  __shared__ __attribute__((aligned(1024))) int8_t lds_k[KW * 64 * D];
  __shared__ __attribute__((aligned(1024))) int8_t lds_v[KW * 64 * D];
  __shared__ float ml[2 * KW * 64];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = a.nh / a.nkv;
  // The blocks of rows that read the same keys run on one XCD (workgroups go round the eight), next to each other in
  // time, so that its L2 has the keys for all but the first: items (part, kv head) in eights, their blocks 8 apart.
  const int items = a.np * a.nkv, pre = items * a.rblocks;
  int b0 = blockIdx.x, rb = 0;
  if (b0 < pre) {
    const int eights = items / 8 * 8, whole = eights * a.rblocks, left = items - eights;
    const int i = b0 < whole ? b0 % 8 : (b0 - whole) % left, j = b0 < whole ? b0 / 8 : (b0 - whole) / left;
    rb = j % a.rblocks;
    b0 = (b0 < whole ? j / a.rblocks * 8 : eights) + i;
  } else {
    b0 -= pre;
  }
  const int kvh = b0 % a.nkv, rest = b0 / a.nkv;
  Keys ks;
  ks.kp = 2 * a.kpt;
  ks.vp = 2 * a.vpt;
  ks.kp2 = ks.vp2 = 0;
  ks.k2 = ks.v2 = nullptr;
  ks.n2 = 0;
  const Seen seen = {};
  i32x4 qf[D / 16];
  auto write = [&](int part, int64_t out_row, bool mine) {
    return [=](int chunk, const f32x4& o, float m, float l) {
      const int dim = 8 * chunk + 4 * half;
      if (!mine || dim >= a.d) return;
      if (part < 0) {
        store4<DT>(a.out + out_row * a.d + dim, o, l == 0.0f ? 0.0f : 1.0f / l);
      } else {
        const int64_t at = (int64_t)part * a.B * a.nh + out_row;
        *reinterpret_cast<f32x4*>(a.po + at * a.d + dim) = o;
        if (dim == 0) *reinterpret_cast<float2*>(a.pml + at * 2) = make_float2(m, l);
      }
    };
  };
  if ((int)blockIdx.x < pre) {
    const int part = rest, nrows = a.B * grp;
    const int want = rb * (32 * QW) + 32 * (wave % QW) + (lane & 31), idx = min(want, nrows - 1);
    const int b = idx / grp, head = kvh * grp + idx - b * grp;
    load_q<D>(qf, a.q + b * a.qb + head * a.qh, half, a.d, a.sign);
    const int k0 = part * a.pkeys;
    ks.k = reinterpret_cast<const char*>(a.kp + k0 * a.kpt + kvh * a.kph);
    ks.v = reinterpret_cast<const char*>(a.vp + k0 * a.vpt + kvh * a.vph);
    ks.n = max(0, min(a.pkeys, a.P - k0));
    const auto out = write(part, (int64_t)b * a.nh + head, want < nrows);
    if constexpr (WIDE) {
      attend_wide<DT, D, false, 1, 0>(lds_k, lds_v, ks, a.d, qf, seen, rb * 128 + 32 * wave >= nrows, a.c, out);
    } else {
      attend_split<DT, D, KW, false>(lds_k, lds_v, ml, ks, a.d, qf, seen, a.c, out);
    }
    return;
  }
  // rows: the q heads of one (sequence, kv head), 32 at a time
  const int hb = (grp + 31) / 32, own = rest, parts = max(1, a.no);
  const int b = own / (hb * parts), at = own - b * (hb * parts), part = at / hb, want = (at - part * hb) * 32 + (lane & 31);
  const int head = kvh * grp + min(want, grp - 1);
  load_q<D>(qf, a.q + b * a.qb + head * a.qh, half, a.d, a.sign);
  const int len = min(max(a.lens[b], 0), a.S);
  const char* kc = reinterpret_cast<const char*>(a.kc + b * a.kcb + kvh * a.kch);
  const char* vc = reinterpret_cast<const char*>(a.vc + b * a.vcb + kvh * a.vch);
  const bool all = a.no == 0;
  if (all) {
    ks.k = reinterpret_cast<const char*>(a.kp + kvh * a.kph);
    ks.v = reinterpret_cast<const char*>(a.vp + kvh * a.vph);
    ks.n = a.P;
    ks.k2 = kc;
    ks.v2 = vc;
    ks.kp2 = 2 * a.kct;
    ks.vp2 = 2 * a.vct;
    ks.n2 = len;
  } else {
    const int64_t k0 = (int64_t)part * a.okeys;
    ks.k = kc + k0 * a.kct * 2;
    ks.v = vc + k0 * a.vct * 2;
    ks.kp = 2 * a.kct;
    ks.vp = 2 * a.vct;
    ks.n = (int)max<int64_t>(0, min<int64_t>(a.okeys, len - k0));
  }
  attend_split<DT, D, KW, false>(lds_k, lds_v, ml, ks, a.d, qf, seen, a.c,
                                 write(all ? -1 : a.np + part, (int64_t)b * a.nh + head, want < grp));
}

// The parts of a row joined: a workgroup per row, wave w the parts w, w + 4, .., then the waves in their order; lane
// l dims 2 l, 2 l + 1.
template <int DT>
__global__ __launch_bounds__(256) void prefix_join_kernel(const float* __restrict__ po, const float* __restrict__ pml,
                                                          int parts, int64_t rows, int d, float c,
                                                          uint16_t* __restrict__ out) {
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
  for (int g = 1; g < 4; ++g) {
    l += lv[g];
    x += ov[g][lane].x;
    y += ov[g][lane].y;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint32_t*>(out + row * d + 2 * lane) = pack2<DT>(x * inv, y * inv);
}

// How a call is split. Up to 512 keys for few sequences: a workgroup of eight waves for each (sequence, kv head), one
// launch and nothing to join (4 sequences, 8 kv heads, 264 + 64 keys 9.3 us, in parts 10.7; 64 sequences, 500 + 100:
// 20.5 / 16.5). Else the prefix in parts that make a workgroup a CU in the 32-row form, two in the 128-row one, none
// under 256 keys, and own keys in parts of 128 at least as far as two workgroups a CU take them (1 sequence, 32768
// keys, 8 kv heads: 16 / 32 / 64 parts 29.1 / 28.0 / 30.7 us; 24 x 32 heads over 100000: 32 / 64 / 128 parts 50.2 /
// 46.3 / 53.1; 16 sequences of 1000 own keys, 2 kv heads: 1 / 2 / 4 / 8 parts 16.7 / 13.7 / 11.8 / 11.1).
void prefix_plan(PrefixArgs& a) {
  const int64_t grp = a.nh / a.nkv, hb = cdiv(grp, 32), cus = device_cus(), rows = a.B * grp;
  a.rblocks = (int)cdiv(rows, rows <= 32 ? 32 : 128);
  if ((int64_t)a.P + a.S <= 512 && a.B * hb * a.nkv <= cus) {
    a.np = a.no = 0;
    a.pkeys = a.okeys = 0;
    return;
  }
  const int64_t np = std::max<int64_t>(1, std::min((rows <= 32 ? cus : 2 * cus) / (a.rblocks * a.nkv), cdiv(a.P, 256)));
  const int64_t no = std::max<int64_t>(1, std::min(2 * cus / (a.B * hb * a.nkv), cdiv(a.S, 128)));
  a.pkeys = (int)(cdiv(cdiv(a.P, np), 64) * 64);
  a.okeys = (int)(cdiv(cdiv(a.S, no), 32) * 32);
  a.np = a.P ? (int)cdiv(a.P, a.pkeys) : 0;
  a.no = a.S ? (int)cdiv(a.S, a.okeys) : 1;
}

template <int DT, int D>
int prefix_go(const PrefixArgs& a, hipStream_t st) {
  const int64_t grp = a.nh / a.nkv, hb = cdiv(grp, 32), rows = a.B * grp;
  const int64_t grid = (a.np * (int64_t)a.rblocks + a.B * hb * std::max(1, a.no)) * a.nkv;
  if (a.np + a.no == 0) prefix_kernel<DT, D, false, 8><<<(unsigned)grid, 512, 0, st>>>(a);
  else if (rows <= 32 || a.np == 0) prefix_kernel<DT, D, false, 4><<<(unsigned)grid, 256, 0, st>>>(a);
  else prefix_kernel<DT, D, true, 4><<<(unsigned)grid, 256, 0, st>>>(a);
  if (a.np + a.no > 0)
    prefix_join_kernel<DT><<<(unsigned)((int64_t)a.B * a.nh), 256, 0, st>>>(a.po, a.pml, a.np + a.no, (int64_t)a.B * a.nh, a.d, a.c, a.out);
  return launch_status("attention_prefix");
}

// above 0, so that an unseen key's -inf stays one: scale 0 weighs all keys alike with it
float scale_c(float scale) { return std::max(fabsf(scale) * 1.44269504088896340736f, 1.17549435e-38f); }

// A stride in elements that keeps 16-byte alignment; one from token to token: whose offsets within a tile of 64 keys fit
// 31 bits besides. All others are multiplied in 64 bits.
bool stride_ok(int64_t s, bool token) { return s >= 0 && s % 8 == 0 && (!token || s < (1ll << 24)); }

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_attention_causal(const void* q, const void* k, const void* v, int dtype, const int64_t* strides,
                          const int32_t* starts, int64_t nseq, int64_t T, int nh, int nkv, int d, float scale, void* out,
                          void* stream) {
  XDNA_REQUIRE(dtype == XDNA_BF16 || dtype == XDNA_F16, "dtype must be BF16/F16");
  XDNA_REQUIRE(T >= 0 && nseq >= 0 && nseq < (1ll << 30) && nh >= 1 && nkv >= 1 && nh % nkv == 0, "bad sizes");
  XDNA_REQUIRE(d >= 8 && d <= 128 && d % 8 == 0, "head dims must be a multiple of 8, at most 128");
  if (T == 0) return XDNA_OK;
  XDNA_REQUIRE(q && k && v && strides && starts && out, "null pointer");
  XDNA_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16), "operands must be 16-byte aligned");
  for (int i = 0; i < 6; ++i)
    XDNA_REQUIRE(stride_ok(strides[i], i == 2 || i == 4), "strides must be multiples of 8, from key to key below 2^24");
  XDNA_REQUIRE(strides[2] >= d && strides[4] >= d, "a token's keys and values must not overlap the next one's");
  // 31-bit row numbers, and the launch's threads
  XDNA_REQUIRE(T * (nh / nkv) < (1ll << 31) - 128 && cdiv(T * (nh / nkv), 128) * nkv <= MAX_LAUNCH_THREADS / 256, "too many tokens");
  CausalArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
               strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], starts, (int)nseq + 1, (int)T, nh, nkv, d,
               scale_c(scale), scale < 0.0f ? 0x80008000u : 0u, static_cast<uint16_t*>(out)};
  if (dtype == XDNA_BF16) return d > 64 ? causal_go<XDNA_BF16, 128>(a, as_stream(stream)) : causal_go<XDNA_BF16, 64>(a, as_stream(stream));
  return d > 64 ? causal_go<XDNA_F16, 128>(a, as_stream(stream)) : causal_go<XDNA_F16, 64>(a, as_stream(stream));
}

static bool prefix_sizes_ok(int64_t P, int64_t S, int64_t B, int nh, int nkv, int d) {
  return P >= 0 && S >= 0 && B >= 0 && P < (1ll << 30) && S < (1ll << 30) && nh >= 1 && nkv >= 1 && nh % nkv == 0 &&
         nh < (1 << 16) && B * nh < (1ll << 22) && d >= 8 && d <= 128 && d % 8 == 0;
}

int64_t xdna_attention_prefix_ws_bytes(int64_t P, int64_t S, int64_t B, int nh, int nkv, int d) {
  XDNA_REQUIRE(prefix_sizes_ok(P, S, B, nh, nkv, d), "bad sizes");
  if (B == 0) return 0;
  PrefixArgs a{};
  a.P = (int)P, a.S = (int)S, a.B = (int)B, a.nh = nh, a.nkv = nkv, a.d = d;
  prefix_plan(a);
  return (int64_t)(a.np + a.no) * B * nh * (d + 2) * 4;
}

int xdna_attention_prefix(const void* q, const void* kp, const void* vp, const void* kc, const void* vc, int dtype,
                          const int64_t* strides, const int32_t* lens, int64_t P, int64_t S, int64_t B, int nh, int nkv,
                          int d, float scale, void* out, void* ws, int64_t ws_bytes, void* stream) {
  XDNA_REQUIRE(dtype == XDNA_BF16 || dtype == XDNA_F16, "dtype must be BF16/F16");
  XDNA_REQUIRE(prefix_sizes_ok(P, S, B, nh, nkv, d), "bad sizes (head dims: a multiple of 8, at most 128)");
  if (B == 0) return XDNA_OK;
  XDNA_REQUIRE(q && strides && lens && out && (P == 0 || (kp && vp)) && (S == 0 || (kc && vc)), "null pointer");
  XDNA_REQUIRE(aligned(q, 16) && aligned(kp, 16) && aligned(vp, 16) && aligned(kc, 16) && aligned(vc, 16) && aligned(out, 16),
               "operands must be 16-byte aligned");
  for (int i = 0; i < 12; ++i)
    XDNA_REQUIRE(stride_ok(strides[i], i == 2 || i == 4 || i == 7 || i == 10), "strides must be multiples of 8, from key to key below 2^24");
  XDNA_REQUIRE(strides[2] >= d && strides[4] >= d && strides[7] >= d && strides[10] >= d,
               "a token's keys and values must not overlap the next one's");
  PrefixArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(kp), static_cast<const uint16_t*>(vp),
               static_cast<const uint16_t*>(kc), static_cast<const uint16_t*>(vc), strides[0], strides[1], strides[2],
               strides[3], strides[4], strides[5], strides[6], strides[7], strides[8], strides[9], strides[10], strides[11],
               lens, (int)P, (int)S, (int)B, nh, nkv, d, 0, 0, 0, 0, 0, scale_c(scale), scale < 0.0f ? 0x80008000u : 0u,
               nullptr, nullptr, static_cast<uint16_t*>(out)};
  prefix_plan(a);
  const int64_t rows = B * nh, need = (int64_t)(a.np + a.no) * rows * (d + 2) * 4;
  XDNA_REQUIRE(need == 0 || (ws && aligned(ws, 16) && ws_bytes >= need), "workspace too small or misaligned");
  a.po = static_cast<float*>(ws);
  a.pml = a.po + (int64_t)(a.np + a.no) * rows * d;
  if (dtype == XDNA_BF16) return d > 64 ? prefix_go<XDNA_BF16, 128>(a, as_stream(stream)) : prefix_go<XDNA_BF16, 64>(a, as_stream(stream));
  return d > 64 ? prefix_go<XDNA_F16, 128>(a, as_stream(stream)) : prefix_go<XDNA_F16, 64>(a, as_stream(stream));
}

}  // extern "C"
