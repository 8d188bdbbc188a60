// A decoder layer's rows between its products, for gfx950 (MI355X), float32, bfloat16 and float16:
//
//   rotary          queries and keys turned to their positions
//   residual_norm   x' = x + s g n(o), y = w x' / rms(x')     (n: the norm of the block's output, or nothing; g: its gate)
//
// Both read and write each value once and compute in float32; what bounds them is memory, and for few rows the launch.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xdna_common.h"
#include "xdna_hip.h"
#include "xdna_rotate.h"

namespace xdna {
namespace {

// ------------------------------------------------------------------------------ rotary
struct RotaryArgs {
  const void* x;
  int64_t xt, xh;             // elements from token to token and from head to head
  const void* positions;
  int wide;
  const double* freqs;
  int half, d, heads, tokens; // tokens of a workgroup
  Divisor by_head, by_token, by_half;           // units of a head, of a token; pairs
  int64_t T;
  float magnitude;
  void* y;
};

constexpr int MAX_TURNS = 1024;

// A workgroup has a few tokens: their angles go to LDS once (256 threads, one each), then every thread takes units of up to 16
// values of their heads, 64 bytes of 16-bit values read and written. 16384 tokens, 24 heads of 128 in bfloat16, 201 MB: 31.4 us
// where the caches hold them (6.3 TB/s), 41.6 with new ones each time (4.8, a large copy's rate); 4 tokens 3.0 us, the
// launch and two round trips.
template <int DT, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  __shared__ float cs[MAX_TURNS], sn[MAX_TURNS];
  const int64_t t0 = (int64_t)blockIdx.x * a.tokens;
  const int n = (int)min<int64_t>(a.tokens, a.T - t0);
  for (int i = threadIdx.x; i < n * a.half; i += 256) {
    const int tok = a.by_half.of(i), j = i - tok * a.half;
    const double pos = a.wide ? (double)static_cast<const int64_t*>(a.positions)[t0 + tok]
                              : (double)static_cast<const int32_t*>(a.positions)[t0 + tok];
    const Turn t = turn_of(pos, a.freqs[j] * QUARTERS);
    cs[i] = t.cos * a.magnitude;
    sn[i] = t.sin * a.magnitude;
  }
  __syncthreads();
  const int per_head = a.by_head.d, per_token = a.by_token.d;
  for (int i = threadIdx.x; i < n * per_token; i += 256) {
    const int tok = a.by_token.of(i), at = i - tok * per_token, head = a.by_head.of(at);
    const Unit u = unit_of<INTER>(at - head * per_head, a.d, a.half);
    const int64_t from = (t0 + tok) * a.xt + head * a.xh, to = ((t0 + tok) * a.heads + head) * a.d;
    float p[8], q[8];
    load_upto8<DT>(a.x, from + u.a, u.na, p);
    load_upto8<DT>(a.x, from + u.b, u.nb, q);
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
    store_upto8<DT>(a.y, to + u.a, u.na, p);
    store_upto8<DT>(a.y, to + u.b, u.nb, q);
  }
}

template <int DT>
int rotary_go(RotaryArgs a, bool interleaved, hipStream_t st) {
  const int most = a.half ? std::max(1, 256 / a.half) : 16;
  a.tokens = (int)std::min<int64_t>(most, std::max<int64_t>(1, a.T / (4 * device_cus())));
  a.by_head = Divisor(units_of(a.d, a.half)), a.by_token = Divisor((int64_t)units_of(a.d, a.half) * a.heads), a.by_half = Divisor(std::max(1, a.half));
  const int64_t grid = cdiv(a.T, a.tokens), step = MAX_LAUNCH_THREADS / 256;
  const int64_t esz = DT == XDNA_F32 ? 4 : 2;
  for (int64_t b = 0; b < grid; b += step) {
    RotaryArgs p = a;
    const int64_t t = b * a.tokens;
    p.x = static_cast<const char*>(a.x) + t * a.xt * esz;
    p.positions = static_cast<const char*>(a.positions) + t * (a.wide ? 8 : 4);
    p.y = static_cast<char*>(a.y) + t * a.heads * a.d * esz;
    p.T = a.T - t;
    const unsigned g = (unsigned)std::min(step, grid - b);
    if (interleaved) rotary_kernel<DT, true><<<g, 256, 0, st>>>(p);
    else rotary_kernel<DT, false><<<g, 256, 0, st>>>(p);
  }
  return launch_status("rotary");
}

// ------------------------------------------------------------------------------ residual_norm
struct NormArgs {
  const void* x;
  const void *o, *gate, *post, *weight;
  int64_t x0, x1, o0, o1, g0, g1, inner;      // where row r starts: r / inner and r % inner times these
  int wdt, pdt;               // types of weight and post
  int64_t row0, rows;         // rows of this launch: row0 .., up to the last
  int width;
  float scale, eps;
  void *sum, *y;
};

// eight values of a weight of any type
__device__ __forceinline__ void load_weight8(const void* w, int dt, int at, int n, float (&x)[8]) {
  if (dt == XDNA_F32) load_upto8<XDNA_F32>(w, at, n, x);
  else if (dt == XDNA_BF16) load_upto8<XDNA_BF16>(w, at, n, x);
  else load_upto8<XDNA_F16>(w, at, n, x);
}

// the sum of v over the L lanes that share a row; all of them get it
template <int L>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int off = (L < 64 ? L : 64) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (L > 64) {
    __syncthreads();                     // the last sum's parts have been read
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) v += part[w];
  }
  return v;
}

// L lanes have a row, C times eight values each in registers between the sums; workgroups of max(L, 256) threads. 8192 rows of 4096,
// a float32 stream, a bfloat16 block with its norm and a gate a row, 470 MB: 93 us (5.0 TB/s; a large copy 4.8); 4 rows of 1024
// 3.3 us, the launch and a round trip. Widths of 513 to 1024 leave half of a row's 256 lanes and more without values: 20000 rows of
// 768 in bfloat16 2.8 TB/s, of 1024 3.9, where 16384 of 1536 have 5.0 and 60000 of 512 5.2.
template <int DTX, int DTO, int L, int C>
__global__ __launch_bounds__(L > 256 ? L : 256) void norm_kernel(NormArgs a) {
  constexpr int THREADS = L > 256 ? L : 256, ROWS = THREADS / L;
  __shared__ float part[THREADS / 64];
  const int lane = threadIdx.x % L;
  const int64_t row = a.row0 + (int64_t)blockIdx.x * ROWS + threadIdx.x / L, r = min(row, a.rows - 1);
  const int64_t ro = r / a.inner, ri = r - ro * a.inner, xr = ro * a.x0 + ri * a.x1, orow = ro * a.o0 + ri * a.o1, gr = ro * a.g0 + ri * a.g1;
  float x[C][8];
  int n[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int at = (c * L + lane) * 8;
    n[c] = max(0, min(8, a.width - at));
    load_upto8<DTX>(a.x, xr + at, n[c], x[c]);
  }
  if (a.o) {
    float o[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) load_upto8<DTO>(a.o, orow + (c * L + lane) * 8, n[c], o[c]);
    if (a.post) {
      float s = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(o[c][e], o[c][e], s);
      const float inv = 1.0f / sqrtf(row_sum<L>(s, part) / (float)a.width + a.eps);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float w[8];
        load_weight8(a.post, a.pdt, (c * L + lane) * 8, n[c], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c][e] *= inv * w[e];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (a.gate) {
        float g[8];
        load_upto8<DTO>(a.gate, gr + (c * L + lane) * 8, n[c], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[c][e] *= g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] = __builtin_fmaf(o[c][e], a.scale, x[c][e]);
      if (row < a.rows) store_upto8<DTX>(a.sum, r * a.width + (c * L + lane) * 8, n[c], x[c]);
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[c][e], x[c][e], s);
  const float inv = 1.0f / sqrtf(row_sum<L>(s, part) / (float)a.width + a.eps);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (a.weight) {
      float w[8];
      load_weight8(a.weight, a.wdt, (c * L + lane) * 8, n[c], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[c][e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[c][e] *= inv;
    if (row < a.rows) store_upto8<DTO>(a.y, r * a.width + (c * L + lane) * 8, n[c], x[c]);
  }
}

constexpr int64_t MAX_WIDTH = 1024 * 8 * 4;

template <int DTX, int DTO, int L, int C>
void norm_launch(NormArgs a, hipStream_t st) {
  constexpr int THREADS = L > 256 ? L : 256, ROWS = THREADS / L;
  constexpr int64_t STEP = MAX_LAUNCH_THREADS / THREADS * ROWS;
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += STEP)
    norm_kernel<DTX, DTO, L, C><<<(unsigned)cdiv(std::min(STEP, a.rows - a.row0), ROWS), THREADS, 0, st>>>(a);
}

template <int DTX, int DTO>
int norm_go(const NormArgs& a, hipStream_t st) {
  if (a.width <= 128) norm_launch<DTX, DTO, 16, 1>(a, st);
  else if (a.width <= 512) norm_launch<DTX, DTO, 64, 1>(a, st);
  else if (a.width <= 2048) norm_launch<DTX, DTO, 256, 1>(a, st);
  else if (a.width <= 4096) norm_launch<DTX, DTO, 256, 2>(a, st);
  else if (a.width <= 8192) norm_launch<DTX, DTO, 256, 4>(a, st);
  else if (a.width <= 16384) norm_launch<DTX, DTO, 1024, 2>(a, st);
  else norm_launch<DTX, DTO, 1024, 4>(a, st);
  return launch_status("residual_norm");
}

bool is_float(int t) { return t == XDNA_F32 || t == XDNA_BF16 || t == XDNA_F16; }

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" {

int xdna_rotary(const void* x, int dtype, int64_t x_token, int64_t x_head, const void* positions, int wide, const double* freqs,
                int64_t half, float magnitude, int interleaved, void* y, int64_t T, int64_t heads, int64_t d, void* stream) {
  XDNA_REQUIRE(is_float(dtype), "dtype must be F32/BF16/F16");
  XDNA_REQUIRE(T >= 0 && heads >= 0 && d >= 0 && heads * d < (1ll << 24) && T < (1ll << 40), "bad sizes");
  XDNA_REQUIRE(half >= 0 && half <= MAX_TURNS && 2 * half <= d, "at most 1024 pairs, and no more than half the dims");
  if (T == 0 || heads == 0 || d == 0) return XDNA_OK;
  XDNA_REQUIRE(x && positions && y && (freqs || half == 0), "null pointer");
  XDNA_REQUIRE(x_token >= 0 && x_head >= 0, "strides must not be negative");
  RotaryArgs a{x, x_token, x_head, positions, wide, freqs, (int)half, (int)d, (int)heads, 0, {}, {}, {}, T, magnitude, y};
  if (dtype == XDNA_F32) return rotary_go<XDNA_F32>(a, interleaved, as_stream(stream));
  if (dtype == XDNA_BF16) return rotary_go<XDNA_BF16>(a, interleaved, as_stream(stream));
  return rotary_go<XDNA_F16>(a, interleaved, as_stream(stream));
}

int xdna_residual_norm(const void* x, int x_dtype, const void* o, int dtype, const void* gate, const int64_t* strides, int64_t inner,
                       const void* post, int post_dtype, const void* weight, int weight_dtype, float scale, float eps, void* sum,
                       void* y, int64_t rows, int64_t width, void* stream) {
  XDNA_REQUIRE(is_float(x_dtype) && (x_dtype == dtype || x_dtype == XDNA_F32) && is_float(dtype),
               "dtype must be F32/BF16/F16, and x's the same or F32");
  XDNA_REQUIRE(is_float(post_dtype) && is_float(weight_dtype), "weights must be F32/BF16/F16");
  XDNA_REQUIRE(rows >= 0 && width >= 0 && width <= MAX_WIDTH && rows < (1ll << 40), "bad sizes (width: at most 32768)");
  if (rows == 0 || width == 0) return XDNA_OK;
  XDNA_REQUIRE(x && y && strides && (!o || sum) && (o || (!gate && !post)), "null pointer, or a gate or norm of nothing");
  XDNA_REQUIRE(inner >= 1, "inner must be at least 1");
  for (int i = 0; i < 6; ++i) XDNA_REQUIRE(strides[i] >= 0, "strides must not be negative");
  NormArgs a{x, o, gate, post, weight, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], inner, weight_dtype,
             post_dtype, 0, rows, (int)width, scale, eps, sum, y};
  hipStream_t st = as_stream(stream);
  if (x_dtype == XDNA_F32) {
    if (dtype == XDNA_F32) return norm_go<XDNA_F32, XDNA_F32>(a, st);
    return dtype == XDNA_BF16 ? norm_go<XDNA_F32, XDNA_BF16>(a, st) : norm_go<XDNA_F32, XDNA_F16>(a, st);
  }
  return dtype == XDNA_BF16 ? norm_go<XDNA_BF16, XDNA_BF16>(a, st) : norm_go<XDNA_F16, XDNA_F16>(a, st);
}

}  // extern "C"
