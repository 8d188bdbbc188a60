// Logits before a token is chosen, for gfx950 (MI355X): penalties for the tokens of each row's history, a bias, and a
// grammar's mask, in one pass over the logits.
//
//   n[b, v] = how often v is in row b's history
//   x' = n ? (x > 0 ? x / r : x * r) : x;   x' - f n - p (n > 0) + bias;   -inf where the mask's bit is 0
//
// A workgroup has CHUNK tokens of one row's vocabulary: it counts the history's tokens that fall into its chunk in LDS
// (whole numbers: the order of the atomics changes nothing), then streams its chunk. The row's history is read
// once per chunk, from L2: at 4096 tokens 16 KB against the chunk's own 8 to 40 KB of logits, bias and mask, which
// are loaded before the count so that their latency hides behind it. Bound by memory: 64 x 128259 logits in bfloat16
// with a float32 bias each, 67 MB, 16.4 us (4.1 TB/s; a large copy reaches 4.8); 8200 logits 3.6 us, the launch and two
// round trips.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xdna_common.h"
#include "xdna_hip.h"

namespace xdna {
namespace {

// rows start wherever the vocabulary's size puts them
typedef uint32_t u32x4e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4w __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4w __attribute__((ext_vector_type(4), aligned(4)));

struct LogitsArgs {
  const void* x;
  int64_t ld;
  const void* tokens;
  int wide;
  int64_t ldt;
  int L;
  const int32_t* lens;
  const float *rep, *pres, *freq, *bias;
  int64_t ldb;
  const uint8_t* allowed;
  int64_t lda;               // bytes
  void* y;
  int64_t V;
  int chunks;
};

// U groups of E consecutive tokens per thread
template <int DT, int U>
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs a) {
  constexpr int E = 8, CHUNK = 256 * U * E;
  __shared__ __attribute__((aligned(16))) uint32_t cnt[CHUNK];
  const int64_t b = blockIdx.x / a.chunks;
  const int64_t v0 = (int64_t)(blockIdx.x - b * a.chunks) * CHUNK;
  const int n = (int)min<int64_t>(CHUNK, a.V - v0);
  constexpr int esz = DT == XDNA_F32 ? 4 : 2;
  const char* xrow = static_cast<const char*>(a.x) + (b * a.ld + v0) * esz;
  char* yrow = static_cast<char*>(a.y) + (b * a.V + v0) * esz;
  const float* brow = a.bias ? a.bias + b * a.ldb + v0 : nullptr;
  float x[U][E], bias[U][E];
  uint32_t ok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * 256 + threadIdx.x) * E;
    ok[u] = 0xffu;
#pragma unroll
    for (int e = 0; e < E; ++e) x[u][e] = bias[u][e] = 0.0f;
    if (i + E <= n) {
      if constexpr (DT == XDNA_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4w w = *reinterpret_cast<const f32x4w*>(xrow + i * 4 + 16 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][4 * h + e] = w[e];
        }
      } else {
        const u32x4e w = *reinterpret_cast<const u32x4e*>(xrow + i * 2);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
          x[u][e] = DT == XDNA_F16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
      }
      if (brow) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4w w = *reinterpret_cast<const f32x4w*>(brow + i + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) bias[u][4 * h + e] = w[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < n) {
          x[u][e] = load_as_f32<DT>(xrow, i + e);
          if (brow) bias[u][e] = brow[i + e];
        }
    }
    if (a.allowed && i < n) ok[u] = a.allowed[b * a.lda + (v0 + i) / 8];
  }
  const int len = a.tokens ? min(max(a.lens[b], 0), a.L) : 0;     // uniform
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (len) {
    if (a.rep) rep = a.rep[b];
    if (a.pres) pres = a.pres[b];
    if (a.freq) freq = a.freq[b];
    for (int i = threadIdx.x * 4; i < CHUNK; i += 1024) *reinterpret_cast<u32x4*>(cnt + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    auto count = [&](int64_t tok) {
      if (tok >= v0 && tok - v0 < n) atomicAdd(cnt + (tok - v0), 1u);
    };
    if (a.wide) {
      const int64_t* t = static_cast<const int64_t*>(a.tokens) + b * a.ldt;
#pragma unroll 4
      for (int i = threadIdx.x; i < len; i += 256) count(t[i]);
    } else {
      const int32_t* t = static_cast<const int32_t*>(a.tokens) + b * a.ldt;
      const int whole = len & ~3;
#pragma unroll 2
      for (int i = threadIdx.x * 4; i < whole; i += 1024) {
        const u32x4w w = *reinterpret_cast<const u32x4w*>(t + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) count((int32_t)w[e]);
      }
      if (whole + (int)threadIdx.x < len) count(t[whole + threadIdx.x]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (u * 256 + threadIdx.x) * E;
    if (i >= n) break;
    if (len) {
      uint32_t k[E];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(cnt + i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) k[4 * h + e] = w[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (k[e]) {
          float v = x[u][e];
          v = v > 0.0f ? v / rep : v * rep;
          v -= freq * (float)k[e];
          x[u][e] = v - pres;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (brow) x[u][e] += bias[u][e];
      if (!(ok[u] >> e & 1u)) x[u][e] = -INFINITY;
    }
    if (i + E <= n) {
      if constexpr (DT == XDNA_F32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4w w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = x[u][4 * h + e];
          *reinterpret_cast<f32x4w*>(yrow + i * 4 + 16 * h) = w;
        }
      } else {
        u32x4e w;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = DT == XDNA_F16 ? f32x2_to_f16x2_bits(x[u][2 * e], x[u][2 * e + 1])
                                : f32x2_to_bf16x2_bits(x[u][2 * e], x[u][2 * e + 1]);
        *reinterpret_cast<u32x4e*>(yrow + i * 2) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < n) store_from_f32<DT>(yrow, i + e, x[u][e]);
    }
  }
}

template <int DT>
int logits_go(LogitsArgs a, int64_t B, hipStream_t st) {
  const bool wide = B * cdiv(a.V, 4096) >= 2 * (int64_t)device_cus();
  const int64_t chunk = wide ? 4096 : 2048, chunks = cdiv(a.V, chunk);
  a.chunks = (int)chunks;
  const int64_t step = std::max<int64_t>(1, MAX_LAUNCH_THREADS / 256 / chunks);      // rows of a launch
  const int esz = DT == XDNA_F32 ? 4 : 2;
  for (int64_t b = 0; b < B; b += step) {
    LogitsArgs p = a;
    p.x = static_cast<const char*>(a.x) + b * a.ld * esz;
    p.y = static_cast<char*>(a.y) + b * a.V * esz;
    if (a.tokens) {
      p.tokens = static_cast<const char*>(a.tokens) + b * a.ldt * (a.wide ? 8 : 4);
      p.lens = a.lens + b;
    }
    if (a.rep) p.rep = a.rep + b;
    if (a.pres) p.pres = a.pres + b;
    if (a.freq) p.freq = a.freq + b;
    if (a.bias) p.bias = a.bias + b * a.ldb;
    if (a.allowed) p.allowed = a.allowed + b * a.lda;
    const unsigned grid = (unsigned)(std::min(step, B - b) * chunks);
    if (wide) logits_kernel<DT, 2><<<grid, 256, 0, st>>>(p);
    else logits_kernel<DT, 1><<<grid, 256, 0, st>>>(p);
  }
  return launch_status("logits_adjust");
}

}  // namespace
}  // namespace xdna

using namespace xdna;

extern "C" int xdna_logits_adjust(const void* logits, int dtype, int64_t ld, const void* tokens, int wide, int64_t ldt,
                                  int64_t L, const int32_t* lens, const float* repetition, const float* presence,
                                  const float* frequency, const float* bias, int64_t ldb, const int32_t* allowed,
                                  int64_t lda, void* y, int64_t B, int64_t V, void* stream) {
  XDNA_REQUIRE(dtype == XDNA_F32 || dtype == XDNA_BF16 || dtype == XDNA_F16, "dtype must be F32/BF16/F16");
  XDNA_REQUIRE(B >= 0 && V >= 0 && L >= 0 && L < (1ll << 30) && V < (1ll << 31), "bad sizes");
  if (B == 0 || V == 0) return XDNA_OK;
  XDNA_REQUIRE(logits && y && ld >= V, "null pointer, or ld < V");
  XDNA_REQUIRE(!tokens || (lens && ldt >= L), "tokens need lens, and ldt >= L");
  XDNA_REQUIRE(!bias || ldb == 0 || ldb >= V, "ldb must be 0 or at least V");
  XDNA_REQUIRE(!allowed || lda >= cdiv(V, 32), "lda must hold V bits");
  LogitsArgs a{logits, ld, tokens, wide, ldt, (int)L, lens, repetition, presence, frequency, bias, ldb,
               reinterpret_cast<const uint8_t*>(allowed), lda * 4, y, V, 0};
  if (dtype == XDNA_F32) return logits_go<XDNA_F32>(a, B, as_stream(stream));
  if (dtype == XDNA_BF16) return logits_go<XDNA_BF16>(a, B, as_stream(stream));
  return logits_go<XDNA_F16>(a, B, as_stream(stream));
}
