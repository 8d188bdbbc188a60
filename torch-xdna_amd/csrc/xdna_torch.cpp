// The language model operators' GPU kernels of torch.ops.xdna.*, from the dispatcher to the library's C ABI without a
// trip through Python: the checks, the output, the workspace, the stream. A small call is all host time: one row
// through 1024 x 4096 4-bit weights takes 4.5 us on the GPU, and took 15 to issue from Python.
//
// Registered for CUDA (the work), AutogradCUDA and AutogradCPU (nothing but the dispatch below them; outputs of inputs
// that need a gradient get a node that raises when it is asked for, and a tangent raises at once). Python's registrations of the ops give them their schemas,
// their host kernels and their shapes under fake tensors.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <atomic>
#include <chrono>
#include <cmath>
#include <vector>

#include "xdna_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------------------ what report() shows
struct Counts {
  std::atomic<int64_t> calls{0}, macs{0}, launches{0}, nanoseconds{0};
} counts;

struct Record {
  std::chrono::steady_clock::time_point since = std::chrono::steady_clock::now();
  int64_t macs = 0;
  bool launched = false;
  ~Record() {
    counts.calls.fetch_add(1, std::memory_order_relaxed);
    counts.macs.fetch_add(macs, std::memory_order_relaxed);
    if (launched) counts.launches.fetch_add(1, std::memory_order_relaxed);
    counts.nanoseconds.fetch_add((std::chrono::steady_clock::now() - since).count(), std::memory_order_relaxed);
  }
};

// ------------------------------------------------------------------------------ arguments
int code(at::ScalarType t) { return t == at::kFloat ? XDNA_F32 : t == at::kBFloat16 ? XDNA_BF16 : t == at::kHalf ? XDNA_F16 : -1; }

void check_float(const char* name, const Tensor& t) {
  TORCH_CHECK_TYPE(code(t.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}

void check_device(const Tensor& x, const Tensor& t) {
  TORCH_CHECK_VALUE(t.device() == x.device(), "all tensors must be on one device, got ", x.device(), " and ", t.device());
}
void check_device(const Tensor& x, const OptTensor& t) {
  if (t) check_device(x, *t);
}

void check_shape(const char* name, const Tensor& t, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}

void check_whole(const char* name, const Tensor& t, int64_t dims, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dims, name, " must be ", what, ", got ", t.sizes());
}

const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

void done(int status, const char* what) {
  // sizes past what the kernels' indexes reach: wrong arguments like those that are refused above
  TORCH_CHECK_VALUE(status != XDNA_EINVAL, "xdna ", what, ": ", xdna_last_error());
  TORCH_CHECK(status == 0, "xdna ", what, " failed (status ", status, "): ", xdna_last_error());
}

struct Launch {       // the tensors' device made current, and its current stream
  c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard;
  void* stream;
  explicit Launch(const Tensor& x)
      : guard(x.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream()) {}
};

Tensor bytes(const Tensor& x, int64_t n) { return at::empty({n}, x.options().dtype(at::kByte)); }

// ------------------------------------------------------------------------------ linear_w4
Tensor linear_w4(const Tensor& x, const Tensor& qweight, const Tensor& scales, const OptTensor& zeros, const OptTensor& bias) {
  Record rec;
  check_float("x", x);
  check_float("scales", scales);
  TORCH_CHECK_TYPE(qweight.scalar_type() == at::kByte && (!zeros || zeros->scalar_type() == at::kByte),
                   "qweight and zeros must be uint8");
  TORCH_CHECK_VALUE(x.dim() >= 1 && qweight.dim() == 2 && scales.dim() == 2,
                    "linear_w4 takes x [..., K], qweight [N, K / 2] and scales [N, K / G]");
  const int64_t n = qweight.size(0), k = 2 * qweight.size(1), groups = scales.size(1);
  TORCH_CHECK_VALUE(k && groups && x.size(-1) == k && scales.size(0) == n && k % groups == 0 && k / groups % 32 == 0, "linear_w4: x ",
                    x.sizes(), ", qweight ", qweight.sizes(), " and scales ", scales.sizes(),
                    " do not fit (K / G groups, G a multiple of 32)");
  if (zeros) check_shape("zeros", *zeros, scales.sizes());
  if (bias) {
    check_float("bias", *bias);
    check_shape("bias", *bias, {n});
  }
  TORCH_CHECK_VALUE(qweight.is_contiguous() && scales.is_contiguous() && (!zeros || zeros->is_contiguous()),
                    "linear_w4: qweight, scales and zeros must be contiguous");
  check_device(x, qweight), check_device(x, scales), check_device(x, zeros), check_device(x, bias);
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(qweight.const_data_ptr()) % 16 == 0, "linear_w4: qweight must be 16-byte aligned");
  const Launch go(x);
  at::DimVector shape(x.sizes());
  shape.back() = n;
  Tensor y = at::empty(shape, x.options());
  const int64_t m = x.numel() / k;
  rec.macs = m * n * k;
  if (m == 0 || n == 0) return y;
  Tensor x2 = x.dim() == 2 ? x : x.reshape({m, k});
  const auto fits = [&](const Tensor& t) {
    return t.stride(1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 &&
           (m == 1 || t.stride(0) * t.element_size() % 16 == 0);
  };
  // rows that overlap, or lie further apart than the kernels' offsets reach, are read from a copy
  if (!fits(x2) || (m > 1 && (x2.stride(0) < k || x2.stride(0) > (1 << 22)))) x2 = x2.clone(at::MemoryFormat::Contiguous);
  const int xc = code(x.scalar_type());
  const Tensor b = bias ? bias->contiguous() : Tensor();
  const int64_t need = xdna_linear_w4_ws_bytes(xc, m, n, k);
  const Tensor ws = need > 0 ? bytes(x, need) : Tensor();
  done(xdna_linear_w4_ws(x2.const_data_ptr(), xc, m > 1 ? x2.stride(0) : k, qweight.const_data_ptr(), scales.const_data_ptr(),
                         code(scales.scalar_type()), ptr(zeros), bias ? b.const_data_ptr() : nullptr,
                         bias ? code(b.scalar_type()) : XDNA_F32, y.mutable_data_ptr(), m, n, k, k / groups,
                         need > 0 ? ws.mutable_data_ptr() : nullptr, need > 0 ? need : 0, go.stream),
       "linear_w4");
  rec.launched = true;
  return y;
}

// ------------------------------------------------------------------------------ attention
double attention_args(const char* name, const Tensor& q, std::initializer_list<const Tensor*> kvs, std::optional<double> scale) {
  TORCH_CHECK_TYPE(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, name, " takes bfloat16 or float16, got ",
                   q.scalar_type());
  for (const Tensor* t : kvs)
    TORCH_CHECK_TYPE(t->scalar_type() == q.scalar_type(), name, ": q, keys and values must be of one dtype, got ", q.scalar_type(),
                     " and ", t->scalar_type());
  const int64_t d = q.size(-1), nkv = (*kvs.begin())->size(-2);
  TORCH_CHECK_VALUE(d >= 8 && d <= 128 && d % 8 == 0, name, ": head dims must be a multiple of 8, at most 128, got ", d);
  TORCH_CHECK_VALUE(nkv && q.size(-2) && q.size(-2) % nkv == 0, name, ": ", q.size(-2), " q heads do not share ", nkv,
                    " key heads evenly");
  return scale ? *scale : 1.0 / std::sqrt((double)d);
}

// t [.., heads, d] as the library reads it, and its strides but the last's (of dims of one, any will do): itself
// where the last dim is dense, it starts on 16 bytes, no token's values overlap the next one's, the strides are
// multiples of 8 and that of tokens fits the kernels' offsets; else a copy.
Tensor heads(Tensor t, int64_t* st) {
  const int64_t n = t.dim() - 1, d = t.size(n);
  for (int pass = 0; pass < 2; ++pass) {
    bool ok = t.stride(n) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int64_t i = 0; i < n; ++i) {
      st[i] = t.size(i) == 1 ? d : t.stride(i);
      ok = ok && st[i] % 8 == 0;
    }
    if (ok && st[n - 2] >= d && st[n - 2] < (1 << 24)) break;
    t = t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

Tensor attention_causal(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts, std::optional<double> scale_) {
  Record rec;
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes(),
                    "attention_causal takes q [T, H, D] and k, v [T, KV, D], got ", q.sizes(), ", ", k.sizes(), " and ", v.sizes());
  const int64_t t = q.size(0), h = q.size(1), d = q.size(2), nkv = k.size(1);
  check_shape("k", k, {t, nkv, d});
  const double scale = attention_args("attention_causal", q, {&k, &v}, scale_);
  check_whole("starts", starts, 1, "[S + 1]");
  TORCH_CHECK_VALUE(starts.size(0) >= 1, "starts must be [S + 1], got []");
  check_device(q, k), check_device(q, v), check_device(q, starts);
  rec.macs = t * t * h * d;              // at most: the sequences' lengths are not read
  const Launch go(q);
  Tensor out = at::empty({t, h, d}, q.options());
  if (t == 0) return out;
  int64_t st[6];
  const Tensor qs = heads(q, st), ks = heads(k, st + 2), vs = heads(v, st + 4), ss = starts.contiguous();
  done(xdna_attention_causal(qs.const_data_ptr(), ks.const_data_ptr(), vs.const_data_ptr(), code(q.scalar_type()), st,
                             ss.const_data_ptr<int32_t>(), ss.size(0) - 1, t, (int)h, (int)nkv, (int)d, (float)scale,
                             out.mutable_data_ptr(), go.stream),
       "attention_causal");
  rec.launched = true;
  return out;
}

Tensor attention_prefix(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& kc, const Tensor& vc, const Tensor& lens,
                        std::optional<double> scale_) {
  Record rec;
  TORCH_CHECK_VALUE(q.dim() == 3 && kp.dim() == 3 && kc.dim() == 4 && vp.sizes() == kp.sizes() && vc.sizes() == kc.sizes(),
                    "attention_prefix takes q [B, H, D], kp, vp [P, KV, D] and kc, vc [B, S, KV, D], got ", q.sizes(), ", ", kp.sizes(),
                    ", ", vp.sizes(), ", ", kc.sizes(), " and ", vc.sizes());
  const int64_t b = q.size(0), h = q.size(1), d = q.size(2), p = kp.size(0), nkv = kp.size(1), s = kc.size(1);
  check_shape("kp", kp, {p, nkv, d});
  check_shape("kc", kc, {b, s, nkv, d});
  const double scale = attention_args("attention_prefix", q, {&kp, &vp, &kc, &vc}, scale_);
  check_whole("lens", lens, 1, "[B]");
  check_shape("lens", lens, {b});
  check_device(q, kp), check_device(q, vp), check_device(q, kc), check_device(q, vc), check_device(q, lens);
  rec.macs = 2 * b * (p + s) * h * d;
  const Launch go(q);
  Tensor out = at::empty({b, h, d}, q.options());
  if (b == 0) return out;
  int64_t st[12];
  const Tensor qs = heads(q, st), kps = heads(kp, st + 2), vps = heads(vp, st + 4), kcs = heads(kc, st + 6), vcs = heads(vc, st + 9),
               ls = lens.contiguous();
  const int64_t need = xdna_attention_prefix_ws_bytes(p, s, b, (int)h, (int)nkv, (int)d);
  const Tensor ws = need > 0 ? bytes(q, need) : Tensor();
  done(need < 0 ? (int)need
                : xdna_attention_prefix(qs.const_data_ptr(), kps.const_data_ptr(), vps.const_data_ptr(), kcs.const_data_ptr(),
                                        vcs.const_data_ptr(), code(q.scalar_type()), st, ls.const_data_ptr<int32_t>(), p, s, b, (int)h,
                                        (int)nkv, (int)d, (float)scale, out.mutable_data_ptr(),
                                        need > 0 ? ws.mutable_data_ptr() : nullptr, need, go.stream),
       "attention_prefix");
  rec.launched = true;
  return out;
}

// ------------------------------------------------------------------------------ logits_adjust
Tensor logits_adjust(const Tensor& logits, const OptTensor& tokens, const OptTensor& lens, const OptTensor& repetition,
                     const OptTensor& presence, const OptTensor& frequency, const OptTensor& bias, const OptTensor& allowed) {
  Record rec;
  check_float("logits", logits);
  TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [B, V], got ", logits.sizes());
  const int64_t b = logits.size(0), v = logits.size(1);
  TORCH_CHECK_VALUE(tokens.has_value() == lens.has_value(), "logits_adjust: tokens and lens go together");
  if (tokens) {
    TORCH_CHECK_TYPE(tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong, "tokens must be int32 or int64, got ",
                     tokens->scalar_type());
    TORCH_CHECK_VALUE(tokens->dim() == 2 && tokens->size(0) == b, "tokens must be [B, L], got ", tokens->sizes());
    check_whole("lens", *lens, 1, "[B]");
    check_shape("lens", *lens, {b});
  }
  const auto values = [&](const char* name, const OptTensor& t, at::IntArrayRef shape) {
    if (!t) return;
    TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ", t->scalar_type());
    check_shape(name, *t, shape);
  };
  values("repetition", repetition, {b});
  values("presence", presence, {b});
  values("frequency", frequency, {b});
  if (bias && bias->dim() == 1) values("bias", bias, {v});
  else values("bias", bias, {b, v});
  if (allowed) {
    check_whole("allowed", *allowed, 2, "[B, ceil(V / 32)]");
    check_shape("allowed", *allowed, {b, (v + 31) / 32});
  }
  for (const OptTensor* t : {&tokens, &lens, &repetition, &presence, &frequency, &bias, &allowed}) check_device(logits, *t);
  const Launch go(logits);
  Tensor y = at::empty({b, v}, logits.options());
  if (b == 0 || v == 0) return y;
  // rows that are dense and apart, and the elements from one to the next
  const auto rows = [](const Tensor& t) {
    const int64_t w = t.size(1);
    return (t.stride(1) == 1 || w == 1) && (t.size(0) == 1 || t.stride(0) >= w) ? t : t.contiguous();
  };
  const auto ld = [](const Tensor& t) { return !t.defined() ? 0 : t.size(0) == 1 ? t.size(1) : t.stride(0); };
  const auto flat = [](const OptTensor& t) { return t ? t->contiguous() : Tensor(); };
  const Tensor x = rows(logits), tk = tokens ? rows(*tokens) : Tensor(), al = allowed ? rows(*allowed) : Tensor(), ls = flat(lens),
               rp = flat(repetition), pr = flat(presence), fr = flat(frequency);
  Tensor bs;
  int64_t ldb = 0;
  if (bias) {
    // one bias for all rows, or an expanded one, is read as one row
    const bool one = bias->dim() == 1 || b == 1 || bias->stride(0) == 0;
    bs = !one ? rows(*bias) : bias->dim() == 1 ? bias->contiguous() : bias->select(0, 0).contiguous();
    ldb = one ? 0 : ld(bs);
  }
  const auto at = [](const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; };
  done(xdna_logits_adjust(x.const_data_ptr(), code(x.scalar_type()), ld(x), at(tk), tokens && tk.scalar_type() == at::kLong, ld(tk),
                          tokens ? tk.size(1) : 0, (const int32_t*)at(ls), (const float*)at(rp), (const float*)at(pr),
                          (const float*)at(fr), (const float*)at(bs), ldb, (const int32_t*)at(al), ld(al), y.mutable_data_ptr(), b, v,
                          go.stream),
       "logits_adjust");
  rec.launched = true;
  return y;
}

// ------------------------------------------------------------------------------ rotary
void check_freqs(const Tensor& freqs, int64_t d) {
  TORCH_CHECK_TYPE(freqs.scalar_type() == at::kDouble, "freqs must be float64, got ", freqs.scalar_type());
  TORCH_CHECK_VALUE(freqs.dim() == 1 && 2 * freqs.size(0) <= d, "freqs must be [R / 2] with R at most the heads' ", d, " dims, got ",
                    freqs.sizes());
}

// t whose last dim is dense and whose strides are not negative: itself, or a copy
Tensor dense(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.clone(at::MemoryFormat::Contiguous); }

Tensor rotary(const Tensor& x, const Tensor& positions, const Tensor& freqs, double magnitude, bool interleaved) {
  Record rec;
  check_float("x", x);
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must be int32 or int64, got ",
                   positions.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 3, "rotary takes x [.., H, D], got ", x.sizes());
  const int64_t d = x.size(-1), h = x.size(-2);
  check_freqs(freqs, d);
  TORCH_CHECK_VALUE(freqs.size(0) <= 1024, "rotary turns at most 1024 pairs, got ", freqs.size(0));
  check_shape("positions", positions, x.sizes().slice(0, x.dim() - 2));
  check_device(x, positions), check_device(x, freqs);
  const Launch go(x);
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return y;
  const int64_t t = x.numel() / (h * d);
  rec.macs = 2 * t * h * freqs.size(0);
  const Tensor xs = dense(x.dim() == 3 ? x : x.reshape({t, h, d})), ps = positions.contiguous(), fs = freqs.contiguous();
  done(xdna_rotary(xs.const_data_ptr(), code(x.scalar_type()), xs.stride(0), xs.stride(1), ps.const_data_ptr(),
                   ps.scalar_type() == at::kLong, fs.const_data_ptr<double>(), fs.size(0), (float)magnitude, interleaved,
                   y.mutable_data_ptr(), t, h, d, go.stream),
       "rotary");
  rec.launched = true;
  return y;
}

// ------------------------------------------------------------------------------ residual_norm
std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& o, const OptTensor& weight, const OptTensor& post,
                                         const OptTensor& gate, double scale, double eps) {
  Record rec;
  check_float("x", x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) <= 32768, "residual_norm takes x [.., W] with W at most 32768, got ", x.sizes());
  TORCH_CHECK_VALUE(o || (!post && !gate), "residual_norm: post and gate need o");
  const int64_t w = x.size(-1);
  if (o) {
    check_float("o", *o);
    TORCH_CHECK_TYPE(x.scalar_type() == o->scalar_type() || x.scalar_type() == at::kFloat, "x must be of o's type or float32, got ",
                     x.scalar_type(), " and ", o->scalar_type());
    check_shape("o", *o, x.sizes());
  }
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor*>{"weight", &weight}, {"post", &post}})
    if (*t) {
      check_float(name, **t);
      check_shape(name, **t, {w});
    }
  if (gate) {
    TORCH_CHECK_TYPE(gate->scalar_type() == o->scalar_type(), "gate must be of o's type, got ", gate->scalar_type());
    TORCH_CHECK_VALUE(gate->sizes() == x.sizes() || (gate->dim() == 1 && gate->size(0) == w), "gate must have shape ", x.sizes(), " or [",
                      w, "], got ", gate->sizes());
  }
  for (const OptTensor* t : {&o, &weight, &post, &gate}) check_device(x, *t);
  const Launch go(x);
  const auto ot = o ? o->options() : x.options();
  Tensor sum = o ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options()), y = at::empty(x.sizes(), ot);
  if (x.numel() == 0) return {sum, y};
  const int64_t rows = x.numel() / w, inner = x.dim() >= 2 ? x.size(-2) : 1;
  // as [outer, inner, W]: where that is no view of it, or the last dim is not dense, a copy
  int64_t st[6] = {0, 0, 0, 0, 0, 0};
  const auto shaped = [&](const Tensor& t, int64_t* s) {
    const Tensor v = dense(t.dim() == 3 ? t : t.reshape({rows / inner, inner, w}));
    s[0] = v.stride(0), s[1] = v.stride(1);
    return v;
  };
  const Tensor xs = shaped(x, st), os = o ? shaped(*o, st + 2) : Tensor();
  Tensor gs;
  if (gate && gate->dim() == 1 && x.dim() != 1) gs = gate->contiguous();
  else if (gate) gs = shaped(*gate, st + 4);
  const Tensor ws = weight ? weight->contiguous() : Tensor(), ps = post ? post->contiguous() : Tensor();
  const auto at = [](const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; };
  const auto type = [](const Tensor& t) { return t.defined() ? code(t.scalar_type()) : XDNA_F32; };
  done(xdna_residual_norm(at(xs), type(xs), at(os), code(y.scalar_type()), at(gs), st, inner, at(ps), type(ps), at(ws), type(ws),
                          (float)scale, (float)eps, o ? sum.mutable_data_ptr() : nullptr, y.mutable_data_ptr(), rows, w, go.stream),
       "residual_norm");
  rec.launched = true;
  return {sum, y};
}

// ------------------------------------------------------------------------------ the 8-bit cache
struct CacheSizes {
  int64_t b, p, pages, kv, g, d, r;
};

CacheSizes check_cache(const char* name, const Tensor& x, const Tensor& kpages, const Tensor& vpages, const Tensor& kscales,
                       const Tensor& vscales, const Tensor& ktail, const Tensor& vtail, const Tensor& table, const Tensor& lens) {
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name, " takes bfloat16 or float16, got ",
                   x.scalar_type());
  TORCH_CHECK_TYPE(kpages.scalar_type() == at::kChar && vpages.scalar_type() == at::kChar, "kpages and vpages must be int8");
  TORCH_CHECK_TYPE(kscales.scalar_type() == at::kFloat && vscales.scalar_type() == at::kFloat, "kscales and vscales must be float32");
  TORCH_CHECK_TYPE(ktail.scalar_type() == x.scalar_type() && vtail.scalar_type() == x.scalar_type(), "ktail and vtail must be ",
                   x.scalar_type(), ", got ", ktail.scalar_type(), " and ", vtail.scalar_type());
  TORCH_CHECK_VALUE(kpages.dim() == 4 && ktail.dim() == 4, "kpages must be [pages, KV, G, D] and ktail [B, KV, R, D], got ", kpages.sizes(),
                    " and ", ktail.sizes());
  check_whole("table", table, 2, "[B, P]");
  const CacheSizes s{ktail.size(0), table.size(1), kpages.size(0), kpages.size(1), kpages.size(2), kpages.size(3), ktail.size(2)};
  TORCH_CHECK_VALUE(s.g == 16 || s.g == 32 || s.g == 64 || s.g == 128, name, ": pages hold 16, 32, 64 or 128 tokens, got ", s.g);
  TORCH_CHECK_VALUE(s.d >= 16 && s.d <= 128 && s.d % 16 == 0, name, ": head dims must be a multiple of 16, at most 128, got ", s.d);
  TORCH_CHECK_VALUE(s.r >= s.g && s.r % s.g == 0 && s.r < 65536, name, ": R must be a multiple of ", s.g, " below 65536, got ", s.r);
  TORCH_CHECK_VALUE(s.kv >= 1, name, ": no key heads");
  TORCH_CHECK_VALUE(s.pages >= 1 || s.p == 0, name, ": a table of no pages");
  check_shape("vpages", vpages, {s.pages, s.kv, s.d, s.g});
  check_shape("kscales", kscales, {s.pages, s.kv});
  check_shape("vscales", vscales, {s.pages, s.kv});
  check_shape("ktail", ktail, {s.b, s.kv, s.r, s.d});
  check_shape("vtail", vtail, {s.b, s.kv, s.d, s.r});
  check_shape("table", table, {s.b, s.p});
  check_whole("lens", lens, 1, "[B]");
  check_shape("lens", lens, {s.b});
  for (const Tensor* t : {&kpages, &vpages, &kscales, &vscales, &ktail, &vtail}) {
    TORCH_CHECK_VALUE(t->is_contiguous() && reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0, name,
                      ": the cache must be contiguous and 16-byte aligned");
    check_device(x, *t);
  }
  check_device(x, table), check_device(x, lens);
  return s;
}

Tensor cache_append(const Tensor& k, const Tensor& v, const Tensor& kpages, const Tensor& vpages, const Tensor& kscales,
                    const Tensor& vscales, const Tensor& ktail, const Tensor& vtail, const Tensor& table, const Tensor& lens,
                    const OptTensor& starts, const OptTensor& q, const OptTensor& freqs, double magnitude, bool interleaved) {
  Record rec;
  const CacheSizes s = check_cache("cache_append", k, kpages, vpages, kscales, vscales, ktail, vtail, table, lens);
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type() && (!q || q->scalar_type() == k.scalar_type()),
                   "cache_append: q, k and v must be of one dtype");
  TORCH_CHECK_VALUE(k.dim() == 3 && k.sizes() == v.sizes(), "cache_append takes k, v [T, KV, D], got ", k.sizes(), " and ", v.sizes());
  const int64_t t = k.size(0);
  check_shape("k", k, {t, s.kv, s.d});
  if (starts) {
    check_whole("starts", *starts, 1, "[B + 1]");
    check_shape("starts", *starts, {s.b + 1});
  } else {
    TORCH_CHECK_VALUE(s.b ? t % s.b == 0 : t == 0, "cache_append: ", t, " tokens are not the same number for each of ", s.b,
                      " texts; starts must say which are whose");
  }
  if (freqs) check_freqs(*freqs, s.d);
  if (q) {
    TORCH_CHECK_VALUE(freqs, "cache_append: q turns with freqs, and there are none");
    TORCH_CHECK_VALUE(q->dim() == 3 && q->size(1) >= 1 && q->size(1) < 65536, "q must be [T, H, D], H at most 65535, got ", q->sizes());
    check_shape("q", *q, {t, q->size(1), s.d});
  }
  check_device(k, v), check_device(k, starts), check_device(k, q), check_device(k, freqs);
  const Launch go(k);
  Tensor out = q ? at::empty(q->sizes(), k.options()) : at::empty({0}, k.options());
  if (t == 0) return out;
  if (s.b == 0) return out.zero_();
  rec.macs = 2 * t * s.kv * s.d;
  const Tensor ks = dense(k), vs = dense(v), qs = q ? dense(*q) : Tensor(), ls = lens.contiguous(), fs = freqs ? freqs->contiguous() : Tensor(),
               ss = starts ? starts->contiguous() : Tensor(), ts = dense(table);
  const int64_t st[6] = {ks.stride(0), ks.stride(1), vs.stride(0), vs.stride(1), q ? qs.stride(0) : 0, q ? qs.stride(1) : 0};
  done(xdna_cache_append(ks.const_data_ptr(), vs.const_data_ptr(), code(k.scalar_type()), st, kpages.mutable_data_ptr(),
                         vpages.mutable_data_ptr(), (float*)kscales.mutable_data_ptr(), (float*)vscales.mutable_data_ptr(),
                         ktail.mutable_data_ptr(), vtail.mutable_data_ptr(), ts.const_data_ptr<int32_t>(), ts.stride(0),
                         ls.const_data_ptr<int32_t>(), starts ? ss.const_data_ptr<int32_t>() : nullptr,
                         q ? qs.const_data_ptr() : nullptr, freqs ? fs.const_data_ptr<double>() : nullptr, freqs ? fs.size(0) : 0,
                         (float)magnitude, interleaved, q ? out.mutable_data_ptr() : nullptr, t, s.b, s.p, s.pages, s.g, s.r,
                         q ? (int)q->size(1) : 0, (int)s.kv, (int)s.d, go.stream),
       "cache_append");
  rec.launched = true;
  return out;
}

Tensor attention_cache(const Tensor& q, const Tensor& kpages, const Tensor& vpages, const Tensor& kscales, const Tensor& vscales,
                       const Tensor& ktail, const Tensor& vtail, const Tensor& table, const Tensor& lens, std::optional<double> scale_) {
  Record rec;
  const CacheSizes s = check_cache("attention_cache", q, kpages, vpages, kscales, vscales, ktail, vtail, table, lens);
  TORCH_CHECK_VALUE(q.dim() == 4, "attention_cache takes q [B, N, H, D], got ", q.sizes());
  const int64_t n = q.size(1), h = q.size(2);
  check_shape("q", q, {s.b, n, h, s.d});
  TORCH_CHECK_VALUE(h && h < 65536 && h % s.kv == 0, "attention_cache: ", h, " q heads, at most 65535, do not share ", s.kv,
                    " key heads evenly");
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)s.d);
  const Launch go(q);
  Tensor out = at::empty(q.sizes(), q.options());
  if (s.b == 0 || n == 0) return out;
  rec.macs = 2 * s.b * n * h * s.d * s.p * s.g;        // at most: the lengths are not read
  int64_t st[3];
  const Tensor qs = heads(q, st), ls = lens.contiguous(), ts = dense(table);
  const int64_t need = xdna_attention_cache_ws_bytes(s.b, n, (int)h, (int)s.kv, (int)s.d, s.p, s.g);
  const Tensor ws = need > 0 ? bytes(q, need) : Tensor();
  done(need < 0 ? (int)need
                : xdna_attention_cache(qs.const_data_ptr(), code(q.scalar_type()), st, kpages.const_data_ptr(), vpages.const_data_ptr(),
                                       kscales.const_data_ptr<float>(), vscales.const_data_ptr<float>(), ktail.const_data_ptr(),
                                       vtail.const_data_ptr(), ts.const_data_ptr<int32_t>(), ts.stride(0), ls.const_data_ptr<int32_t>(),
                                       s.b, n, s.p, s.pages, s.g, s.r, (int)h, (int)s.kv, (int)s.d, (float)scale, out.mutable_data_ptr(),
                                       need > 0 ? ws.mutable_data_ptr() : nullptr, need, go.stream),
       "attention_cache");
  rec.launched = true;
  return out;
}

// ------------------------------------------------------------------------------ autograd
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <class T>
bool has_tangent(const T&) { return false; }
bool needs_grad(const Tensor& t) { return t.requires_grad(); }
bool needs_grad(const OptTensor& t) { return t && t->requires_grad(); }
template <class T>
bool needs_grad(const T&) { return false; }
void take(std::vector<Tensor>& v, const Tensor& t) { v.push_back(t); }
void take(std::vector<Tensor>& v, const OptTensor& t) { if (t) v.push_back(*t); }
template <class T>
void take(std::vector<Tensor>&, const T&) {}

void each(const Tensor& t, const std::shared_ptr<torch::autograd::Node>& node) { torch::autograd::set_history(t, node); }
void each(const std::tuple<Tensor, Tensor>& t, const std::shared_ptr<torch::autograd::Node>& node) {
  for (const Tensor& x : {std::get<0>(t), std::get<1>(t)}) torch::autograd::set_history(x, node);
}

template <class F>
struct Below;
template <class R, class... A>
struct Below<R(A...)> {
  template <int OP>
  static R call(c10::DispatchKeySet ks, A... a);
};

constexpr const char* NAMES[] = {"xdna::linear_w4", "xdna::attention_causal", "xdna::attention_prefix", "xdna::logits_adjust",
                                 "xdna::rotary", "xdna::residual_norm", "xdna::attention_cache", "xdna::cache_append"};
constexpr int APPEND = 7;      // writes to its arguments 2 .. 7

template <class... A>
void written(const A&... a) {
  const std::tuple<const A&...> t(a...);
  for (const Tensor* x : {&std::get<2>(t), &std::get<3>(t), &std::get<4>(t), &std::get<5>(t), &std::get<6>(t), &std::get<7>(t)})
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
}

template <class R, class... A>
template <int OP>
R Below<R(A...)>::call(c10::DispatchKeySet ks, A... a) {
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(NAMES[OP], "").typed<R(A...)>();
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(a) || ...), NAMES[OP], " has no forward-mode derivative");
  const bool grad = at::GradMode::is_enabled() && (needs_grad(a) || ...);
  // what it writes would hold values of such inputs, with no way back to them
  if (OP == APPEND) TORCH_CHECK_NOT_IMPLEMENTED(!grad, NAMES[OP], " has no derivative, and an input needs a gradient: call it under torch.no_grad()");
  R out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    // past ADInplaceOrView too, which for an op that writes is a kernel in Python: what it would count, written() counts
    out = op.redispatch(ks & c10::after_ADInplaceOrView_keyset, a...);
  }
  if constexpr (OP == APPEND) written(a...);
  if (grad) {
    std::vector<Tensor> in;
    (take(in, a), ...);
    auto node = std::shared_ptr<torch::autograd::NotImplemented>(new torch::autograd::NotImplemented(NAMES[OP]), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(in));
    each(out, node);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(xdna, CUDA, m) {
  m.impl("linear_w4", linear_w4);
  m.impl("attention_causal", attention_causal);
  m.impl("attention_prefix", attention_prefix);
  m.impl("logits_adjust", logits_adjust);
  m.impl("rotary", rotary);
  m.impl("residual_norm", residual_norm);
  m.impl("attention_cache", attention_cache);
  m.impl("cache_append", cache_append);
}

void autograd(torch::Library& m) {
  m.impl("linear_w4", TORCH_FN((&Below<decltype(linear_w4)>::call<0>)));
  m.impl("attention_causal", TORCH_FN((&Below<decltype(attention_causal)>::call<1>)));
  m.impl("attention_prefix", TORCH_FN((&Below<decltype(attention_prefix)>::call<2>)));
  m.impl("logits_adjust", TORCH_FN((&Below<decltype(logits_adjust)>::call<3>)));
  m.impl("rotary", TORCH_FN((&Below<decltype(rotary)>::call<4>)));
  m.impl("residual_norm", TORCH_FN((&Below<decltype(residual_norm)>::call<5>)));
  m.impl("attention_cache", TORCH_FN((&Below<decltype(attention_cache)>::call<6>)));
  m.impl("cache_append", TORCH_FN((&Below<decltype(cache_append)>::call<APPEND>)));
}

TORCH_LIBRARY_IMPL(xdna, AutogradCUDA, m) { autograd(m); }
TORCH_LIBRARY_IMPL(xdna, AutogradCPU, m) { autograd(m); }     // Python's own way past autograd drops tangents there too

extern "C" {

// {calls, multiply-accumulates, launches, nanoseconds} since the last call with reset.
void xdna_torch_counts(int64_t* out, int reset) {
  std::atomic<int64_t>* all[4] = {&counts.calls, &counts.macs, &counts.launches, &counts.nanoseconds};
  for (int i = 0; i < 4; ++i) out[i] = reset ? all[i]->exchange(0) : all[i]->load();
}

}
