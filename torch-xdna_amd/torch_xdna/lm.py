"""Operators of a language model that serves several continuations of one prompt:

  linear_w4         a linear whose weight is 4-bit with scales (and zero points) per group of inputs
  attention_causal  causal grouped-query attention of packed prompts of different lengths
  attention_prefix  one decode step's attention over a prefix that the batch shares and each sequence's own keys
  logits_adjust     penalties for repeated tokens, biases and a grammar's mask on logits, before a token is chosen
  quantize_w4       a float weight as linear_w4 takes it

Each is also the op torch.ops.xdna.<name>, opaque to torch.compile. Tensors on a GPU go to the HIP
kernels (csrc/xdna_torch.cpp checks the arguments there as the functions here do), on torch's current stream, without
synchronizing; a GPU tensor with the library missing raises. Host tensors are computed here with plain torch in
float32. The ops have no derivatives, on the GPU and on the host: a gradient raises where it is asked for, a
forward-mode tangent at the call. (Called here with host tensors the functions are plain torch, derivatives
included.) Wrong arguments raise ValueError or TypeError before anything is launched; what lies in GPU memory (lengths,
starts, token ids) is not read on the host, and the kernels clamp it, so that no value of it reads or writes out of
range.
"""

import math
import time

import torch

from . import kernels
from .runtime import stats

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _on_gpu(name, *args):
    kernels.torch_lib()
    return getattr(torch.ops.xdna, name)(*args)


def _floats(name, t):
    if t.dtype not in FLOATS:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _same_device(x, *ts):
    for t in ts:
        if t is not None and t.device != x.device:
            raise ValueError(f"all tensors must be on one device, got {x.device} and {t.device}")


def _shape(name, t, shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")


# ------------------------------------------------------------------------------ 4-bit weights
def quantize_w4(weight, group=128, symmetric=False):
    """A float weight [N, K] as (qweight uint8 [N, K / 2], scales [N, K / group] of the weight's dtype, zeros uint8
    [N, K / group], or None if symmetric): weight ~= (q - zero) * scale, q in 0..15, two a byte with the even k in the
    low nibble. The range of a group is its smallest to its largest value and 0; symmetric: 7 scales to either side
    and the zero point 8."""
    _floats("weight", weight)
    if weight.dim() != 2 or group < 32 or group % 32 or weight.shape[1] % group or not weight.shape[1]:
        raise ValueError(f"quantize_w4 takes [N, K] with K a multiple of the group and the group one of 32, got "
                         f"{list(weight.shape)} in groups of {group}")
    n, k = weight.shape
    w = weight.detach().float().view(n, k // group, group)
    if symmetric:
        s = (w.abs().amax(-1) / 7).to(weight.dtype)
        z = torch.full_like(s, 8, dtype=torch.float32)
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).to(weight.dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)         # a group of zeros
    sf = s.float()
    if not symmetric:
        z = torch.round(-lo / sf).clamp(0, 15)
    q = (torch.round(w / sf.unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0, 15).to(torch.uint8).view(n, k)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), s.contiguous(), None if symmetric else z.to(torch.uint8)


def linear_w4(x, qweight, scales, zeros=None, bias=None):
    """y [..., N] = x [..., K] times the transpose of (q - zero) * scale, plus bias [N], summed in float32 and rounded
    once to x's dtype. qweight uint8 [N, K / 2] (the even k of a byte in its low nibble), scales [N, K / G] with G a
    multiple of 32, zeros uint8 [N, K / G] or None for 8; qweight, scales and zeros contiguous.
    On the GPU x is read where it lies if its rows are dense, start on 16 bytes, do not overlap and are at most 2^22
    elements apart, else copied first. Rows whose x is not finite, or next to its type's largest, take long: their sums
    are formed a second time, value by value."""
    if x.is_cuda:
        return _on_gpu("linear_w4", x, qweight, scales, zeros, bias)
    _floats("x", x)
    _floats("scales", scales)
    if qweight.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
        raise TypeError("qweight and zeros must be uint8")
    if x.dim() < 1 or qweight.dim() != 2 or scales.dim() != 2:
        raise ValueError("linear_w4 takes x [..., K], qweight [N, K / 2] and scales [N, K / G]")
    n, k = qweight.shape[0], 2 * qweight.shape[1]
    groups = scales.shape[1]
    if x.shape[-1] != k or scales.shape[0] != n or not groups or k % groups or (k // groups) % 32 or not k:
        raise ValueError(f"linear_w4: x {list(x.shape)}, qweight {list(qweight.shape)} and scales {list(scales.shape)} do "
                         "not fit (K / G groups, G a multiple of 32)")
    if zeros is not None:
        _shape("zeros", zeros, scales.shape)
    if bias is not None:
        _floats("bias", bias)
        _shape("bias", bias, (n,))
    if not (qweight.is_contiguous() and scales.is_contiguous() and (zeros is None or zeros.is_contiguous())):
        raise ValueError("linear_w4: qweight, scales and zeros must be contiguous")
    _same_device(x, qweight, scales, zeros, bias)
    t0 = time.perf_counter()
    z = 8.0 if zeros is None else zeros.float().unsqueeze(-1)
    q = torch.stack([qweight & 15, qweight >> 4], dim=-1).view(n, groups, -1).float()
    y = x.reshape(-1, k).float() @ ((q - z) * scales.float().unsqueeze(-1)).view(n, k).t()
    y = (y if bias is None else y + bias.float()).to(x.dtype)
    stats.record("cpu", t0, y.shape[0] * n * k)
    return y.view(*x.shape[:-1], n)


# ------------------------------------------------------------------------------ attention
def _attention_args(name, q, kvs, scale):
    """The checks that both attentions share; the scale as a float."""
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} takes bfloat16 or float16, got {q.dtype}")
    for t in kvs:
        if t.dtype != q.dtype:
            raise TypeError(f"{name}: q, keys and values must be of one dtype, got {q.dtype} and {t.dtype}")
    d = q.shape[-1]
    if not 8 <= d <= 128 or d % 8:
        raise ValueError(f"{name}: head dims must be a multiple of 8, at most 128, got {d}")
    nkv = kvs[0].shape[-2]
    if not nkv or q.shape[-2] % nkv or not q.shape[-2]:
        raise ValueError(f"{name}: {q.shape[-2]} q heads do not share {nkv} key heads evenly")
    return d ** -0.5 if scale is None else float(scale)


def _whole(name, t, dims, what):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must be {what}, got {list(t.shape)}")


def _softmax_v(scores, seen, v):
    """softmax over the seen scores times v; rows that see nothing, or only -inf, are zero. What a value of v that no
    row's mask lets through holds does not matter."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True) if scores.shape[-1] else scores.new_full((*scores.shape[:-1], 1), -math.inf)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ torch.where(v.isfinite(), v, 0.0)
    if not bool(v.isfinite().all()):                   # 0 times an infinity that the row does not see is nothing
        for j in (~v.isfinite()).any(-1).flatten(0, -2).any(0).nonzero().flatten().tolist():
            bad = torch.where(v[..., j:j + 1, :].isfinite(), 0.0, v[..., j:j + 1, :])
            o = o + torch.where(seen[..., j:j + 1] & (bad != 0), p[..., j:j + 1] * bad, 0.0)
    return o


def attention_causal(q, k, v, starts, scale=None):
    """Causal attention of packed prompts: out [T, H, D] of q [T, H, D] and k, v [T, KV, D] (bfloat16 or float16; H a
    multiple of KV, q head h with kv head h / (H / KV); D a multiple of 8, at most 128). starts int32 [S + 1]: the first
    token of each sequence, ascending, and T. A token sees its own sequence's tokens up to itself. scale: 1 / sqrt(D) if
    None. Float32 sums, and the result rounded once; on the GPU the softmax's weights are rounded to q's dtype for their
    product with v, on the host they are not.
    Any strides; but on the GPU a tensor is copied at every call, a whole cache too, unless its last dim is dense, it starts
    on 16 bytes, its other strides are multiples of 8, and its tokens lie D to 2^24 - 1 elements apart."""
    if q.is_cuda:
        return _on_gpu("attention_causal", q, k, v, starts, scale)
    if q.dim() != 3 or k.dim() != 3 or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"attention_causal takes q [T, H, D] and k, v [T, KV, D], got {list(q.shape)}, {list(k.shape)} and "
                         f"{list(v.shape)}")
    t, h, d = q.shape
    _shape("k", k, (t, k.shape[1], d))
    scale = _attention_args("attention_causal", q, (k, v), scale)
    _whole("starts", starts, 1, "[S + 1]")
    if starts.shape[0] < 1:
        raise ValueError("starts must be [S + 1], got []")
    _same_device(q, k, v, starts)
    t0 = time.perf_counter()
    at = torch.arange(t)
    seq = torch.searchsorted(starts, at, right=True)
    seen = (seq[:, None] == seq[None, :]) & (at[None, :] <= at[:, None])
    kv = k.shape[1]
    qf, kf, vf = (x.float().transpose(0, 1) for x in (q, k, v))
    qf = qf.reshape(kv, h // kv, t, d)
    o = _softmax_v(qf @ kf[:, None].transpose(-1, -2) * scale, seen, vf[:, None])
    o = o.reshape(h, t, d).transpose(0, 1).contiguous().to(q.dtype)
    stats.record("cpu", t0, t * t * h * d)     # at most: the sequences' lengths are not read
    return o


def attention_prefix(q, kp, vp, kc, vc, lens, scale=None):
    """One decode step's attention of B sequences that share a prefix: out [B, H, D] of q [B, H, D] (the new tokens'), kp, vp
    [P, KV, D] (the prefix's, held once) and kc, vc [B, S, KV, D], of which sequence b sees the first lens[b] (int32 [B]; clamped to
    0 .. S; the new token's own among them). P and S may be 0. Types, scale, rounding and strides (those of sequences: any
    multiple of 8) as in attention_causal."""
    if q.is_cuda:
        return _on_gpu("attention_prefix", q, kp, vp, kc, vc, lens, scale)
    if q.dim() != 3 or kp.dim() != 3 or kc.dim() != 4 or tuple(vp.shape) != tuple(kp.shape) or tuple(vc.shape) != tuple(kc.shape):
        raise ValueError(f"attention_prefix takes q [B, H, D], kp, vp [P, KV, D] and kc, vc [B, S, KV, D], got {list(q.shape)}, "
                         f"{list(kp.shape)}, {list(vp.shape)}, {list(kc.shape)} and {list(vc.shape)}")
    b, h, d = q.shape
    p, kv = kp.shape[:2]
    _shape("kp", kp, (p, kv, d))
    _shape("kc", kc, (b, kc.shape[1], kv, d))
    scale = _attention_args("attention_prefix", q, (kp, vp, kc, vc), scale)
    _whole("lens", lens, 1, "[B]")
    _shape("lens", lens, (b,))
    _same_device(q, kp, vp, kc, vc, lens)
    t0 = time.perf_counter()
    n = kc.shape[1]
    qf = q.float().reshape(b, kv, h // kv, d)
    k = torch.cat([kp.float().expand(b, p, kv, d), kc.float()], 1).permute(0, 2, 1, 3)
    v = torch.cat([vp.float().expand(b, p, kv, d), vc.float()], 1).permute(0, 2, 1, 3)
    seen = torch.arange(p + n)[None, :] < p + lens.clamp(0, n)[:, None]
    o = _softmax_v(qf @ k.transpose(2, 3) * scale, seen[:, None, None, :].expand(b, kv, h // kv, p + n), v)
    o = o.reshape(b, h, d).to(q.dtype)
    stats.record("cpu", t0, 2 * b * (p + n) * h * d)
    return o


# ------------------------------------------------------------------------------ logits
def logits_adjust(logits, tokens=None, lens=None, repetition=None, presence=None, frequency=None, bias=None, allowed=None):
    """logits [B, V] as the next token is to be chosen from: where token v is n > 0 times among the first lens[b] of tokens [b],
    x / repetition if x > 0 else x * repetition, then - frequency * n, then - presence; for every v + bias; -inf where
    the grammar's bit is 0. In float32, rounded once to logits' dtype (float32, bfloat16 or float16).
    tokens int32 or int64 [B, L] with lens int32 [B] (clamped to 0 .. L; ids outside 0 .. V - 1 count nowhere); repetition,
    presence, frequency float32 [B]; bias float32 [V] or [B, V]; allowed int32 [B, ceil(V / 32)], token v at bit v % 32 of
    word v / 32. Each may be None. All three penalties count the same history."""
    if logits.is_cuda:
        return _on_gpu("logits_adjust", logits, tokens, lens, repetition, presence, frequency, bias, allowed)
    _floats("logits", logits)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], got {list(logits.shape)}")
    b, v = logits.shape
    if (tokens is None) != (lens is None):
        raise ValueError("logits_adjust: tokens and lens go together")
    if tokens is not None:
        if tokens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
        if tokens.dim() != 2:
            raise ValueError(f"tokens must be [B, L], got {list(tokens.shape)}")
        _shape("tokens", tokens, (b, tokens.shape[1]))
        _whole("lens", lens, 1, "[B]")
        _shape("lens", lens, (b,))
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency), ("bias", bias)):
        if t is not None and t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t is not None:
            _shape(name, t, (v,) if name == "bias" and t.dim() == 1 else (b, v) if name == "bias" else (b,))
    if allowed is not None:
        _whole("allowed", allowed, 2, "[B, ceil(V / 32)]")
        _shape("allowed", allowed, (b, -(-v // 32)))
    _same_device(logits, tokens, lens, repetition, presence, frequency, bias, allowed)
    t0 = time.perf_counter()
    x = logits.float()
    if tokens is not None:
        t = tokens.long()
        inside = (torch.arange(t.shape[1])[None, :] < lens[:, None]) & (t >= 0) & (t < v)
        count = torch.zeros(b, v + 1, dtype=torch.int64).scatter_add_(1, torch.where(inside, t, v), torch.ones_like(t))[:, :v]
        y = x
        if repetition is not None:
            y = torch.where(y > 0, y / repetition[:, None], y * repetition[:, None])
        if frequency is not None:
            y = y - frequency[:, None] * count.float()
        if presence is not None:
            y = y - presence[:, None]
        x = torch.where(count > 0, y, x)
    if bias is not None:
        x = x + bias
    if allowed is not None:
        ok = (allowed.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32)) & 1
        x = x.masked_fill(ok.view(b, -1)[:, :v] == 0, -math.inf)
    stats.record("cpu", t0, 0)
    return x.to(logits.dtype)
