"""Operators of a language model that serves several continuations of one prompt, or different prompts together:

  linear_w4         a linear whose weight is 4-bit with scales (and zero points) per group of inputs
  attention_causal  causal grouped-query attention of packed prompts of different lengths
  attention_prefix  one decode step's attention over a prefix that the batch shares and each sequence's own keys
  attention_cache   the attention of each text's newest tokens over its paged 8-bit cache
  cache_append      new tokens' keys and values into that cache, keys (and queries) turned to their positions on the way
  rotary            heads turned to their positions
  residual_norm     a block's output added to the residual stream, with the norms before and after, a gate and a scale
  logits_adjust     penalties for repeated tokens, biases and a grammar's mask on logits, before a token is chosen
  quantize_w4       a float weight as linear_w4 takes it
  cache8            an empty cache (Cache8) for cache_append and attention_cache
  rotary_freqs      the frequencies that rotary and cache_append take

Each but the last three is also the op torch.ops.xdna.<name>, opaque to torch.compile (those of the cache take its
tensors one by one). Tensors on a GPU go to the HIP
kernels (csrc/xdna_torch.cpp checks the arguments there as the functions here do), on torch's current stream, without
synchronizing; a GPU tensor with the library missing raises. Host tensors are computed here with plain torch in
float32. The ops have no derivatives, on the GPU and on the host: a gradient raises where it is asked for, a
forward-mode tangent at the call, and cache_append, which writes to the cache, raises at the call either way. (Called here
with host tensors the functions are plain torch, derivatives included; what goes into a cache is detached.) Wrong arguments raise ValueError or TypeError before anything is launched; what lies in GPU memory (lengths,
starts, token ids) is not read on the host, and the kernels clamp it, so that no value of it reads or writes out of
range.
"""

import math
import time
from typing import NamedTuple

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
    y = x.to(logits.dtype).contiguous()
    return y.clone() if y is logits else y


# ------------------------------------------------------------------------------ positions
def rotary_freqs(dim, base=10000.0, factor=1.0, original=None, slow=1.0, fast=32.0, device=None):
    """(radians a position, float64 [dim / 2], and the magnitude) for heads of which `dim` dims turn: base^(-2 j / dim). Scaled for
    contexts `factor` times as long as the model was made for: all frequencies by 1 / factor if `original` is None; else,
    with `original` positions then, those that turn at least `fast` times over them stay, those that turn at most `slow`
    times go by 1 / factor, those between by a share of each, and the magnitude is 0.1 ln(factor) + 1. The share is linear in the
    number of turns, as the YaRN paper has it. Programs that make it linear in the index of the dim have other frequencies
    between the two: a checkpoint of theirs needs those, given as freqs."""
    if dim < 0 or dim % 2 or factor <= 0:
        raise ValueError(f"rotary_freqs takes an even number of dims and a factor above 0, got {dim} and {factor}")
    f = float(base) ** -(torch.arange(0, dim, 2, dtype=torch.float64, device=device) / max(dim, 1))
    if original is None:
        return f / factor, 1.0
    keep = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1 if factor > 1 else 1.0


def _check_freqs(freqs, d):
    if freqs.dtype != torch.float64:
        raise TypeError(f"freqs must be float64, got {freqs.dtype}")
    if freqs.dim() != 1 or 2 * freqs.shape[0] > d:
        raise ValueError(f"freqs must be [R / 2] with R at most the heads' {d} dims, got {list(freqs.shape)}")


def _turn(x, positions, freqs, magnitude, interleaved):
    """x [T, H, D] turned, in x's type."""
    n = freqs.shape[0]
    angle = positions.double()[:, None, None] * freqs
    cos, sin = angle.cos().float() * magnitude, angle.sin().float() * magnitude
    f = x.float()
    a, b = (f[..., 0:2 * n:2], f[..., 1:2 * n:2]) if interleaved else (f[..., :n], f[..., n:2 * n])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, f[..., 2 * n:]], -1).to(x.dtype)


def rotary(x, positions, freqs, magnitude=1.0, interleaved=False):
    """Heads x [.., H, D] (float32, bfloat16 or float16) turned to the positions [..] (int32 or int64) of their tokens: pair j of
    the first 2 R' dims, R' = len(freqs) (float64, radians a position, at most 1024), by theta = position * freqs[j]: (a, b) ->
    magnitude * (a cos - b sin, b cos + a sin). Pairs are dims (j, R' + j), or (2 j, 2 j + 1) if interleaved; the other dims
    are copied. theta in float64 (off by up to 2^-52 of itself: good to float32 up to 2^28 radians, on the GPU of no meaning from
    2^50 on), the rest in float32, rounded once. A contiguous
    result; on the GPU x is read where it lies if its last dim is dense and its leading dims can be seen as one, and H D is below
    2^24."""
    if x.is_cuda:
        return _on_gpu("rotary", x, positions, freqs, magnitude, interleaved)
    _floats("x", x)
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if x.dim() < 3:
        raise ValueError(f"rotary takes x [.., H, D], got {list(x.shape)}")
    _check_freqs(freqs, x.shape[-1])
    if freqs.shape[0] > 1024:
        raise ValueError(f"rotary turns at most 1024 pairs, got {freqs.shape[0]}")
    _shape("positions", positions, x.shape[:-2])
    _same_device(x, positions, freqs)
    t0 = time.perf_counter()
    y = _turn(x.reshape(positions.numel(), *x.shape[-2:]), positions.reshape(-1), freqs, magnitude, interleaved)
    stats.record("cpu", t0, 2 * positions.numel() * x.shape[-2] * freqs.shape[0])
    return y.view(x.shape)


# ------------------------------------------------------------------------------ residual stream
def residual_norm(x, o=None, weight=None, post=None, gate=None, scale=1.0, eps=1e-6):
    """(s, y): a block's output o [.., W] added to the residual stream x [.., W], and the norm that the next block reads:
    n = post * o / sqrt(mean(o^2) + eps) (o itself if post is None), s = x + scale * gate * n (gate 1 if None),
    y = weight * s / sqrt(mean(s^2) + eps) (weight 1 if None), y from s before it is rounded. In float32, each
    rounded once: s to x's type, y to o's. x is of o's type or float32 (float32, bfloat16 or float16); weight and post [W] of any
    of them, gate of o's type, [W] or of x's shape (any strides: one that a sequence's tokens share can be expanded). Results
    are contiguous; o None: (x, y), y of x's type. W at most 32768."""
    if x.is_cuda:
        s, y = _on_gpu("residual_norm", x, o, weight, post, gate, scale, eps)
        return (x if o is None else s), y
    _floats("x", x)
    if x.dim() < 1 or x.shape[-1] > 32768:
        raise ValueError(f"residual_norm takes x [.., W] with W at most 32768, got {list(x.shape)}")
    if o is None and (post is not None or gate is not None):
        raise ValueError("residual_norm: post and gate need o")
    w = x.shape[-1]
    if o is not None:
        _floats("o", o)
        if x.dtype not in (o.dtype, torch.float32):
            raise TypeError(f"x must be of o's type or float32, got {x.dtype} and {o.dtype}")
        _shape("o", o, x.shape)
    for name, t in (("weight", weight), ("post", post)):
        if t is not None:
            _floats(name, t)
            _shape(name, t, (w,))
    if gate is not None:
        if gate.dtype != o.dtype:
            raise TypeError(f"gate must be of o's type, got {gate.dtype}")
        if gate.shape != x.shape and tuple(gate.shape) != (w,):
            raise ValueError(f"gate must have shape {list(x.shape)} or [{w}], got {list(gate.shape)}")
    _same_device(x, o, weight, post, gate)
    t0 = time.perf_counter()
    s = x.float()
    if o is not None:
        n = o.float()
        if post is not None:
            n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + eps) * post.float()
        s = s + scale * (n if gate is None else n * gate.float())
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    y = (y if weight is None else y * weight.float()).to(x.dtype if o is None else o.dtype).contiguous()
    stats.record("cpu", t0, 0)
    return (x if o is None else s.to(x.dtype).contiguous()), y


# ------------------------------------------------------------------------------ a paged cache in 8 bits
class Cache8(NamedTuple):
    """Keys and values of B texts in 8 bits, in pages of G = 16, 32, 64 or 128 tokens, and in 16 bits where a page is not full.

    kpages int8 [pages, KV, G, D], vpages int8 [pages, KV, D, G]; kscales, vscales float32 [pages, KV]: a page of a head stands for
    q * scale, scale its largest magnitude / 127 (0: all zero; NaN: a value was not finite, and all of it reads as NaN). ktail
    [B, KV, R, D] and vtail [B, KV, D, R] (bfloat16 or float16): each text's last R tokens, position p at place p % R; R a
    multiple of G. table int32 [B, P]: the page of a text's positions G j .. G j + G - 1, a text's capacity P G.

    A page is written once, when its last token comes, from the 16-bit tokens: the cache holds the same whatever calls its
    tokens came in. A text's length is the program's to keep; it may go back by R - G tokens (drafts that were not
    taken) and tokens be appended there anew. The program gives out the pages: one that is going to be written belongs to one
    text, one that is only read may be in many (a shared prompt). The table is read on the device alone."""

    kpages: torch.Tensor
    vpages: torch.Tensor
    kscales: torch.Tensor
    vscales: torch.Tensor
    ktail: torch.Tensor
    vtail: torch.Tensor
    table: torch.Tensor


def cache8(batch, pages, kv, dim, capacity, page=64, places=None, dtype=torch.bfloat16, device=None):
    """An empty Cache8 for `batch` texts of up to `capacity` tokens each over a pool of `pages` pages (zeros), the table all -1:
    no page. places: R, 2 pages' tokens if None."""
    if page not in (16, 32, 64, 128) or dim % 16 or not 16 <= dim <= 128 or dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"cache8 takes pages of 16, 32, 64 or 128 tokens, dims that are a multiple of 16, at most 128, and bfloat16 or "
                         f"float16, got {page}, {dim} and {dtype}")
    r = 2 * page if places is None else places
    if r < page or r % page or r >= 65536:
        raise ValueError(f"cache8: places must be a multiple of {page} below 65536, got {r}")
    z = dict(device=device)
    return Cache8(torch.zeros(pages, kv, page, dim, dtype=torch.int8, **z), torch.zeros(pages, kv, dim, page, dtype=torch.int8, **z),
                  torch.zeros(pages, kv, **z), torch.zeros(pages, kv, **z), torch.zeros(batch, kv, r, dim, dtype=dtype, **z),
                  torch.zeros(batch, kv, dim, r, dtype=dtype, **z),
                  torch.full((batch, -(-capacity // page)), -1, dtype=torch.int32, **z))


def _check_cache(name, x, cache, lens):
    kp, vp, ks, vs, kt, vt, table = cache
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{name} takes bfloat16 or float16, got {x.dtype}")
    if kp.dtype != torch.int8 or vp.dtype != torch.int8:
        raise TypeError("kpages and vpages must be int8")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError("kscales and vscales must be float32")
    if kt.dtype != x.dtype or vt.dtype != x.dtype:
        raise TypeError(f"ktail and vtail must be {x.dtype}, got {kt.dtype} and {vt.dtype}")
    if kp.dim() != 4 or kt.dim() != 4:
        raise ValueError(f"kpages must be [pages, KV, G, D] and ktail [B, KV, R, D], got {list(kp.shape)} and {list(kt.shape)}")
    _whole("table", table, 2, "[B, P]")
    (pages, kv, g, d), b, r = kp.shape, kt.shape[0], kt.shape[2]
    if g not in (16, 32, 64, 128):
        raise ValueError(f"{name}: pages hold 16, 32, 64 or 128 tokens, got {g}")
    if d < 16 or d > 128 or d % 16:
        raise ValueError(f"{name}: head dims must be a multiple of 16, at most 128, got {d}")
    if r < g or r % g or r >= 65536:
        raise ValueError(f"{name}: R must be a multiple of {g} below 65536, got {r}")
    if not kv:
        raise ValueError(f"{name}: no key heads")
    if not pages and table.shape[1]:
        raise ValueError(f"{name}: a table of no pages")
    _shape("vpages", vp, (pages, kv, d, g))
    _shape("kscales", ks, (pages, kv))
    _shape("vscales", vs, (pages, kv))
    _shape("ktail", kt, (b, kv, r, d))
    _shape("vtail", vt, (b, kv, d, r))
    _shape("table", table, (b, table.shape[1]))
    _whole("lens", lens, 1, "[B]")
    _shape("lens", lens, (b,))
    for t in cache[:6]:
        if not t.is_contiguous():
            raise ValueError(f"{name}: the cache must be contiguous and 16-byte aligned")
    _same_device(x, *cache, lens)
    return b, table.shape[1], pages, kv, g, d, r


def _to_page(block, pages, scales, page):
    """One page of every head: block [KV, .., ..] in float32."""
    top = block.abs().amax((1, 2))
    scale = torch.where(top.isfinite(), top / 127, math.nan)
    q = torch.round(block / torch.where(scale > 0, scale, 1.0)[:, None, None]).clamp(-127, 127)
    pages[page] = torch.where((scale > 0)[:, None, None], q, 0.0).to(torch.int8)
    scales[page] = scale


def cache_append(cache, lens, k, v, starts=None, q=None, freqs=None, magnitude=1.0, interleaved=False):
    """New tokens' keys and values k, v [T, KV, D] (bfloat16 or float16; any strides with a dense last dim) go into the cache, to the
    positions lens[b] (int32 [B]; clamped to 0 .. P G) and on of their texts; lens stays as it is. starts int32 [B + 1]: the
    first token of each text, ascending, and behind the last; None: T / B tokens each. Keys are turned to their positions as
    by rotary (freqs None: they are already) and rounded to their type. q [T, H, D]: queries of the same tokens, turned the same
    way (to max(lens[b], 0) and on, also where keys are dropped) and returned (contiguous; rows of no text are zero); None is
    returned without.
    Dropped: tokens that no text has or that its capacity has no room for. A page outside the pool is not written. On the GPU
    T + 2 KV (T / G + 2 B) is below 2^24, P G below 2^30, H below 2^16."""
    if k.is_cuda:
        out = _on_gpu("cache_append", k, v, *cache, lens, starts, q, freqs, magnitude, interleaved)
        return None if q is None else out
    b, p, pages, kv, g, d, r = _check_cache("cache_append", k, cache, lens)
    for t in (v, q):
        if t is not None and t.dtype != k.dtype:
            raise TypeError("cache_append: q, k and v must be of one dtype")
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"cache_append takes k, v [T, KV, D], got {list(k.shape)} and {list(v.shape)}")
    n = k.shape[0]
    _shape("k", k, (n, kv, d))
    if starts is not None:
        _whole("starts", starts, 1, "[B + 1]")
        _shape("starts", starts, (b + 1,))
    elif n % b if b else n:
        raise ValueError(f"cache_append: {n} tokens are not the same number for each of {b} texts; starts must say which are whose")
    if freqs is not None:
        _check_freqs(freqs, d)
    if q is not None:
        if freqs is None:
            raise ValueError("cache_append: q turns with freqs, and there are none")
        if q.dim() != 3 or not q.shape[1]:
            raise ValueError(f"q must be [T, H, D], got {list(q.shape)}")
        _shape("q", q, (n, q.shape[1], d))
    _same_device(k, v, starts, q, freqs)
    t0 = time.perf_counter()
    out = None if q is None else torch.zeros(q.shape, dtype=q.dtype)
    first = starts.tolist() if starts is not None else [i * (n // b) for i in range(b + 1)] if b else []
    with torch.no_grad():
        for i in range(b):
            s0 = min(max(first[i], 0), n)
            s1 = min(max(first[i + 1], s0), n)
            before = min(max(int(lens[i]), 0), p * g)
            end = min(before + s1 - s0, p * g)
            if end == before:
                continue
            pos = torch.arange(before, end)
            kn, vn = k[s0:s0 + end - before].detach(), v[s0:s0 + end - before].detach()
            if freqs is not None:
                kn = _turn(kn, pos, freqs, magnitude, interleaved)
            base = before // g * g
            past = torch.arange(base, before) % r
            kall = torch.cat([cache.ktail[i][:, past].transpose(0, 1), kn]).float()                # [tokens from base on, KV, D]
            vall = torch.cat([cache.vtail[i][:, :, past].permute(2, 0, 1), vn]).float()
            for j in range((end - base) // g):
                page = int(cache.table[i, base // g + j])
                if 0 <= page < pages:
                    _to_page(kall[j * g:(j + 1) * g].transpose(0, 1), cache.kpages, cache.kscales, page)
                    _to_page(vall[j * g:(j + 1) * g].permute(1, 2, 0), cache.vpages, cache.vscales, page)
            at = pos[-r:] % r
            cache.ktail[i][:, at] = kn[-r:].transpose(0, 1)
            cache.vtail[i][:, :, at] = vn[-r:].permute(1, 2, 0)
    if q is not None and b:
        at = torch.arange(n)
        st = torch.tensor(first)
        mine = (at >= st[0]) & (at < st[b])
        seq = (torch.searchsorted(st[:b], at, right=True) - 1).clamp(min=0)
        turned = _turn(q, lens.clamp(min=0)[seq] + at - st[seq], freqs, magnitude, interleaved)
        out = torch.where(mine[:, None, None], turned, 0.0)
    stats.record("cpu", t0, 2 * n * kv * d)
    return out


def attention_cache(q, cache, lens, scale=None):
    """Attention of the newest N tokens of each of B texts over its cache, which holds their keys already (cache_append): out
    [B, N, H, D] of q [B, N, H, D] (bfloat16 or float16; H a multiple of KV, q head h with kv head h / (H / KV)). Token n of text b
    sees its positions 0 .. lens[b] - N + n (lens int32 [B], clamped to 0 .. P G, the new tokens counted): a text with fewer new
    ones has them last, and rows before the first position are zero. Full pages are read in 8 bits, the open one from the
    16-bit places; a page that is none of the pool is seen by no one. scale: 1 / sqrt(D) if None. Float32 sums, the
    result rounded once; on the GPU the softmax's weights are rounded for their product with the values, a page's, times the
    values' scale, to float16, the open page's to q's dtype, on the host they are not.
    On the GPU q is copied unless its last dim is dense, it starts on 16 bytes and its strides are multiples of 8; the work is
    split for texts as long as the table is wide, so a table that is cut to its longest text (table[:, :pages]) is read
    best; B N H is below 2^23, H below 2^16, P G below 2^30."""
    if q.is_cuda:
        return _on_gpu("attention_cache", q, *cache, lens, scale)
    b, p, pages, kv, g, d, r = _check_cache("attention_cache", q, cache, lens)
    if q.dim() != 4:
        raise ValueError(f"attention_cache takes q [B, N, H, D], got {list(q.shape)}")
    n, h = q.shape[1:3]
    _shape("q", q, (b, n, h, d))
    if not h or h % kv:
        raise ValueError(f"attention_cache: {h} q heads do not share {kv} key heads evenly")
    scale = d ** -0.5 if scale is None else float(scale)
    t0 = time.perf_counter()
    out = torch.zeros(q.shape, dtype=q.dtype)
    for i in range(b):
        length = min(max(int(lens[i]), 0), p * g)
        whole = length // g
        ids = cache.table[i, :whole].long()
        good = (ids >= 0) & (ids < pages)
        ids = torch.where(good, ids, 0)
        k = (cache.kpages[ids].float() * cache.kscales[ids][..., None, None]).transpose(0, 1).reshape(kv, -1, d)
        v = (cache.vpages[ids].float() * cache.vscales[ids][..., None, None]).permute(1, 0, 3, 2).reshape(kv, -1, d)
        at = torch.arange(whole * g, length) % r
        k = torch.cat([k, cache.ktail[i][:, at].float()], 1)
        v = torch.cat([v, cache.vtail[i][:, :, at].transpose(1, 2).float()], 1)
        seen = torch.cat([good.repeat_interleave(g), torch.ones(length - whole * g, dtype=torch.bool)])
        seen = seen & (torch.arange(length)[None, :] <= length - n + torch.arange(n)[:, None])
        qf = q[i].float().view(n, kv, h // kv, d).permute(1, 2, 0, 3)                              # [KV, H / KV, N, D]
        o = _softmax_v(qf @ k[:, None].transpose(-1, -2) * scale, seen, v[:, None])
        out[i] = o.permute(2, 0, 1, 3).reshape(n, h, d).to(q.dtype)
    stats.record("cpu", t0, 2 * b * n * h * d * p * g)
    return out
