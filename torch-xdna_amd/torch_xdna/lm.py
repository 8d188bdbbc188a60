"""Operators of a language model that serves several continuations of one prompt:

  linear_w4         a linear whose weight is 4-bit with scales (and zero points) per group of inputs
  attention_causal  causal grouped-query attention of packed prompts of different lengths
  attention_prefix  one decode step's attention over a prefix that the batch shares and each sequence's own keys
  logits_adjust     penalties for repeated tokens, biases and a grammar's mask on logits, before a token is chosen
  quantize_w4       a float weight as linear_w4 takes it

Each is also the op torch.ops.xdna.<name>, opaque to torch.compile. Tensors on a GPU go to the HIP
kernels (kernels.py), on torch's current stream, without synchronizing; a GPU tensor with the library missing raises.
Host tensors are computed here with plain torch in float32. There is no backward pass: a call that needs a
gradient raises where the gradient is asked for. Wrong arguments raise ValueError or TypeError before anything is
launched; what lies in GPU memory (lengths, starts, token ids) is not read on the host, and the kernels
clamp it, so that no value of it reads or writes out of range.
"""

import time

import torch

from . import kernels
from .runtime import stats

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


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
    multiple of 32, zeros uint8 [N, K / G] or None for 8; qweight, scales and zeros contiguous."""
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
    if x.is_cuda:
        y = kernels.linear_w4(x.reshape(-1, k), qweight, scales, zeros, bias)
        stats.launches += 1
    else:
        z = 8.0 if zeros is None else zeros.float().unsqueeze(-1)
        q = torch.stack([qweight & 15, qweight >> 4], dim=-1).view(n, groups, -1).float()
        y = x.reshape(-1, k).float() @ ((q - z) * scales.float().unsqueeze(-1)).view(n, k).t()
        y = (y if bias is None else y + bias.float()).to(x.dtype)
    stats.record("gpu" if x.is_cuda else "cpu", t0, y.shape[0] * n * k)
    return y.view(*x.shape[:-1], n)
