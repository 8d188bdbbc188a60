"""float64 references, inputs and error bounds of the language model operators -- TEST INFRASTRUCTURE.

Rounding to a type moves a value by at most half a step, torch.finfo(t).eps / 2 of it; a float32 sum of n terms is off
by at most n / 2 steps (2^-24 each) of the sum of the terms' sizes, in any order.
"""
import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------ linear_w4
def w4_case(m, n, k, group, zeros, bias, dtype, seed=0, dev="cpu", scales="same"):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    x = torch.randn(m, k, generator=g).to(dt)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((0.5 + torch.rand(n, k // group, generator=g)) * 0.005).to(dt if scales == "same" else DTYPES[scales])
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g).to(dt) if bias else None
    return tuple(None if t is None else t.to(dev) for t in (x, q, s, z, b))


def w4_weight(q, s, z):
    n, groups = s.shape
    w = torch.stack([q % 16, q // 16], dim=-1).view(n, groups, -1).double()
    return (w - (8 if z is None else z.double().unsqueeze(-1))), s.double().unsqueeze(-1)


def w4_reference(x, q, s, z, b):
    """(y, the sum of the sizes of y's terms as the kernels hold them: |x| times 128 + q and 128 + z at the most)."""
    x, q, s, z, b = (None if t is None else t.cpu() for t in (x, q, s, z, b))
    n = q.shape[0]
    w, sd = w4_weight(q, s, z)
    y = x.double() @ (w * sd).view(n, -1).t()
    size = x.double().abs() @ (torch.full_like(w, 2 * 143.0) * sd.abs()).view(n, -1).t()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs()
    return y, size


def w4_tolerance(want, size, dtype, k, biased=False):
    """One rounding to the output's type, and float32 sums: of k terms, a scale and a bias. biased: the terms may be
    128 + q and 128 + z times x (bfloat16), else they are at most 16 / 286 of that."""
    return half_step(dtype) * want.abs() * (1 + 2.0 ** -6) + (k + 8) * U32 * size * (1 if biased else 16 / 286) + 1e-30


# ------------------------------------------------------------------------------ attention
def attention_reference(q, k, v, seen, scale):
    """One head group in float64: q [R, D], k and v [N, D], seen [R, N] -> (out, its error bound for inputs of q's dtype).
    Rows that see nothing are zero.

    The bound: a score is a float32 sum of D products, so off by (D + 4) 2^-24 of the sum of their sizes, and p by as
    much of itself, p's exponent and the power by 2^-22 more; p rounds to the inputs' type (half a step), the sums are
    float32 over N terms, and the result rounds once. Numerator and denominator both carry p's error."""
    dt, d, n = q.dtype, q.shape[1], max(1, k.shape[0])
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out, size = p @ v, p @ v.abs()
    score = ((q.abs() @ k.abs().t()) * abs(scale)).masked_fill(~seen, 0.0)
    score = score.amax(-1, keepdim=True) if k.shape[0] else torch.zeros_like(top)
    rel = half_step(dt) + 2 * ((d + 4) * U32 * score + 4 * U32) + 2 * n * U32
    return out, half_step(dt) * out.abs() * (1 + 2.0 ** -6) + size * rel * (1 + 2.0 ** -6) + torch.finfo(dt).tiny


def causal_reference(q, k, v, lens, scale):
    """attention_causal in float64 with its error bound, [T, H, D] each."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    h, kv, at = q.shape[1], k.shape[1], 0
    for n in lens:
        seen = torch.ones(n, n, dtype=torch.bool).tril()
        for i in range(h):
            g = i // (h // kv)
            out[at:at + n, i], tol[at:at + n, i] = attention_reference(q[at:at + n, i], k[at:at + n, g], v[at:at + n, g], seen, scale)
        at += n
    return out, tol


def causal_case(lens, h, kv, d, dtype, seed=0, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(sum(lens), n, d, generator=g).to(DTYPES[dtype]).to(dev) for n in (h, kv, kv))
    return q, k, v, torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)


def prefix_reference(q, kp, vp, kc, vc, lens, scale):
    """attention_prefix in float64 with its error bound, [B, H, D] each."""
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    b, h, _ = q.shape
    kv = kp.shape[1]
    for i in range(b):
        n = max(0, min(int(lens[i]), kc.shape[1]))
        for g in range(kv):
            heads = slice(g * h // kv, (g + 1) * h // kv)
            k, v = torch.cat([kp[:, g], kc[i, :n, g]]), torch.cat([vp[:, g], vc[i, :n, g]])
            seen = torch.ones(h // kv, k.shape[0], dtype=torch.bool)
            out[i, heads], tol[i, heads] = attention_reference(q[i, heads], k, v, seen, scale)
    return out, tol


def prefix_case(b, p, s, h, kv, d, dtype, seed=0, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    t = [torch.randn(*shape, generator=g).to(dt) for shape in
         ((b, h, d), (p, kv, d), (p, kv, d), (b, s, kv, d), (b, s, kv, d))]
    return (*(x.to(dev) for x in t), torch.randint(0, s + 1, (b,), generator=g).to(torch.int32).to(dev))


# ------------------------------------------------------------------------------ logits_adjust
def logits_case(b, v, length, dtype, bias="", mask=True, seed=0, dev="cpu", wide=False):
    g = torch.Generator().manual_seed(seed)
    tokens = (torch.rand(b, length, generator=g) ** 3 * v).long().clamp(max=v - 1)
    shape = {"": None, "one": (v,), "row": (b, v)}[bias]
    args = ((3 * torch.randn(b, v, generator=g)).to(DTYPES[dtype]), tokens if wide else tokens.to(torch.int32),
            torch.randint(0, length + 1, (b,), generator=g).to(torch.int32), 1 + torch.rand(b, generator=g),
            torch.rand(b, generator=g), torch.rand(b, generator=g), None if shape is None else torch.randn(*shape, generator=g),
            torch.randint(-2 ** 31, 2 ** 31, (b, -(-v // 32)), generator=g).to(torch.int32) if mask else None)
    return tuple(None if t is None else t.to(dev) for t in args)


def logits_reference(logits, tokens=None, lens=None, repetition=None, presence=None, frequency=None, bias=None, allowed=None):
    """(y in float64, its error bound): five float32 operations of half a step each on values no larger than the terms' sum,
    and the output's rounding."""
    dt = logits.dtype
    x = logits.double().cpu()
    size = x.abs()
    b, v = x.shape
    for i in range(b if tokens is not None else 0):
        t = tokens[i, :max(0, min(int(lens[i]), tokens.shape[1]))].long().cpu()
        said, n = torch.unique(t[(t >= 0) & (t < v)], return_counts=True)
        at, n = x[i, said], n.double()
        r = 1.0 if repetition is None else repetition[i].double().item()
        f, p = (0.0 if t is None else t[i].double().item() for t in (frequency, presence))
        at = torch.where(at > 0, at / r, at * r)
        size[i, said] = at.abs() + f * n + p
        x[i, said] = at - f * n - p
    if bias is not None:
        x, size = x + bias.double().cpu(), size + bias.double().cpu().abs()
    if allowed is not None:
        for j in range(32):
            x[:, j::32] = torch.where((allowed.long().cpu() >> j & 1).bool()[:, :x[:, j::32].shape[1]], x[:, j::32], -math.inf)
    return x, half_step(dt) * x.abs().nan_to_num(posinf=0.0) + 6 * U32 * size + torch.finfo(dt).tiny
