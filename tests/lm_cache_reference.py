"""float64 references, inputs and error bounds of rotary, residual_norm and the 8-bit cache's operators -- TEST INFRASTRUCTURE.

Bounds count roundings as lm_reference.py does: half a step, torch.finfo(t).eps / 2 of the value, for each rounding to t, and
2^-24 for each float32 operation.
"""
import math

import torch

from lm_reference import DTYPES, U32, attention_reference, half_step
from torch_xdna import lm


# ------------------------------------------------------------------------------ rotary
def rotary_reference(x, positions, freqs, magnitude=1.0, interleaved=False):
    """(y in float64, its bound): cos and sin are off by at most 4 2^-24 (the quarter turn's rounding to float32, the series, the
    magnitude), the two products and their sum by 2 more, and the result rounds once."""
    dt, half = x.dtype, freqs.shape[0]
    x = x.double().cpu()
    angle = (positions.double().cpu()[..., None] * freqs.double().cpu())[..., None, :]
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude
    y, size = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(magnitude)
    return y, (half_step(dt) * y.abs() * (1 + 2.0 ** -6) + torch.finfo(dt).tiny) * (size > 0) + 6 * U32 * size


# ------------------------------------------------------------------------------ residual_norm
def norm_case(rows, width, dtype, stream=None, post=True, gate="row", weight=True, seed=0, dev="cpu"):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (2 * rnd(rows, width)).to(DTYPES[stream or dtype])
    shape = {"": None, "one": (width,), "row": (rows, width)}[gate]
    args = (x, rnd(rows, width).to(dt), (1 + 0.2 * rnd(width)).to(dt) if weight else None,
            (1 + 0.2 * rnd(width)).to(dt) if post else None, None if shape is None else rnd(*shape).to(dt), 0.7)
    return tuple(t.to(dev) if isinstance(t, torch.Tensor) else t for t in args)


def norm_reference(x, o=None, weight=None, post=None, gate=None, scale=1.0, eps=1e-6):
    """((s, y) in float64, their bounds). A mean of squares comes from chains of at most 64 float32 sums, so it is off by (64 + 8)
    2^-24 of itself, its inverse root by half of that and 4 more; then six float32 operations, and one rounding each."""
    xt, yt = x.dtype, x.dtype if o is None else o.dtype
    d = [None if t is None else t.double().cpu() for t in (x, o, weight, post, gate)]
    x, o, weight, post, gate = d
    root = (72 / 2 + 4) * U32
    s, off = x, torch.zeros_like(x)
    if o is not None:
        n, rel = o, 0.0
        if post is not None:
            n, rel = o / (o.square().mean(-1, keepdim=True) + eps).sqrt() * post, root
        n = scale * (n if gate is None else n * gate)
        s = x + n
        off = (rel + 6 * U32) * n.abs() + U32 * s.abs()
    inv = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    w = 1.0 if weight is None else weight
    y = s * inv * w
    # y's own value's error, and that of the root, which the errors of all of s move by at most their rms
    ytol = (off * inv) * (w if weight is None else w.abs()) + y.abs() * (root + 3 * U32 + off.square().mean(-1, keepdim=True).sqrt() * inv)
    return (s, y), (off + half_step(xt) * s.abs() * (1 + 2.0 ** -6) + torch.finfo(xt).tiny,
                    ytol + half_step(yt) * y.abs() * (1 + 2.0 ** -6) + torch.finfo(yt).tiny)


# ------------------------------------------------------------------------------ the cache
def random_cache(batch, kv, dim, capacity, page, dtype, places=None, seed=0, dev="cpu", spare=3):
    """A cache whose table names distinct pages in any order, and whose memory holds anything."""
    g = torch.Generator().manual_seed(seed)
    cols = -(-capacity // page)
    pages = batch * cols + spare
    c = lm.cache8(batch, pages, kv, dim, capacity, page, places, DTYPES[dtype])
    c.kpages.copy_(torch.randint(-128, 128, c.kpages.shape, generator=g))
    c.vpages.copy_(torch.randint(-128, 128, c.vpages.shape, generator=g))
    c.kscales.copy_(0.01 + 0.03 * torch.rand(c.kscales.shape, generator=g))
    c.vscales.copy_(0.01 + 0.03 * torch.rand(c.vscales.shape, generator=g))
    c.ktail.copy_(torch.randn(c.ktail.shape, generator=g))
    c.vtail.copy_(torch.randn(c.vtail.shape, generator=g))
    c.table.copy_(torch.randperm(pages, generator=g)[:batch * cols].view(batch, cols))
    return lm.Cache8(*(t.to(dev) for t in c))


def clone(cache):
    return lm.Cache8(*(t.clone() for t in cache))


def tokens(n, heads, kv, dim, dtype, seed=0, dev="cpu"):
    """(q, k, v) [n, .., dim] as views of one fused projection."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads + 2 * kv, dim, generator=g).to(DTYPES[dtype]).to(dev)
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]


def page_of(block):
    """A page of one head as it is held: (int8, scale) of block (16-bit values), in float32 as the definition has it."""
    x = block.float().cpu()
    scale = x.abs().max() / torch.tensor(127.0)
    if not bool(scale.isfinite()):
        return torch.zeros_like(x, dtype=torch.int8), torch.tensor(math.nan)
    q = torch.round(x / scale) if scale > 0 else torch.zeros_like(x)
    return q.clamp(-127, 127).to(torch.int8), scale


def cache_reference(q, cache, lens, scale=None):
    """attention_cache in float64 with its error bound, [B, N, H, D] each: attention_reference's on the values that the cache
    stands for, and 6 2^-24 more for the share of the values' scale in p."""
    q, cache = q.cpu(), [t.cpu() for t in cache]
    kp, vp, ks, vs, kt, vt, table = cache
    b, n, h, d = q.shape
    pages, kv, g, _ = kp.shape
    r = kt.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for i in range(b):
        length = max(0, min(int(lens[i]), table.shape[1] * g))
        whole = length // g
        ids = [int(t) for t in table[i, :whole]]
        good = torch.tensor([0 <= t < pages for t in ids] + [], dtype=torch.bool).repeat_interleave(g)
        ids = [t if 0 <= t < pages else 0 for t in ids]
        at = torch.arange(whole * g, length) % r
        for c in range(kv):
            k = torch.cat([(kp[ids, c].double() * ks[ids, c].double()[:, None, None]).reshape(-1, d), kt[i, c, at].double()])
            v = torch.cat([(vp[ids, c].double() * vs[ids, c].double()[:, None, None]).transpose(1, 2).reshape(-1, d),
                           vt[i, c][:, at].t().double()])
            for j in range(n):
                heads = slice(c * h // kv, (c + 1) * h // kv)
                m = max(0, min(length, length - n + j + 1))
                seen = torch.cat([good, torch.ones(length - whole * g, dtype=torch.bool)])[:m].expand(h // kv, m)
                # what no row sees does not matter
                kk, vv = (torch.where(seen[0][:, None], t[:m], 0.0) for t in (k, v))
                o, e = attention_reference(q[i, j, heads], kk, vv, seen, scale)
                p = torch.softmax((q[i, j, heads].double() @ kk.t() * scale).masked_fill(~seen, -math.inf), -1) if bool(seen.any()) else 0.0
                out[i, j, heads] = o
                tol[i, j, heads] = e + (6 * U32 * (p @ vv.abs()) if bool(seen.any()) else 0.0)
    return out, tol
