"""attention_cache, residual_norm and logits_adjust at values and strides where a route can part from the definition, on host
tensors; test_gpu_lm_cache_edges.py runs the same functions on the GPU."""
import math

import pytest
import torch

from lm_cache_reference import random_cache
from lm_reference import DTYPES, attention_reference
from torch_xdna import lm


def within(y, want, tol):
    y, want, tol = y.double().cpu(), want.cpu(), tol.cpu()
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------ infinite keys
def infinite_keys(dev, dim, dtype, page=32):
    """A key in the open page with an infinity against q's sign has the score -inf and the weight 0, in whatever dim it lies: the
    others' attention is left. A row of such keys only is zero."""
    dt, old, n, heads = DTYPES[dtype], 2 * page, 3, 4
    for at in (0, dim // 2, dim - 16, dim - 9, dim - 1):
        cache = random_cache(2, 2, dim, 4 * page, page, dtype, seed=dim + at, dev=dev)
        g = torch.Generator().manual_seed(at)
        q = torch.randn(2, n, heads, dim, generator=g).to(dt)
        q[..., at] = 1 + q[..., at].abs()
        q = q.to(dev)
        lens, low = [old + 9, 3], [[old + 2, old + 7], [0, 1, 2]]
        places = cache.ktail.shape[2]
        for i in range(2):
            for p in low[i]:
                cache.ktail[i, :, p % places, at] = -math.inf
        o = lm.attention_cache(q, cache, _i32(lens, dev))
        assert bool((o[1] == 0).all())
        ids = cache.table[0, :2].long()
        for head in range(heads):
            kv = head // 2
            k = (cache.kpages[ids, kv].double() * cache.kscales[ids, kv].double()[:, None, None]).reshape(-1, dim)
            v = (cache.vpages[ids, kv].double() * cache.vscales[ids, kv].double()[:, None, None]).transpose(1, 2).reshape(-1, dim)
            ring = torch.arange(old, lens[0], device=dev) % places
            k = torch.cat([k, cache.ktail[0, kv, ring].double()]).cpu()
            v = torch.cat([v, cache.vtail[0, kv][:, ring].t().double()]).cpu()
            seen = torch.arange(lens[0])[None, :] <= lens[0] - n + torch.arange(n)[:, None]
            seen[:, low[0]] = False
            within(o[0, :, head], *attention_reference(q[0, :, head], torch.where(k.isfinite(), k, 0.0), v, seen, dim ** -0.5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 80, 128])
def test_infinite_keys(dim, dtype):
    infinite_keys("cpu", dim, dtype)


# ------------------------------------------------------------------------------ large scores
def large_scores(dev, dtype, dim, n, group, page, length, power, scale):
    """Scores up to where float32 has no fraction, and differences that are all or nothing: a row's output is the value of its best
    key, or the mean of two that are as good, in pages whose scales differ and in the open page."""
    dt, g = DTYPES[dtype], torch.Generator().manual_seed(page + length)
    kv = 2
    cache = random_cache(1, kv, dim, length, page, dtype, seed=length, dev="cpu")
    whole, places = length // page, cache.ktail.shape[2]
    at = torch.arange(whole * page, length)
    sign = -1.0 if scale < 0 else 1.0
    for c in range(kv):
        best = torch.randint(0, length - n, (2,), generator=g).tolist()      # every row sees them
        value = torch.randint(-100, 60, (length,), generator=g).double()     # of all of a key's dims: its score's sign and size
        value[best] = 64.0
        if c == 1:
            value[best[1]] = -100.0
        value *= sign
        for j in range(whole):
            e, ids = j % 3, int(cache.table[0, j])                            # the page's scale: value = int8 * 2^e
            part = value[j * page:(j + 1) * page]
            part = torch.where(part.abs() == 64, part, torch.trunc(part / 2 ** e) * 2 ** e)
            cache.kpages[ids, c] = (part / 2 ** e).to(torch.int8)[:, None]
            cache.kscales[ids, c] = 2.0 ** e * power[1]
        cache.ktail[0, c][at % places] = (value[at] * power[1]).to(dt)[:, None]
        best = [b for b in best if value[b] == 64.0 * sign]
        v = []
        for b in best:
            if b < whole * page:
                i = int(cache.table[0, b // page])
                v.append(cache.vpages[i, c, :, b % page].double() * cache.vscales[i, c].double())
            else:
                v.append(cache.vtail[0, c][:, b % places].double())
        if c == 0:
            want = [torch.stack(v)]
        else:
            want.append(torch.stack(v))
    cache = lm.Cache8(*(t.to(dev) for t in cache))
    q = torch.full((1, n, kv * group, dim), power[0], dtype=dt, device=dev)
    o = lm.attention_cache(q, cache, _i32([length], dev), scale)
    for c in range(kv):
        mean, size = want[c].mean(0), want[c].abs().mean(0)
        # the weights (1 or 1/2, times the values' scale) round to 16 bits, the result once; float32 in between
        tol = torch.finfo(dt).eps / 2 * (mean.abs() * (1 + 2.0 ** -6) + size * (1 + 2.0 ** -6)) + 16 * 2.0 ** -24 * size + torch.finfo(dt).tiny
        rows = o[0, :, c * group:(c + 1) * group].reshape(-1, dim)
        within(rows, mean.expand_as(rows), tol.expand_as(rows))


# (q's values, keys' unit): scores of about 64 x dim x their product x scale
LARGE = [("f16", (2.0 ** 13, 2.0 ** 8)), ("bf16", (2.0 ** 13, 2.0 ** 8)), ("bf16", (2.0 ** 40, 2.0 ** 30)), ("f16", (2.0 ** 8, 2.0 ** 5))]


@pytest.mark.parametrize("dtype,power", LARGE)
@pytest.mark.parametrize("page,length,scale", [(16, 45, 0.125), (64, 300, -0.3), (32, 70, 0.17)])
def test_large_scores(dtype, power, page, length, scale):
    large_scores("cpu", dtype, 32, 2, 2, page, length, power, scale)


# ------------------------------------------------------------------------------ permuted inputs
def permuted(dev):
    """Results are contiguous, as their shape functions say, whatever the inputs' strides; in a compiled function too."""
    g = torch.Generator().manual_seed(0)
    x, o, gate = (torch.randn(4, 3, 16, generator=g).to(dev).transpose(0, 1) for _ in range(3))
    for args in ((x, o), (x, o, None, None, gate), (x.bfloat16(), o.bfloat16()), (x, o.half(), None, x[0, 0].contiguous()), (x,)):
        got = torch.ops.xdna.residual_norm(*args)
        want = torch.ops.xdna.residual_norm(*(None if t is None else t.contiguous() for t in args))
        for a, b in zip(got, want):
            assert a.is_contiguous() and torch.equal(a, b)
        if len(args) > 1:
            assert all(t.is_contiguous() for t in lm.residual_norm(*args))
    backend = "inductor" if dev != "cpu" else "aot_eager"
    with torch.no_grad():
        both = torch.compile(lambda a, b: [t + 1 for t in torch.ops.xdna.residual_norm(a, b)], fullgraph=True, backend=backend)(x, o)
        for a, b in zip(both, torch.ops.xdna.residual_norm(x, o)):
            assert torch.equal(a, b + 1) and a.stride() == b.stride()


def test_permuted():
    permuted("cpu")


def logits_as_they_are(dev):
    """Nothing to adjust, and permuted logits: a result of its own, contiguous."""
    for dtype in DTYPES.values():
        x = torch.randn(4, 40, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
        for logits in (x, x.t().contiguous().t()):
            for y in (lm.logits_adjust(logits), torch.ops.xdna.logits_adjust(logits)):
                assert torch.equal(y, x) and y.data_ptr() != logits.data_ptr() and y.is_contiguous()
            y = torch.ops.xdna.logits_adjust(logits, None, None, None, None, None, torch.ones(40, device=dev))
            assert y.is_contiguous() and torch.equal(y, (x.float() + 1).to(dtype))


def test_logits_as_they_are():
    logits_as_they_are("cpu")
