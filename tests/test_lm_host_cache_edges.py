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
