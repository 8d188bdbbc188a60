"""attention_causal and attention_prefix on the MI355X for scores up to where float32 has no fraction: differences are all or
nothing, and a row's output is the mean of the values of its best keys."""
import pytest
import torch

from lm_reference import DTYPES, U32, half_step
from torch_xdna import lm

pytestmark = pytest.mark.gpu

# (q's values, keys' unit): scores of up to 127 x dim x their product x scale
LARGE = [("f16", (2.0 ** 13, 2.0 ** 8)), ("bf16", (2.0 ** 13, 2.0 ** 8)), ("bf16", (2.0 ** 40, 2.0 ** 30)), ("f16", (2.0 ** 8, 2.0 ** 5))]


def _within(y, best, v, dtype):
    """best [R, N]: which keys are the best of those that row r sees."""
    p = best.double() / best.sum(-1, keepdim=True)
    want, size = p @ v.double(), p @ v.double().abs()
    # p is 1 for each of them; float32 sums of as many terms, and one rounding
    tol = half_step(dtype) * want.abs() * (1 + 2.0 ** -6) + (best.sum(-1, keepdim=True) + 4) * U32 * size + torch.finfo(dtype).tiny
    off = int((~((y.double() - want).abs() <= tol)).sum())
    assert off == 0, f"{off} of {y.numel()} off"


def _keys(n, kv, dim, unit, sign, dt, gpu, seed):
    g = torch.Generator().manual_seed(seed)
    value = torch.randint(-127, 128, (n, kv), generator=g)
    k = (value * unit * sign)[:, :, None].expand(n, kv, dim).to(dt).to(gpu).contiguous()
    return value.to(gpu), k, torch.randn(n, kv, dim, generator=g).to(dt).to(gpu)


@pytest.mark.parametrize("dtype,power", LARGE)
@pytest.mark.parametrize("lens,h,kv,dim,scale", [([70, 1, 33], 4, 2, 64, 0.17), ([300], 16, 8, 128, -0.09), ([2100], 16, 8, 128, 0.11),
                                                 ([100] * 40, 16, 8, 128, 0.125), ([2500, 60], 12, 4, 64, 0.19)])
def test_causal(gpu, dtype, power, lens, h, kv, dim, scale):
    """Few rows, and 128 rows to a workgroup by one and by two groups of waves."""
    dt, t = DTYPES[dtype], sum(lens)
    value, k, v = _keys(t, kv, dim, power[1], 1 if scale > 0 else -1, dt, gpu, t)
    q = torch.full((t, h, dim), power[0], dtype=dt, device=gpu)
    starts = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(gpu)
    o = lm.attention_causal(q, k, v, starts, scale)
    for s, n in zip(starts.tolist(), lens):
        some = torch.arange(0, n, max(1, n // 300), device=gpu)
        seen = torch.arange(n, device=gpu)[None, :] <= some[:, None]
        for i in range(h):
            x = value[s:s + n, i // (h // kv)].expand(some.shape[0], n).masked_fill(~seen, -1000)
            _within(o[s + some, i], x == x.amax(-1, keepdim=True), v[s:s + n, i // (h // kv)], dt)


@pytest.mark.parametrize("dtype,power", LARGE)
@pytest.mark.parametrize("b,p,n,h,kv,dim,scale", [(3, 40, 17, 4, 2, 64, 0.17), (4, 264, 64, 16, 8, 128, -0.09), (48, 4096, 300, 16, 8, 128, 0.11),
                                                  (24, 20000, 10, 32, 4, 64, 0.13), (64, 500, 100, 16, 8, 128, 0.1)])
def test_prefix(gpu, dtype, power, b, p, n, h, kv, dim, scale):
    """One workgroup for all keys, parts of the prefix, 32 and 128 rows to a workgroup."""
    dt, sign = DTYPES[dtype], 1 if scale > 0 else -1
    pv, kp, vp = _keys(p, kv, dim, power[1], sign, dt, gpu, p)
    ov, kc, vc = _keys(b * n, kv, dim, power[1], sign, dt, gpu, b)
    q = torch.full((b, h, dim), power[0], dtype=dt, device=gpu)
    lens = torch.randint(0, n + 1, (b,), generator=torch.Generator().manual_seed(n)).to(torch.int32).to(gpu)
    o = lm.attention_prefix(q, kp, vp, kc.view(b, n, kv, dim), vc.view(b, n, kv, dim), lens, scale)
    for i in range(0, b, max(1, b // 6)):
        m = int(lens[i])
        for c in range(kv):
            x = torch.cat([pv[:, c], ov[i * n:i * n + m, c]])[None]
            rows = o[i, c * h // kv:(c + 1) * h // kv]
            best = (x == x.amax()).expand(rows.shape[0], -1)
            _within(rows, best, torch.cat([vp[:, c], vc[i * n:i * n + m, c]]), dt)
