"""rotary and residual_norm on the MI355X against float64 (lm_cache_reference.py)."""
import math

import pytest
import torch

from lm_cache_reference import norm_case, norm_reference, rotary_reference
from lm_reference import DTYPES
from torch_xdna import lm

pytestmark = pytest.mark.gpu


def _within(y, want, tol):
    y, want, tol = y.double().cpu(), want.cpu(), tol.cpu()
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,h,d,turned", [(1, 1, 2, 2), (1, 16, 128, 128), (5, 3, 80, 32), (33, 2, 7, 6), (700, 24, 64, 20), (3, 1, 64, 0),
                                          (2, 2, 2050, 2048), (4100, 5, 96, 96), (9, 2, 20, 18)])
def test_rotary(gpu, t, h, d, turned, interleaved, dtype):
    g = torch.Generator().manual_seed(t + d)
    x = torch.randn(t, h, d, generator=g).to(DTYPES[dtype]).to(gpu)
    pos = torch.randint(-5, 200000, (t,), generator=g).to(gpu)
    freqs, magnitude = lm.rotary_freqs(turned, factor=8.0, original=4096, device=gpu)
    y = lm.rotary(x, pos, freqs, magnitude, interleaved)
    assert y.dtype == x.dtype and y.is_contiguous()
    _within(y, *rotary_reference(x, pos, freqs, magnitude, interleaved))
    assert torch.equal(y, lm.rotary(x, pos.int(), freqs, magnitude, interleaved))
    assert torch.equal(y[..., turned:], x[..., turned:])


def test_rotary_positions_and_strides(gpu):
    """The far ends of both integer types, odd frequencies, batches, views, no tokens."""
    x = torch.randn(6, 2, 64, device=gpu)
    freqs, _ = lm.rotary_freqs(64, device=gpu)
    for pos in ([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 999999], [2 ** 40, -2 ** 40, 2 ** 45 + 1, 2 ** 46, 3, 2 ** 33 + 5]):
        p = torch.tensor(pos, device=gpu)
        want, tol = rotary_reference(x, p, freqs)
        # theta itself, a float64 product, is off by 2^-53 of its size in the reference and by twice that in the kernel
        _within(lm.rotary(x, p, freqs), want, tol + 4 * 2.0 ** -53 * p.abs().double().cpu()[:, None, None] * x.abs().sum(-1, keepdim=True).double().cpu())
    odd = torch.tensor([0.0, math.pi, math.pi / 2, -3.3, 1e-300, 100.0], dtype=torch.float64, device=gpu)
    p = torch.arange(6, device=gpu)
    _within(lm.rotary(x, p, odd), *rotary_reference(x, p, odd))
    y = lm.rotary(x, p, torch.tensor([math.nan, math.inf, 1.0], dtype=torch.float64, device=gpu))
    assert bool(y[1:, :, [0, 1, 3, 4]].isnan().all()) and bool(y[..., 2].isfinite().all())
    p = torch.arange(6, device=gpu).view(2, 3)
    want = lm.rotary(x, p.flatten(), freqs)
    assert torch.equal(lm.rotary(x.view(2, 3, 2, 64), p, freqs), want.view(2, 3, 2, 64))
    assert torch.equal(lm.rotary(x.view(2, 3, 2, 64).transpose(0, 1), p.t(), freqs), want.view(2, 3, 2, 64).transpose(0, 1))
    wide = torch.full((6, 5, 67), math.nan, device=gpu)
    for dt in DTYPES.values():
        w = wide.to(dt)
        w[:, 2:4, 1:65] = x.to(dt)
        assert torch.equal(lm.rotary(w[:, 2:4, 1:65], p.flatten(), freqs), lm.rotary(x.to(dt), p.flatten(), freqs))
    assert torch.equal(lm.rotary(x.transpose(1, 2).contiguous().transpose(1, 2), p.flatten(), freqs), want)
    assert lm.rotary(x[:0], p.flatten()[:0], freqs).shape == (0, 2, 64) and lm.rotary(x[:, :0], p.flatten(), freqs).shape == (6, 0, 64)


@pytest.mark.parametrize("dtype,stream", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,width,post,gate,weight", [
    (1, 1, True, "row", True), (3, 7, True, "", True), (5, 64, False, "one", True), (17, 128, True, "row", False), (4, 129, False, "", True),
    (9, 512, True, "one", True), (3, 1001, True, "row", True), (2, 2048, False, "row", True), (7, 2055, True, "", True),
    (5, 4096, True, "row", True), (2, 8184, True, "one", False), (3, 16384, True, "row", True), (2, 32767, False, "one", True)])
def test_norm(gpu, rows, width, post, gate, weight, dtype, stream):
    args = norm_case(rows, width, dtype, stream, post, gate, weight, seed=width, dev=gpu)
    got = lm.residual_norm(*args)
    want, tol = norm_reference(*args)
    assert got[0].dtype == args[0].dtype and got[1].dtype == args[1].dtype
    for a, w, t in zip(got, want, tol):
        _within(a, w, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_norm_alone_and_views(gpu, dtype):
    """Without a block's output; heads of a fused projection; rows that are not dense, batches, gates that a batch's tokens
    share, weights of another type."""
    x, o, w, post, gate, scale = norm_case(12, 96, dtype, seed=5, dev=gpu)
    s, y = lm.residual_norm(x, weight=w)
    assert s is x
    (_, want), (_, tol) = norm_reference(x, weight=w)
    _within(y, want, tol)
    qkv = torch.randn(10, 7, 128, device=gpu).to(x.dtype)
    for part in (qkv[:, 1:5], qkv[:, ::2], qkv.transpose(0, 1)[2:4], qkv[:, :, 3:100], qkv[:, :, ::2], qkv[0], qkv[0, 0], qkv[:0]):
        _, y = lm.residual_norm(part)
        assert torch.equal(y, lm.residual_norm(part.contiguous())[1])
    args = (x, o, w, post, gate, scale)
    want = lm.residual_norm(*args)
    b = [t.view(3, 4, 96) for t in (x, o, gate)]
    odd = []
    for t in b:
        z = torch.full((4, 3, 101), math.nan, dtype=t.dtype, device=gpu)
        z[..., 2:98] = t.transpose(0, 1)
        odd.append(z[..., 2:98].transpose(0, 1))
    for v in (b, odd, [t.transpose(1, 2).contiguous().transpose(1, 2) for t in b]):
        got = lm.residual_norm(v[0], v[1], w, post, v[2], scale)
        assert torch.equal(got[0], want[0].view(3, 4, 96)) and torch.equal(got[1], want[1].view(3, 4, 96))
    shared = gate[:3].view(3, 1, 96).expand(3, 4, 96)
    a, c = (lm.residual_norm(b[0], b[1], w, post, g, scale) for g in (shared, shared.contiguous()))
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    for dt in DTYPES.values():
        other = (x, o, w.to(dt), post.to(dt), gate, scale)
        for p, q, t in zip(lm.residual_norm(*other), *norm_reference(*other)):
            _within(p, q, t)
    assert torch.equal(lm.residual_norm(x[0], o[0], w, post, gate[0], scale)[1], want[1][0])
    z = lm.residual_norm(torch.zeros_like(x), torch.zeros_like(o), w, post, gate)
    assert bool((z[0] == 0).all()) and bool((z[1] == 0).all())
    n = lm.residual_norm(torch.where(torch.arange(12, device=gpu)[:, None] == 3, math.nan, x), o, w)
    assert bool(n[1][3].isnan().all()) and bool(n[1][:3].isfinite().all()) and bool(n[1][4:].isfinite().all())


def test_rows_in_a_graph_and_on_a_stream(gpu):
    x, o, w, post, gate, scale = norm_case(5, 1024, "bf16", "f32", seed=1, dev=gpu)
    freqs, _ = lm.rotary_freqs(128, device=gpu)
    pos = torch.tensor([1, 7, 100, 5000, 70000], device=gpu)

    def step():
        s, y = lm.residual_norm(x, o, w, post, gate, scale)
        return s, lm.rotary(y.view(5, 8, 128), pos, freqs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.normal_(), o.normal_()
        pos += 1
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
