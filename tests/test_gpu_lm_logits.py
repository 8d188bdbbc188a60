"""logits_adjust on the MI355X against float64 (lm_reference.py)."""
import math

import pytest
import torch

from lm_reference import logits_case, logits_reference
from torch_xdna import lm

pytestmark = pytest.mark.gpu


def _within(y, ref):
    want, tol = ref
    y = y.double().cpu()
    ok = torch.where(want.isinf(), y == want, (y - want).abs() <= tol)
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off"


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,v,length,bias,mask,wide", [
    (1, 1, 1, "", True, False), (2, 31, 7, "one", False, False), (3, 33, 1, "row", True, True), (1, 2047, 300, "one", True, False),
    (2, 2048, 5, "", False, True), (5, 2049, 999, "row", True, False), (1, 8200, 264, "", True, False),
    (64, 32771, 70, "one", True, False), (70, 32773, 33, "row", False, True)])
def test_logits(gpu, b, v, length, bias, mask, wide, dtype):
    args = logits_case(b, v, length, dtype, bias, mask, seed=v, dev=gpu, wide=wide)
    y = lm.logits_adjust(*args)
    assert y.dtype == args[0].dtype
    _within(y, logits_reference(*args))


def test_logits_options(gpu):
    """Each option alone, none at all, strided rows, token ids and lengths of any value, one token said very often."""
    full = logits_case(4, 3001, 50, "bf16", "row", True, seed=1, dev=gpu)
    x, tokens, lens, rep, pres, freq, bias, allowed = full
    assert torch.equal(lm.logits_adjust(x), x)
    for kw in (dict(tokens=tokens, lens=lens), dict(tokens=tokens, lens=lens, repetition=rep), dict(bias=bias), dict(allowed=allowed),
               dict(tokens=tokens, lens=lens, presence=pres), dict(tokens=tokens, lens=lens, frequency=freq),
               dict(repetition=rep, presence=pres)):
        _within(lm.logits_adjust(x, **kw), logits_reference(x, **kw))
    want = lm.logits_adjust(*full)
    wide = torch.full((4, 3100), math.nan, dtype=x.dtype, device=gpu)
    wide[:, 3:3004] = x
    for t in (wide[:, 3:3004], x.t().contiguous().t()):
        assert torch.equal(lm.logits_adjust(t, *full[1:]), want)
    assert torch.equal(torch.ops.xdna.logits_adjust(x, tokens.t().contiguous().t(), lens, rep.repeat_interleave(2)[::2], pres, freq,
                                                    bias.t().contiguous().t(), allowed.repeat(1, 2)[:, :94]), want)
    row = bias[:1]
    same = lm.logits_adjust(x, bias=row[0])
    assert torch.equal(lm.logits_adjust(x, bias=row.expand(4, 3001)), same)
    odd = torch.tensor([[5, -1, 3001, 5, 2 ** 31 - 1, -2 ** 31, 3000, 5]] * 4, dtype=torch.int32, device=gpu)
    n = torch.tensor([8, 10 ** 6, -4, 4], dtype=torch.int32, device=gpu)
    for t in (odd, odd.long(), odd.long() + (odd.long() == 2 ** 31 - 1) * 2 ** 40):
        _within(lm.logits_adjust(x, t, n, rep, pres, freq), logits_reference(x, t, n, rep, pres, freq))
    often = torch.full((4, 70001), 17, dtype=torch.int32, device=gpu)
    n = torch.tensor([70001, 70000, 1, 0], dtype=torch.int32, device=gpu)
    xf = x.float()
    _within(lm.logits_adjust(xf, often, n, None, None, freq), logits_reference(xf, often, n, None, None, freq))
    assert lm.logits_adjust(x[:0], tokens[:0], lens[:0]).shape == (0, 3001) and lm.logits_adjust(x[:, :0]).shape == (4, 0)


def test_logits_not_finite(gpu):
    """NaN and infinities stay what they are, but not behind the mask."""
    x = torch.zeros(1, 64, device=gpu)
    x[0, :4] = torch.tensor([math.nan, math.inf, -math.inf, math.nan])
    tokens = torch.arange(64, device=gpu, dtype=torch.int32)[None]
    one = torch.ones(1, device=gpu)
    mask = torch.tensor([[~8, 0]], dtype=torch.int32, device=gpu)
    y = lm.logits_adjust(x, tokens, 64 * one.int(), 2 * one, one, one, None, mask)[0]
    assert bool(y[0].isnan()) and y[1] == math.inf and y[2] == -math.inf and y[3] == -math.inf
    assert bool((y[4:32] == -2).all()) and bool((y[32:] == -math.inf).all())


def test_logits_stream_and_graph(gpu):
    args = logits_case(7, 9001, 400, "f16", "one", True, seed=4, dev=gpu)
    want = lm.logits_adjust(*args)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(lm.logits_adjust(*args), want)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = lm.logits_adjust(*args)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(lm.logits_adjust(*args), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with pytest.raises(RuntimeError):
        torch.ops.xdna.logits_adjust(args[0].clone().requires_grad_()).float().sum().backward()
