"""attention_causal, attention_prefix and logits_adjust on host tensors: the plain route against float64, the refusals, the
shape functions under fake tensors, and the entry points' argument checks. No GPU is needed."""
import ctypes
import math

import pytest
import torch

from lm_reference import (causal_case, causal_reference, logits_case, logits_reference, prefix_case, prefix_reference)
from torch_xdna import kernels, lm


def _within(y, ref):
    want, tol = ref
    y = y.double()
    assert bool(torch.where(want.isinf(), y == want, (y - want).abs() <= tol).all())


@pytest.mark.parametrize("lens,h,kv,d,dtype", [([1], 1, 1, 8, "bf16"), ([5, 1, 0, 30], 4, 2, 24, "f16"), ([40], 6, 1, 128, "bf16")])
def test_causal_host(lens, h, kv, d, dtype):
    q, k, v, starts = causal_case(lens, h, kv, d, dtype, seed=1)
    y = lm.attention_causal(q, k, v, starts)
    assert y.dtype == q.dtype
    _within(y, causal_reference(q, k, v, lens, d ** -0.5))
    torch.library.opcheck(torch.ops.xdna.attention_causal.default, (q, k, v, starts, 0.2),
                          test_utils=("test_schema", "test_faketensor"))


def test_causal_host_not_finite():
    q, k, v, starts = causal_case([6, 9], 4, 2, 16, "bf16", seed=2)
    want = lm.attention_causal(q, k, v, starts)
    v = v.clone()
    v[8, 1, 3], v[14, 0, 0] = math.inf, math.nan
    got = lm.attention_causal(q, k, v, starts)
    assert torch.equal(got[:8], want[:8]) and torch.equal(got[8:14, :2], want[8:14, :2])
    assert bool((got[8:, 2:, 3] == math.inf).all()) and bool(got[14, :2, 0].isnan().all())


@pytest.mark.parametrize("b,p,s,h,kv,d", [(1, 1, 0, 1, 1, 8), (3, 0, 4, 4, 2, 16), (2, 30, 5, 6, 1, 64), (2, 0, 0, 2, 2, 8)])
def test_prefix_host(b, p, s, h, kv, d):
    args = prefix_case(b, p, s, h, kv, d, "bf16", seed=3)
    args[3][:, max(1, s):] = math.nan
    _within(lm.attention_prefix(*args), prefix_reference(*args, d ** -0.5))
    torch.library.opcheck(torch.ops.xdna.attention_prefix.default, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_logits_host(dtype):
    for b, v, length, bias in ((1, 1, 1, ""), (3, 77, 9, "one"), (2, 200, 40, "row")):
        args = logits_case(b, v, length, dtype, bias, seed=v)
        _within(lm.logits_adjust(*args), logits_reference(*args))
        torch.library.opcheck(torch.ops.xdna.logits_adjust.default, args, test_utils=("test_schema", "test_faketensor"))
    x, tokens, lens, rep, pres, freq, bias, allowed = args
    assert torch.equal(lm.logits_adjust(x), x)
    tokens = torch.tensor([[3, -1, 200, 3], [0, 0, 0, 0]])
    for kw in (dict(tokens=tokens, lens=lens), dict(tokens=tokens, lens=lens, frequency=freq), dict(bias=bias), dict(allowed=allowed)):
        _within(lm.logits_adjust(x, **kw), logits_reference(x, **kw))


def test_attention_refusals():
    q, k, v, starts = causal_case([5, 4], 4, 2, 16, "bf16", seed=4)
    for args in ((q.float(), k.float(), v.float(), starts), (q, k.half(), v, starts), (q, k, v, starts.long())):
        with pytest.raises(TypeError):
            lm.attention_causal(*args)
    for args in ((q[0], k, v, starts), (q, k[:8], v[:8], starts), (q, k, v[:, :1], starts), (q[:, :3], k, v, starts),
                 (q[..., :12], k[..., :12], v[..., :12], starts), (q, k[:, :0], v[:, :0], starts), (q[:, :0], k, v, starts),
                 (q.repeat(1, 1, 9), k.repeat(1, 1, 9), v.repeat(1, 1, 9), starts), (q, k, v, starts[None]), (q, k, v, starts[:0]),
                 (q, k, v, starts.to("meta"))):
        with pytest.raises(ValueError):
            lm.attention_causal(*args)
    q, kp, vp, kc, vc, lens = prefix_case(3, 6, 4, 4, 2, 16, "f16", seed=5)
    for args in ((q.bfloat16(), kp, vp, kc, vc, lens), (q, kp, vp, kc, vc.bfloat16(), lens), (q, kp, vp, kc, vc, lens.long())):
        with pytest.raises(TypeError):
            lm.attention_prefix(*args)
    for args in ((q[0], kp, vp, kc, vc, lens), (q, kp[..., :8], vp[..., :8], kc, vc, lens), (q, kp, vp[:3], kc, vc, lens),
                 (q, kp, vp, kc[:2], vc[:2], lens), (q, kp, vp, kc[:, :, :1], vc[:, :, :1], lens), (q, kp, vp, kc, vc, lens[:2]),
                 (q, kp, vp, kc, vc, lens[None]), (q[:, :3], kp, vp, kc, vc, lens), (q, kp, vp, kc.to("meta"), vc, lens)):
        with pytest.raises(ValueError):
            lm.attention_prefix(*args)


def test_logits_refusals():
    x, tokens, lens, rep, pres, freq, bias, allowed = logits_case(2, 70, 5, "f32", "row", seed=6)
    for kw in (dict(logits=x.double()), dict(tokens=tokens.short()), dict(lens=lens.long()), dict(repetition=rep.double()),
               dict(bias=bias.half()), dict(allowed=allowed.long())):
        with pytest.raises(TypeError):
            lm.logits_adjust(**{**dict(logits=x, tokens=tokens, lens=lens), **kw})
    for kw in (dict(logits=x[0]), dict(tokens=tokens[0]), dict(tokens=tokens[:1]), dict(lens=lens[:1]), dict(lens=None),
               dict(tokens=None), dict(repetition=rep[:1]), dict(presence=pres[None]), dict(bias=bias[:, :3]), dict(bias=bias[:1]),
               dict(allowed=allowed[:, :2]), dict(frequency=freq.to("meta"))):
        with pytest.raises(ValueError):
            lm.logits_adjust(**{**dict(logits=x, tokens=tokens, lens=lens), **kw})


def test_attention_entry_point_checks():
    lib, p = kernels.lib(), ctypes.c_void_p(16)

    def causal(q=p, k=p, v=p, dt=1, st=(64, 8, 64, 8, 64, 8), starts=p, nseq=1, T=4, nh=8, nkv=2, d=8, out=p):
        return lib.xdna_attention_causal(q, k, v, dt, (ctypes.c_int64 * 6)(*st), starts, nseq, T, nh, nkv, d, 1.0, out, None)

    assert causal(T=0) == 0
    for bad in (dict(dt=0), dict(dt=3), dict(T=-1), dict(nseq=-1), dict(nh=7), dict(nkv=0), dict(d=4), dict(d=20), dict(d=136),
                dict(q=None), dict(starts=None), dict(out=None), dict(q=ctypes.c_void_p(8)), dict(v=ctypes.c_void_p(24)),
                dict(st=(64, 8, 60, 8, 64, 8)), dict(st=(64, 8, 64, 8, 1 << 24, 8)), dict(st=(64, 8, 0, 8, 64, 8)),
                dict(st=(-64, 8, 64, 8, 64, 8)), dict(T=1 << 30)):
        assert causal(**bad) == -1, bad

    def prefix(q=p, kp=p, vp=p, kc=p, vc=p, dt=1, st=(64, 8) * 3 + (1 << 40, 64, 8) * 2, lens=p, P=4, S=4, B=1, nh=8, nkv=2, d=8, out=p,
               ws=None, wsb=0):
        return lib.xdna_attention_prefix(q, kp, vp, kc, vc, dt, (ctypes.c_int64 * 12)(*st), lens, P, S, B, nh, nkv, d, 1.0, out, ws,
                                         wsb, None)

    assert prefix(B=0) == 0
    for bad in (dict(dt=0), dict(P=-1), dict(S=-1), dict(B=-1), dict(nh=7), dict(d=12), dict(q=None), dict(kp=None), dict(vc=None),
                dict(lens=None), dict(out=None), dict(kc=ctypes.c_void_p(8)), dict(st=(64, 8) * 3 + (4, 64, 8) * 2),
                dict(st=(64, 8, 0, 8) + (64, 8) + (64, 64, 8) * 2), dict(P=1 << 20), dict(P=1 << 20, ws=p, wsb=64), dict(B=1 << 22)):
        assert prefix(**bad) == -1, bad
    size = lib.xdna_attention_prefix_ws_bytes
    assert size(1 << 40, 1, 1, 8, 2, 64) == -1 and size(100, 100, 0, 8, 2, 64) == 0

    def logits(x=p, dt=0, ld=9, tokens=p, ldt=4, L=4, lens=p, bias=None, ldb=0, allowed=None, lda=1, y=p, B=1, V=9):
        return lib.xdna_logits_adjust(x, dt, ld, tokens, 0, ldt, L, lens, None, None, None, bias, ldb, allowed, lda, y, B, V, None)

    assert logits(B=0) == 0 and logits(V=0) == 0
    for bad in (dict(dt=3), dict(B=-1), dict(V=1 << 31), dict(L=-1), dict(x=None), dict(y=None), dict(ld=8), dict(lens=None),
                dict(ldt=3), dict(bias=p, ldb=8), dict(allowed=p, lda=0)):
        assert logits(**bad) == -1, bad
    assert "logits_adjust" in lib.xdna_last_error().decode()
