"""rotary, residual_norm and the paged 8-bit cache on host tensors: the plain route against float64, pages and lengths that are
none, the refusals, the shape functions under fake tensors, and the entry points' argument checks. No GPU is needed."""
import ctypes
import math

import pytest
import torch

from lm_cache_reference import cache_reference, clone, norm_case, norm_reference, page_of, random_cache, rotary_reference, tokens
from lm_reference import DTYPES
from torch_xdna import kernels, lm

ops = torch.ops.xdna


def _within(y, want, tol):
    bad = ~((y.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y.double() - want).abs() / tol).max())} bounds"


def _other(dev):
    return "meta" if dev == "cpu" else "cpu"


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------------------ rotary
def test_rotary_freqs():
    f, m = lm.rotary_freqs(8, base=100.0)
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, 100.0 ** -(torch.arange(4, dtype=torch.float64) / 4))
    assert torch.equal(lm.rotary_freqs(8, base=100.0, factor=4.0)[0], f / 4)
    g, m = lm.rotary_freqs(64, factor=8.0, original=4096)
    plain = lm.rotary_freqs(64)[0]
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(g[turns >= 32], plain[turns >= 32]) and torch.allclose(g[turns <= 1], plain[turns <= 1] / 8)
    mid = (turns < 32) & (turns > 1)
    assert bool((g[mid] < plain[mid]).all()) and bool((g[mid] > plain[mid] / 8).all()) and m == 0.1 * math.log(8) + 1
    assert lm.rotary_freqs(0)[0].shape == (0,)
    for bad in (dict(dim=7), dict(dim=-2), dict(dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            lm.rotary_freqs(**bad)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_host(dtype, interleaved):
    x = torch.randn(2, 3, 4, 40, generator=torch.Generator().manual_seed(0)).to(DTYPES[dtype])
    pos = torch.tensor([[0, 5, -7], [100000, 2 ** 31 - 1, 12]])
    freqs, _ = lm.rotary_freqs(24)
    y = lm.rotary(x, pos, freqs, 1.1, interleaved)
    _within(y, *rotary_reference(x, pos, freqs, 1.1, interleaved))
    assert torch.equal(ops.rotary(x, pos.int(), freqs, 1.1, interleaved), y)
    torch.library.opcheck(ops.rotary.default, (x, pos, freqs, 1.1, interleaved), test_utils=("test_schema", "test_faketensor"))


def rotary_refusals(dev):
    x, pos, f = torch.randn(3, 2, 16, device=dev), torch.arange(3, device=dev), lm.rotary_freqs(16, device=dev)[0]
    for args in ((x.double(), pos, f), (x, pos.float(), f), (x, pos.short(), f), (x, pos, f.float())):
        with pytest.raises(TypeError):
            lm.rotary(*args)
    for args in ((x[0], pos[:2], f), (x, pos[:2], f), (x, pos[None], f), (x, pos, f[None]), (x[..., :14], pos, f), (x, pos, f.to(_other(dev))),
                 (x, pos.to(_other(dev)), f), (torch.randn(1, 1, 4000, device=dev), pos[:1], torch.ones(1025, dtype=torch.float64, device=dev))):
        with pytest.raises(ValueError):
            lm.rotary(*args)


def test_rotary_refusals():
    rotary_refusals("cpu")


# ------------------------------------------------------------------------------ residual_norm
@pytest.mark.parametrize("dtype,stream", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("width,post,gate,weight", [(1, True, "row", True), (129, True, "one", False), (1000, False, "", True)])
def test_norm_host(width, post, gate, weight, dtype, stream):
    args = norm_case(5, width, dtype, stream, post, gate, weight, seed=width)
    for got, want, tol in zip(lm.residual_norm(*args), *norm_reference(*args)):
        _within(got, want, tol)
    for a, b in zip(ops.residual_norm(*args), lm.residual_norm(*args)):
        assert torch.equal(a, b)
    s, y = lm.residual_norm(args[0], weight=args[2])
    assert s is args[0] and y.dtype == args[0].dtype
    empty, same = ops.residual_norm(args[0], None, args[2])
    assert empty.shape == (0,) and torch.equal(same, y)
    for a in (args, (args[0], None, args[2])):
        torch.library.opcheck(ops.residual_norm.default, a, test_utils=("test_schema", "test_faketensor"))


def norm_refusals(dev):
    x, o, w, post, gate, _ = norm_case(4, 32, "bf16", dev=dev)
    for args in ((x.double(), o), (x, o.half()), (x.half(), o), (x, o, w.int()), (x, o, w, post.double()), (x, o, w, post, gate.float())):
        with pytest.raises(TypeError):
            lm.residual_norm(*args)
    for args in ((x, o[:3]), (x, o, w[:3]), (x, o, w, post[None]), (x, o, w, post, gate[:1]), (x, o, w, post, gate[..., :8]),
                 (x, None, w, post), (x, None, w, None, gate), (x[0, 0], None), (x, o.to(_other(dev))), (x, o, w.to(_other(dev))),
                 (torch.zeros(1, 32769, device=dev),)):
        with pytest.raises(ValueError):
            lm.residual_norm(*args)


def test_norm_refusals():
    norm_refusals("cpu")


# ------------------------------------------------------------------------------ the cache
@pytest.mark.parametrize("page,turned,interleaved,dtype", [(16, 32, False, "bf16"), (32, 20, True, "f16")])
def test_append_host(page, turned, interleaved, dtype):
    """Pages are those of the turned keys, in whatever calls the tokens come; the rest of the pool stays."""
    kv, dim, new = 2, 32, [2 * page + 3, 0, 1, page]
    start = random_cache(4, kv, dim, 4 * page, page, dtype, places=4 * page)
    q, k, v = tokens(sum(new), 4, kv, dim, dtype)
    freqs, _ = lm.rotary_freqs(turned)
    lens = _i32(0, 3, page - 1, 5)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    cache = clone(start)
    out = lm.cache_append(cache, lens, k, v, starts, q, freqs, 1.0, interleaved)
    written = set()
    for i, n in enumerate(new):
        at, pos = int(starts[i]), int(lens[i]) + torch.arange(n)
        _within(cache.ktail[i][:, pos].transpose(0, 1), *rotary_reference(k[at:at + n], pos, freqs, 1.0, interleaved))
        _within(out[at:at + n], *rotary_reference(q[at:at + n], pos, freqs, 1.0, interleaved))
        for j in range(int(lens[i]) // page, (int(lens[i]) + n) // page):
            p = int(start.table[i, j])
            written.add(p)
            for c in range(kv):
                cut = slice(j * page, (j + 1) * page)
                for pages, scales, block in ((cache.kpages, cache.kscales, cache.ktail[i, c, cut]), (cache.vpages, cache.vscales, cache.vtail[i, c][:, cut])):
                    whole, scale = page_of(block)
                    assert torch.equal(pages[p, c], whole) and float(scales[p, c]) == float(scale)
    assert len(written) == 4
    rest = [p for p in range(start.kpages.shape[0]) if p not in written]
    for a, b in zip(cache[:4], start[:4]):
        assert torch.equal(a[rest], b[rest])
    other = clone(start)
    ops.cache_append(k, v, *other, lens, starts, q, freqs, 1.0, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(other, cache))
    for args in ((None, None, None), (starts, q, freqs)):
        torch.library.opcheck(ops.cache_append.default, (k[:84] if args[0] is None else k, v[:84] if args[0] is None else v, *clone(start), lens, *args),
                              test_utils=("test_schema", "test_faketensor"))
    small = random_cache(1, kv, dim, 4 * page, page, dtype, places=page)
    want, got = clone(small), clone(small)
    lm.cache_append(want, _i32(0), k[:3 * page], v[:3 * page], None, None, freqs)
    for i in range(3 * page):
        lm.cache_append(got, _i32(i), k[i:i + 1], v[i:i + 1], None, None, freqs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_host_limits():
    page = 16
    start = random_cache(3, 1, 16, 48, page, "bf16")
    start.table[0, 1], start.table[1, 0], start.table[2, 2] = -1, start.kpages.shape[0], 2 ** 31 - 1
    q, k, v = tokens(180, 1, 1, 16, "bf16")
    cache = clone(start)
    lm.cache_append(cache, _i32(-5, 0, 0), k, v)
    assert torch.equal(cache.ktail[:, :, torch.arange(16, 48) % 32], k.view(3, 60, 1, 16)[:, 16:48].transpose(1, 2))
    full = clone(cache)
    lm.cache_append(full, _i32(48, 60, 2 ** 31 - 1), k, v)
    lm.cache_append(full, _i32(0, 0, 0), k, v, _i32(0, 0, 0, 0))
    assert lm.cache_append(full, _i32(0, 0, 0), k[:0], v[:0]) is None
    assert all(torch.equal(a, b) for a, b in zip(full, cache))
    for st in ([5, 3, 200, 190], [-7, 20, 10, 4], [50, 60, 70, 80]):
        out = lm.cache_append(full, _i32(0, 1, 2), k, v, _i32(*st), torch.ones_like(q), lm.rotary_freqs(0)[0])
        assert bool(((out == 0) | (out == 1)).all())
    assert bool((out[50:80] == 1).all()) and bool((out[:50] == 0).all()) and bool((out[80:] == 0).all())
    none = lm.cache8(0, 4, 1, 16, 48, page)
    assert lm.cache_append(none, _i32(), k[:0], v[:0]) is None
    assert lm.attention_cache(torch.zeros(0, 1, 1, 16, dtype=k.dtype), none, _i32()).shape == (0, 1, 1, 16)
    empty = lm.cache8(2, 0, 1, 16, 0, page)
    assert bool((lm.attention_cache(torch.ones(2, 1, 1, 16, dtype=k.dtype), empty, _i32(5, 0)) == 0).all())


@pytest.mark.parametrize("page,dim,n,lens", [(16, 16, 1, [1, 16, 17, 0, 40]), (32, 48, 3, [2, 3, 31, 64, 65])])
def test_attention_host(page, dim, n, lens):
    cache = random_cache(len(lens), 2, dim, 100, page, "bf16")
    q = torch.randn(len(lens), n, 6, dim, generator=torch.Generator().manual_seed(3)).bfloat16()
    o = lm.attention_cache(q, cache, _i32(*lens))
    _within(o, *cache_reference(q, cache, lens))
    assert torch.equal(ops.attention_cache(q, *cache, _i32(*lens)), o)
    torch.library.opcheck(ops.attention_cache.default, (q, *cache, _i32(*lens)), test_utils=("test_schema", "test_faketensor"))
    cache.table[0, 0], cache.table[1, 0], cache.table[-1, 1] = -1, 10 ** 6, -2 ** 31
    _within(lm.attention_cache(q, cache, _i32(*lens), -0.3), *cache_reference(q, cache, lens, -0.3))
    bad = clone(cache)
    for i, length in enumerate(lens):
        gone = [p for p in range(2 * page) if p not in (torch.arange(length // page * page, length) % (2 * page)).tolist()]
        bad.ktail[i][:, gone], bad.vtail[i][:, :, gone] = math.nan, math.inf
    assert torch.equal(lm.attention_cache(q, bad, _i32(*lens)), lm.attention_cache(q, cache, _i32(*lens)))


def cache_refusals(dev):
    cache, lens = random_cache(2, 2, 32, 64, 16, "bf16", dev=dev), torch.tensor([3, 4], dtype=torch.int32, device=dev)
    q, k, v = tokens(6, 4, 2, 32, "bf16", dev=dev)
    st, f = torch.tensor([0, 2, 6], dtype=torch.int32, device=dev), lm.rotary_freqs(32, device=dev)[0]
    lm.cache_append(clone(cache), lens, k, v, st, q, f)
    types = [cache._replace(kpages=cache.kpages.short()), cache._replace(vpages=cache.vpages.to(torch.uint8)),
             cache._replace(kscales=cache.kscales.double()), cache._replace(vscales=cache.vscales.half()),
             cache._replace(ktail=cache.ktail.half()), cache._replace(vtail=cache.vtail.float()), cache._replace(table=cache.table.long())]
    shapes = [cache._replace(kpages=cache.kpages[:3]), cache._replace(vpages=cache.vpages.transpose(2, 3)), cache._replace(kscales=cache.kscales[:, :1]),
              cache._replace(vscales=cache.vscales[None]), cache._replace(ktail=cache.ktail[:1]), cache._replace(vtail=cache.vtail[..., :16]),
              cache._replace(table=cache.table[:1]), cache._replace(table=cache.table[0]), cache._replace(ktail=cache.ktail[:, :, :24], vtail=cache.vtail[..., :24]),
              cache._replace(kpages=cache.kpages.transpose(2, 3).contiguous().transpose(2, 3)), cache._replace(vtail=cache.vtail.to(_other(dev))),
              cache._replace(table=cache.table.to(_other(dev))), cache._replace(kpages=cache.kpages[0]), cache._replace(ktail=cache.ktail[0]),
              cache._replace(kpages=cache.kpages[:, :, :8].contiguous(), vpages=cache.vpages[..., :8].contiguous()),
              cache._replace(kpages=cache.kpages[:0], vpages=cache.vpages[:0], kscales=cache.kscales[:0], vscales=cache.vscales[:0])]
    calls = [lambda c: lm.cache_append(c, lens, k, v), lambda c: lm.attention_cache(q[:2, None], c, lens)]
    for call in calls:
        for c in types:
            with pytest.raises(TypeError):
                call(c)
        for c in shapes:
            with pytest.raises(ValueError):
                call(c)
    for args in ((lens, k.float(), v.float()), (lens, k, v.half()), (lens, k, v, st.long()), (lens, k, v, st, q.half(), f),
                 (lens, k, v, st, q, f.float()), (lens.long(), k, v)):
        with pytest.raises(TypeError):
            lm.cache_append(cache, *args)
    for args in ((lens[:1], k, v), (lens, k[:5], v[:5]), (lens, k, v[:5]), (lens, k[..., :16], v[..., :16]), (lens, k[:, :1], v[:, :1]),
                 (lens, k, v, st[:2]), (lens, k, v, st[None]), (lens, k, v, st, q), (lens, k, v, st, q[:5], f), (lens, k, v, st, q[0], f),
                 (lens, k, v, st, q[..., :16], f), (lens, k, v, st, q[:, :0], f), (lens, k, v, st, q, f.repeat(2)), (lens, k[0], v[0]),
                 (lens, k, v.to(_other(dev))), (lens, k, v, st, q, f.to(_other(dev))), (lens.to(_other(dev)), k, v)):
        with pytest.raises(ValueError):
            lm.cache_append(cache, *args)
    x = q[:2, None]
    with pytest.raises(TypeError):
        lm.attention_cache(x.half(), cache, lens)
    for args in ((q, cache, lens), (x[:1], cache, lens), (x[:, :, :3], cache, lens), (x[..., :16], cache, lens), (x[:, :, :0], cache, lens),
                 (x, cache, lens[:1])):
        with pytest.raises(ValueError):
            lm.attention_cache(*args)
    big = lm.cache8(1, 2, 1, 16, 32, 16, device=dev)
    for kw in (dict(page=24), dict(page=256), dict(dim=20), dict(dim=144), dict(dim=0), dict(dtype=torch.float32), dict(places=24), dict(places=16, page=32)):
        with pytest.raises(ValueError):
            lm.cache8(**{**dict(batch=1, pages=2, kv=1, dim=16, capacity=32, page=16), **kw})
    assert big.ktail.shape == (1, 1, 32, 16) and bool((big.table == -1).all()) and big.table.shape == (1, 2)


def test_cache_refusals():
    cache_refusals("cpu")


def derivatives(dev):
    """None: gradients raise where they are asked for, tangents and the cache's writes at the call."""
    x = torch.randn(4, 2, 16, device=dev).bfloat16()
    cache, lens = random_cache(4, 2, 16, 64, 16, "bf16", dev=dev), torch.full((4,), 20, dtype=torch.int32, device=dev)
    pos, f = torch.arange(4, device=dev), lm.rotary_freqs(16, device=dev)[0]
    calls = {"rotary": lambda t: ops.rotary(t, pos, f), "norm": lambda t: ops.residual_norm(t, x)[1], "sum": lambda t: ops.residual_norm(t, x)[0],
             "block": lambda t: ops.residual_norm(x, t)[0], "attention": lambda t: ops.attention_cache(t[:, None], *cache, lens)}
    for name, call in calls.items():
        want, first = call(x), x.clone().requires_grad_()
        got = call(first)
        assert got.requires_grad and torch.equal(got, want), name
        with pytest.raises(RuntimeError):
            got.float().sum().backward()
        with torch.no_grad():
            assert not call(first).requires_grad
        with torch.inference_mode():
            assert torch.equal(call(x), want)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    append = lambda t, c: ops.cache_append(t, x, *c, lens, None, x, f)  # noqa: E731
    first = x.clone().requires_grad_()
    mine = clone(cache)
    with pytest.raises(NotImplementedError):
        append(first, mine)
    assert all(torch.equal(a, b) for a, b in zip(mine, cache))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        append(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), mine)
    before = [t._version for t in mine[:6]]
    with torch.no_grad():
        q = append(first, mine)
    assert not q.requires_grad and all(t._version > v for t, v in zip(mine[:6], before))
    again = clone(cache)
    with torch.inference_mode():
        assert torch.equal(append(x, again), q)
    assert all(torch.equal(a, b) for a, b in zip(again, mine))


def test_derivatives():
    derivatives("cpu")


def compiled(dev):
    """A step of the operators in one compiled function gives what they give alone, the cache's tensors written."""
    cache, lens = random_cache(3, 2, 16, 64, 16, "bf16", dev=dev), torch.tensor([15, 31, 2], dtype=torch.int32, device=dev)
    q, k, v = tokens(3, 4, 2, 16, "bf16", dev=dev)
    f = lm.rotary_freqs(16, device=dev)[0]

    def step(c):
        turned = ops.cache_append(k, v, *c, lens, None, q, f)
        o = ops.attention_cache(turned[:, None], *c, lens + 1).view(3, 64)
        s, y = ops.residual_norm(o, o * 2)
        return s + 1, ops.rotary(y.view(3, 4, 16), lens, f) * 2

    a, b = clone(cache), clone(cache)
    with torch.no_grad():
        want = step(a)
        got = torch.compile(step, fullgraph=True, backend="inductor" if dev != "cpu" else "aot_eager")(b)
    for x, y in zip((*got, *b), (*want, *a)):
        torch.testing.assert_close(x, y, rtol=0, atol=0)


def test_compiled():
    compiled("cpu")


# ------------------------------------------------------------------------------ the C ABI
def test_entry_point_checks():
    L, p, odd = kernels.lib(), ctypes.c_void_p(16), ctypes.c_void_p(24)
    st = (ctypes.c_int64 * 6)(*[64] * 6)

    def rotary(x=p, dt=1, xt=64, xh=16, pos=p, f=p, half=8, y=p, t=2, h=4, d=16):
        return L.xdna_rotary(x, dt, xt, xh, pos, 0, f, half, 1.0, 0, y, t, h, d, None)

    assert rotary(t=0) == 0 and rotary(h=0) == 0 and rotary(d=0, half=0) == 0
    for bad in (dict(dt=3), dict(half=9), dict(half=-1), dict(half=1025, d=4000), dict(x=None), dict(pos=None), dict(f=None), dict(y=None),
                dict(xt=-1), dict(t=-1), dict(h=1 << 24)):
        assert rotary(**bad) == -1, bad
    assert "rotary" in L.xdna_last_error().decode()

    def norm(x=p, xd=1, o=p, dt=1, gate=None, s=st, inner=1, post=None, pd=0, wd=0, total=p, y=p, rows=2, width=64):
        return L.xdna_residual_norm(x, xd, o, dt, gate, s, inner, post, pd, None, wd, 1.0, 1e-6, total, y, rows, width, None)

    assert norm(rows=0) == 0 and norm(width=0) == 0
    neg = (ctypes.c_int64 * 6)(64, 64, 64, -64, 64, 64)
    for bad in (dict(xd=2), dict(dt=3), dict(pd=3), dict(wd=7), dict(x=None), dict(y=None), dict(total=None), dict(s=None), dict(s=neg), dict(inner=0),
                dict(o=None, gate=p), dict(o=None, post=p), dict(width=32769), dict(rows=-1), dict(rows=1 << 40)):
        assert norm(**bad) == -1, bad

    def append(k=p, v=p, dt=1, s=st, kp=p, vt=p, table=p, lens=p, starts=p, q=None, f=p, half=8, out=p, t=4, b=2, P=4, pages=8, g=16, r=32, nh=4,
               kv=2, d=16):
        return L.xdna_cache_append(k, v, dt, s, kp, p, p, p, p, vt, table, 4, lens, starts, q, f, half, 1.0, 0, out, t, b, P, pages, g, r, nh, kv,
                                   d, None)

    assert append(t=0) == 0
    for bad in (dict(dt=0), dict(k=None), dict(v=None), dict(s=None), dict(kp=None), dict(kp=odd), dict(vt=None), dict(vt=odd), dict(table=None),
                dict(lens=None), dict(starts=None, t=5), dict(f=None), dict(half=9), dict(q=p, out=None), dict(q=p, nh=0), dict(t=-1), dict(g=24),
                dict(r=24), dict(r=1 << 16), dict(d=24), dict(d=144), dict(kv=0), dict(P=1 << 28), dict(pages=-1), dict(b=0, q=p), dict(s=neg)):
        assert append(**bad) == -1, bad

    ws_bytes = L.xdna_attention_cache_ws_bytes
    assert ws_bytes(0, 1, 4, 2, 16, 4, 16) == 0
    for bad in ((1, 1, 3, 2, 16, 4, 16), (1, 1, 4, 2, 20, 4, 16), (1, 1, 4, 2, 16, 4, 48), (-1, 1, 4, 2, 16, 4, 16), (1, -1, 4, 2, 16, 4, 16),
                (1 << 21, 1, 4, 2, 16, 4, 16)):
        assert ws_bytes(*bad) == -1, bad

    def attend(q=p, dt=1, s=st, kp=p, kt=p, table=p, lens=p, b=2, n=1, P=4, pages=8, g=16, r=32, nh=4, kv=2, d=16, out=p):
        return L.xdna_attention_cache(q, dt, s, kp, p, p, p, kt, p, table, 4, lens, b, n, P, pages, g, r, nh, kv, d, 0.25, out, None, 0, None)

    assert attend(b=0) == 0 and attend(n=0) == 0
    uneven = (ctypes.c_int64 * 6)(64, 64, 20, 64, 64, 64)
    for bad in (dict(dt=0), dict(q=None), dict(q=odd), dict(s=None), dict(s=uneven), dict(kp=None), dict(kp=odd), dict(kt=None), dict(table=None),
                dict(lens=None), dict(out=None), dict(out=odd), dict(pages=0), dict(nh=3), dict(d=136), dict(g=8), dict(r=40)):
        assert attend(**bad) == -1, bad
    assert "attention_cache" in L.xdna_last_error().decode()
