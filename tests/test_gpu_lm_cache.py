"""The paged 8-bit cache (cache_append, attention_cache) on the MI355X against float64 (lm_cache_reference.py), at the sizes,
masks and contents where it can go wrong."""
import math

import pytest
import torch

from lm_cache_reference import cache_reference, clone, page_of, random_cache, rotary_reference, tokens
from torch_xdna import lm

pytestmark = pytest.mark.gpu


def _within(y, want, tol):
    y, want, tol = y.double().cpu(), want.cpu(), tol.cpu()
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


def _starts(counts, dev):
    return torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32).to(dev)


def _lens(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------ cache_append
@pytest.mark.parametrize("page,kv,heads,dim,turned,interleaved,dtype", [
    (16, 1, 1, 16, 16, False, "bf16"), (16, 2, 6, 48, 20, True, "f16"), (32, 4, 4, 64, 64, True, "bf16"), (64, 2, 14, 96, 96, False, "f16"),
    (64, 8, 16, 128, 128, False, "bf16"), (128, 3, 3, 128, 114, False, "bf16"), (128, 2, 2, 80, 0, False, "f16"),
    (128, 1, 4, 128, 2, True, "f16")])
def test_append(gpu, page, kv, heads, dim, turned, interleaved, dtype):
    """Ragged texts into caches that hold tokens already: the ring is wide enough to show every key as it was turned, pages are
    exactly those of the ring's values, and nothing else changes."""
    old, new = [0, 5, page - 1, page, 2 * page + 3, 7], [page + 2, 1, 1, 2 * page, 0, 3 * page - 7]
    before = random_cache(6, kv, dim, 6 * page, page, dtype, places=6 * page, seed=page + dim, dev=gpu)
    cache = clone(before)
    q, k, v = tokens(sum(new) + 2, heads, kv, dim, dtype, seed=dim, dev=gpu)          # two tokens of no text
    freqs, magnitude = lm.rotary_freqs(turned, factor=4.0, original=512, device=gpu)
    out = lm.cache_append(cache, _lens(old, gpu), k, v, _starts(new, gpu), q, freqs, magnitude, interleaved)
    starts, written = [0] + torch.tensor(new).cumsum(0).tolist(), set()
    kt, vt = before.ktail.cpu(), before.vtail.cpu()
    for i, (o, n) in enumerate(zip(old, new)):
        rows, pos = slice(starts[i], starts[i] + n), torch.arange(o, o + n)
        _within(out[rows], *rotary_reference(q[rows], pos, freqs, magnitude, interleaved))
        want, tol = rotary_reference(k[rows], pos, freqs, magnitude, interleaved)
        _within(cache.ktail[i][:, o:o + n].transpose(0, 1), want, tol)
        kt[i][:, o:o + n] = cache.ktail[i][:, o:o + n].cpu()
        vt[i][:, :, o:o + n] = v[rows].permute(1, 2, 0).cpu()
        for j in range(o // page, (o + n) // page):
            at, cut = int(before.table[i, j]), slice(j * page, (j + 1) * page)
            written.add(at)
            for c in range(kv):
                for pages, scales, block in ((cache.kpages, cache.kscales, cache.ktail[i, c, cut]),
                                             (cache.vpages, cache.vscales, cache.vtail[i, c][:, cut])):
                    whole, scale = page_of(block)
                    assert torch.equal(pages[at, c].cpu(), whole) and float(scales[at, c]) == float(scale), (i, j, c)
    assert torch.equal(cache.ktail.cpu(), kt) and torch.equal(cache.vtail.cpu(), vt)
    rest = [p for p in range(before.kpages.shape[0]) if p not in written]
    for a, b in zip(cache[:4], before[:4]):
        assert torch.equal(a[rest], b[rest])
    assert torch.equal(cache.table, before.table)
    assert bool((out[starts[-1]:] == 0).all())


@pytest.mark.parametrize("page,places,dtype,interleaved", [(16, 16, "bf16", False), (16, 48, "f16", True), (32, 64, "bf16", True),
                                                            (64, 64, "bf16", False), (128, 128, "f16", False)])
def test_append_does_not_depend_on_the_calls(gpu, page, places, dtype, interleaved):
    """All at once, in chunks that end anywhere, longer than the ring among them, and token by token: the same bits."""
    total, kv, dim = 3 * page + 5, 2, 64
    start = random_cache(2, kv, dim, 4 * page, page, dtype, places=places, dev=gpu)
    q, k, v = tokens(2 * total, 4, kv, dim, dtype, seed=page, dev=gpu)
    q, k, v = (t.reshape(2, total, -1, dim) for t in (q, k, v))
    freqs, _ = lm.rotary_freqs(48, device=gpu)

    def put(cuts):
        cache, at, out = clone(start), 0, []
        for n in cuts:
            part = [t[:, at:at + n].reshape(2 * n, -1, dim) for t in (k, v, q)]
            out.append(lm.cache_append(cache, _lens([at, at], gpu), part[0], part[1], None, part[2], freqs, 1.0, interleaved).view(2, n, 4, dim))
            at += n
        assert at == total
        return (*cache, torch.cat(out, 1))

    want = put([total])
    for cuts in ([1] * total, [page - 1, 2 * page + 6], [page + 3, 1, 2 * page + 1], [5, total - 5], [page, page, page, 5], [7, page - 7, total - page]):
        for a, b in zip(put(cuts), want):
            assert torch.equal(a, b), cuts


def test_append_back_and_again(gpu):
    """A length that goes back by R - G tokens and new tokens there: as if the others had never come."""
    page, kv, dim = 16, 2, 32
    start = random_cache(1, kv, dim, 128, page, "bf16", places=3 * page, dev=gpu)
    _, k, v = tokens(100, 1, kv, dim, "bf16", seed=2, dev=gpu)
    for first in (33, 37, 48, 50):
        a, b = clone(start), clone(start)
        back = first - 2 * page
        for c in (a, b):
            lm.cache_append(c, _lens([0], gpu), k[:back], v[:back])
        lm.cache_append(a, _lens([back], gpu), k[60:60 + first - back], v[60:60 + first - back])      # drafts
        for c in (a, b):
            lm.cache_append(c, _lens([back], gpu), k[back:60], v[back:60])
        whole = [int(p) for p in start.table[0, :60 // page]]
        for x, y in zip(a[:4], b[:4]):
            assert torch.equal(x[whole], y[whole])
        at = torch.arange(60 // page * page, 60) % (3 * page)
        assert torch.equal(a.ktail[:, :, at], b.ktail[:, :, at]) and torch.equal(a.vtail[..., at], b.vtail[..., at])


def test_append_bad_pages_and_limits(gpu):
    """Pages outside the pool are not written, tokens past the capacity dropped, negative lengths are 0, any starts are read in
    range; an empty call does nothing."""
    page, kv, dim = 16, 2, 32
    start = random_cache(3, kv, dim, 48, page, "bf16", dev=gpu)
    start.table[0, 1], start.table[1, 0], start.table[2, 2] = -1, start.kpages.shape[0], 2 ** 31 - 1
    _, k, v = tokens(3 * 60, 1, kv, dim, "bf16", seed=3, dev=gpu)
    cache = clone(start)
    lm.cache_append(cache, _lens([-5, 0, 0], gpu), k, v)
    for i in range(3):
        for j in range(3):
            at = int(start.table[i, j])
            if 0 <= at < start.kpages.shape[0]:
                for c in range(kv):
                    whole, scale = page_of(k[60 * i + page * j:60 * i + page * (j + 1), c])
                    assert torch.equal(cache.kpages[at, c].cpu(), whole) and float(cache.kscales[at, c]) == float(scale)
    used = {int(p) for p in start.table.flatten()}
    rest = [p for p in range(start.kpages.shape[0]) if p not in used]
    for a, b in zip(cache[:4], start[:4]):
        assert torch.equal(a[rest], b[rest])
    # 48 tokens fit: the ring (32 places) has the last 32 of them
    assert torch.equal(cache.ktail[:, :, torch.arange(16, 48) % 32], k.view(3, 60, kv, dim)[:, 16:48].transpose(1, 2))
    full = clone(cache)
    lm.cache_append(full, _lens([48, 60, 2 ** 31 - 1], gpu), k, v)
    for a, b in zip(full, cache):
        assert torch.equal(a, b)
    lm.cache_append(full, _lens([0, 0, 0], gpu), k[:0], v[:0])
    lm.cache_append(full, _lens([0, 0, 0], gpu), k, v, _starts([0, 0, 0], gpu))
    for a, b in zip(full, cache):
        assert torch.equal(a, b)
    q = torch.ones(180, 1, dim, dtype=k.dtype, device=gpu)
    for st in ([5, 3, 200, 190], [-7, 20, 10, 4], [180, 180, 180, 180], [100, 110, 105, 2 ** 31 - 1], [50, 60, 70, 80]):
        out = lm.cache_append(full, _lens([0, 1, 2], gpu), k, v, _lens(st, gpu), q, lm.rotary_freqs(0, device=gpu)[0])
        assert bool(((out == 0) | (out == 1)).all())
    assert bool((out[50:80] == 1).all()) and bool((out[:50] == 0).all()) and bool((out[80:] == 0).all())
    # ascending starts that begin late: text b's tokens are its own
    fresh = clone(start)
    lm.cache_append(fresh, _lens([0, 0, 0], gpu), k, v, _lens([50, 60, 70, 80], gpu))
    for i in range(3):
        assert torch.equal(fresh.ktail[i][:, :10].transpose(0, 1), k[50 + 10 * i:60 + 10 * i])


def test_append_many_texts(gpu):
    """More texts than a wave has lanes, empty ones among them."""
    page, kv, dim = 16, 1, 16
    counts = [(7 * i) % 23 for i in range(150)]
    cache = random_cache(150, kv, dim, 32, page, "f16", dev=gpu)
    q, k, v = tokens(sum(counts), 1, kv, dim, "f16", dev=gpu)
    old = [i % 9 for i in range(150)]
    freqs, _ = lm.rotary_freqs(dim, device=gpu)
    out = lm.cache_append(cache, _lens(old, gpu), k, v, _starts(counts, gpu), q, freqs)
    at = 0
    for i, (o, n) in enumerate(zip(old, counts)):
        want, tol = rotary_reference(k[at:at + n], torch.arange(o, o + n), freqs)
        _within(cache.ktail[i][:, o:o + n].transpose(0, 1), want, tol)
        _within(out[at:at + n], *rotary_reference(q[at:at + n], torch.arange(o, o + n), freqs))
        assert torch.equal(cache.vtail[i][:, :, o:o + n], v[at:at + n].permute(1, 2, 0))
        at += n


def test_append_values(gpu):
    """Zeros, the smallest and largest values, infinities and NaN."""
    page, kv, dim = 16, 1, 16
    for dtype in (torch.bfloat16, torch.float16):
        k = torch.randn(page * 6, kv, dim, dtype=torch.float32).to(dtype)
        k[:page] = 0
        k[page:2 * page] = torch.where(k[page:2 * page] > 0, 1, -1) * torch.finfo(dtype).smallest_normal * 2.0 ** -7
        k[2 * page:3 * page] *= torch.finfo(dtype).max / 8
        k[3 * page, 0, 3], k[4 * page + 1, 0, 5] = math.inf, math.nan
        k[5 * page, 0, 0] = -torch.finfo(dtype).max
        k = k.to(gpu)
        cache = random_cache(1, kv, dim, 6 * page, page, "bf16" if dtype == torch.bfloat16 else "f16", dev=gpu)
        lm.cache_append(cache, _lens([0], gpu), k, k)
        for j in range(6):
            at = int(cache.table[0, j])
            whole, scale = page_of(k[j * page:(j + 1) * page, 0])
            assert torch.equal(cache.kpages[at, 0].cpu(), whole) and torch.equal(cache.vpages[at, 0].cpu(), whole.t())
            for s in (cache.kscales, cache.vscales):
                assert float(s[at, 0]) == float(scale) or (math.isnan(float(s[at, 0])) and math.isnan(float(scale)))
        o = lm.attention_cache(torch.ones(1, 1, 1, dim, dtype=dtype, device=gpu), cache, _lens([page], gpu))
        assert bool((o == 0).all())
        for n in (4 * page, 5 * page, 6 * page):
            assert bool(lm.attention_cache(torch.ones(1, 1, 1, dim, dtype=dtype, device=gpu), cache, _lens([n], gpu)).isnan().all())


def test_append_strides(gpu):
    """Heads before tokens, unaligned rows, expanded values."""
    page, kv, dim = 32, 2, 48
    start = random_cache(2, kv, dim, 64, page, "bf16", dev=gpu)
    q, k, v = tokens(80, 4, kv, dim, "bf16", dev=gpu)
    freqs, _ = lm.rotary_freqs(20, device=gpu)
    want = clone(start)
    out = lm.cache_append(want, _lens([3, 9], gpu), k, v, None, q, freqs)

    def odd(t):
        x = torch.zeros(t.shape[1], t.shape[0], dim + 3, dtype=t.dtype, device=gpu)
        x[..., 3:] = t.transpose(0, 1)
        return x[..., 3:].transpose(0, 1)

    for args in ((odd(k), odd(v), odd(q)), (k.flip(-1).flip(-1), v.transpose(1, 2).contiguous().transpose(1, 2), q.contiguous())):
        got = clone(start)
        assert torch.equal(lm.cache_append(got, _lens([3, 9], gpu), args[0], args[1], None, args[2], freqs), out)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    one = v[:, :1].expand(80, kv, dim)
    a, b = clone(start), clone(start)
    lm.cache_append(a, _lens([3, 9], gpu), k, one)
    lm.cache_append(b, _lens([3, 9], gpu), k, one.contiguous())
    assert torch.equal(a.vpages, b.vpages) and torch.equal(a.vtail, b.vtail)


# ------------------------------------------------------------------------------ attention_cache
def _query(b, n, h, d, dtype, gpu, seed=1):
    return torch.randn(b, n, h, d, generator=torch.Generator().manual_seed(seed)).to({"bf16": torch.bfloat16, "f16": torch.float16}[dtype]).to(gpu)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,kv,group,dim,n,lens", [
    (16, 1, 1, 16, 1, [1, 2, 15, 16, 17, 33, 0]), (16, 2, 3, 64, 2, [1, 2, 3, 63, 64, 65, 200]), (32, 1, 16, 48, 1, [31, 32, 96, 97, 500]),
    (32, 4, 7, 96, 5, [3, 5, 64, 260, 700]), (64, 8, 2, 128, 1, [64, 63, 65, 129, 1000]), (64, 2, 8, 80, 3, [1, 190, 192, 300]),
    (128, 4, 8, 64, 1, [127, 128, 129, 2000]), (128, 1, 71, 128, 1, [5, 255, 513]), (128, 2, 4, 112, 20, [10, 130, 400])])
def test_attention(gpu, page, kv, group, dim, n, lens, dtype):
    cache = random_cache(len(lens), kv, dim, max(lens) + page, page, dtype, seed=page + dim, dev=gpu)
    q = _query(len(lens), n, kv * group, dim, dtype, gpu)
    o = lm.attention_cache(q, cache, _lens(lens, gpu))
    assert o.dtype == q.dtype and o.shape == q.shape
    _within(o, *cache_reference(q, cache, lens))
    assert torch.equal(o, lm.attention_cache(q, cache, _lens(lens, gpu)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_long(gpu, dtype):
    """Texts that many workgroups share out, next to short and empty ones in a table as wide."""
    lens = [20000, 1, 0, 777]
    cache = random_cache(4, 2, 64, 20000, 64, dtype, dev=gpu)
    q = _query(4, 1, 8, 64, dtype, gpu)
    _within(lm.attention_cache(q, cache, _lens(lens, gpu)), *cache_reference(q, cache, lens))
    q = _query(4, 6, 8, 64, dtype, gpu)
    _within(lm.attention_cache(q, cache, _lens(lens, gpu), 0.3), *cache_reference(q, cache, lens, 0.3))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_scales(gpu, dtype):
    """Values' scales that grow and fall by powers of ten from page to page, scales of zero, and the softmax's scale: none, zero,
    negative."""
    for seed in range(8):
        page, g = (16, 32, 64, 128)[seed % 4], torch.Generator().manual_seed(seed)
        cache = random_cache(2, 2, 32, 400, page, dtype, seed=seed, dev=gpu)
        cache.vscales.copy_(10.0 ** torch.randint(-6, 3, cache.vscales.shape, generator=g))
        cache.vscales[::5] = 0
        cache.kscales[::7] = 0
        q = _query(2, 2, 4, 32, dtype, gpu, seed=seed)
        lens = [390, 401]
        for scale in (None, 0.0, -0.2, 1e-3, 1.5):
            _within(lm.attention_cache(q, cache, _lens(lens, gpu), scale), *cache_reference(q, cache, lens, scale))
    tiny = cache._replace(vscales=torch.full_like(cache.vscales, 1e-30))
    # under the open page's values such a page is next to nothing; without it, it is all there is
    for n in ([384, 400], [390, 395]):
        if dtype == "bf16":
            _within(lm.attention_cache(q, tiny, _lens(n, gpu)), *cache_reference(q, tiny, n))


def test_attention_unseen(gpu):
    """What no row sees does not matter: places behind the last token, pages past it, pages that are none; nor what some rows do
    not see to those: keys and values that are not finite."""
    page, dim = 16, 32
    lens = [37, 50, 5]
    for dtype, dt in (("bf16", torch.bfloat16), ("f16", torch.float16)):
        cache = random_cache(3, 2, dim, 64, page, dtype, dev=gpu)
        q = _query(3, 4, 4, dim, dtype, gpu)
        want = lm.attention_cache(q, cache, _lens(lens, gpu))
        bad = clone(cache)
        for i, n in enumerate(lens):
            keep = torch.arange(n // page * page, n) % 32
            gone = [p for p in range(32) if p not in keep.tolist()]
            bad.ktail[i][:, gone], bad.vtail[i][:, :, gone] = math.nan, math.inf
            bad.table[i, n // page:] = torch.tensor([-1, 10 ** 9, -2 ** 31, 2 ** 31 - 1][:4 - n // page], dtype=torch.int32)
        used = {int(p) for i, n in enumerate(lens) for p in cache.table[i, :n // page]}
        rest = [p for p in range(cache.kpages.shape[0]) if p not in used]
        bad.kscales[rest], bad.vscales[rest] = math.nan, math.inf
        assert torch.equal(lm.attention_cache(q, bad, _lens(lens, gpu)), want)
        # a page that is none is left out
        holes = clone(cache)
        holes.table[0, 1], holes.table[1, 0], holes.table[1, 2] = -3, cache.kpages.shape[0], 2 ** 30
        _within(lm.attention_cache(q, holes, _lens(lens, gpu)), *cache_reference(q, holes, lens))
        # the last token's key and value, which only the last row sees
        last = clone(cache)
        for i, n in enumerate(lens):
            last.ktail[i][:, (n - 1) % 32, 3], last.vtail[i][0, 5, (n - 1) % 32] = math.nan, math.inf
        o = lm.attention_cache(q, last, _lens(lens, gpu))
        assert torch.equal(o[:, :3], want[:, :3]) and bool(o[:, 3].isnan().all())
        last = clone(cache)
        for i, n in enumerate(lens):
            last.vtail[i][0, 5, (n - 1) % 32], last.vtail[i][1, 7, (n - 2) % 32] = math.inf, -math.inf
        o = lm.attention_cache(q, last, _lens(lens, gpu))
        assert torch.equal(o[:, :2], want[:, :2])
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[:, 3, :2, 5] = hit[:, 2:, 2:, 7] = True
        assert bool((o[:, 3, :2, 5] == math.inf).all()) and bool((o[:, 2:, 2:, 7] == -math.inf).all())
        torch.testing.assert_close(o[~hit], want[~hit], rtol=0, atol=0)


def test_attention_strides_streams_and_graphs(gpu):
    cache = random_cache(3, 2, 64, 300, 32, "bf16", dev=gpu)
    lens = _lens([300, 129, 64], gpu)
    q = _query(3, 2, 6, 64, "bf16", gpu)
    want = lm.attention_cache(q, cache, lens)
    wide = torch.zeros(3, 2, 11, 64 + 8, dtype=q.dtype, device=gpu)
    wide[:, :, 3:9, 8:] = q
    odd = torch.zeros(3, 2, 6, 64 + 1, dtype=q.dtype, device=gpu)
    odd[..., 1:] = q
    for x in (wide[:, :, 3:9, 8:], odd[..., 1:], q.permute(1, 3, 0, 2).contiguous().permute(2, 0, 3, 1), q[:, :1].expand(3, 2, 6, 64)):
        ref = want if x.stride(1) else lm.attention_cache(x.contiguous(), cache, lens)
        assert torch.equal(lm.attention_cache(x, cache, lens), ref)
    table = torch.full((3, 40), -1, dtype=torch.int32, device=gpu)
    table[:, :20:2] = cache.table
    assert torch.equal(lm.attention_cache(q, cache._replace(table=table[:, ::2][:, :10]), lens), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lm.attention_cache(q, cache, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    # a step of appending and attending in a graph, replayed over growing texts, against the same calls outside
    freqs, _ = lm.rotary_freqs(64, device=gpu)
    qs, k, v = tokens(3, 6, 2, 64, "bf16", dev=gpu)
    qs, k, v, n = qs.clone(), k.clone(), v.clone(), _lens([14, 62, 31], gpu)

    def step(c):
        turned = lm.cache_append(c, n, k, v, None, qs, freqs)
        return lm.attention_cache(turned[:, None], c, n + 1)

    eager, replayed = clone(cache), clone(cache)
    scratch = clone(cache)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(scratch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(replayed)
    for x, y in zip(replayed, cache):
        x.copy_(y)
    for i in range(20):
        for t in (qs, k, v):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(i)))
        ref = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref), i
        for x, y in zip(eager, replayed):
            assert torch.equal(x, y), i
        n += 1


@pytest.mark.parametrize("b,n,group,kv,dim,page,longest", [(1, 30, 4, 2, 64, 64, 3000), (1, 150, 3, 1, 128, 32, 700), (2, 40, 1, 3, 96, 16, 5000),
                                                           (3000, 1, 2, 1, 32, 16, 40), (300, 2, 3, 4, 128, 64, 300), (40, 1, 4, 8, 128, 64, 5000)])
def test_attention_blocks_and_parts(gpu, b, n, group, kv, dim, page, longest):
    """Several blocks of rows, parts of keys, both, and as many texts as make four waves a workgroup: some rows of each."""
    g = torch.Generator().manual_seed(b + n)
    lens = torch.randint(0, longest + 1, (b,), generator=g).tolist()
    cache = random_cache(b, kv, dim, longest, page, "bf16", seed=n, dev=gpu)
    q = _query(b, n, kv * group, dim, "bf16", gpu)
    o = lm.attention_cache(q, cache, _lens(lens, gpu))
    some = list(range(b))[::max(1, b // 7)]
    part = cache._replace(ktail=cache.ktail[some], vtail=cache.vtail[some], table=cache.table[some])
    _within(o[some], *cache_reference(q[some], part, [lens[i] for i in some]))
    # every text alone, split another way: the same up to the order of sums
    if b <= 300:
        for i in some:
            one = cache._replace(ktail=cache.ktail[i:i + 1], vtail=cache.vtail[i:i + 1], table=cache.table[i:i + 1])
            torch.testing.assert_close(lm.attention_cache(q[i:i + 1], one, _lens(lens[i:i + 1], gpu)), o[i:i + 1], rtol=2 ** -6, atol=2 ** -6)


@pytest.mark.parametrize("seed", range(24))
def test_random_steps(gpu, seed):
    """Texts of any lengths get a few tokens each, then all of them attend: the cache's own contents in float64 beside it."""
    g = torch.Generator().manual_seed(seed)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=g))]  # noqa: E731
    page, kv, dim, group, dtype = pick(16, 32, 64, 128), pick(1, 2, 3, 8), pick(16, 32, 48, 64, 80, 96, 112, 128), pick(1, 2, 5, 8, 16, 17), pick("bf16", "f16")
    b, n = pick(1, 2, 5, 9), pick(1, 1, 2, 3, 7)
    old = [int(v) for v in torch.randint(0, pick(3 * page, 900, 2500), (b,), generator=g)]
    cache = random_cache(b, kv, dim, max(old) + n, page, dtype, places=page * pick(1, 2, 3), seed=seed, dev=gpu)
    q, k, v = tokens(b * n, kv * group, kv, dim, dtype, seed=seed, dev=gpu)
    freqs, magnitude = lm.rotary_freqs(dim // 2 // 2 * 2, factor=pick(1.0, 4.0), original=2048, device=gpu)
    inter = pick(False, True)
    turned = lm.cache_append(cache, _lens(old, gpu), k, v, None, q, freqs, magnitude, inter)
    pos = torch.cat([torch.arange(o, o + n) for o in old])
    _within(turned, *rotary_reference(q, pos, freqs, magnitude, inter))
    want = rotary_reference(k, pos, freqs, magnitude, inter)
    ring = torch.cat([cache.ktail[i][:, torch.arange(o, o + n) % cache.ktail.shape[2]].transpose(0, 1) for i, o in enumerate(old)])
    if n <= cache.ktail.shape[2]:
        _within(ring, *want)
    lens = [o + n for o in old]
    o = lm.attention_cache(turned.view(b, n, kv * group, dim), cache, _lens(lens, gpu))
    _within(o, *cache_reference(turned.view(b, n, kv * group, dim), cache, lens))


def test_far_pages(gpu):
    """Pages past 2^32 bytes of the pool are written and read where they lie."""
    page, kv, dim = 64, 8, 128
    pages = 70000                                      # 4.6 GB each of keys and values
    c = lm.cache8(1, 0, kv, dim, 0, page, device=gpu)
    cache = lm.Cache8(torch.empty(pages, kv, page, dim, dtype=torch.int8, device=gpu), torch.empty(pages, kv, dim, page, dtype=torch.int8, device=gpu),
                      torch.zeros(pages, kv, device=gpu), torch.zeros(pages, kv, device=gpu), c.ktail, c.vtail,
                      torch.tensor([[69999, 3, 66000, 40000]], dtype=torch.int32, device=gpu))
    small = random_cache(1, kv, dim, 256, page, "bf16", dev=gpu, spare=0)
    small = small._replace(ktail=torch.zeros_like(c.ktail), vtail=torch.zeros_like(c.vtail))
    q, k, v = tokens(200, 16, kv, dim, "bf16", dev=gpu)
    for x in (cache, small):
        lm.cache_append(x, _lens([0], gpu), k, v)
    a, b = (lm.attention_cache(q[None, -1:], x, _lens([200], gpu)) for x in (cache, small))
    assert torch.equal(a, b)


def test_refusals_derivatives_and_compiled(gpu):
    import test_lm_host_cache as host

    host.rotary_refusals(gpu)
    host.norm_refusals(gpu)
    host.cache_refusals(gpu)
    host.derivatives(gpu)
    host.compiled(gpu)
    x = torch.zeros(2 * 16 * 2 * 32 + 16, dtype=torch.int8, device=gpu)
    cache = random_cache(1, 2, 32, 32, 16, "bf16", dev=gpu, spare=0)
    with pytest.raises(ValueError):
        lm.attention_cache(_query(1, 1, 2, 32, "bf16", gpu), cache._replace(kpages=x[8:8 + 2048].view(2, 2, 16, 32)), _lens([3], gpu))
