"""attention_causal and attention_prefix on the MI355X against float64 (lm_reference.py), at the sizes, strides, masks and
values where they can go wrong."""
import math

import pytest
import torch

from lm_reference import causal_case, causal_reference, prefix_case, prefix_reference
from torch_xdna import lm

pytestmark = pytest.mark.gpu


def _within(y, ref):
    want, tol = ref
    y = y.double().cpu()
    assert y.shape == want.shape
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


def _replays(call, want):
    """A captured call, replayed with eager work between the replays, gives the eager result every time."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = call()
        torch.cuda.current_stream().synchronize()
        assert torch.equal(got, want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        out.fill_(7)
        graph.replay()
        assert torch.equal(call(), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------------------ causal
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,h,kv,d", [
    ([1], 1, 1, 8), ([1, 1, 1], 4, 2, 64), ([2, 1], 3, 1, 24), ([31], 2, 2, 128), ([33], 4, 2, 64), ([64, 65], 8, 8, 128),
    ([31, 32, 33, 64, 65, 127, 129], 4, 2, 128), ([300, 5], 7, 1, 96), ([257], 16, 1, 64), ([3, 260, 1, 1, 90], 16, 8, 128),
    ([20] * 40, 4, 2, 64), ([1] * 70, 2, 1, 128), ([0, 17, 0, 0, 40, 0], 4, 4, 64)])
def test_causal(gpu, lens, h, kv, d, dtype):
    q, k, v, starts = causal_case(lens, h, kv, d, dtype, seed=len(lens) + d, dev=gpu)
    _within(lm.attention_causal(q, k, v, starts), causal_reference(q, k, v, lens, d ** -0.5))


@pytest.mark.parametrize("lens,h,kv,d,dtype", [([1300, 1, 801], 16, 8, 128, "bf16"), ([1030, 980, 100], 12, 12, 64, "f16"),
                                               ([30] * 70, 16, 8, 80, "f16"), ([1100, 1000], 12, 12, 40, "bf16"),
                                               ([700], 35, 5, 128, "f16")])
def test_causal_many_rows(gpu, lens, h, kv, d, dtype):
    """Enough rows for the form with 128 of them to a workgroup."""
    q, k, v, starts = causal_case(lens, h, kv, d, dtype, seed=3, dev=gpu)
    _within(lm.attention_causal(q, k, v, starts), causal_reference(q, k, v, lens, d ** -0.5))


@pytest.mark.parametrize("lens,h,kv,d,dtype", [([1600], 16, 8, 128, "bf16"), ([1057, 1300], 12, 12, 64, "f16"), ([1100], 28, 28, 72, "bf16"),
                                               ([2049, 1], 16, 8, 64, "bf16"), ([4000], 1, 1, 128, "f16"), ([7000], 7, 1, 64, "bf16")])
def test_causal_long_rows(gpu, lens, h, kv, d, dtype):
    """Few long sequences: keys shared out between two groups of waves."""
    q, k, v, starts = causal_case(lens, h, kv, d, dtype, seed=4, dev=gpu)
    _within(lm.attention_causal(q, k, v, starts), causal_reference(q, k, v, lens, d ** -0.5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_causal_not_finite_long_rows(gpu, dtype):
    """As test_causal_not_finite, where two groups of waves share out the keys."""
    q, k, v, starts = causal_case([1600], 16, 8, 128, dtype, seed=9, dev=gpu)
    want = lm.attention_causal(q, k, v, starts)
    for at, value in ((1500, math.nan), (1599, math.inf), (70, math.nan)):
        v2 = v.clone()
        v2[at, 2, 9] = value
        got = lm.attention_causal(q, k, v2, starts)
        assert torch.equal(got[:at], want[:at])
        assert torch.equal(got[at:, :4], want[at:, :4]) and torch.equal(got[at:, 6:], want[at:, 6:])
        assert not bool(got[at:, 4:6, 9].isfinite().any())


@pytest.mark.parametrize("t", [100, 2100])
def test_causal_strides(gpu, t):
    """Views of a fused projection, heads outermost, an expanded head, unaligned and reversed-stride layouts."""
    q, k, v, starts = causal_case([t - 40, 40], 16, 8, 64, "bf16", seed=5, dev=gpu)
    want = lm.attention_causal(q, k, v, starts)
    fused = torch.cat([q, k, v], 1)
    assert torch.equal(lm.attention_causal(fused[:, :16], fused[:, 16:24], fused[:, 24:], starts), want)
    assert torch.equal(torch.ops.xdna.attention_causal(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)),
                                                       starts), want)
    odd = torch.full((t, 3 * 64 * 16 + 3), math.nan, dtype=q.dtype, device=gpu)
    odd[:, 1:1 + 64 * 8] = k.reshape(t, -1)
    assert torch.equal(lm.attention_causal(q, odd[:, 1:1 + 64 * 8].view(t, 8, 64), v, starts), want)
    assert torch.equal(lm.attention_causal(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, starts.repeat(2)[:3]), want)
    one = k[:, :1].expand(t, 8, 64)
    assert torch.equal(lm.attention_causal(q, one, v, starts), lm.attention_causal(q, one.contiguous(), v, starts))
    same = k[:1].expand(t, 8, 64)
    assert torch.equal(lm.attention_causal(q, same, v, starts), lm.attention_causal(q, same.contiguous(), v, starts))


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_causal_scales(gpu, scale):
    q, k, v, starts = causal_case([150, 30], 4, 2, 128, "bf16", seed=6, dev=gpu)
    _within(lm.attention_causal(q, k, v, starts, scale), causal_reference(q, k, v, [150, 30], scale))


def test_causal_large_scores(gpu):
    """Scores in the thousands: the maximum is found and taken off before the power."""
    q, k, v, starts = causal_case([200], 2, 2, 64, "f16", seed=7, dev=gpu)
    q, k = q * 30, k * 30
    _within(lm.attention_causal(q, k, v, starts), causal_reference(q, k, v, [200], 64 ** -0.5))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[40, 70, 90], [700, 900, 500]])
def test_causal_not_finite(gpu, lens, dtype):
    """NaN and infinities in keys and values reach the rows that see them and no others."""
    h, kv = 16, 8
    q, k, v, starts = causal_case(lens, h, kv, 64, dtype, seed=8, dev=gpu)
    want = lm.attention_causal(q, k, v, starts)
    t = sum(lens)
    for name, at, value in (("v", lens[0] + 25, math.inf), ("v", lens[0] + 25, math.nan), ("k", lens[0] + 25, math.nan),
                            ("v", t - 1, math.nan), ("v", 0, -math.inf)):
        k2, v2 = k.clone(), v.clone()
        (k2 if name == "k" else v2)[at, 3, 5] = value
        got = lm.attention_causal(q, k2, v2, starts)
        hit = torch.zeros(t, h, dtype=torch.bool, device=gpu)
        end = next(int(e) for e in starts[1:] if int(e) > at)
        hit[at:end, 6:8] = True
        assert torch.equal(got[~hit], want[~hit]), (name, at, value)
        if name == "k":
            assert bool(got[hit].isnan().all())
        else:
            dims = torch.arange(64, device=gpu) != 5
            assert torch.equal(got[hit][:, dims], want[hit][:, dims])
            seen = got[hit][:, 5]
            # a weight that has sunk to zero makes NaN of an infinity, as the formula has it
            assert bool(seen.isnan().all() if math.isnan(value) else ((seen == value) | seen.isnan()).all())


def test_causal_rows_of_minus_infinity(gpu):
    """A row whose every score is -inf is zero; one that also sees another key is not."""
    q, k, v, starts = causal_case([3], 2, 1, 64, "bf16", seed=9, dev=gpu)
    q, k = q.abs(), k.clone()
    k[0] = 0
    k[0, :, 0] = -math.inf
    got = lm.attention_causal(q, k, v, starts)
    assert bool((got[0] == 0).all())
    torch.testing.assert_close(got[1], v[1].expand(2, 64), rtol=0, atol=0)


def test_causal_starts_of_any_value(gpu):
    """What the starts hold reads nothing out of range: each token sees itself at least."""
    for lens in ([50], [2100]):
        q, k, v, starts = causal_case(lens, 16, 8, 128, "bf16", seed=10, dev=gpu)
        want = lm.attention_causal(q, k, v, starts)
        for bad in ([0], [-5, 10 ** 9], [2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, 7] * 9, [40, 3, 20]):
            got = lm.attention_causal(q, k, v, torch.tensor(bad, dtype=torch.int32, device=gpu))
            assert bool(got.isfinite().all()), bad
            if bad in ([0], [-5, 10 ** 9], [2 ** 31 - 1]):
                assert torch.equal(got, want)


def test_causal_empty_stream_and_graph(gpu):
    q, k, v, starts = causal_case([70, 200], 4, 2, 128, "bf16", seed=11, dev=gpu)
    assert lm.attention_causal(q[:0], k[:0], v[:0], starts[:1]).shape == (0, 4, 128)
    want = lm.attention_causal(q, k, v, starts)
    _replays(lambda: lm.attention_causal(q, k, v, starts), want)
    with pytest.raises(RuntimeError):
        torch.ops.xdna.attention_causal(q.clone().requires_grad_(), k, v, starts).float().sum().backward()
    with pytest.raises(ValueError):
        lm.attention_causal(q, k.cpu(), v, starts)


# ------------------------------------------------------------------------------ prefix
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("b,p,s,h,kv,d", [
    (1, 1, 0, 1, 1, 8), (1, 0, 1, 2, 1, 64), (3, 1, 1, 4, 4, 128), (4, 264, 64, 16, 8, 128), (2, 31, 33, 7, 1, 64),
    (1, 1000, 300, 8, 8, 96), (5, 1025, 7, 40, 1, 128), (20, 1200, 50, 16, 8, 128), (70, 1100, 10, 4, 2, 64),
    (2, 0, 1500, 8, 2, 128), (3, 2000, 0, 8, 2, 64), (33, 65, 1100, 2, 1, 64), (1, 3000, 1, 64, 8, 128),
    (9, 700, 20, 40, 1, 72)])
def test_prefix(gpu, b, p, s, h, kv, d, dtype):
    args = prefix_case(b, p, s, h, kv, d, dtype, seed=b + p, dev=gpu)
    _within(lm.attention_prefix(*args), prefix_reference(*args, d ** -0.5))


@pytest.mark.parametrize("p,s", [(100, 60), (1500, 90)])
def test_prefix_strides_and_unseen(gpu, p, s):
    """Caches that are parts of larger ones, with NaN in every slot that no row sees, keys and values interleaved."""
    b, h, kv, d = 5, 8, 4, 64
    q, kp, vp, kc, vc, lens = prefix_case(b, p, s, h, kv, d, "bf16", seed=12, dev=gpu)
    lens[0], lens[1] = 0, s
    want = lm.attention_prefix(q, kp, vp, kc, vc, lens)
    big = torch.full((2, b, kv, s + 37, 2 * d), math.nan, dtype=q.dtype, device=gpu)     # heads before tokens, k | v
    pre = torch.full((p + 50, 2, kv, d), math.nan, dtype=q.dtype, device=gpu)
    pre[:p, 0], pre[:p, 1] = kp, vp
    for i in range(b):
        big[1, i, :, :int(lens[i]), :d] = kc[i, :int(lens[i])].transpose(0, 1)
        big[1, i, :, :int(lens[i]), d:] = vc[i, :int(lens[i])].transpose(0, 1)
    own = big[1].transpose(1, 2)[:, :s]
    got = lm.attention_prefix(q, pre[:p, 0], pre[:p, 1], own[..., :d], own[..., d:], lens)
    assert torch.equal(got, want)
    assert torch.equal(torch.ops.xdna.attention_prefix(q.transpose(0, 1).contiguous().transpose(0, 1), kp, vp, kc, vc,
                                                       lens.repeat_interleave(2)[::2], d ** -0.5), want)
    wide = torch.zeros(b, h, d + 1, dtype=q.dtype, device=gpu)
    wide[..., 1:] = q
    assert torch.equal(lm.attention_prefix(wide[..., 1:], kp, vp, kc, vc, lens), want)
    # lengths past the cache, and below zero, are those of its ends
    lens[1], lens[0] = s + 1000, -3
    assert torch.equal(lm.attention_prefix(q, kp, vp, kc, vc, lens), want)


def test_prefix_nothing_seen(gpu):
    """No prefix and no own keys: a row of zeros."""
    for s in (0, 5, 1500):
        q, kp, vp, kc, vc, lens = prefix_case(3, 0, s, 4, 2, 128, "f16", seed=13, dev=gpu)
        lens.zero_()
        kc.fill_(math.nan)
        vc.fill_(math.nan)
        assert bool((lm.attention_prefix(q, kp, vp, kc, vc, lens) == 0).all())
    assert lm.attention_prefix(q[:0], kp, vp, kc[:0], vc[:0], lens[:0]).shape == (0, 4, 128)


@pytest.mark.parametrize("p", [200, 2000])
def test_prefix_not_finite_stays_in_its_sequence(gpu, p):
    q, kp, vp, kc, vc, lens = prefix_case(6, p, 40, 8, 2, 64, "bf16", seed=14, dev=gpu)
    lens.fill_(40)
    want = lm.attention_prefix(q, kp, vp, kc, vc, lens)
    kc, vc = kc.clone(), vc.clone()
    vc[2, 30, 1, 7], kc[4, 3, 0, 0] = math.inf, math.nan
    got = lm.attention_prefix(q, kp, vp, kc, vc, lens)
    hit = torch.zeros(6, 8, dtype=torch.bool, device=gpu)
    hit[2, 4:], hit[4, :4] = True, True
    assert torch.equal(got[~hit], want[~hit])
    assert bool((got[2, 4:, 7] == math.inf).all()) and bool(got[4, :4].isnan().all())


@pytest.mark.parametrize("p,scale", [(100, -0.25), (3000, 0.3), (3000, 0.0)])
def test_prefix_scales_stream_and_graph(gpu, p, scale):
    args = prefix_case(6, p, 40, 8, 2, 128, "bf16", seed=15, dev=gpu)
    want = lm.attention_prefix(*args, scale)
    _within(want, prefix_reference(*args, scale))
    _replays(lambda: lm.attention_prefix(*args, scale), want)


def test_prefix_offsets_past_32_bits(gpu):
    """Caches whose tokens, and whose sequences, lie so far apart that byte offsets pass 32 bits."""
    p, s, kv, d = 700, 300, 2, 64
    q, kp, vp, kc, vc, lens = prefix_case(2, p, s, 4, kv, d, "bf16", seed=16, dev=gpu)
    want = lm.attention_prefix(q, kp, vp, kc, vc, lens)
    far = torch.empty(p, 1 << 22, dtype=q.dtype, device=gpu)                      # 8 MB from token to token: 5.9 GB
    kf, vf = far[:, :kv * d].view(p, kv, d), far[:, kv * d:2 * kv * d].view(p, kv, d)
    kf.copy_(kp), vf.copy_(vp)
    apart = far.view(-1)[5 << 20:].as_strided((2, s, kv, d), ((p // 2) << 22, 1024, 256, 1))     # 2.9 GB from sequence to sequence
    apart.copy_(kc)
    kf.copy_(kp), vf.copy_(vp)
    assert torch.equal(lm.attention_prefix(q, kf, vf, apart, vc, lens), want)    # the views do not overlap
    assert torch.equal(lm.attention_prefix(q, kf, vf, kc, vc, lens), want)
    c = causal_case([p - 200, 200], 4, kv, d, "bf16", seed=17, dev=gpu)
    kf.copy_(c[1])
    assert torch.equal(lm.attention_causal(c[0], kf, c[2], c[3]), lm.attention_causal(*c))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_caches_of_one_head_after_another(gpu, dtype):
    """Keys and values laid out [heads, tokens, dims]: heads 2^24 elements apart and more are read where they lie, without a
    copy of the cache."""
    b, p, h, kv, d = 2, 131200, 4, 2, 128
    q, kp, vp, kc, vc, lens = prefix_case(b, 300, 8, h, kv, d, dtype, seed=12, dev=gpu)
    want = lm.attention_prefix(q, kp, vp, kc, vc, lens)
    cache = torch.zeros(2, kv, p, d, dtype=q.dtype, device=gpu)
    cache[0, :, -300:], cache[1, :, -300:] = kp.transpose(0, 1), vp.transpose(0, 1)
    k, v = (t[:, -300:].transpose(0, 1) for t in cache)
    assert k.stride(1) > 1 << 24
    assert torch.equal(lm.attention_prefix(q, k, v, kc, vc, lens), want)
    causal = lm.attention_causal(kp.repeat_interleave(2, 1), kp, vp, torch.tensor([0, 300], dtype=torch.int32, device=gpu))
    assert torch.equal(lm.attention_causal(kp.repeat_interleave(2, 1), k, v, torch.tensor([0, 300], dtype=torch.int32, device=gpu)), causal)
    k, v = (t.transpose(0, 1) for t in cache)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = lm.attention_prefix(q, k, v, kc, vc, lens)
    assert torch.cuda.max_memory_allocated() - before < cache.nbytes // 4
    assert torch.equal(out, lm.attention_prefix(q, k.contiguous(), v.contiguous(), kc, vc, lens))
