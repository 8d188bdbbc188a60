"""The operators together: a prompt's continuations step by step against the whole sequences at once."""
import pytest
import torch

from torch_xdna import continuations as C


def _check(dev, **sizes):
    torch.manual_seed(0)
    model = C.Decoder(**sizes).to(dev)
    prompt = torch.randint(0, model.vocab, (37,)).to(torch.int32).to(dev)
    batch, steps = 3, 6
    odd = torch.full((-(-model.vocab // 32),), -1431655766, dtype=torch.int32, device=dev)       # 0xaaaaaaaa: odd tokens only
    out = C.continuations(model, prompt, batch, steps, allowed=odd)
    assert out.shape == (batch, steps) and bool((out % 2 == 1).all()) and bool((out < model.vocab).all())
    assert len(set(out[:, 0].tolist())) == batch
    assert torch.equal(out, C.continuations(model, prompt, batch, steps, allowed=odd))
    # the same logits from all sequences, packed, in one pass: two routes of bfloat16 roundings through the layers
    with torch.no_grad():
        whole = torch.cat([torch.cat([prompt, row]) for row in out])
        n = prompt.shape[0] + steps
        starts = torch.arange(0, n * batch + 1, n, dtype=torch.int32, device=dev)
        want, _ = model.prefill(whole, starts)
        want = want.view(batch, n, -1)[:, prompt.shape[0] - 1:-1]
        logits, prefix = model.prefill(prompt)
        own = [tuple(torch.zeros(batch, steps, *t.shape[1:], dtype=t.dtype, device=dev) for t in kv) for kv in prefix]
        got = [logits[-1:].expand(batch, -1)]
        for i in range(steps - 1):
            got.append(model.step(out[:, i], prefix, own, torch.full((batch,), i, dtype=torch.int32, device=dev)))
        got = torch.stack(got, 1)
    err = (got.float() - want.float()).norm() / want.float().norm()
    assert err < 0.02, err


def test_continuations_host():
    _check("cpu", vocab=300, width=128, layers=2, heads=4, kv=2, dim=32, inner=192)


@pytest.mark.gpu
def test_continuations(gpu):
    _check(gpu)
    _check(gpu, vocab=1001, width=256, layers=3, heads=6, kv=1, dim=64, inner=512, dtype=torch.float16)


def _small(**sizes):
    return C.Decoder(**{**dict(vocab=300, width=128, layers=1, heads=4, kv=2, dim=32, inner=64), **sizes})


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_fewer_tokens_allowed_than_continuations(device):
    """Every token is one that may be chosen, also where fewer may than there are continuations (or tokens at all): the
    others begin with the likeliest."""
    torch.manual_seed(0)
    model = _small().to(device)
    prompt = torch.randint(0, 300, (11,)).to(torch.int32).to(device)
    for tokens in ([5], [299], [5, 64, 200]):
        allowed = torch.zeros(10, dtype=torch.int64)
        for t in tokens:
            allowed[t // 32] |= 1 << t % 32
        allowed = allowed.to(torch.int32).to(device)
        out = C.continuations(model, prompt, 5, 4, allowed=allowed)
        assert set(out.flatten().tolist()) <= set(tokens)
        first = out[:, 0].tolist()
        assert set(first) == set(tokens) and first[len(tokens):] == first[:1] * (5 - len(tokens))
    out = C.continuations(_small(vocab=3).to(device), prompt % 3, 5, 2)
    assert set(out[:, 0].tolist()) == {0, 1, 2} and bool((out < 3).all())


def test_no_token_allowed():
    model, prompt = _small(), torch.arange(7, dtype=torch.int32)
    none = torch.zeros(10, dtype=torch.int32)
    with pytest.raises(ValueError):
        C.continuations(model, prompt, 2, 3, allowed=none)
    none[9] = -1 << 12                                  # tokens 300 .. 319, which there are not
    with pytest.raises(ValueError):
        C.continuations(model, prompt, 2, 3, allowed=none)
    none[9] = 1 << 11
    assert bool((C.continuations(model, prompt, 2, 3, allowed=none) == 299).all())
