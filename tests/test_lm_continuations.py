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
