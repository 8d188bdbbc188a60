"""The operators over the paged 8-bit cache together: texts step by step against the whole texts at once."""
import pytest
import torch

from torch_xdna import serving as S


def _prompts(vocab, lengths, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).to(torch.int32).to(dev) for n in lengths]


def _check(dev, page, **sizes):
    model = S.Server(**sizes).to(dev)
    lengths, steps = [37, 1, 2 * page, page - 1], 5
    prompts = _prompts(model.vocab, lengths, dev)
    out = S.serve(model, prompts, steps, page)
    assert out.shape == (4, steps) and bool(((out >= 0) & (out < model.vocab)).all())
    assert torch.equal(out, S.serve(model, prompts, steps, page))
    # each alone: the batch changes nothing but the order of sums
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(dev)
    with torch.no_grad():
        texts = S.Texts(model, 4, max(lengths) + steps, page, device=dev)
        for i, n in enumerate(lengths):
            texts.reserve(i, n + steps)
        logits = [model.start(texts, torch.cat(prompts), starts)[starts[1:].long() - 1]]
        for i in range(steps - 1):
            logits.append(model.step(texts, out[:, i:i + 1])[:, 0])
        got = torch.stack(logits, 1)
        # the same tokens as one draft of steps - 1: each row sees what it saw before, from the same cache in the end
        again = S.Texts(model, 4, max(lengths) + steps, page, device=dev)
        for i, n in enumerate(lengths):
            again.reserve(i, n + steps)
        model.start(again, torch.cat(prompts), starts)
        draft = model.step(again, out[:, :steps - 1])
        # and all at once in 16 bits, without a cache
        whole = [torch.cat([p, row]) for p, row in zip(prompts, out)]
        ends = torch.tensor([0] + [w.shape[0] for w in whole]).cumsum(0).to(torch.int32).to(dev)
        empty = S.Texts(model, 4, max(lengths) + steps, page, device=dev)
        for i, w in enumerate(whole):
            empty.reserve(i, w.shape[0])
        want = model.start(empty, torch.cat(whole), ends)
        want = torch.stack([want[int(e) - steps - 1:int(e) - 1] for e in ends[1:]])
    assert torch.equal(texts.lens.cpu(), torch.tensor(lengths, dtype=torch.int32) + steps - 1)
    # a page's values are off by up to half of 1 / 127 of its largest, 0.8% of them in the mean where that is 3.5 times their rms:
    # with the softmax's weights' the same through keys, 1.1% of what attention adds in a layer, and bfloat16's roundings
    for a, b in ((draft, got[:, 1:]), (got, want)):
        err = (a.float() - b.float()).norm() / b.float().norm()
        assert err < 0.05, err
    pages = 4 * texts.columns
    texts.release(2)
    texts.reserve(2, 3)
    assert sorted(texts.free + sum(texts.given, [])) == list(range(pages)) and len(texts.given[2]) == 1
    assert texts.layers[-1].table[2].tolist() == texts.given[2] + [-1] * (texts.columns - 1) and int(texts.lens[2]) == 0
    with pytest.raises(ValueError):
        texts.reserve(1, 10 ** 6)


def test_serving_host():
    _check("cpu", 16, vocab=300, width=128, layers=2, heads=4, kv=2, dim=32, inner=192)


@pytest.mark.gpu
def test_serving(gpu):
    _check(gpu, 64)


@pytest.mark.gpu
def test_serving_gpu_and_host(gpu):
    """The GPU's logits are the host's, up to the roundings of bfloat16 through the layers."""
    sizes = dict(vocab=300, width=128, layers=2, heads=4, kv=2, dim=32, inner=192)
    got = []
    for dev in ("cpu", gpu):
        model = S.Server(**sizes).to(dev)
        prompts = _prompts(300, [20, 33, 5], dev)
        texts = S.Texts(model, 3, 64, 16, device=dev)
        for i in range(3):
            texts.reserve(i, 64)
        with torch.no_grad():
            model.start(texts, torch.cat(prompts), torch.tensor([0, 20, 53, 58], dtype=torch.int32, device=dev))
            out = [model.step(texts, torch.tensor([[i, i + 1], [2 * i, 5], [7, 9]], dtype=torch.int32, device=dev)) for i in range(6)]
        got.append(torch.stack(out).float().cpu())
    assert (got[0] - got[1]).norm() / got[0].norm() < 0.02


def test_main(capsys):
    S.main(["--texts", "2", "--prompt", "6", "--steps", "3", "--page", "16", "--device", "cpu"])
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 3 and [len(line.split()) for line in lines[:2]] == [3, 3]
