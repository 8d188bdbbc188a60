"""serving.Texts and Server as texts come and go: rows without a text, texts that grow past their pages, and past their capacity."""
import pytest
import torch

from torch_xdna import serving as S

SIZES = dict(vocab=300, width=128, layers=2, heads=4, kv=2, dim=32, inner=192)


def _prompt(n, dev):
    return torch.randint(0, 300, (n,), generator=torch.Generator().manual_seed(n)).to(torch.int32).to(dev)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _text_after_idle_steps(dev, page):
    """A row whose text ended while the others went on, and which has a new one now, is as a row that nobody had."""
    model, first, new = S.Server(**SIZES).to(dev), [_prompt(2 * page + 5, dev), _prompt(9, dev)], _prompt(page + 4, dev)
    got = []
    for idle in (0, 5, 2 * page):
        texts = S.Texts(model, 2, 6 * page, page, device=dev)
        with torch.no_grad():
            for i, p in enumerate(first):
                texts.reserve(i, p.shape[0] + 3 * page)
            n = first[0].shape[0]
            model.start(texts, torch.cat(first), _i32([0, n, n + 9], dev))
            model.step(texts, _i32([[1], [2]], dev))
            texts.release(1)
            for i in range(idle):
                model.step(texts, _i32([[i], [7]], dev))
            assert texts.lens.tolist() == [n + 1 + idle, 0]
            texts.reserve(1, new.shape[0] + 3)
            out = [model.start(texts, new, _i32([0, 0, new.shape[0]], dev))]
            for i in range(3):
                out.append(model.step(texts, _i32([[i], [i + 4]], dev))[1])
            assert texts.lens.tolist() == [n + 1 + idle + 3, new.shape[0] + 3]
        got.append(torch.cat(out))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_text_after_idle_steps():
    _text_after_idle_steps("cpu", 16)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_text_after_idle_steps_gpu(gpu, page):
    _text_after_idle_steps(gpu, page)
