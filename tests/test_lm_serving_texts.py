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


def _steps_past_pages_and_capacity(dev, page):
    """Steps get the pages that their tokens need, and raise, before anything is written, where there are none."""
    model, prompt = S.Server(**SIZES).to(dev), _prompt(page + 4, dev)
    got = []
    for reserved, draft in ((3 * page, 1), (0, 1), (page + 4, 4)):
        texts = S.Texts(model, 2, 3 * page, page, pages=5, device=dev)
        texts.reserve(1, page)
        if reserved:
            texts.reserve(0, reserved)
        with torch.no_grad():
            model.start(texts, prompt, _i32([0, page + 4, page + 4], dev))
            out = []
            for i in range(0, 2 * page - 4, draft):
                tokens = _i32([list(range(i, i + draft)), [0] * draft], dev)
                if int(texts.lens[1]) + draft > page:                 # the pool's last page is text 0's
                    texts.release(1)
                out.append(model.step(texts, tokens)[0])
            got.append(torch.cat(out))
            assert int(texts.lens[0]) == 3 * page and len(texts.given[0]) == 3
            before = [t.clone() for t in (*texts.layers[0], *texts.layers[1], texts.lens)]
            with pytest.raises(ValueError):
                model.step(texts, tokens)                             # no capacity
            for t, b in zip((*texts.layers[0], *texts.layers[1], texts.lens), before):
                assert torch.equal(t, b)
            assert texts.held[0] == 3 * page
    assert torch.equal(got[0], got[1])
    # drafts: the same cache, up to the order of sums
    assert (got[2].float() - got[0].float()).norm() < 0.05 * got[0].float().norm()


def _refusals(dev):
    page, model = 16, S.Server(**SIZES).to(dev)
    texts = S.Texts(model, 2, 2 * page, page, pages=3, device=dev)
    long, short = _prompt(2 * page + 1, dev), _prompt(page + 1, dev)
    with torch.no_grad():
        for tokens, starts in ((long, [0, 2 * page + 1, 2 * page + 1]), (torch.cat([short, short]), [0, page + 1, 2 * page + 2]),
                               (short, [0, page + 1]), (short, [0, 5, 3]), (short, [0, 5, page + 2]), (short, [-1, 5, page + 1])):
            with pytest.raises(ValueError):
                model.start(texts, tokens, _i32(starts, dev))
        assert len(texts.free) == 3 and texts.lens.tolist() == [0, 0] and texts.held == [0, 0] and bool((texts.layers[0].table == -1).all())
        model.start(texts, short, _i32([0, page + 1, page + 1], dev))
        with pytest.raises(ValueError):
            model.start(texts, short, _i32([0, page + 1, page + 1], dev))          # not empty
        with pytest.raises(ValueError):
            model.step(texts, _i32([[1]], dev))
        model.start(texts, short[:page], _i32([0, 0, page], dev))
        with pytest.raises(ValueError):
            model.step(texts, _i32([[1], [2]], dev))                               # the pool has no page for the second
        assert texts.lens.tolist() == [page + 1, page] == texts.held and not texts.free
        texts.release(0)
        model.step(texts, _i32([[1], [2]], dev))
        assert texts.lens.tolist() == [0, page + 1] == texts.held and len(texts.free) == 1


def test_steps_past_pages_and_capacity():
    _steps_past_pages_and_capacity("cpu", 16)


def test_refusals():
    _refusals("cpu")


@pytest.mark.gpu
def test_steps_past_pages_and_capacity_gpu(gpu):
    _steps_past_pages_and_capacity(gpu, 16)
    _steps_past_pages_and_capacity(gpu, 64)
    _refusals(gpu)


@pytest.mark.gpu
def test_captured_step(gpu):
    """A step in a graph: the pages given before, the count kept beside the replays."""
    model, prompt = S.Server(**SIZES).to(gpu), _prompt(13, gpu)
    eager, replayed = (S.Texts(model, 2, 80, 16, device=gpu) for _ in range(2))
    tokens = _i32([[1], [2]], gpu)
    with torch.no_grad():
        for texts in (eager, replayed):
            texts.reserve(0, 70)
            model.start(texts, prompt, _i32([0, 13, 13], gpu))
            model.step(texts, tokens)                                 # (the first call of everything is outside)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = model.step(replayed, tokens)
        for i in range(30):
            tokens.copy_(_i32([[i], [2 * i]], gpu))
            want = model.step(eager, tokens)
            if i:                                                     # the capture has counted the first
                replayed.grow([1, 0])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]), i
            assert eager.held == replayed.held == eager.lens.tolist() == replayed.lens.tolist()
        with pytest.raises(ValueError):
            replayed.grow([80 - replayed.held[0] + 1, 0])


def _drafts_taken_back(dev, page):
    """Steps of drafts of which some are not taken: the program sets lens back, and only what is held counts against the capacity.
    The tokens that were taken have the logits that they have one by one; a row set to 0 takes a new prompt."""
    model, prompt = S.Server(**SIZES).to(dev), _prompt(page + 3, dev)
    plain, drafts = (S.Texts(model, 1, 3 * page, page, device=dev) for _ in range(2))
    with torch.no_grad():
        for texts in (plain, drafts):
            model.start(texts, prompt, _i32([0, page + 3], dev))
        for i in range(2 * page - 7):
            want = model.step(plain, _i32([[i]], dev))[0, 0]
            got = model.step(drafts, _i32([[i, 250, 251, 252, 253]], dev))[0, 0]
            drafts.lens -= 4
            assert (got.float() - want.float()).norm() < 0.03 * want.float().norm(), i
        assert drafts.lens.tolist() == plain.lens.tolist() == [3 * page - 4]
        with pytest.raises(ValueError):
            model.step(drafts, _i32([[1, 2, 3, 4, 5]], dev))
        model.step(drafts, _i32([[1, 2, 3, 4]], dev))
        with pytest.raises(ValueError):
            model.start(drafts, prompt, _i32([0, page + 3], dev))
        drafts.lens.zero_()
        model.start(drafts, prompt, _i32([0, page + 3], dev))
        assert drafts.lens.tolist() == [page + 3] == drafts.held


def test_drafts_taken_back():
    _drafts_taken_back("cpu", 16)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_drafts_taken_back_gpu(gpu, page):
    _drafts_taken_back(gpu, page)
