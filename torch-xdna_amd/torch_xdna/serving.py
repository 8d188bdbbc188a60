"""Different texts continued together, as a program that serves a language model runs them: the operators of lm.py over a paged
8-bit cache.

    python -m torch_xdna.serving [--texts 8] [--prompt 300] [--steps 16] [--page 64] [--device cuda]

The decoder of continuations.py (random weights: there is no checkpoint here). Prompts of different lengths go in packed, once:
rotary, attention_causal, cache_append. Then every text gets a token a step: cache_append puts its key and value into the
text's pages and turns the query to its place, attention_cache reads them, residual_norm joins block to block, logits_adjust
weighs what was said. The program's side of a cache is here too: which pages are whose, and how long each text is.
"""

import argparse
import time

import torch
import torch.nn.functional as F

from . import lm
from .continuations import Decoder


class Texts:
    """The caches of `batch` texts in all layers: a Cache8 a layer over one table, and the texts' lengths. A row of the batch has a
    text from the time that it has pages until they are given back; the tokens that a step has for the other rows go nowhere, and
    its logits for those mean nothing. What a text holds is counted on the host too, so that nothing grows past its pages: a program
    that replays a captured step gives the pages out before (reserve), and counts each replay but the first (grow). A program may
    set lens back (drafts that were not taken): the host's count, too high then, is read from it again before anything is refused."""

    def __init__(self, model, batch, capacity, page=64, pages=None, device=None):
        layer = model.layers[0]
        columns = -(-capacity // page)
        pages = batch * columns if pages is None else pages
        dtype = model.embed.dtype
        first = lm.cache8(batch, pages, layer.kv, layer.dim, capacity, page, dtype=dtype, device=device)
        self.layers = [first] + [lm.cache8(batch, pages, layer.kv, layer.dim, capacity, page, dtype=dtype, device=device)
                                 ._replace(table=first.table) for _ in model.layers[1:]]
        self.page, self.columns = page, columns
        self.free = list(range(pages))
        self.given = [[] for _ in range(batch)]
        self.held = [0] * batch
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.live = torch.zeros(batch, dtype=torch.int32, device=device)       # 1: a text's row

    def reserve(self, text, tokens):
        """Pages for the first `tokens` tokens of a text."""
        columns = -(-tokens // self.page)
        missing = columns - len(self.given[text])
        if columns > self.columns or missing > len(self.free):
            raise ValueError(f"no room for {tokens} tokens of text {text}: {len(self.free)} pages are free, of {self.columns} a text")
        if missing > 0:
            new = [self.free.pop() for _ in range(missing)]
            at = len(self.given[text])
            self.layers[0].table[text, at:at + missing] = torch.tensor(new, dtype=torch.int32).to(self.lens.device)
            self.given[text] += new
            self.live[text] = 1

    def grow(self, new):
        """Counts new[i] more tokens of each text i, and gives out the pages that they need; without room for all, it raises and
        nothing changes."""
        for again in (False, True):
            held = [h + n for h, n in zip(self.held, new)]
            missing = sum(max(0, -(-h // self.page) - len(g)) for h, n, g in zip(held, new, self.given) if n)
            if max(held, default=0) <= self.columns * self.page and missing <= len(self.free):
                break
            if again:
                raise ValueError(f"no room for texts of {held} tokens: {missing} pages are missing and {len(self.free)} free, of "
                                 f"{self.columns} a text")
            self.held = self.lens.tolist()
        for text, n in enumerate(new):
            if n:
                self.reserve(text, held[text])
        self.held = held

    def release(self, text):
        """A text that has ended gives its pages back, and its place can have a new one."""
        self.free += self.given[text]
        self.given[text] = []
        self.held[text] = 0
        self.layers[0].table[text] = -1
        self.lens[text] = self.live[text] = 0


class Server(Decoder):
    """continuations.Decoder with its layers on lm's operators."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        self.register_buffer("freqs", lm.rotary_freqs(self.dim)[0])

    def heads(self, layer, y):
        """(q and k [rows, heads, dim] of unit variance, v) of the rows y."""
        h, kv, d = layer.heads, layer.kv, layer.dim
        qkv = layer.qkv(y).view(-1, h + 2 * kv, d)
        return lm.residual_norm(qkv[:, :h + kv])[1], qkv[:, h + kv:]

    def finish(self, layer, x, o):
        x, y = lm.residual_norm(x, layer.out(o.flatten(1)))
        g, u = layer.gate_up(y).chunk(2, -1)
        return lm.residual_norm(x, layer.down((F.silu(g.float()) * u.float()).to(x.dtype)))

    def start(self, texts, tokens, starts):
        """Logits of every token [T] of the packed prompts, whose keys and values go into the texts' empty caches. A text without a
        prompt (two equal starts) stays as it is."""
        first = starts.tolist()
        new = [b - a for a, b in zip(first, first[1:])]
        if len(new) != len(texts.held) or min(new, default=0) < 0 or first[0] < 0 or first[-1] > tokens.shape[0]:
            raise ValueError(f"starts must be [{len(texts.held) + 1}], ascending, within the {tokens.shape[0]} tokens")
        if any(n and h for n, h in zip(new, texts.held)):
            texts.held = texts.lens.tolist()
            if any(n and h for n, h in zip(new, texts.held)):
                raise ValueError("a prompt is for a text that holds nothing: release it first")
        texts.grow(new)
        at = torch.arange(tokens.shape[0], device=tokens.device)
        place = at - starts.long()[torch.searchsorted(starts.long(), at, right=True) - 1]
        x = self.embed[tokens.long()]
        _, y = lm.residual_norm(x)
        for layer, cache in zip(self.layers, texts.layers):
            qk, v = self.heads(layer, y)
            qk = lm.rotary(qk, place, self.freqs)
            q, k = qk[:, :layer.heads], qk[:, layer.heads:]
            lm.cache_append(cache, texts.lens, k, v, starts)
            x, y = self.finish(layer, x, lm.attention_causal(q, k, v, starts))
        texts.lens += starts[1:] - starts[:-1]
        return self.head(y)

    def step(self, texts, tokens):
        """Logits [B, N, V] of N new tokens [B, N] of every text, which go into their caches."""
        b, n = tokens.shape
        if b != len(texts.held):
            raise ValueError(f"a step takes tokens [{len(texts.held)}, N], got {list(tokens.shape)}")
        texts.grow([n if given else 0 for given in texts.given])
        x = self.embed[tokens.long().flatten()]
        _, y = lm.residual_norm(x)
        seen = texts.lens + n
        for layer, cache in zip(self.layers, texts.layers):
            qk, v = self.heads(layer, y)
            q = lm.cache_append(cache, texts.lens, qk[:, layer.heads:], v, None, qk[:, :layer.heads], self.freqs)
            x, y = self.finish(layer, x, lm.attention_cache(q.view(b, n, layer.heads, self.dim), cache, seen).flatten(0, 1))
        texts.lens.add_(texts.live, alpha=n)
        return self.head(y).view(b, n, -1)


@torch.no_grad()
def serve(model, prompts, steps, page=64, repetition=1.1, presence=0.1, frequency=0.1):
    """`steps` tokens [B, steps] (int32) after each of the prompts (int32 tensors of at least one token each)."""
    dev, lengths = model.embed.device, [p.shape[0] for p in prompts]
    if not lengths or min(lengths) < 1:
        raise ValueError("serve takes prompts of at least one token each")
    b = len(prompts)
    texts = Texts(model, b, max(lengths) + steps, page, sum(-(-(n + steps) // page) for n in lengths), dev)
    for i, n in enumerate(lengths):
        texts.reserve(i, n + steps)
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(dev)
    logits = model.start(texts, torch.cat(list(prompts)).to(dev), starts)[starts[1:].long() - 1]
    said = torch.zeros(b, max(lengths) + steps, dtype=torch.int32, device=dev)
    for i, p in enumerate(prompts):
        said[i, :lengths[i]] = p
    settings = [torch.full((b,), float(v), device=dev) for v in (repetition, presence, frequency)]
    rows, out = torch.arange(b, device=dev), []
    for i in range(steps):
        tokens = lm.logits_adjust(logits, said, texts.lens, *settings).argmax(-1).to(torch.int32)
        said[rows, texts.lens.long()] = tokens
        out.append(tokens)
        if i + 1 < steps:
            logits = model.step(texts, tokens[:, None])[:, 0]
    return torch.stack(out, 1) if out else torch.zeros(b, 0, dtype=torch.int32, device=dev)


def main(argv=None):
    a = argparse.ArgumentParser(description="Different texts continued together by a decoder of random weights.")
    a.add_argument("--texts", type=int, default=8)
    a.add_argument("--prompt", type=int, default=300)
    a.add_argument("--steps", type=int, default=16)
    a.add_argument("--page", type=int, default=64)
    a.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    o = a.parse_args(argv)
    model = Server().to(o.device)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.vocab, (max(1, o.prompt * (i + 1) // o.texts),), generator=g).to(torch.int32).to(o.device)
               for i in range(o.texts)]
    serve(model, prompts, 2, o.page)
    t0 = time.perf_counter()
    out = serve(model, prompts, o.steps, o.page).cpu()
    t = time.perf_counter() - t0
    for row in out.tolist():
        print(*row)
    print(f"{o.texts} texts of up to {o.prompt} tokens by {o.steps}: {t * 1e3:.1f} ms, {o.texts * o.steps / t:.0f} tokens/s on {o.device}")


if __name__ == "__main__":
    main()
