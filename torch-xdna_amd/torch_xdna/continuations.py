"""Several continuations of one prompt, as a program that serves a language model runs them: the operators of lm.py together.

    python -m torch_xdna.continuations [--batch 4] [--prompt 264] [--steps 16] [--device cuda]

A small decoder of random weights (there is no checkpoint here): 4-bit projections (linear_w4), the prompt once through
attention_causal, whose keys and values every continuation then shares (attention_prefix, with each one's own keys
beside them), and tokens chosen from logits with penalties for what was said and a mask of what may be (logits_adjust).
The sizes are the defaults of `Decoder`; anything with the same parts can be run the same way.
"""

import argparse
import time

import torch
import torch.nn.functional as F

from . import lm


class W4(torch.nn.Module):
    """A linear without bias whose weight is 4-bit with scales and zero points per group of 64 inputs."""

    def __init__(self, n, k, dtype, generator):
        super().__init__()
        w = torch.randn(n, k, generator=generator) * k ** -0.5
        q, s, z = lm.quantize_w4(w.to(dtype), 64)
        self.register_buffer("q", q), self.register_buffer("s", s), self.register_buffer("z", z)

    def forward(self, x):
        return lm.linear_w4(x, self.q, self.s, self.z)


class Layer(torch.nn.Module):
    def __init__(self, width, heads, kv, dim, inner, dtype, generator):
        super().__init__()
        self.heads, self.kv, self.dim = heads, kv, dim
        self.qkv = W4((heads + 2 * kv) * dim, width, dtype, generator)
        self.out = W4(width, heads * dim, dtype, generator)
        self.gate_up = W4(2 * inner, width, dtype, generator)
        self.down = W4(width, inner, dtype, generator)

    def project(self, x, cos, sin):
        """(q, k, v) [rows, heads, dim] of the rows x, q and k of unit variance and rotated to the rows' positions."""
        h, kv, d = self.heads, self.kv, self.dim
        qkv = self.qkv(norm(x)).view(-1, h + 2 * kv, d)
        qk = norm(qkv[:, :h + kv]).float()
        a, b = qk[..., :d // 2], qk[..., d // 2:]
        qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)
        return qk[:, :h], qk[:, h:], qkv[:, h + kv:]

    def finish(self, x, o):
        x = x + self.out(o.flatten(1))
        g, u = self.gate_up(norm(x)).chunk(2, -1)
        return x + self.down((F.silu(g.float()) * u.float()).to(x.dtype))


def norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Decoder(torch.nn.Module):
    def __init__(self, vocab=8200, width=1024, layers=4, heads=16, kv=8, dim=128, inner=2048, dtype=torch.bfloat16, seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.vocab, self.dim = vocab, dim
        self.register_buffer("embed", torch.randn(vocab, width, generator=g).to(dtype))
        self.layers = torch.nn.ModuleList(Layer(width, heads, kv, dim, inner, dtype, g) for _ in range(layers))
        self.head = W4(vocab, width, dtype, g)
        self.register_buffer("freq", 10000.0 ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim))

    def angles(self, pos):
        t = pos.double()[:, None, None] * self.freq               # in 64 bits: far positions turn many times
        return t.cos().float(), t.sin().float()

    def prefill(self, tokens, starts=None):
        """Logits of every token [T] of the packed prompts that start at `starts` (one prompt if None), and each layer's (k, v)."""
        t = tokens.shape[0]
        if starts is None:
            starts = torch.tensor([0, t], dtype=torch.int32, device=tokens.device)
        at = torch.arange(t, device=tokens.device)
        first = starts.long()[torch.searchsorted(starts.long(), at, right=True) - 1]
        cos, sin = self.angles(at - first)
        x, cache = self.embed[tokens.long()], []
        for layer in self.layers:
            q, k, v = layer.project(x, cos, sin)
            x = layer.finish(x, lm.attention_causal(q, k, v, starts))
            cache.append((k, v))
        return self.head(norm(x)), cache

    def step(self, tokens, prefix, own, lens):
        """Logits [B, V] of one new token [B] of each continuation; its keys and values go to place lens[b] of own."""
        p = prefix[0][0].shape[0]
        cos, sin = self.angles(p + lens)
        rows, seen = torch.arange(tokens.shape[0], device=tokens.device), lens + 1
        x = self.embed[tokens.long()]
        for layer, (kp, vp), (kc, vc) in zip(self.layers, prefix, own):
            q, k, v = layer.project(x, cos, sin)
            kc[rows, lens.long()], vc[rows, lens.long()] = k, v
            x = layer.finish(x, lm.attention_prefix(q, kp, vp, kc, vc, seen))
        return self.head(norm(x))


def likeliest(scores, n):
    """The n likeliest tokens of the scores [V]; past those that there are, and that may be chosen, the first of them again."""
    top = scores.topk(min(n, scores.shape[0]))
    tokens = torch.where(top.values == -torch.inf, top.indices[:1], top.indices)
    return torch.cat([tokens, tokens[:1].expand(n - tokens.shape[0])])


@torch.no_grad()
def continuations(model, prompt, batch, steps, repetition=1.1, presence=0.1, frequency=0.1, allowed=None):
    """`batch` continuations [batch, steps] (int32) of the tokens `prompt` [P]: the first tokens are the `batch` likeliest (where
    there are fewer, the likeliest again), each later one the likeliest after its own. allowed: a mask [ceil(V / 32)] of the
    tokens that may be chosen, at least one (read on the host, once), or None."""
    dev, p = prompt.device, prompt.shape[0]
    if allowed is not None:
        bits = allowed.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=dev) & 1
        if not bool(bits.flatten()[:model.vocab].any()):
            raise ValueError("the mask allows no token")
    logits, prefix = model.prefill(prompt)
    own = [tuple(torch.zeros(batch, steps, *t.shape[1:], dtype=t.dtype, device=dev) for t in kv) for kv in prefix]
    said = torch.zeros(batch, p + steps, dtype=torch.int32, device=dev)
    said[:, :p] = prompt
    settings = [torch.full((batch,), float(v), device=dev) for v in (repetition, presence, frequency)]
    mask = None if allowed is None else allowed.expand(batch, -1)
    lens = torch.zeros(batch, dtype=torch.int32, device=dev)
    logits = logits[-1:].expand(batch, -1)
    for i in range(steps):
        scores = lm.logits_adjust(logits, said, lens + p, *settings, None, mask)
        tokens = likeliest(scores[0], batch) if i == 0 else scores.argmax(-1)
        said[:, p + i] = tokens.to(torch.int32)
        if i + 1 < steps:
            logits = model.step(tokens, prefix, own, lens)
            lens = lens + 1
    return said[:, p:]


def main(argv=None):
    a = argparse.ArgumentParser(description="Several continuations of one prompt by a decoder of random weights.")
    a.add_argument("--batch", type=int, default=4)
    a.add_argument("--prompt", type=int, default=264)
    a.add_argument("--steps", type=int, default=16)
    a.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    o = a.parse_args(argv)
    model = Decoder().to(o.device)
    prompt = torch.randint(0, model.vocab, (o.prompt,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(o.device)
    continuations(model, prompt, o.batch, 2)
    t0 = time.perf_counter()
    out = continuations(model, prompt, o.batch, o.steps).cpu()
    t = time.perf_counter() - t0
    for row in out.tolist():
        print(*row)
    print(f"{o.batch} continuations of {o.prompt} tokens by {o.steps}: {t * 1e3:.1f} ms, {o.batch * o.steps / t:.0f} tokens/s on {o.device}")


if __name__ == "__main__":
    main()
