"""The operators of a language model that serves several continuations of one prompt, as cases that can be
timed and compared: products with 4-bit weights, causal attention over packed prompts, one decode step's
attention over a prefix that the batch shares and each sequence's own keys, and the adjustment of the logits
before a token is chosen.

`prepare` makes what the program holds before the call, `run` is one call (the framework's own where `own` is
set, else elementary torch operations in float32, rounded once), `exact` the same values in 64 bits.

Activations are N(0, 1) with 0.1% outliers of 20 times that; 4-bit weights are uniform in 0..15 with scales
around 0.02 / 4; queries and keys have unit variance, as a norm over a head leaves them; logits are
N(0, 3).
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-xdna_amd")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESZ = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one token through the fused q | k | v projection of a small model: the smallest product, all latency
        {"name": "w4 one row", "kind": "w4", "m": 1, "k": 1024, "n": 4096, "group": 128, "dtype": "bf16", "zeros": False,
         "bias": False},
        # one token through a wide MLP projection with zero points and a bias: bound by the weight stream
        {"name": "w4 one wide row", "kind": "w4", "m": 1, "k": 4096, "n": 14336, "group": 128, "dtype": "bf16",
         "zeros": True, "bias": True},
        # a decode step of 40 sequences through the projection back, in float16 with short groups
        {"name": "w4 40 rows", "kind": "w4", "m": 40, "k": 14336, "n": 4096, "group": 64, "dtype": "f16", "zeros": True,
         "bias": False},
        # three rows of a float32 model whose widths are multiples of nothing but the shortest group
        {"name": "w4 odd sizes", "kind": "w4", "m": 3, "k": 1504, "n": 1001, "group": 32, "dtype": "f32", "zeros": True,
         "bias": True},
        # a handful of short prompts, one of a single token: a small, ragged, latency-bound call
        {"name": "causal short prompts", "kind": "causal", "lens": "264 1 222 33 97", "heads": 16, "kv": 8, "dim": 128,
         "dtype": "bf16"},
        # prompts of very different lengths in one call, every head with its own keys, in float16
        {"name": "causal heads of 64", "kind": "causal", "lens": "4096 1500 700", "heads": 12, "kv": 12, "dim": 64,
         "dtype": "f16"},
        # one long prompt: the largest call, bound by the matrix units
        {"name": "causal 16384", "kind": "causal", "lens": "16384", "heads": 16, "kv": 8, "dim": 128, "dtype": "bf16"},
        # four continuations of a short prompt: a decode step that is all latency
        {"name": "prefix 264", "kind": "prefix", "batch": 4, "prefix": 264, "own": 64, "heads": 16, "kv": 8, "dim": 128,
         "dtype": "bf16"},
        # a batch of 48 over a system prompt of ordinary length, own parts of up to 700 tokens
        {"name": "prefix 4096", "kind": "prefix", "batch": 48, "prefix": 4096, "own": 700, "heads": 16, "kv": 8,
         "dim": 128, "dtype": "bf16"},
        # 24 continuations of a very long document, eight query heads to a key head, float16 heads of 64
        {"name": "prefix 100000", "kind": "prefix", "batch": 24, "prefix": 100000, "own": 333, "heads": 32, "kv": 4,
         "dim": 64, "dtype": "f16"},
        # one sequence's logits over a small vocabulary with its prompt as history
        {"name": "logits 8200", "kind": "logits", "batch": 1, "vocab": 8200, "history": 264, "dtype": "f32", "bias": "",
         "mask": True},
        # 64 sequences over a large, odd vocabulary with long histories, a bias for each sequence and a grammar
        {"name": "logits 64 rows", "kind": "logits", "batch": 64, "vocab": 128259, "history": 4096, "dtype": "bf16",
         "bias": "row", "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "w4", "causal", "prefix", "logits"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        k = max(1, _log(rng, 256, 14336) // group) * group
        n = _log(rng, 64, 14336)
        n = n // 64 * 64 if rng.random() < 0.5 else n
        return {"kind": "w4", "m": rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 64)]), "k": k, "n": max(64, n),
                "group": group, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "zeros": rng.random() < 0.5,
                "bias": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 7, 8])
    dim, dtype = rng.choice([64, 128, 128]), rng.choice(["bf16", "f16"])
    if kind == "causal":
        while True:
            lens = [_log(rng, 1, 8192) for _ in range(rng.randint(1, 6))]
            if sum(lens) ** 2 * heads <= 16384 ** 2 * 16 and sum(n * n for n in lens) * heads * dim <= 16384 ** 2 * 16 * 128:
                break
        return {"kind": "causal", "lens": " ".join(map(str, lens)), "heads": heads, "kv": kv, "dim": dim, "dtype": dtype}
    if kind == "prefix":
        while True:
            batch, prefix, length = _log(rng, 1, 64), _log(rng, 1, 100000), _log(rng, 1, 1000)
            if batch * (prefix + length) * heads <= 24 * 100333 * 32:
                break
        return {"kind": "prefix", "batch": batch, "prefix": prefix, "own": length, "heads": heads, "kv": kv, "dim": dim,
                "dtype": dtype}
    return {"kind": "logits", "batch": _log(rng, 1, 64), "vocab": _log(rng, 1000, 128259), "history": _log(rng, 1, 4096),
            "dtype": rng.choice(["f32", "bf16", "f16"]), "bias": rng.choice(["", "one", "row"]), "mask": rng.random() < 0.7}


# ------------------------------------------------------------------------------ inputs
class _Rand:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype="f32"):
        return (torch.randn(*shape, generator=self.g, device=self.dev) * std).to(DTYPES[dtype])

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=self.dev)

    def whole(self, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.g, device=self.dev, dtype=dtype)


def _lens(case):
    return [int(v) for v in case["lens"].split()]


def prepare(case, seed):
    r, kind, dt = _Rand(seed), case["kind"], case["dtype"]
    if kind == "w4":
        m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
        x = r.normal(m, k)
        x = torch.where(r.uniform(m, k) < 1e-3, 20 * x, x).to(DTYPES[dt])
        return {"kind": kind, "x": x, "qweight": r.whole(0, 256, n, k // 2, dtype=torch.uint8),
                "scales": ((0.5 + r.uniform(n, groups)) * 0.005).to(DTYPES[dt]),
                "zeros": r.whole(5, 12, n, groups, dtype=torch.uint8) if case["zeros"] else None,
                "bias": r.normal(n, std=0.01, dtype=dt) if case["bias"] else None}
    if kind == "logits":
        b, v, length = case["batch"], case["vocab"], case["history"]
        # tokens of a text: a few of them frequent, most of them rare
        tokens = (r.uniform(b, length) ** 4 * v).to(torch.int32).clamp(max=v - 1)
        bias = {"": None, "one": (v,), "row": (b, v)}[case["bias"]]
        return {"kind": kind, "logits": r.normal(b, v, std=3.0, dtype=dt), "tokens": tokens,
                "lens": r.whole(0, length + 1, b), "repetition": 1 + 0.3 * r.uniform(b), "presence": 0.5 * r.uniform(b),
                "frequency": 0.2 * r.uniform(b), "bias": None if bias is None else r.normal(*bias, std=0.5),
                "allowed": r.whole(-2 ** 31, 2 ** 31, b, -(-v // 32)) if case["mask"] else None}
    h, kv, d = case["heads"], case["kv"], case["dim"]
    if kind == "causal":
        lens = _lens(case)
        qkv = r.normal(sum(lens), h + 2 * kv, d, dtype=dt)     # as the fused projection leaves them
        starts = torch.tensor([0] + lens, device=r.dev).cumsum(0).to(torch.int32)
        return {"kind": kind, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:], "starts": starts,
                "scale": d ** -0.5}
    b, p, s = case["batch"], case["prefix"], case["own"]
    return {"kind": kind, "q": r.normal(b, h, d, dtype=dt), "kp": r.normal(p, kv, d, dtype=dt),
            "vp": r.normal(p, kv, d, dtype=dt), "kc": r.normal(b, s, kv, d, dtype=dt), "vc": r.normal(b, s, kv, d, dtype=dt),
            "lens": r.whole(1, s + 1, b), "scale": d ** -0.5}


# ------------------------------------------------------------------------------ one call
def run(state):
    s, kind = state, state["kind"]
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import torch_xdna  # noqa: F401  (registers the ops)
        ops = torch.ops.xdna
        with torch.no_grad():
            if kind == "w4":
                return ops.linear_w4(s["x"], s["qweight"], s["scales"], s["zeros"], s["bias"])
            if kind == "causal":
                return ops.attention_causal(s["q"], s["k"], s["v"], s["starts"], s["scale"])
            if kind == "prefix":
                return ops.attention_prefix(s["q"], s["kp"], s["vp"], s["kc"], s["vc"], s["lens"], s["scale"])
            return ops.logits_adjust(s["logits"], s["tokens"], s["lens"], s["repetition"], s["presence"], s["frequency"],
                                     s["bias"], s["allowed"])
    with torch.no_grad():
        return {"w4": _w4, "causal": _causal, "prefix": _prefix, "logits": _logits}[kind](s)


def _w4(s):
    q, x = s["qweight"], s["x"]
    n, groups = s["scales"].shape
    w = torch.stack([q & 15, q >> 4], dim=-1).view(n, groups, -1).float()
    z = 8.0 if s["zeros"] is None else s["zeros"].float().unsqueeze(-1)
    w = ((w - z) * s["scales"].float().unsqueeze(-1)).view(n, -1)
    y = x.float() @ w.t()
    return (y if s["bias"] is None else y + s["bias"].float()).to(x.dtype)


def _softmax_times(scores, seen, v):
    """softmax over the seen scores, times v; zero for a row that sees nothing."""
    top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top)).masked_fill(~seen, 0.0)
    total = p.sum(-1, keepdim=True)
    return (p / torch.where(total == 0, 1.0, total)) @ v


def _causal(s):
    q, k, v = (s[c].float().transpose(0, 1) for c in "qkv")        # [heads, tokens, dim]
    h, t, d = q.shape
    at = torch.arange(t, device=q.device)
    seq = torch.searchsorted(s["starts"].long(), at, right=True)
    seen = (seq[:, None] == seq[None, :]) & (at[None, :] <= at[:, None])
    q = q.reshape(k.shape[0], -1, t, d)
    o = _softmax_times((q @ k[:, None].transpose(-1, -2)) * s["scale"], seen, v[:, None])
    return o.reshape(h, t, d).transpose(0, 1).contiguous().to(s["q"].dtype)


def _prefix(s):
    b, h, d = s["q"].shape
    p, kv, _ = s["kp"].shape
    n = s["kc"].shape[1]
    q = s["q"].float().view(b, kv, h // kv, d)
    kp, vp = s["kp"].float().permute(1, 0, 2), s["vp"].float().permute(1, 0, 2)                    # [kv, p, d]
    kc, vc = s["kc"].float().permute(0, 2, 1, 3), s["vc"].float().permute(0, 2, 1, 3)              # [b, kv, n, d]
    seen = (torch.arange(n, device=q.device)[None, :] < s["lens"][:, None])[:, None, None, :]
    first = (q.transpose(0, 1).reshape(kv, -1, d) @ kp.transpose(1, 2)).view(kv, b, -1, p).transpose(0, 1) * s["scale"]
    rest = ((q @ kc.transpose(2, 3)) * s["scale"]).masked_fill(~seen, -math.inf)
    top = torch.maximum(first.amax(-1, keepdim=True), rest.amax(-1, keepdim=True))
    first, rest = torch.exp(first - top), torch.exp(rest - top)
    total = first.sum(-1, keepdim=True) + rest.sum(-1, keepdim=True)
    o = (first.transpose(0, 1).reshape(kv, -1, p) @ vp).view(kv, b, -1, d).transpose(0, 1) + rest @ vc
    return (o / total).reshape(b, h, d).to(s["q"].dtype)


def _logits(s):
    x = s["logits"].float()
    b, v = x.shape
    tokens = s["tokens"].long()
    valid = torch.arange(tokens.shape[1], device=x.device)[None, :] < s["lens"][:, None]
    count = torch.zeros(b, v, device=x.device).scatter_add_(1, tokens, valid.float())
    rep = s["repetition"][:, None]
    x = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"].float()
    if s["allowed"] is not None:
        bits = torch.arange(32, device=x.device, dtype=torch.int32)
        ok = ((s["allowed"].unsqueeze(-1) >> bits) & 1).view(b, -1)[:, :v].bool()
        x = x.masked_fill(~ok, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, esz = case["kind"], ESZ[case["dtype"]]
    if kind == "w4":
        m, k, n, groups = case["m"], case["k"], case["n"], case["k"] // case["group"]
        return {"bytes": n * k // 2 + n * groups * (esz + case["zeros"]) + (m * (k + n) + n * case["bias"]) * esz,
                "flops": 2 * m * n * k}
    if kind == "logits":
        b, v = case["batch"], case["vocab"]
        # on average half of a history's slots are taken
        return {"bytes": 2 * b * v * esz + b * case["history"] // 2 * 4 + {"": 0, "one": v, "row": b * v}[case["bias"]] * 4
                + case["mask"] * b * v // 8, "flops": 4 * b * v}
    h, kv, d = case["heads"], case["kv"], case["dim"]
    if kind == "causal":
        lens = _lens(case)
        return {"bytes": sum(lens) * (2 * h + 2 * kv) * d * esz, "flops": sum(2 * n * (n + 1) for n in lens) * h * d}
    b, p, mean = case["batch"], case["prefix"], (case["own"] + 1) / 2
    return {"bytes": (2 * b * h + 2 * p * kv + 2 * b * mean * kv) * d * esz, "flops": 4 * b * (p + mean) * h * d}


# ------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in float64, a head or a sequence at a time."""
    with torch.no_grad():
        s, kind = prepare(case, seed), case["kind"]
        if kind == "w4":
            x, g = s["x"].double(), case["group"]
            byte = s["qweight"].int()
            y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=x.device)
            for i in range(case["k"] // g):
                part = byte[:, i * g // 2:(i + 1) * g // 2]
                low, high = (part % 16).double(), (part // 16).double()
                xs = x[:, i * g:(i + 1) * g]
                z = s["zeros"][:, i].double() if case["zeros"] else torch.full_like(low[:, 0], 8.0)
                whole = xs[:, 0::2] @ low.t() + xs[:, 1::2] @ high.t() - xs.sum(1, keepdim=True) * z
                y += whole * s["scales"][:, i].double()
            return y + s["bias"].double() if case["bias"] else y
        if kind == "logits":
            x = s["logits"].double()
            for b in range(case["batch"]):
                said, times = torch.unique(s["tokens"][b, :int(s["lens"][b])].long(), return_counts=True)
                rep = s["repetition"][b].double()
                at = x[b, said]
                at = torch.where(at > 0, at / rep, at * rep)
                x[b, said] = at - s["frequency"][b].double() * times - s["presence"][b].double()
            if s["bias"] is not None:
                x += s["bias"].double()
            if s["allowed"] is not None:
                for j in range(32):
                    part = x[:, j::32]
                    part[((s["allowed"].long() >> j) & 1)[:, :part.shape[1]] == 0] = -math.inf
            return x
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        h, kv = case["heads"], case["kv"]
        if kind == "causal":
            at = 0
            for n in _lens(case):
                later = torch.ones(n, n, dtype=torch.bool, device=out.device).triu(1)
                for i in range(h):
                    q, k, v = (s[c][at:at + n, j].double() for c, j in (("q", i), ("k", i * kv // h), ("v", i * kv // h)))
                    p = torch.softmax((q @ k.t() * s["scale"]).masked_fill_(later, -math.inf), dim=-1)
                    out[at:at + n, i] = p @ v
                at += n
            return out
        for g in range(kv):
            kp, vp = s["kp"][:, g].double(), s["vp"][:, g].double()
            for b in range(case["batch"]):
                n = int(s["lens"][b])
                k = torch.cat([kp, s["kc"][b, :n, g].double()])
                v = torch.cat([vp, s["vc"][b, :n, g].double()])
                heads = slice(g * h // kv, (g + 1) * h // kv)
                out[b, heads] = torch.softmax(s["q"][b, heads].double() @ k.t() * s["scale"], dim=-1) @ v
        return out
