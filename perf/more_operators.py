"""The operators of a language model that serves different prompts together, as cases that can be timed and compared:
rotary positions, the residual sum with the norms around it, keys and values that go into a paged 8-bit cache, and the
attention of new tokens over that cache.

`prepare` makes what the program holds before the call, `run` is one call (the framework's own where `own` is
set, else elementary torch operations in float32, angles in 64 bits, rounded once), `exact` the same values in 64 bits.

Queries, keys and values have unit variance, as a norm over a head leaves them; the residual stream is N(0, 4), with
0.1% outliers of 20 times that, norm weights lie around 1, gates are N(0, 1). Pages of the 8-bit cache have scales of a
3 to 4.5 sigma maximum; pages of a sequence lie anywhere in the pool.

The cache: kpages int8 [pages, KV, G, D] and vpages int8 [pages, KV, D, G] with a float32 scale for each page and head;
the tokens of a sequence's open page, and some before, in 16 bits at place position % R of ktail [B, KV, R, D] and vtail
[B, KV, D, R]; table [B, P] names the pages of a sequence.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-xdna_amd")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESZ = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the query heads of four sequences' next tokens, far into their texts: the smallest call, all latency
        {"name": "rotary 4 tokens", "kind": "rotary", "tokens": 4, "heads": 16, "dim": 128, "turned": 128, "dtype": "bf16",
         "interleaved": False, "scaled": False, "far": 100000},
        # query and key heads of a long prompt, frequencies scaled for long contexts: bound by memory
        {"name": "rotary 16384 tokens", "kind": "rotary", "tokens": 16384, "heads": 24, "dim": 128, "turned": 128,
         "dtype": "bf16", "interleaved": False, "scaled": True, "far": 0},
        # a float32 model that turns 32 of its heads' 80 dims, neighbours as pairs, over an odd number of tokens
        {"name": "rotary part of a head", "kind": "rotary", "tokens": 1501, "heads": 12, "dim": 80, "turned": 32, "dtype": "f32",
         "interleaved": True, "scaled": False, "far": 0},
        # four sequences' next tokens between attention and MLP of a small model: all latency
        {"name": "norm 4 rows", "kind": "norm", "rows": 4, "width": 1024, "dtype": "bf16", "stream": "bf16", "post": False,
         "gate": ""},
        # a long prompt through a block with norms on both sides and a gate per row, float32 residual stream
        {"name": "norm 8192 rows", "kind": "norm", "rows": 8192, "width": 4096, "dtype": "bf16", "stream": "f32", "post": True,
         "gate": "row"},
        # one new token of each of 48 sequences goes into the cache, its queries turn on the way; no page becomes full
        {"name": "append 48 tokens", "kind": "append", "new": " ".join(["1"] * 48), "before": 4000, "heads": 16, "kv": 8,
         "dim": 128, "turned": 128, "page": 64, "dtype": "bf16", "interleaved": False, "values": False},
        # a handful of short prompts of different lengths into empty caches, half of each head turned, float16
        {"name": "append short prompts", "kind": "append", "new": "264 1 222 33 97", "before": 0, "heads": 12, "kv": 4, "dim": 64,
         "turned": 32, "page": 32, "dtype": "f16", "interleaved": True, "values": True},
        # one long prompt into an empty cache
        {"name": "append 16384 tokens", "kind": "append", "new": "16384", "before": 0, "heads": 16, "kv": 8, "dim": 128,
         "turned": 128, "page": 64, "dtype": "bf16", "interleaved": False, "values": True},
        # four sequences of a short text each: a decode step that is all latency
        {"name": "cache 4 x 330", "kind": "cache", "batch": 4, "new": 1, "longest": 330, "heads": 16, "kv": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # a batch of 48 sequences of up to 8192 tokens: bound by the stream of keys and values
        {"name": "cache 48 x 8192", "kind": "cache", "batch": 48, "new": 1, "longest": 8192, "heads": 16, "kv": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # one sequence over a very long document, eight query heads to a key head, float16 heads of 64
        {"name": "cache 1 x 131000", "kind": "cache", "batch": 1, "new": 1, "longest": 131000, "heads": 32, "kv": 4, "dim": 64,
         "page": 128, "dtype": "f16"},
        # five drafted tokens of each of 16 sequences are looked over at once, short pages, heads of 96
        {"name": "cache 16 x 5 tokens", "kind": "cache", "batch": 16, "new": 5, "longest": 5000, "heads": 28, "kv": 4, "dim": 96,
         "page": 32, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "norm", "append", "cache", "cache"])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128])
        tokens, heads = _log(rng, 1, 16384), rng.choice([1, 3, 8, 12, 24])
        return {"kind": kind, "tokens": tokens, "heads": heads, "dim": dim, "turned": rng.choice([dim, dim, dim // 2, 20]),
                "dtype": rng.choice(["bf16", "bf16", "f16"] if tokens > 8192 else ["bf16", "f16", "f32"]),
                "interleaved": rng.random() < 0.5, "scaled": rng.random() < 0.5, "far": rng.choice([0, 1000000])}
    if kind == "norm":
        while True:
            rows, width = _log(rng, 1, 20000), _log(rng, 64, 16384)
            if rows * width <= 8192 * 4096:
                break
        dtype = rng.choice(["bf16", "f16", "f32"])
        width = width // 8 * 8 if rng.random() < 0.7 else width
        return {"kind": kind, "rows": rows, "width": width, "dtype": dtype, "stream": rng.choice([dtype, "f32"]),
                "post": rng.random() < 0.5, "gate": rng.choice(["", "one", "row"])}
    kv, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128, 128]), rng.choice([16, 32, 64, 128])
    heads, dtype = kv * rng.choice([1, 2, 4, 7]), rng.choice(["bf16", "f16"])
    if kind == "append":
        step = rng.random() < 0.4
        if step:
            new, before = [1] * _log(rng, 1, 64), _log(rng, 1, 8000)
        elif rng.random() < 0.3:                                    # a few more tokens of sequences that are there
            new, before = [rng.randint(1, page) for _ in range(rng.randint(1, 8))], _log(rng, 1, 300)
        else:
            new, before = [_log(rng, 1, 4096) for _ in range(rng.randint(1, 4))], 0
        return {"kind": kind, "new": " ".join(map(str, new)), "before": before, "heads": heads, "kv": kv, "dim": dim,
                "turned": rng.choice([dim, dim, dim // 2]), "page": page, "dtype": dtype, "interleaved": rng.random() < 0.3,
                "values": not step}
    while True:
        batch, longest, new = _log(rng, 1, 64), _log(rng, 8, 131000), rng.choice([1, 1, 1, rng.randint(2, 8)])
        if batch * longest * kv * dim <= 48 * 8192 * 8 * 128 and batch * longest * heads * new * dim <= 48 * 8192 * 16 * 128:
            return {"kind": kind, "batch": batch, "new": new, "longest": longest, "heads": heads, "kv": kv, "dim": dim,
                    "page": page, "dtype": dtype}


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

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=self.dev).to(torch.int32)


def _freqs(turned, scaled, dev):
    """Radians a position [turned / 2] (float64) and the factor on the turned values; scaled: slow dims eight times as slow."""
    f = 10000.0 ** -(torch.arange(0, turned, 2, dtype=torch.float64, device=dev) / turned)
    if not scaled:
        return f, 1.0
    turns = 8192 * f / (2 * math.pi)                  # over the length that the model was made for
    keep = ((turns - 1) / 31).clamp(0, 1)
    return f * keep + f / 8 * (1 - keep), 0.1 * math.log(8) + 1


def _new(case):
    return [int(v) for v in case["new"].split()]


def _columns(case):
    """Pages of a sequence's row of the table: those that `before` tokens, and the new ones, may lie in."""
    return case["before"] // case["page"] + -(-max(_new(case)) // case["page"]) + 1


def prepare(case, seed):
    r, kind, dt = _Rand(seed), case["kind"], case["dtype"]
    if kind == "rotary":
        t = case["tokens"]
        freqs, magnitude = _freqs(case["turned"], case["scaled"], r.dev)
        at = r.whole(0, case["far"] + 1, t) if case["far"] else torch.arange(t, device=r.dev, dtype=torch.int32)
        return {"kind": kind, "x": r.normal(t, case["heads"], case["dim"], dtype=dt), "positions": at, "freqs": freqs,
                "magnitude": magnitude, "interleaved": case["interleaved"]}
    if kind == "norm":
        n, w = case["rows"], case["width"]
        x = r.normal(n, w, std=2.0)
        x = torch.where(r.uniform(n, w) < 1e-3, 20 * x, x).to(DTYPES[case["stream"]])
        gate = {"": None, "one": (w,), "row": (n, w)}[case["gate"]]
        return {"kind": kind, "x": x, "o": r.normal(n, w, dtype=dt), "weight": (1 + r.normal(w, std=0.2)).to(DTYPES[dt]),
                "post": (1 + r.normal(w, std=0.2)).to(DTYPES[dt]) if case["post"] else None,
                "gate": None if gate is None else r.normal(*gate, dtype=dt), "scale": 0.7}
    kv, d, g, h = case["kv"], case["dim"], case["page"], case["heads"]
    slots = 2 * g
    if kind == "append":
        new, p, before = _new(case), _columns(case), case["before"]
        b, t = len(new), sum(new)
        qkv = r.normal(t, h + 2 * kv, d, dtype=dt)     # as the fused projection leaves them
        lens = r.whole(before // 2, before + 1, b) if before else torch.zeros(b, dtype=torch.int32, device=r.dev)
        if not case["values"]:                         # no page becomes full
            lens = torch.where(lens % g == g - 1, lens - 1, lens)
        freqs, _ = _freqs(case["turned"], False, r.dev)
        same = min(new) == max(new)
        return {"kind": kind, "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:],
                "kpages": torch.zeros(b * p, kv, g, d, dtype=torch.int8, device=r.dev),
                "vpages": torch.zeros(b * p, kv, d, g, dtype=torch.int8, device=r.dev),
                "kscales": torch.zeros(b * p, kv, device=r.dev), "vscales": torch.zeros(b * p, kv, device=r.dev),
                "ktail": r.normal(b, kv, slots, d, dtype=dt), "vtail": r.normal(b, kv, d, slots, dtype=dt),
                "table": r.order(b * p).view(b, p), "lens": lens, "freqs": freqs, "interleaved": case["interleaved"],
                "starts": torch.tensor([0] + new, device=r.dev).cumsum(0).to(torch.int32),
                "ragged": not same, "values": case["values"], "touched": min(p, -(-(max(new) + g - 1) // g)),
                "kvalues": torch.empty(b * p, kv, g, d, dtype=DTYPES[dt], device=r.dev) if case["values"] else None,
                "vvalues": torch.empty(b * p, kv, d, g, dtype=DTYPES[dt], device=r.dev) if case["values"] else None}
    b, n, longest = case["batch"], case["new"], case["longest"]
    p = -(-longest // g)
    whole = lambda *shape: r.normal(*shape, std=36.0).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    qkv = r.normal(b, n, h + 2 * kv, d, dtype=dt)
    return {"kind": kind, "q": qkv[:, :, :h], "kpages": whole(b * p, kv, g, d), "vpages": whole(b * p, kv, d, g),
            "kscales": (0.75 + 0.5 * r.uniform(b * p, kv)) / 36, "vscales": (0.75 + 0.5 * r.uniform(b * p, kv)) / 36,
            "ktail": r.normal(b, kv, slots, d, dtype=dt), "vtail": r.normal(b, kv, d, slots, dtype=dt),
            "table": r.order(b * p).view(b, p), "lens": r.whole(max(n, longest // 2), max(n, longest) + 1, b).clamp_(max=p * g),
            "scale": d ** -0.5}


# ------------------------------------------------------------------------------ one call
def run(state):
    s, kind = state, state["kind"]
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import torch_xdna  # noqa: F401  (registers the ops)
        ops = torch.ops.xdna
        with torch.no_grad():
            if kind == "rotary":
                return ops.rotary(s["x"], s["positions"], s["freqs"], s["magnitude"], s["interleaved"])
            if kind == "norm":
                return ops.residual_norm(s["x"], s["o"], s["weight"], s["post"], s["gate"], s["scale"], EPS)
            if kind == "append":
                q = ops.cache_append(s["k"], s["v"], s["kpages"], s["vpages"], s["kscales"], s["vscales"], s["ktail"], s["vtail"],
                                     s["table"], s["lens"], s["starts"] if s["ragged"] else None, s["q"], s["freqs"], 1.0,
                                     s["interleaved"])
                return _held(s, q)
            return ops.attention_cache(s["q"], s["kpages"], s["vpages"], s["kscales"], s["vscales"], s["ktail"], s["vtail"],
                                       s["table"], s["lens"], s["scale"])
    with torch.no_grad():
        return {"rotary": _rotary, "norm": _norm, "append": _append, "cache": _cache}[kind](s)


def _held(s, q):
    """What the cache holds after an append: the open pages as they are, the whole ones as the values they stand for."""
    if not s["values"]:
        return q, s["ktail"], s["vtail"]
    torch.mul(s["kpages"], s["kscales"][:, :, None, None], out=s["kvalues"])
    torch.mul(s["vpages"], s["vscales"][:, :, None, None], out=s["vvalues"])
    return q, s["ktail"], s["vtail"], s["kvalues"], s["vvalues"]


def _turn(x, positions, freqs, magnitude, interleaved):
    """x [T, H, D] in float32, its first 2 len(freqs) dims turned."""
    n = 2 * freqs.shape[0]
    angle = positions.double()[:, None, None] * freqs
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    f = x.float()
    a, b = (f[..., 0:n:2], f[..., 1:n:2]) if interleaved else (f[..., :n // 2], f[..., n // 2:n])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, f[..., n:]], -1)


def _rotary(s):
    return _turn(s["x"], s["positions"], s["freqs"], s["magnitude"], s["interleaved"]).to(s["x"].dtype)


def _norm(s):
    f = s["o"].float()
    if s["post"] is not None:
        f = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        f = f * s["gate"].float()
    x = s["x"].float() + s["scale"] * f
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    return x.to(s["x"].dtype), y.to(s["o"].dtype)


def _fill(pages, scales, page, full, dense):
    """The dense pages [b, n, kv, ..] that are full go into the pool as whole numbers with a scale."""
    scale = dense.abs().amax((-1, -2)) / 127
    whole = torch.round(dense / torch.where(scale == 0, 1.0, scale)[..., None, None]).to(torch.int8)
    scales[page] = torch.where(full[..., None], scale, scales[page])
    pages[page] = torch.where(full[..., None, None, None], whole, pages[page])


def _append(s):
    k, v, lens, starts, table = s["k"], s["v"], s["lens"].long(), s["starts"].long(), s["table"].long()
    t, kv, d = k.shape
    b, slots, g = lens.shape[0], s["ktail"].shape[2], s["kpages"].shape[2]
    at = torch.arange(t, device=k.device)
    seq = torch.searchsorted(starts, at, right=True) - 1
    pos = lens[seq] + at - starts[seq]
    q = _turn(s["q"], pos, s["freqs"], 1.0, s["interleaved"]).to(s["q"].dtype)
    k = _turn(k, pos, s["freqs"], 1.0, s["interleaved"]).to(k.dtype)
    end = (lens + starts[1:] - starts[:-1])[:, None]
    # the pages that new tokens fall into, dense: old tokens from the open page, new ones from the call
    first = lens[:, None] // g * g
    p = first + torch.arange(s["touched"] * g, device=k.device)                                     # [b, touched g]
    token = (starts[:-1, None] + p - lens[:, None]).clamp(0, t - 1)
    old, rows = (p < lens[:, None])[:, :, None, None], torch.arange(b, device=k.device)[:, None]
    kd = torch.where(old, s["ktail"][rows, :, p % slots], k[token]).float().view(b, -1, g, kv, d)
    vd = torch.where(old, s["vtail"][rows, :, :, p % slots], v[token]).float().view(b, -1, g, kv, d)
    column = first // g + torch.arange(s["touched"], device=k.device)
    full = ((column + 1) * g <= end)
    page = table.gather(1, column.clamp(max=table.shape[1] - 1))
    _fill(s["kpages"], s["kscales"], page, full, kd.permute(0, 1, 3, 2, 4))
    _fill(s["vpages"], s["vscales"], page, full, vd.permute(0, 1, 3, 4, 2))
    # each place of the open pages: the last token that falls on it, if it is a new one
    place = torch.arange(slots, device=k.device)
    last = end - 1 - (end - 1 - place) % slots                                                      # [b, slots]
    token, new = (starts[:-1, None] + last - lens[:, None]).clamp(0, t - 1), (last >= lens[:, None])
    s["ktail"].copy_(torch.where(new[:, None, :, None], k[token].transpose(1, 2), s["ktail"]))
    s["vtail"].copy_(torch.where(new[:, None, None, :], v[token].permute(0, 2, 3, 1), s["vtail"]))
    return _held(s, q)


def _cache(s):
    q, table = s["q"].float(), s["table"].long()
    b, n, h, d = q.shape
    kv, g, slots = s["kpages"].shape[1], s["kpages"].shape[2], s["ktail"].shape[2]
    lens = s["lens"].long()[:, None]
    k = s["kpages"][table].float() * s["kscales"][table][..., None, None]                           # [b, pages, kv, g, d]
    v = s["vpages"][table].float() * s["vscales"][table][..., None, None]                           # [b, pages, kv, d, g]
    whole = lens // g * g
    open_ = whole + torch.arange(g, device=q.device)                                                # [b, g]
    rows = torch.arange(b, device=q.device)[:, None]
    k = torch.cat([k.transpose(1, 2).reshape(b, kv, -1, d), s["ktail"][rows, :, open_ % slots].transpose(1, 2).float()], 2)
    v = torch.cat([v.permute(0, 2, 1, 4, 3).reshape(b, kv, -1, d), s["vtail"][rows, :, :, open_ % slots].transpose(1, 2).float()], 2)
    p = torch.arange(table.shape[1] * g, device=q.device).expand(b, -1)
    p = torch.cat([torch.where(p < whole, p, 1 << 40), open_], 1)                                   # a key's place
    seen = p[:, None, :] <= (lens - n + torch.arange(n, device=q.device))[:, :, None]               # [b, n, keys]
    qg = q.view(b, n, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    scores = (qg @ k.transpose(2, 3)).view(b, kv, n, h // kv, -1) * s["scale"]
    seen = seen[:, None, :, None, :]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total == 0, 1.0, total)).view(b, kv, n * (h // kv), -1)
    o = (w @ v).view(b, kv, n, h // kv, d).permute(0, 2, 1, 3, 4)
    return o.reshape(b, n, h, d).to(s["q"].dtype)


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, esz = case["kind"], ESZ[case["dtype"]]
    if kind == "rotary":
        t, h, d, n = (case[c] for c in ("tokens", "heads", "dim", "turned"))
        return {"bytes": 2 * t * h * d * esz + 4 * t + 4 * n, "flops": 3 * t * h * n}
    if kind == "norm":
        n, w = case["rows"], case["width"]
        gate = {"": 0, "one": w, "row": n * w}[case["gate"]]
        return {"bytes": n * w * (2 * ESZ[case["stream"]] + 2 * esz) + (gate + w * (1 + case["post"])) * esz,
                "flops": n * w * (6 + 4 * case["post"] + bool(gate))}
    h, kv, d, g = case["heads"], case["kv"], case["dim"], case["page"]
    if kind == "append":
        new = _new(case)
        t = sum(new)
        # the open pages' 16-bit tokens, and the whole pages' 8-bit ones (of old tokens too, on average)
        return {"bytes": t * (2 * h + 2 * kv) * d * esz + sum(min(n, 2 * g) for n in new) * 2 * kv * d * esz
                + case["values"] * sum(n // g * g for n in new) * 2 * kv * d, "flops": 3 * t * (h + kv) * case["turned"] + 2 * t * kv * d}
    b, n, longest = case["batch"], case["new"], case["longest"]
    mean = (max(n, longest // 2) + max(n, longest)) / 2
    return {"bytes": int(2 * b * mean * kv * d + 2 * b * n * h * d * esz), "flops": int(4 * b * n * mean * h * d)}


# ------------------------------------------------------------------------------ in 64 bits
def _turn64(x, positions, freqs, magnitude, interleaved):
    """x [T, H, D] as complex numbers times m e^(i theta)."""
    half = freqs.shape[0]
    z = torch.polar(torch.full((x.shape[0], 1, half), magnitude, dtype=torch.float64, device=x.device),
                    positions.double().view(-1, 1, 1) * freqs.view(1, 1, -1))
    y = x.double().clone()
    part = y[..., :2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    part = part if interleaved else part.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(part.contiguous()) * z)
    y[..., :2 * half] = (turned if interleaved else turned.transpose(-1, -2)).flatten(-2)
    return y


def exact(case, seed):
    """The definitions in float64, a sequence or a head at a time. Turned keys are rounded to their type before they are
    put into 8 bits, and a page's scale to float32, as the cache holds them."""
    with torch.no_grad():
        s, kind = prepare(case, seed), case["kind"]
        if kind == "rotary":
            return _turn64(s["x"], s["positions"], s["freqs"], s["magnitude"], s["interleaved"])
        if kind == "norm":
            o = s["o"].double()
            if case["post"]:
                o = o / (o.pow(2).sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * s["post"].double()
            o = o * s["gate"].double() if case["gate"] else o
            x = s["x"].double() + o * s["scale"]
            return x, x / (x.pow(2).sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * s["weight"].double()
        kv, d, g = case["kv"], case["dim"], case["page"]
        slots = s["ktail"].shape[2]
        if kind == "append":
            new, q, at, dt = _new(case), [], 0, s["k"].dtype
            ktail, vtail = s["ktail"].double(), s["vtail"].double()
            kvalues = torch.zeros(s["kpages"].shape, dtype=torch.float64, device=ktail.device)
            vvalues = torch.zeros(s["vpages"].shape, dtype=torch.float64, device=ktail.device)
            for i, n in enumerate(new):
                before = int(s["lens"][i])
                pos = torch.arange(before, before + n, device=ktail.device)
                q.append(_turn64(s["q"][at:at + n], pos, s["freqs"], 1.0, s["interleaved"]))
                k = _turn64(s["k"][at:at + n], pos, s["freqs"], 1.0, s["interleaved"])
                v = s["v"][at:at + n].double()
                first = before // g * g
                past = torch.arange(first, before, device=ktail.device) % slots
                kall = torch.cat([s["ktail"][i][:, past].transpose(0, 1).double(), k.to(dt).double()])
                vall = torch.cat([s["vtail"][i][:, :, past].permute(2, 0, 1).double(), v])
                for j in range((before + n - first) // g if case["values"] else 0):
                    page = int(s["table"][i, first // g + j])
                    for part, values, dims in ((kall, kvalues, (1, 0, 2)), (vall, vvalues, (1, 2, 0))):
                        block = part[j * g:(j + 1) * g].permute(dims)
                        scale = (block.abs().flatten(1).max(1).values / 127).float().double()[:, None, None]
                        values[page] = torch.round(block / scale.masked_fill(scale == 0, 1)) * scale
                keep = pos[-slots:]
                ktail[i][:, keep % slots] = k[-slots:].transpose(0, 1)
                vtail[i][:, :, keep % slots] = v[-slots:].permute(1, 2, 0)
                at += n
            return (torch.cat(q), ktail, vtail, kvalues, vvalues) if case["values"] else (torch.cat(q), ktail, vtail)
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        n, group = case["new"], case["heads"] // kv
        for i in range(case["batch"]):
            length = int(s["lens"][i])
            whole = length // g
            pages, place = s["table"][i, :whole].long(), torch.arange(whole * g, length, device=out.device) % slots
            for c in range(kv):
                k = s["kpages"][pages, c].double() * s["kscales"][pages, c].double()[:, None, None]
                v = (s["vpages"][pages, c].double() * s["vscales"][pages, c].double()[:, None, None]).transpose(1, 2)
                k = torch.cat([k.reshape(-1, d), s["ktail"][i, c, place].double()])
                v = torch.cat([v.reshape(-1, d), s["vtail"][i, c][:, place].t().double()])
                for j in range(n):
                    m, heads = length - n + j + 1, slice(c * group, (c + 1) * group)
                    out[i, j, heads] = torch.softmax(s["q"][i, j, heads].double() @ k[:m].t() * s["scale"], dim=-1) @ v[:m]
        return out
