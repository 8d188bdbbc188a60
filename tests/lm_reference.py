"""float64 references, inputs and error bounds of the language model operators -- TEST INFRASTRUCTURE.

Rounding to a type moves a value by at most half a step, torch.finfo(t).eps / 2 of it; a float32 sum of n terms is off
by at most n / 2 steps (2^-24 each) of the sum of the terms' sizes, in any order.
"""
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------ linear_w4
def w4_case(m, n, k, group, zeros, bias, dtype, seed=0, dev="cpu", scales="same"):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    x = torch.randn(m, k, generator=g).to(dt)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((0.5 + torch.rand(n, k // group, generator=g)) * 0.005).to(dt if scales == "same" else DTYPES[scales])
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g).to(dt) if bias else None
    return tuple(None if t is None else t.to(dev) for t in (x, q, s, z, b))


def w4_weight(q, s, z):
    n, groups = s.shape
    w = torch.stack([q % 16, q // 16], dim=-1).view(n, groups, -1).double()
    return (w - (8 if z is None else z.double().unsqueeze(-1))), s.double().unsqueeze(-1)


def w4_reference(x, q, s, z, b):
    """(y, the sum of the sizes of y's terms as the kernels hold them: |x| times 128 + q and 128 + z at the most)."""
    x, q, s, z, b = (None if t is None else t.cpu() for t in (x, q, s, z, b))
    n = q.shape[0]
    w, sd = w4_weight(q, s, z)
    y = x.double() @ (w * sd).view(n, -1).t()
    size = x.double().abs() @ (torch.full_like(w, 2 * 143.0) * sd.abs()).view(n, -1).t()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs()
    return y, size


def w4_tolerance(want, size, dtype, k, biased=False):
    """One rounding to the output's type, and float32 sums: of k terms, a scale and a bias. biased: the terms may be
    128 + q and 128 + z times x (bfloat16), else they are at most 16 / 286 of that."""
    return half_step(dtype) * want.abs() * (1 + 2.0 ** -6) + (k + 8) * U32 * size * (1 if biased else 16 / 286) + 1e-30
