"""The language model operators (torch_xdna.lm) on host tensors: the plain route against float64, the refusals, the shape
functions under fake tensors, and the entry points' argument checks. No GPU is needed."""
import ctypes
import math

import pytest
import torch

from lm_reference import w4_case, w4_reference, w4_tolerance
from torch_xdna import kernels, lm


# ------------------------------------------------------------------------------ linear_w4
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group,zeros,bias", [(1, 5, 32, 32, True, True), (3, 17, 192, 64, False, False),
                                                    (7, 33, 256, 128, True, False)])
def test_w4_host(m, n, k, group, zeros, bias, dtype):
    args = w4_case(m, n, k, group, zeros, bias, dtype, seed=m)
    y = lm.linear_w4(*args)
    assert y.dtype == args[0].dtype and y.shape == (m, n)
    want, size = w4_reference(*args)
    assert bool(((y.double() - want).abs() <= w4_tolerance(want, size, args[0].dtype, k)).all())


def test_w4_shapes_and_op():
    x, q, s, z, b = w4_case(6, 40, 64, 32, True, True, "bf16", seed=3)
    want = lm.linear_w4(x, q, s, z, b)
    assert torch.equal(torch.ops.xdna.linear_w4(x.view(2, 3, 64), q, s, z, b), want.view(2, 3, 40))
    assert torch.equal(torch.ops.xdna.linear_w4(x[0], q, s, z, b), want[0])
    assert lm.linear_w4(x[:0], q, s, z, b).shape == (0, 40)
    assert torch.equal(lm.linear_w4(x, q, s, torch.full_like(z, 8), None), lm.linear_w4(x, q, s))
    torch.library.opcheck(torch.ops.xdna.linear_w4.default, (x, q, s, z, b), test_utils=("test_schema", "test_faketensor"))


def test_w4_quantize():
    """Every weight comes back within half a step of its group (the clamps move none), and zeros exactly."""
    g = torch.Generator().manual_seed(0)
    w = torch.randn(24, 256, generator=g) * 0.02
    w[3] = 0
    w[4, :32] = w[4, :32].abs() + 1          # a group of one sign: its range starts at 0
    for sym in (False, True):
        q, s, z = lm.quantize_w4(w, 32, symmetric=sym)
        assert (z is None) == sym and q.shape == (24, 128) and s.shape == (24, 8)
        back = lm.linear_w4(torch.eye(256), q, s, z).t()
        step = s.repeat_interleave(32, dim=1)
        # asymmetric: the rounded zero point moves the range by up to half a step, so its ends clamp by as much again
        assert bool(((back - w).abs() <= (0.5 if sym else 1.0) * step * (1 + 1e-5)).all())
        assert bool((back[3] == 0).all())


def test_w4_refusals():
    x, q, s, z, b = w4_case(2, 8, 128, 32, True, True, "f32", seed=1)
    bad = [(x.double(), q, s, z, b), (x, q.to(torch.int8), s, z, b), (x, q, s, z.int(), b), (x, q, s.double(), z, b),
           (x, q, s, z, b.double())]
    for args in bad:
        with pytest.raises(TypeError):
            lm.linear_w4(*args)
    bad = [(x[:, :64], q, s, z, b), (x, q[:4], s, z, b), (x, q, s[:, :3].contiguous(), z, b), (x, q, s, z[:4], b),
           (x, q, s, z, b[:4]), (x, q.t().contiguous().t(), s, z, b), (x, q, s[:, :0], z, b),
           (x, q, s.repeat(1, 2), None, b), (x[..., None], q, s, z, b), (x, q[0], s, z, b)]
    for args in bad:
        with pytest.raises(ValueError):
            lm.linear_w4(*args)
    with pytest.raises(ValueError):
        lm.linear_w4(x, q.to("meta"), s, z, b)
    for w, group in [(torch.zeros(4, 64), 48), (torch.zeros(4, 64), 128), (torch.zeros(64), 32), (torch.zeros(4, 0), 32)]:
        with pytest.raises(ValueError):
            lm.quantize_w4(w, group)


def test_w4_entry_point_checks():
    f, p = kernels.lib().xdna_linear_w4, ctypes.c_void_p(16)

    def call(x=p, xd=1, ldx=64, q=p, s=p, sd=1, z=None, b=None, bd=0, y=p, m=1, n=4, k=64, g=32):
        return f(x, xd, ldx, q, s, sd, z, b, bd, y, m, n, k, g, None)

    assert call(m=0) == 0 and call(n=0) == 0
    for bad in (dict(xd=3), dict(sd=7), dict(b=p, bd=4), dict(g=16), dict(g=48), dict(k=48, g=32), dict(m=-1), dict(ldx=32),
                dict(x=None), dict(q=None), dict(s=None), dict(y=None), dict(x=ctypes.c_void_p(24)), dict(ldx=68),
                dict(q=ctypes.c_void_p(8)), dict(k=0), dict(k=1 << 23, ldx=1 << 23), dict(ldx=1 << 23), dict(n=1 << 27)):
        assert call(**bad) == -1, bad
    assert "linear_w4" in kernels.lib().xdna_last_error().decode()
