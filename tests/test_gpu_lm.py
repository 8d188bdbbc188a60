"""The language model operators (torch_xdna.lm) on the MI355X against float64 (lm_reference.py), at the sizes and values
where they can go wrong."""
import math

import pytest
import torch

from lm_reference import DTYPES, w4_case, w4_reference, w4_tolerance
from torch_xdna import kernels, lm

pytestmark = pytest.mark.gpu


def _within(y, want, tol):
    y, want, tol = y.double().cpu(), want.cpu(), tol.cpu()
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


# ------------------------------------------------------------------------------ linear_w4
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group,zeros,bias", [
    (1, 1, 32, 32, True, True), (1, 16, 128, 128, False, False), (1, 1001, 1504, 32, True, True),
    (1, 130, 4096, 128, True, False), (2, 31, 96, 96, True, False), (5, 48, 320, 64, False, True),
    (16, 33, 1024, 1024, True, True), (17, 64, 1024, 128, True, False), (33, 40, 2080, 32, False, True),
    (64, 15, 640, 160, True, True), (65, 100, 384, 64, True, True), (200, 17, 4224, 128, True, False)])
def test_w4(gpu, m, n, k, group, zeros, bias, dtype):
    args = w4_case(m, n, k, group, zeros, bias, dtype, seed=m + n, dev=gpu)
    y = lm.linear_w4(*args)
    assert y.dtype == args[0].dtype and y.shape == (m, n)
    want, size = w4_reference(*args)
    _within(y, want, w4_tolerance(want, size, args[0].dtype, k, biased=dtype == "bf16"))


@pytest.mark.parametrize("dtype,scales", [("bf16", "f32"), ("bf16", "f16"), ("f16", "bf16"), ("f16", "f32"), ("f32", "bf16"),
                                          ("f32", "f16")])
def test_w4_scale_types(gpu, dtype, scales):
    args = w4_case(3, 50, 256, 64, True, True, dtype, seed=9, dev=gpu, scales=scales)
    want, size = w4_reference(*args)
    _within(lm.linear_w4(*args), want, w4_tolerance(want, size, args[0].dtype, 256, biased=dtype == "bf16"))


def test_w4_strides_and_zero_points(gpu):
    """Rows of a wider tensor, transposed and unaligned activations, zero points up to 255, the op's own route."""
    x, q, s, z, b = w4_case(6, 40, 256, 64, True, True, "bf16", seed=4, dev=gpu)
    want = lm.linear_w4(x, q, s, z, b)
    wide = torch.full((6, 600), math.nan, dtype=x.dtype, device=gpu)
    for at in (0, 8, 3):
        wide[:, at:at + 256] = x
        assert torch.equal(lm.linear_w4(wide[:, at:at + 256], q, s, z, b), want), at
    assert torch.equal(lm.linear_w4(x.t().contiguous().t(), q, s, z, b), want)
    assert torch.equal(torch.ops.xdna.linear_w4(x.view(2, 3, 256), q, s, z, b).view(6, 40), want)
    assert torch.equal(lm.linear_w4(x, q, s, z, b.repeat_interleave(2)[::2]), want)
    z = torch.randint(0, 256, z.shape, dtype=torch.uint8, device=gpu)
    for dt in DTYPES.values():
        a = (x.to(dt), q, s, z, None)
        ref, size = w4_reference(*a)
        # the sums' terms: (128 + q or 15) + (128 + z or 255) at the most, against the reference's 286
        _within(lm.linear_w4(*a), ref, w4_tolerance(ref, 2 * size, dt, 256, biased=True))
    assert lm.linear_w4(x[:0], q, s, z, b).shape == (0, 40)
    with pytest.raises(ValueError):
        lm.linear_w4(x, q.cpu(), s, z, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_w4_not_finite(gpu, dtype):
    """An infinity or NaN in one row of x reaches that row alone, and as the formula has it."""
    x, q, s, z, b = w4_case(5, 70, 512, 128, True, False, dtype, seed=6, dev=gpu)
    z = z.clamp(max=14)
    x[1, 37], x[3, 300] = math.inf, math.nan
    y = lm.linear_w4(x, q, s, z).cpu()
    clean = x.clone()
    clean[1, 37], clean[3, 300] = 0, 0
    want = lm.linear_w4(clean, q, s, z).cpu()
    assert torch.equal(y[[0, 2, 4]], want[[0, 2, 4]]) and bool(y[3].isnan().all())
    w37 = ((q[:, 18] >> 4).float() - z[:, 0].float()).cpu()          # k = 37: byte 18, high nibble, group 0
    torch.testing.assert_close(y[1], torch.where(w37 == 0, math.nan, w37.sign() * math.inf).to(y.dtype), rtol=0, atol=0,
                               equal_nan=True)


def test_w4_stream_and_repeat(gpu):
    """Another stream than the default one, and the same bits at every call."""
    args = w4_case(40, 500, 2048, 64, True, True, "f16", seed=2, dev=gpu)
    want = lm.linear_w4(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [lm.linear_w4(*args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)
    x = args[0].clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.ops.xdna.linear_w4(x, *args[1:]).sum().backward()
