"""linear_w4 on the MI355X against float64 (lm_reference.py): every form of the kernels that a size selects."""
import math

import pytest
import torch

from lm_reference import w4_case, w4_reference, w4_tolerance
from torch_xdna import kernels, lm

pytestmark = pytest.mark.gpu


def _check(args, biased=False):
    y = lm.linear_w4(*args)
    want, size = w4_reference(*args)
    tol = w4_tolerance(want, size, y.dtype, args[0].shape[1], biased=biased)
    y = y.double().cpu()
    bad = ~((y - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float(((y - want).abs() / tol).max())} bounds"


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group,zeros,bias", [
    # one row: columns and blocks of every remainder, more blocks than LDS holds at once, waves that share columns
    (1, 3, 32, 32, False, True), (1, 67, 992, 32, True, False), (1, 40, 20512, 32, True, True), (1, 9, 17152, 128, False, False),
    (1, 70, 9216, 96, True, False), (1, 8200, 544, 32, True, True), (1, 8193, 160, 160, False, True),
    # two to four rows of few weights, and of many
    (2, 40, 8320, 128, True, True), (3, 77, 4192, 32, False, True), (4, 33, 2048, 64, True, False), (4, 2100, 2048, 128, True, True),
    # tiles: K in one part and in several, windows of scales that end inside a group
    (17, 70, 1376, 32, True, True), (33, 65, 1056, 96, False, False), (64, 130, 4512, 32, True, True), (50, 64, 5120, 160, True, False),
    (5, 70, 512, 32, True, True), (30, 90, 544, 32, False, True), (64, 100, 640, 128, True, False), (20, 50, 20512, 32, True, True),
    (33, 17000, 640, 64, True, True), (16, 200, 9216, 64, False, True), (47, 300, 2240, 64, True, False), (8, 100, 2176, 128, True, True), (70, 40, 3200, 320, True, True)])
def test_w4_forms(gpu, m, n, k, group, zeros, bias, dtype):
    _check(w4_case(m, n, k, group, zeros, bias, dtype, seed=m + k, dev=gpu), biased=dtype == "bf16")


@pytest.mark.parametrize("dtype,scales", [("bf16", "f32"), ("f16", "f32"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("m,n,k,group", [(1, 50, 4096, 64), (4, 60, 1024, 32), (30, 80, 4096, 32)])
def test_w4_forms_scale_types(gpu, m, n, k, group, dtype, scales):
    _check(w4_case(m, n, k, group, True, True, dtype, seed=2, dev=gpu, scales=scales), biased=dtype == "bf16")


@pytest.mark.parametrize("m,n,k", [(1, 50, 4096), (1, 9000, 512), (3, 40, 1024), (40, 64, 4096)])
def test_w4_not_finite_in_every_form(gpu, m, n, k):
    """bfloat16: an infinity, NaN or a value near the type's largest reaches its own row alone, and as the formula has it."""
    x, q, s, z, _ = w4_case(m, n, k, 128, True, False, "bf16", seed=3, dev=gpu)
    want = lm.linear_w4(x, q, s, z)
    r = m - 1
    low = (q[:, 100 // 2] & 15).float()                      # k = 100, group 0
    for value in (math.inf, -math.inf, math.nan, 2.0 ** 126):
        x2 = x.clone()
        x2[r, 100] = value
        y = lm.linear_w4(x2, q, s, z)
        assert torch.equal(y[:r], want[:r])
        d = low - z[:, 0].float()
        if math.isnan(value):
            assert bool(y[r].isnan().all())
        elif math.isinf(value):
            torch.testing.assert_close(y[r].float(), torch.where(d == 0, math.nan, d.sign() * value), rtol=0, atol=0, equal_nan=True)
        else:
            # the rest of the row is far below half a step of this product
            expect = (d.double() * s[:, 0].double() * value)
            assert bool(((y[r].double() - expect).abs()[d != 0] <= expect.abs()[d != 0] * 2.0 ** -7).all())


def test_w4_split_without_workspace(gpu):
    """The entry point without a workspace splits nothing: the same product to the last rounding."""
    x, q, s, z, b = w4_case(40, 200, 8192, 64, True, True, "f16", seed=4, dev=gpu)
    assert kernels.lib().xdna_linear_w4_ws_bytes(2, 40, 200, 8192) > 0
    y = torch.empty(40, 200, dtype=x.dtype, device=gpu)
    st = kernels.lib().xdna_linear_w4(x.data_ptr(), 2, 8192, q.data_ptr(), s.data_ptr(), 2, z.data_ptr(), b.data_ptr(), 2, y.data_ptr(),
                                      40, 200, 8192, 64, torch.cuda.current_stream().cuda_stream)
    assert st == 0
    want, size = w4_reference(x, q, s, z, b)
    tol = w4_tolerance(want, size, x.dtype, 8192)
    assert bool(((y.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("m,n,k", [(1, 100, 2048), (40, 64, 8192)])
def test_w4_graph(gpu, m, n, k):
    args = w4_case(m, n, k, 64, True, True, "bf16", seed=5, dev=gpu)
    want = lm.linear_w4(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(lm.linear_w4(*args), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lm.linear_w4(*args)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(lm.linear_w4(*args), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
