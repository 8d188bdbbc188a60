"""linear_w4 on the MI355X at the edges of its tiles: columns past N and values that are not finite."""
import math

import pytest
import torch

from lm_reference import w4_case
from torch_xdna import lm

pytestmark = pytest.mark.gpu


def _us(f, before=lambda: None):
    """The shortest of ten calls of f, each right after `before`."""
    best = math.inf
    for _ in range(10):
        before()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        f()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end) * 1e3)
    return best


@pytest.mark.parametrize("m", [4, 40])
def test_w4_ragged_columns_take_the_same_time_after_any_kernel(gpu, m):
    """Columns past N have no scales. What a kernel before left in their place in LDS (NaN, from the same kernel with
    scales of NaN) must not send the last columns through the sums for values that are not finite: those take over 100
    times as long."""
    x, q, s, z, _ = w4_case(m, 8200, 1024, 64, True, False, "bf16", seed=1, dev=gpu)
    full = w4_case(m, 16384, 1024, 64, True, False, "bf16", seed=2, dev=gpu)
    bad = torch.full_like(full[2], math.nan)
    want = lm.linear_w4(x, q, s, z)
    clean = _us(lambda: lm.linear_w4(x, q, s, z), lambda: lm.linear_w4(*full))
    dirty = _us(lambda: lm.linear_w4(x, q, s, z), lambda: lm.linear_w4(full[0], full[1], bad, full[3]))
    print(f"after finite scales {clean:.1f} us, after scales of NaN {dirty:.1f} us")
    assert torch.equal(lm.linear_w4(x, q, s, z), want)
    assert dirty < 3 * clean


def test_w4_rows_that_are_not_finite_cost_their_own_sums_only(gpu):
    """One row of 64 with a NaN: its sums are formed again, value by value, and not those of the other rows (a wave would
    do 16 rows' worth for one, in turn)."""
    x, q, s, z, _ = w4_case(64, 4096, 4096, 64, True, False, "bf16", seed=3, dev=gpu)
    one, every = x.clone(), x.clone()
    one[37, 100], every[:, 100] = math.nan, math.nan
    want = lm.linear_w4(x, q, s, z)
    y = lm.linear_w4(one, q, s, z)
    keep = torch.arange(64, device=gpu) != 37
    assert torch.equal(y[keep], want[keep]) and bool(y[37].isnan().all())
    t1, t64 = _us(lambda: lm.linear_w4(one, q, s, z)), _us(lambda: lm.linear_w4(every, q, s, z))
    print(f"one row {t1:.1f} us, every row {t64:.1f} us")
    assert t1 < t64 / 4


@pytest.mark.parametrize("m,n,k,scales", [(1, 50, 4096, "same"), (1, 9000, 512, "same"), (3, 40, 1024, "same"), (2, 30, 8320, "bf16"),
                                          (8, 100, 2176, "same"), (40, 64, 4096, "f16")])
def test_w4_float32_near_the_largest(gpu, m, n, k, scales):
    """float32 x near the type's largest: the product with q - z passes it, the result does not. Its own row is as the
    formula has it, the others are as they were; infinities and NaN too."""
    x, q, s, z, _ = w4_case(m, n, k, 128, True, False, "f32", seed=5, dev=gpu, scales=scales)
    want = lm.linear_w4(x, q, s, z)
    r, at = m - 1, k - 28                                     # in the last group
    d = (q[:, at // 2] & 15).float() - z[:, -1].float()
    w = d.double() * s[:, -1].double()
    for value in (2.0 ** 126, -1.5 * 2.0 ** 127):
        x2 = x.clone()
        x2[r, at] = value
        y = lm.linear_w4(x2, q, s, z)
        assert torch.equal(y[:r], want[:r])
        # the rest of the row is far below half a step of this product; q - z, the scale and the product round once each
        expect = w * value
        assert float(expect.abs().max()) < torch.finfo(torch.float32).max and bool((d.abs() >= 8).any())
        assert bool(((y[r].double() - expect).abs()[d != 0] <= expect.abs()[d != 0] * 2.0 ** -22).all())
    for value in (math.inf, math.nan):
        x2 = x.clone()
        x2[r, at] = value
        y = lm.linear_w4(x2, q, s, z)
        assert torch.equal(y[:r], want[:r])
        expect = torch.where(d == 0, math.nan, d.sign() * value)
        torch.testing.assert_close(y[r], expect, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_w4_rows_far_apart(gpu, dtype):
    """The last token of every prompt, a view whose rows lie further apart than the kernels' offsets reach."""
    x, q, s, z, b = w4_case(3, 40, 4096, 64, True, True, dtype, seed=6, dev=gpu)
    want = lm.linear_w4(x, q, s, z, b)
    states = torch.zeros(3, 1025, 4096, dtype=x.dtype, device=gpu)
    states[:, -1] = x
    assert states[:, -1].stride(0) > 1 << 22
    assert torch.equal(lm.linear_w4(states[:, -1], q, s, z, b), want)
    assert torch.equal(torch.ops.xdna.linear_w4(states[:, -1:], q, s, z, b), want[:, None])
