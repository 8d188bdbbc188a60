"""linear_w4 on the MI355X within bounds that follow its sums (lm_w4_bounds.py), which no lost part of K, no neighbour's
scale and no x of fewer bits would keep (test_lm_w4_bounds.py)."""
import pytest

from lm_reference import w4_case
from lm_w4_bounds import SIZES, w4_bounds, w4_off
from torch_xdna import lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group,zeros,bias", SIZES)
def test_w4_within_bounds(gpu, m, n, k, group, zeros, bias, dtype):
    args = w4_case(m, n, k, group, zeros, bias, dtype, seed=m + k, dev=gpu)
    off = w4_off(lm.linear_w4(*args), w4_bounds(*args))
    assert not off, off


@pytest.mark.parametrize("dtype,scales", [("bf16", "f32"), ("bf16", "f16"), ("f16", "f32"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("m,n,k,group", [(1, 50, 20512, 32), (4, 60, 1024, 32), (30, 80, 9216, 96), (64, 64, 4096, 128)])
def test_w4_scale_types_within_bounds(gpu, m, n, k, group, dtype, scales):
    args = w4_case(m, n, k, group, True, True, dtype, seed=2, dev=gpu, scales=scales)
    off = w4_off(lm.linear_w4(*args), w4_bounds(*args))
    assert not off, off
