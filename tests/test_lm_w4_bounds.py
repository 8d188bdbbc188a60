"""The bounds that linear_w4's results are held to (lm_w4_bounds.py): the exact result, rounded, keeps them at every size, and
every mistake that a kernel of windows, steps and parts could make breaks them. No GPU is needed."""
import pytest
import torch

from lm_reference import DTYPES, w4_case, w4_weight
from lm_w4_bounds import SIZES, w4_bounds, w4_off


def _product(x, q, s, z, b):
    w, sd = w4_weight(q, s, z)
    y = x.double() @ (w * sd).view(q.shape[0], -1).t()
    return y if b is None else y + b.double()


def _mistakes(x, q, s, z, b):
    """(name, the product with the mistake in it)"""
    group = x.shape[1] // s.shape[1]
    yield "all zeros", torch.zeros(x.shape[0], q.shape[0])
    for name, n in (("the last group lost", group), ("the last 8 of K lost", 8)):
        cut = x.clone()
        cut[:, -n:] = 0
        yield name, _product(cut, q, s, z, b)
    if s.shape[1] > 1:
        yield "scales of the next group", _product(x, q, s.roll(1, 1), z, b)
        if z is not None:
            yield "zero points of the next group", _product(x, q, s, z.roll(1, 1), b)
        if z is not None and x.shape[0] > 1:             # of one row it may be next to nothing: the group's x add up to that
            other = z.clone()
            other[:, -1] = z[:, -2]
            yield "the last group's zero points from the one before", _product(x, q, s, other, b)
    if s.shape[0] > 1:
        yield "scales of the next column", _product(x, q, s.roll(1, 0), z, b)
    yield "nibbles swapped", _product(x, (q << 4) | (q >> 4), s, z, b)
    if x.dtype != torch.bfloat16:
        yield "x in bfloat16", _product(x.bfloat16(), q, s, z, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group,zeros,bias", SIZES)
def test_bounds(m, n, k, group, zeros, bias, dtype):
    args = w4_case(m, n, k, group, zeros, bias, dtype, seed=m + k)
    bounds = w4_bounds(*args)
    assert not w4_off(_product(*args).to(DTYPES[dtype]), bounds)
    for name, y in _mistakes(*args):
        assert w4_off(y.to(DTYPES[dtype]), bounds), name
