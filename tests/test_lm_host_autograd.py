"""Derivatives of the language model operators on host tensors: torch.ops.xdna.* have none and raise, in reverse mode where
the gradient is asked for and in forward mode at the call; lm's functions are plain torch there and have them. No GPU is needed."""
import pytest
import torch

from lm_reference import causal_case, logits_case, prefix_case, w4_case
from torch_xdna import lm

CASES = {"linear_w4": lambda: w4_case(3, 40, 128, 32, True, True, "bf16"),
         "attention_causal": lambda: causal_case([5, 9], 4, 2, 16, "bf16") + (None,),
         "attention_prefix": lambda: prefix_case(3, 6, 4, 4, 2, 16, "bf16") + (0.3,),
         "logits_adjust": lambda: logits_case(2, 70, 5, "bf16", "row")}


@pytest.mark.parametrize("name", CASES)
def test_host_ops_have_no_derivative(name):
    args = CASES[name]()
    f = getattr(torch.ops.xdna, name)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(NotImplementedError):
            f(dual, *args[1:])
        plain = getattr(lm, name)(dual, *args[1:])
        assert torch.autograd.forward_ad.unpack_dual(plain).tangent is not None
    first = args[0].clone().requires_grad_()
    got = f(first, *args[1:])
    assert got.requires_grad and torch.equal(got, f(*args))
    with pytest.raises(RuntimeError):
        got.float().sum().backward()
    with torch.no_grad():
        assert not f(first, *args[1:]).requires_grad
    torch.compile(f, fullgraph=True, backend="aot_eager")(*args)
