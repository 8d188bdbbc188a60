"""The language model operators' way from torch.ops.xdna.* to the GPU: refusals, autograd, tracing, registration, the report."""
import pytest
import torch

import torch_xdna
from lm_reference import causal_case, logits_case, prefix_case, w4_case
from torch_xdna import lm, runtime

pytestmark = pytest.mark.gpu
ops = torch.ops.xdna


def _cases(dev):
    return {"linear_w4": w4_case(3, 40, 128, 32, True, True, "bf16", dev=dev),
            "attention_causal": causal_case([5, 9], 4, 2, 16, "bf16", dev=dev) + (None,),
            "attention_prefix": prefix_case(3, 6, 4, 4, 2, 16, "bf16", dev=dev) + (0.3,),
            "logits_adjust": logits_case(2, 70, 5, "bf16", "row", dev=dev)}


NAMES = ("linear_w4", "attention_causal", "attention_prefix", "logits_adjust")


def test_refusals(gpu):
    x, q, s, z, b = w4_case(2, 8, 128, 32, True, True, "f32", dev=gpu)
    for f in (lm.linear_w4, ops.linear_w4):
        for args in ((x.double(), q, s, z, b), (x, q.to(torch.int8), s, z, b), (x, q, s, z.int(), b), (x, q, s.double(), z, b),
                     (x, q, s, z, b.double())):
            with pytest.raises(TypeError):
                f(*args)
        odd = torch.zeros(8 * 64 + 16, dtype=torch.uint8, device=gpu)[1:1 + 8 * 64].view(8, 64)
        for args in ((x[:, :64], q, s, z, b), (x, q[:4], s, z, b), (x, q, s[:, :3].contiguous(), z, b), (x, q, s, z[:4], b),
                     (x, q, s, z, b[:4]), (x, q.t().contiguous().t(), s, z, b), (x, q, s[:, :0], z, b), (x, q, s.repeat(1, 2), None, b),
                     (x[..., None], q, s, z, b), (x, q[0], s, z, b), (x, q.cpu(), s, z, b), (x, q, s, z, b.cpu()), (x, odd, s, z, b),
                     (x.cpu(), q, s, z, b)):
            with pytest.raises(ValueError):
                f(*args)
    q, k, v, starts = causal_case([5, 4], 4, 2, 16, "bf16", dev=gpu)
    for args in ((q.float(), k.float(), v.float(), starts), (q, k.half(), v, starts), (q, k, v, starts.long())):
        with pytest.raises(TypeError):
            lm.attention_causal(*args)
    for args in ((q[0], k, v, starts), (q, k[:8], v[:8], starts), (q, k, v[:, :1], starts), (q[:, :3], k, v, starts),
                 (q[..., :12], k[..., :12], v[..., :12], starts), (q, k[:, :0], v[:, :0], starts), (q[:, :0], k, v, starts),
                 (q.repeat(1, 1, 9), k.repeat(1, 1, 9), v.repeat(1, 1, 9), starts), (q, k, v, starts[None]), (q, k, v, starts[:0]),
                 (q, k, v, starts.cpu())):
        with pytest.raises(ValueError):
            lm.attention_causal(*args)
    q, kp, vp, kc, vc, lens = prefix_case(3, 6, 4, 4, 2, 16, "f16", dev=gpu)
    for args in ((q.bfloat16(), kp, vp, kc, vc, lens), (q, kp, vp, kc, vc.bfloat16(), lens), (q, kp, vp, kc, vc, lens.long())):
        with pytest.raises(TypeError):
            lm.attention_prefix(*args)
    for args in ((q[0], kp, vp, kc, vc, lens), (q, kp[..., :8], vp[..., :8], kc, vc, lens), (q, kp, vp[:3], kc, vc, lens),
                 (q, kp, vp, kc[:2], vc[:2], lens), (q, kp, vp, kc[:, :, :1], vc[:, :, :1], lens), (q, kp, vp, kc, vc, lens[:2]),
                 (q, kp, vp, kc, vc, lens[None]), (q[:, :3], kp, vp, kc, vc, lens), (q, kp, vp, kc.cpu(), vc, lens)):
        with pytest.raises(ValueError):
            lm.attention_prefix(*args)
    x, tokens, lens, rep, pres, freq, bias, allowed = logits_case(2, 70, 5, "f32", "row", dev=gpu)
    for kw in (dict(logits=x.double()), dict(tokens=tokens.short()), dict(lens=lens.long()), dict(repetition=rep.double()),
               dict(bias=bias.half()), dict(allowed=allowed.long())):
        with pytest.raises(TypeError):
            lm.logits_adjust(**{**dict(logits=x, tokens=tokens, lens=lens), **kw})
    for kw in (dict(logits=x[0]), dict(tokens=tokens[0]), dict(tokens=tokens[:1]), dict(lens=lens[:1]), dict(lens=None),
               dict(tokens=None), dict(repetition=rep[:1]), dict(presence=pres[None]), dict(bias=bias[:, :3]), dict(bias=bias[:1]),
               dict(allowed=allowed[:, :2]), dict(frequency=freq.cpu())):
        with pytest.raises(ValueError):
            lm.logits_adjust(**{**dict(logits=x, tokens=tokens, lens=lens), **kw})


@pytest.mark.parametrize("name", NAMES)
def test_autograd_and_modes(gpu, name):
    """The forward pass works with inputs that need a gradient, under no_grad and in inference mode alike; asking for the
    gradient raises. Fake tensors launch nothing."""
    args = _cases(gpu)[name]
    f = getattr(ops, name)
    want = f(*args)
    assert not want.requires_grad
    first = args[0].clone().requires_grad_()
    got = f(first, *args[1:])
    assert got.requires_grad and torch.equal(got, want)
    with pytest.raises(RuntimeError):
        got.float().sum().backward()
    with torch.no_grad():
        assert not f(first, *args[1:]).requires_grad
    with torch.inference_mode():
        assert torch.equal(f(*args), want)
    before = torch_xdna.stats.as_dict()["gpu_launches"]
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = f(*(mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args))
    assert fake.shape == want.shape and fake.dtype == want.dtype
    assert torch_xdna.stats.as_dict()["gpu_launches"] == before
    torch.library.opcheck(getattr(f, "default"), args, test_utils=("test_schema", "test_faketensor"))


def test_compiled_and_report(gpu):
    """A decode step's operators in one compiled function give what they give alone, and the report counts them."""
    w, c, p, s = (_cases(gpu)[n] for n in NAMES)

    def step():
        return (ops.linear_w4(*w) * 2, ops.attention_causal(*c) + 1, ops.attention_prefix(*p), ops.logits_adjust(*s))

    want = step()
    runtime.stats.reset()
    got = torch.compile(step, fullgraph=True)()
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=0, atol=0)
    d = torch_xdna.stats.as_dict()
    assert d["calls"]["gpu"] == 4 and d["gpu_launches"] == 4
    runtime.stats.reset()
    assert torch_xdna.stats.as_dict()["calls"].get("gpu", 0) == 0


def test_without_the_library(gpu, monkeypatch):
    """A GPU tensor with the operators' library missing raises."""
    from torch_xdna import kernels

    monkeypatch.setattr(kernels, "_torch_lib", None)
    monkeypatch.setattr(kernels, "TORCH_LIB_PATH", "/nowhere/libxdna_torch.so")
    with pytest.raises(RuntimeError, match="not built"):
        lm.linear_w4(*_cases(gpu)["linear_w4"])


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode(gpu, name):
    """There is no forward-mode derivative: a tangent raises, on the GPU and on the host, and is not dropped."""
    for dev in (gpu, "cpu"):
        args = _cases(dev)[name]
        f = getattr(ops, name)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(args[0], torch.ones_like(args[0]))
            with pytest.raises(NotImplementedError):
                f(dual, *args[1:])
            with torch.no_grad(), pytest.raises(NotImplementedError):
                f(dual, *args[1:])
            assert f(*args).shape == f(args[0], *args[1:]).shape
        first = args[0].clone().requires_grad_()
        with pytest.raises(RuntimeError):
            f(first, *args[1:]).float().sum().backward()
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda t: f(t, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
