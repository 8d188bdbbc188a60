"""Error bounds of linear_w4 that follow the kernels' sums, in float64, and the sizes they are asked at -- TEST INFRASTRUCTURE.

The kernels form float32 sums over a step of a group (32, 64 or 128 k, the largest that divides the group) before the scale
goes on; the steps' results are then added up over lanes, waves and parts of K. Each addition and product is off by at
most half a step (2^-24) of what has been summed so far:

* in a step, `inner` of them: one for each k (three for float32, whose x is cut in three parts for the matrix units), and
  8 more. The terms are (q - z) x s, or in bfloat16 (128 + q) x s and (128 + z) x s;
* over the steps, `outer`: one for each step, and 32 for lanes, waves, parts, scale and bias. The terms are
  (q - z) x s.

In the worst case what has been summed is the sum of the terms' sizes: the bound of each output. x is drawn from N(0, 1), so the
partial sums' root mean square over many outputs is at most that of the terms' squares: the bound of the outputs'
norm, far tighter for long K (of the steps' norms no cancelling among each other is assumed). The output rounds once.
"""
import torch

from lm_reference import U32, half_step

# m, n, k, group, zeros, bias
SIZES = [
    (1, 3, 32, 32, False, True), (1, 67, 992, 32, True, False), (1, 40, 20512, 32, True, True), (1, 9, 17152, 128, False, False),
    (1, 70, 9216, 96, True, False), (1, 8200, 544, 32, True, True), (1, 8193, 1280, 160, True, True), (1, 130, 4096, 128, True, False),
    (2, 40, 8320, 128, True, True), (3, 77, 4192, 32, False, True), (4, 33, 2048, 64, True, False), (4, 2100, 2048, 128, True, True),
    (17, 70, 1376, 32, True, True), (33, 65, 1056, 96, False, False), (64, 130, 4512, 32, True, True), (50, 64, 5120, 160, True, False),
    (30, 90, 544, 32, False, True), (20, 50, 20512, 32, True, True), (33, 8500, 640, 64, True, True), (16, 200, 9216, 64, True, True),
    (47, 300, 2240, 64, True, False), (8, 100, 2176, 128, True, True), (70, 40, 3200, 320, True, True), (200, 17, 4224, 128, True, False),
    (40, 130, 14336, 64, True, False)]


def w4_bounds(x, q, s, z, b):
    """(y in float64, a bound for each output's error, a bound for the errors' norm)."""
    x, q, s, z, b = (None if t is None else t.cpu() for t in (x, q, s, z, b))
    n, groups = s.shape
    k = x.shape[1]
    group = k // groups
    step = 128 if group % 128 == 0 else 64 if group % 64 == 0 else 32
    inner, outer = (3 if x.dtype == torch.float32 else 1) * step + 8, k // step + 32
    xd, sd = x.double(), s.double().unsqueeze(-1)
    qd = torch.stack([q % 16, q // 16], dim=-1).view(n, groups, group).double()
    zd = torch.full_like(sd, 8.0) if z is None else z.double().unsqueeze(-1)
    w = ((qd - zd) * sd).view(n, k)
    held = ((256 + qd + zd) * sd).view(n, k) if x.dtype == torch.bfloat16 else w.abs()      # a step's terms over x
    y, size, square = xd @ w.t(), xd.abs() @ w.abs().t(), xd.square() @ w.square().t()
    if b is not None:
        y, size, square = y + b.double(), size + b.double().abs(), square + b.double().square()
    steps = torch.zeros_like(y)                                # the sum over steps of the root of the terms' squares
    for i in range(0, k, step):
        steps += (xd[:, i:i + step].square() @ held[:, i:i + step].square().t()).sqrt()
    each = half_step(x.dtype) * y.abs() * (1 + 2.0 ** -6) + U32 * (inner * (xd.abs() @ held.t()) + outer * size) + 1e-30
    norm = half_step(x.dtype) * y.norm() * (1 + 2.0 ** -6) + U32 * (inner * steps.norm() + outer * square.sqrt().norm()) + 1e-30
    return y, each, norm


def w4_off(got, bounds):
    """What of the bounds `got` breaks, as a text; empty if it keeps them."""
    want, each, norm = bounds
    err = (got.double().cpu() - want).abs()
    out = []
    bad = ~(err <= each)
    if bool(bad.any()):
        out.append(f"{int(bad.sum())} of {bad.numel()} off, by up to {float((err / each).max()):.3g} bounds")
    if not bool(err.norm() <= norm):
        out.append(f"the errors' norm is {float(err.norm() / norm):.3g} bounds")
    return "; ".join(out)
