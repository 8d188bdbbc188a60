"""attention_cache on the MI355X at values where a kernel can part from the definition: the functions of
test_lm_host_cache_edges.py."""
import pytest
import torch

import test_lm_host_cache_edges as host
from torch_xdna import lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_infinite_keys(gpu, dim, dtype):
    """Head dims that the kernels hold as they are, and those that they fill up to the next multiple of 32."""
    host.infinite_keys(gpu, dim, dtype)


@pytest.mark.parametrize("dtype,power", host.LARGE)
@pytest.mark.parametrize("dim,n,group,page,length,scale", [
    (32, 2, 2, 16, 45, 0.125), (64, 1, 1, 64, 300, -0.3), (128, 1, 8, 32, 70, 0.17), (96, 5, 7, 32, 1500, 0.11), (48, 3, 6, 128, 5000, 0.125),
    (128, 2, 16, 16, 40, -0.09), (64, 1, 4, 128, 60, 0.2)])
def test_large_scores(gpu, dtype, power, dim, n, group, page, length, scale):
    """In one page, over the waves of a workgroup, over parts, in the open page alone."""
    host.large_scores(gpu, dtype, dim, n, group, page, length, power, scale)


def test_permuted(gpu):
    host.permuted(gpu)


def test_limits(gpu):
    """Sizes past what the kernels' indexes reach are wrong arguments like others: refused as such, before anything is launched."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    cache = lm.cache8(1, 1, 1, 16, 16, 16, device=gpu)
    q = torch.zeros(1, 1, 1, 16, dtype=torch.bfloat16, device=gpu)
    k = torch.zeros(1, 1, 16, dtype=torch.bfloat16, device=gpu)
    f = lm.rotary_freqs(16, device=gpu)[0]
    for x in (q.expand(1, 1 << 23, 1, 16), q.expand(1, 1, 1 << 16, 16), q.expand(1, 1 << 12, 1 << 11, 16)):
        with pytest.raises(ValueError):
            lm.attention_cache(x, cache, i32(1))
    far = cache._replace(table=cache.table[:, :1].expand(1, 1 << 26))
    for call in (lambda: lm.attention_cache(q, far, i32(1)), lambda: lm.cache_append(far, i32(0), k, k),
                 lambda: lm.cache_append(cache, i32(0), k, k, None, k.expand(1, 1 << 16, 16), f),
                 lambda: lm.cache_append(cache, i32(0), k.expand(1 << 24, 1, 16), k.expand(1 << 24, 1, 16)),
                 lambda: lm.rotary(torch.zeros(1, 1 << 20, 16, dtype=torch.bfloat16, device=gpu), i32(0), f)):
        with pytest.raises(ValueError):
            call()


def test_logits_as_they_are(gpu):
    host.logits_as_they_are(gpu)
