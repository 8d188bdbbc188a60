"""attention_cache on the MI355X at values where a kernel can part from the definition: the functions of
test_lm_host_cache_edges.py."""
import pytest

import test_lm_host_cache_edges as host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_infinite_keys(gpu, dim, dtype):
    """Head dims that the kernels hold as they are, and those that they fill up to the next multiple of 32."""
    host.infinite_keys(gpu, dim, dtype)
