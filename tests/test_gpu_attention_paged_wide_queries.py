"""Queries whose numbers lie far apart, over an 8-bit cache whose whole numbers are 0 where the largest is: the scores are those of the others."""
import pytest

torch = pytest.importorskip("torch")
import serving_util as u  # noqa: E402
from test_gpu_attention_paged_far_apart import caches, check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_a_query_whose_largest_number_meets_zeros(dev, pkg, new, d):
    """2^22 times the others."""
    cache, q = caches(pkg, [(new, 700), (new, 90)], d, "bf16", "i8", 4, 47)
    q[..., 0] = 2.0 ** 22
    cache.scales[0].fill_(1 / 8)  # scores that differ: a query without its small numbers would weigh all keys alike
    check(dev, pkg, cache, q, "bf16")


@pytest.mark.parametrize("new,most", [(1, 124), (40, 110)])  # a chunk's scores are sums of queries times whole numbers before a step comes to them
def test_queries_near_the_end_of_bf16(dev, pkg, new, most):
    """All numbers around 2^124, up to the last exponent, or around 2^-100: no infinity, nothing lost."""
    for at in (most, -100):
        cache, q = caches(pkg, [(new, 300)], 64, "bf16", "i8", 4, 48)
        q = (u.normal(u.gen(49), q.shape) * 2.0 ** at).bfloat16()
        if at > 0:
            q[..., 5] = 1.5 * 2.0 ** (at + 3)
        cache.scales[0].fill_(2.0 ** (-2 - at if at > 0 else 97))
        check(dev, pkg, cache, q, "bf16")
