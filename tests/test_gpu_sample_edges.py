"""Token sampling where a filter's border lies at the edge of what its numbers can hold, against the 64-bit definition."""
import math

import pytest

from test_gpu_dense import _check_draw, _rng

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("V", [300, 5000, 70000])
@pytest.mark.parametrize("k", [None, 2000])
def test_min_p_of_one_and_temperatures_that_level_all(gpu, V, k):
    """At T = inf, or so large that exp((x - max) / T) rounds to 1, every weight reaches a min-p of 1: the nucleus alone
    bounds the draw. At T = 1 only the largest logits reach it."""
    x = torch.randn((8, V), generator=_rng(V)) * 3
    x[4, ::3] = -math.inf
    x[5, 7::11] = x[5].max()
    kw = dict(temperature=[math.inf, 1e30, 1e30, 3e38, math.inf, 1.0, 1e30, math.inf],
              top_p=[0.9, 0.47, 0.99, 0.001, 0.8, 0.9, 0.9, 0.3], min_p=[1.0] * 6 + [1 - 2.0 ** -24] * 2)
    if k:
        kw["top_k"] = [k] * 8
    for u in (0.0, 0.3, 0.77, 0.99999):
        print("levelled", V, k, u, flush=True)
        _check_draw(x, [u] * 8, **kw)
        _check_draw(x, [u] * 8, **dict(kw, top_p=[1.0] * 8))
