"""The combination of rows without some of their experts (pos -1)."""
import numpy as np
import pytest
import torch

from promoe_b200 import _lib
from tests.helpers import dev, ptr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_shared", [0, 1])
@pytest.mark.parametrize("weight", [0.0, 0.25, -3.0, float("inf"), float("nan")])
def test_the_weight_of_a_missing_expert_does_not_count(lib, weight, n_shared):
    """At every place among the k, and at all of them; a NaN makes the row NaN and no other."""
    rng = np.random.default_rng(7)
    k, H = 4, 72
    places = [[j] for j in range(k)] + [[0, 2], list(range(k)), []]
    T = len(places)
    yexp = rng.standard_normal((T * k + n_shared * T, H)).astype(np.float32)
    pos = rng.permutation(T * k).astype(np.int32).reshape(T, k)
    w = rng.random((T, k)).astype(np.float32)
    for t, holes in enumerate(places):
        pos[t, holes] = -1
        w[t, holes] = weight
    ref = np.zeros((T, H))
    for t in range(T):
        for j in range(k):
            if pos[t, j] >= 0:
                ref[t] += w[t, j].astype(np.float64) * yexp[pos[t, j]]
        for s in range(n_shared):
            ref[t] += yexp[T * k + s * T + t]
        if np.isnan(weight) and places[t]:
            ref[t] = np.nan
    y = torch.full((T, H), 7.0, dtype=torch.bfloat16, device="cuda")
    yd, pd, wd = dev(yexp), dev(pos), dev(w)
    _lib.call("pm_k_combine", ptr(yd), ptr(pd), ptr(wd), T, H, k, T * k, n_shared, None, ptr(y), None)
    torch.cuda.synchronize()
    # five products and sums in float32 (half a step each of at most 5 terms up to 4) and one rounding to bf16
    np.testing.assert_allclose(y.float().cpu().numpy(), ref, rtol=2.0 ** -8, atol=10 * 20 * 2.0 ** -24)
