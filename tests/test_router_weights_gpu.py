"""Router weights at the ends of their range."""
import numpy as np
import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import F32, gen, randn, route_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("level", [-86.0, -87.0, -88.0, -88.5, -60.0, 0.0, 40.0, 88.0])
def test_sigmoid_weights_of_every_size(lib, level, norm, bias):
    g = gen(1)
    logits = level + 0.2 * randn(g, 20, 64)
    kw = dict(scoring="sigmoid")
    if bias:
        kw["bias"] = randn(g, 64)
    ids, w = ops.Router(64, 6, norm_topk=norm, routed_scale=2.0, **kw)(logits)
    ref_ids, ref_w = route_oracle(logits, 6, norm=norm, scale=2.0, **kw)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    # an exponential (two half steps, its argument is exact), a sum, three quotients and products: 20 half steps of a normal number
    # are generous. Below 2^-126 steps are 2^-149; a weight takes three of them through its quotient and its product with 2.
    small = 6 * 2.0 ** -149 / (1e-20 if norm else 1.0)
    np.testing.assert_allclose(w.cpu().numpy(), ref_w, rtol=20 * 2.0 ** -24, atol=small if level < -80 else 0.0)
