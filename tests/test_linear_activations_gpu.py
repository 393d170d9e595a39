"""The activations of the dense product, value by value: every finite 16-bit number through a product with 1."""
import math

import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import BF16, F16, F32, act64, half_step

pytestmark = pytest.mark.gpu


def exponent(v, act):
    """The largest argument that the activation's exponential takes."""
    return v.square() / 2 if act == "gelu" else (2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)).abs() if act == "gelu_tanh" else v.abs()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("K,rows", [(8, None), (7, None), (8, 16), (7, 5)])  # the tensor cores' kernel, rows off boundaries, few tokens, both
def test_every_value(lib, act, dtype, wide, K, rows):
    v = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v)]
    x, w = torch.zeros((v.numel(), K), dtype=dtype, device="cuda"), torch.zeros((2, K), dtype=dtype, device="cuda")
    x[:, 1], w[:, 1] = v, 1.0
    lin = ops.Linear(w, None, act, F32 if wide else dtype)
    if rows is None:
        y = lin(x)[:, 1]
    else:  # as many values as calls of a few tokens take in reasonable time, those near zero and in the tails among them
        pick = torch.cat([v.double().abs().argsort()[:512], (v.double() + 5).abs().argsort()[:512], torch.arange(0, v.numel(), 97, device="cuda")])
        x, v = x[pick], v[pick]
        y = torch.cat([lin(x[i:i + rows])[:, 0] for i in range(0, len(x), rows)])
    v = v.double()
    ref = act64(v, act)
    z = exponent(v, act).clamp_max(200)
    # Relative errors. 16 bits: the result's rounding, and an exponential that is off by 2 + 1.2 z steps of float32 besides its
    # argument's roundings (3 z half steps). float32: 16 half steps for the polynomial, exponential, division and products, and
    # the argument's roundings where it has any that are not made up for (the cubic's).
    if wide:
        tol = (16 + (4 * z if act == "gelu_tanh" else 0)) * 2.0 ** -24
    else:
        tol = half_step(dtype) + (8 + 4 * z) * 2.0 ** -23
    # below the normal numbers steps are absolute; so they are of exponentials down there
    tiny = torch.finfo(y.dtype).tiny * half_step(y.dtype) * 2.1 + 2.0 ** -126 * (1 + v.abs())
    bad = (y.double() - ref).abs() > tol * ref.abs() + torch.where(z > 80, tiny, torch.finfo(y.dtype).tiny * half_step(y.dtype) * 2.1)
    bad &= ref.abs() <= torch.finfo(y.dtype).max  # beyond: infinite
    assert not bool(bad.any()), [(float(a), float(b), float(c)) for a, b, c in zip(v[bad][:5], y[bad][:5], ref[bad][:5])]


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out", [BF16, F32])
def test_infinities_and_nan(lib, act, out):
    x = torch.zeros((3, 8), dtype=BF16, device="cuda")
    x[:, 0] = torch.tensor([float("inf"), -float("inf"), float("nan")])
    w = torch.zeros((2, 8), dtype=BF16, device="cuda")
    w[:, 0] = 1.0
    for rows in (x, x.repeat(12, 1)):
        y = ops.Linear(w, None, act, out)(rows)[:3, 0]
        assert bool(torch.isposinf(y[0])) and bool(torch.isnan(y[2]))
        assert bool(torch.isnan(y[1]))  # -inf times a sigmoid of 0
