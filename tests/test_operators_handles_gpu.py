"""The operators' torch handles: what they refuse to record, and what becomes of them when their tensors change."""
import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import BF16, F32, gen, randn

pytestmark = pytest.mark.gpu


def calls():
    g = gen(1)
    w, x = randn(g, 24, 16).to(BF16), randn(g, 3, 16).to(BF16)
    lin, router = ops.Linear(w), ops.Router(24, 4)
    targets = torch.zeros(3, dtype=torch.int64, device="cuda")
    return {"linear": (lin, x), "residual": (lambda r: lin(x, residual=r), lin(x)), "route": (lambda t: router(t)[1], lin(x)),
            "logprobs": (lambda t: ops.token_logprobs(t, targets)[0], lin(x))}


@pytest.mark.parametrize("name", ["linear", "residual", "route", "logprobs"])
def test_forward_mode_tangents_are_refused(lib, name):
    import torch.autograd.forward_ad as fw
    f, t = calls()[name]
    f(t)
    with fw.dual_level():
        f(t)  # no tangent, nothing to lose
        with pytest.raises(ValueError, match="tangent"):
            f(fw.make_dual(t, torch.ones_like(t)))
    with pytest.raises(Exception):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("name", ["linear", "residual", "route", "logprobs"])
def test_tracing_is_refused(lib, name):
    f, t = calls()[name]
    with pytest.raises(ValueError, match="trace"):
        torch.jit.trace(lambda v: f(v) * 1, t, check_trace=False)
