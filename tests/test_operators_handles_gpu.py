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


def test_what_a_handle_was_made_from_is_set_once(lib):
    """A weight or bias put in its place would leave the launch with the old one's address and sizes."""
    g = gen(2)
    lin = ops.Linear(randn(g, 24, 16).to(BF16), randn(g, 24).to(BF16))
    router = ops.Router(24, 4, bias=randn(g, 24))
    for handle, name, value in ((lin, "weight", randn(g, 8, 16).to(BF16)), (lin, "bias", None), (lin, "bias", randn(g, 24).to(BF16)),
                                (lin, "N", 8), (lin, "K", 8), (lin, "out_dtype", F32), (lin, "device_index", 1),
                                (router, "bias", randn(g, 24)), (router, "top_k", 8), (router, "num_expert", 16), (router, "device_index", None)):
        with pytest.raises(AttributeError):
            setattr(handle, name, value)
    assert (lin.N, lin.K, lin.out_dtype, router.num_expert, router.top_k) == (24, 16, BF16, 24, 4)


def test_a_handle_keeps_the_memory_it_reads(lib):
    """The caller's tensors get other memory; what they had before must not be given to anyone else."""
    g = gen(3)
    weight, bias, correction = randn(g, 512, 512).to(BF16), randn(g, 512).to(BF16), 0.5 * randn(g, 512)
    lin, router = ops.Linear(weight, bias), ops.Router(512, 4, scoring="sigmoid", bias=correction)
    x, logits = randn(g, 3, 512).to(BF16), randn(g, 3, 512)
    want, ids = lin(x).clone(), router(logits)[0].clone()
    weight.data, bias.data, correction.data = weight * 2, bias * 2, -correction
    fill = [torch.full((n,), 3.0, dtype=t, device="cuda") for n, t in ((512 * 512, BF16), (512, BF16), (512, F32)) for _ in range(4)]
    assert torch.equal(lin(x), want) and torch.equal(router(logits)[0], ids)
    lin.bias.add_(1.0)  # in place: followed
    assert torch.equal(lin(x), ops.Linear(lin.weight, lin.bias)(x)) and not torch.equal(lin(x), want)
    del fill
