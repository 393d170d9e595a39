"""What install_linears does to modules, without a GPU: the library's product is stood in for by torch's, everything around it
is as installed."""
import copy
import io

import pytest
import torch

from promoe_b200 import hf_fused

BF16 = torch.bfloat16


class StandIn:
    """ops.Linear on the CPU. calls counts the products made by all of them."""
    calls = 0

    def __init__(self, weight, bias=None, activation=None, out_dtype=None):
        self.weight, self.bias, self.act, (self.N, self.K) = weight.detach(), bias, activation, weight.shape

    def __call__(self, x, residual=None, out=None):
        StandIn.calls += 1
        assert x.dim() == 2 and x.stride(1) == 1 and not (torch.is_grad_enabled() and x.requires_grad)
        y = torch.nn.functional.linear(x.detach(), self.weight, self.bias)
        return torch.nn.functional.silu(y) if self.act == "silu" else y


@pytest.fixture
def stand_in(monkeypatch):
    def usable(m):
        return isinstance(m, torch.nn.Linear) and m.weight.dtype is BF16
    monkeypatch.setattr(hf_fused, "_usable", usable)
    monkeypatch.setattr(hf_fused.ops, "Linear", StandIn)
    StandIn.calls = 0
    return StandIn


class Mlp(torch.nn.Module):
    def __init__(self, H=32, I=48):
        super().__init__()
        self.gate_proj, self.up_proj = torch.nn.Linear(H, I, bias=False), torch.nn.Linear(H, I, bias=False)
        self.down_proj, self.act_fn = torch.nn.Linear(I, H, bias=False), torch.nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


def installed(m):
    m = m.to(BF16).eval().requires_grad_(False)
    own = copy.deepcopy(m)
    hf_fused.install_linears(m)
    return m, own


def close(a, b):
    return float((a.float() - b.float()).norm()) <= 0.02 * float(b.float().norm()) + 1e-6  # a few roundings to bf16


@pytest.mark.parametrize("make", [lambda: torch.nn.Linear(32, 48), Mlp])
def test_saved_and_copied_modules(stand_in, make):
    torch.manual_seed(0)
    m, own = installed(make())
    x = torch.randn(2, 3, 32).to(BF16)
    assert close(m(x), own(x)) and stand_in.calls > 0
    file = io.BytesIO()
    torch.save(m, file)
    file.seek(0)
    for other in (torch.load(file, weights_only=False), copy.deepcopy(m)):
        assert close(other(x), own(x))
        for p in other.parameters():
            p.mul_(-1.5)
        own2 = copy.deepcopy(own)
        own2.load_state_dict(other.state_dict())
        before = stand_in.calls
        assert close(other(x), own2(x)) and stand_in.calls > before
        assert close(m(x), own(x))


def test_the_name_of_the_argument_stays(stand_in):
    m, own = installed(torch.nn.Linear(32, 48))
    x = torch.randn(5, 32).to(BF16)
    assert close(m(input=x), own(input=x))
