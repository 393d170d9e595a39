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
        self.like, self.act = (weight.shape, weight.stride(), None if bias is None else bias.shape), activation

    def _without_memory(self):
        return self

    def _dense(self, x, M, weight, bias):
        StandIn.calls += 1
        assert self.like == (weight.shape, weight.stride(), None if bias is None else bias.shape)
        assert x.is_contiguous() and x.numel() == M * weight.shape[1] and not (torch.is_grad_enabled() and x.requires_grad)
        y = torch.nn.functional.linear(x.detach(), weight.detach(), bias)
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


class Adapter(torch.nn.Module):
    """A low-rank addition around a layer, which shows the layer's weight as its own."""

    def __init__(self, base, rank=4):
        super().__init__()
        self.base = base
        self.a = torch.nn.Parameter(torch.randn(rank, base.in_features).to(BF16) * 0.3)
        self.b = torch.nn.Parameter(torch.randn(base.out_features, rank).to(BF16) * 0.3)
        self.requires_grad_(False)

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + x @ self.a.T @ self.b.T


@pytest.mark.parametrize("part", ["gate_proj", "up_proj", "down_proj"])
def test_adapters_around_the_parts_of_a_gated_mlp(stand_in, part):
    torch.manual_seed(1)
    m, own = installed(Mlp())
    x = torch.randn(2, 3, 32).to(BF16)
    plain = m(x)
    adapter = Adapter(getattr(m, part))
    theirs = copy.deepcopy(adapter)
    theirs.base = getattr(own, part)
    setattr(m, part, adapter)
    setattr(own, part, theirs)
    assert close(m(x), own(x)) and not close(m(x), plain)


@pytest.mark.parametrize("part", ["gate_proj", "up_proj", "down_proj", "act_fn"])
@pytest.mark.parametrize("kind", ["after", "before", "with kwargs"])
def test_hooks_on_the_parts_run_and_see_what_they_always_saw(stand_in, part, kind):
    torch.manual_seed(2)
    m, own = installed(Mlp())
    x = torch.randn(2, 3, 32).to(BF16)
    m(x)

    def hook_into(model):
        seen = []

        def after(mod, args, out):
            seen.append((args[0].shape, out.shape))
            return out * 2

        def before(mod, args):
            seen.append(args[0].shape)
            return (args[0] + 1,)
        child = getattr(model, part)
        if kind == "after":
            child.register_forward_hook(after)
        elif kind == "before":
            child.register_forward_pre_hook(before)
        else:
            child.register_forward_pre_hook(lambda mod, args, kwargs: (seen.append(args[0].shape), (args, kwargs))[1], with_kwargs=True)
        return seen
    mine, theirs = hook_into(m), hook_into(own)
    assert close(m(x), own(x)) and mine == theirs and len(mine) == 1


def test_hooks_on_every_module(stand_in):
    m, own = installed(Mlp())
    x = torch.randn(3, 32).to(BF16)
    seen = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(type(mod).__name__))
    try:
        m(x)
        mine, seen[:] = list(seen), []
        own(x)
    finally:
        handle.remove()
    assert mine == seen and len(mine) == 5


def test_parts_exchanged_afterwards(stand_in):
    torch.manual_seed(3)
    m, own = installed(Mlp())
    x = torch.randn(3, 32).to(BF16)
    for model in (m, own):
        model.act_fn = torch.nn.GELU()
    assert close(m(x), own(x))
    for model in (m, own):
        model.act_fn = torch.nn.SiLU()
        model.gate_proj.forward = lambda v, g=model.gate_proj: torch.nn.functional.linear(v, g.weight) * 3
    assert close(m(x), own(x))
    m, own = installed(Mlp())
    wide = torch.nn.Linear(32, 48, bias=False).to(BF16).requires_grad_(False)
    m.up_proj, own.up_proj = wide.float(), wide.float()
    for model in (m, own):
        model.up_proj.register_forward_pre_hook(lambda mod, args: (args[0].float(),))
        model.down_proj.register_forward_pre_hook(lambda mod, args: (args[0].to(BF16),))
    assert close(m(x), own(x))


def test_a_gated_mlp_takes_three_products(stand_in):
    m, own = installed(Mlp())
    x = torch.randn(2, 3, 32).to(BF16)
    stand_in.calls = 0
    assert close(m(x), own(x)) and stand_in.calls == 3


def gated(forward, **attrs):
    """An Mlp of another class, whose forward is given; whether it is taken for a gated MLP."""
    m = type("Other", (Mlp,), {"forward": forward})()
    for k, v in attrs.items():
        setattr(m, k, v)
    return hf_fused.install_linears(m.to(BF16)) == 4


def test_what_is_taken_for_a_gated_mlp(stand_in):
    torch.manual_seed(4)
    assert gated(lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)))
    assert gated(lambda self, x: self.down_proj(self.up_proj(x) * self.act_fn(self.gate_proj(x))))
    assert gated(lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x) * self.s) * self.up_proj(x)), s=1.0)

    def by_steps(self, hidden):
        g = self.act_fn(self.gate_proj(hidden))
        y = self.down_proj(g * self.up_proj(hidden))
        return y
    assert gated(by_steps)
    others = [
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)).clamp(max=50.0) * self.up_proj(x)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x).clamp(-7, 7)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * (self.up_proj(x) + 1e-4)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)) * 1.01, {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x * 1.01)) * self.up_proj(x)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.up_proj(x)) * self.gate_proj(x)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * self.gate_proj(x)), {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)) if x.shape[0] < 100 else x, {}),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x) * self.s) * self.up_proj(x)), dict(s=1.01)),
        (lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x) * self.s[0]) * self.up_proj(x)), dict(s=[1.0])),
        (lambda self, x: (self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)),), {}),
        (lambda self, x, more=None: self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x)), {}),
        (lambda self, x: self.down_proj(torch.nn.functional.silu(self.gate_proj(x)) * self.up_proj(x)), {}),
    ]
    for i, (forward, attrs) in enumerate(others):
        assert not gated(forward, **attrs), i


def test_installed_classes_are_recognised(stand_in):
    from transformers.models.deepseek_v3.configuration_deepseek_v3 import DeepseekV3Config
    from transformers.models.deepseek_v3.modeling_deepseek_v3 import DeepseekV3MLP
    from transformers.models.qwen2_moe.configuration_qwen2_moe import Qwen2MoeConfig
    from transformers.models.qwen2_moe.modeling_qwen2_moe import Qwen2MoeMLP
    for m in (DeepseekV3MLP(DeepseekV3Config(hidden_size=32, intermediate_size=48)),
              Qwen2MoeMLP(Qwen2MoeConfig(hidden_size=32, intermediate_size=48), 48)):
        m = m.to(BF16).eval().requires_grad_(False)
        own = copy.deepcopy(m)
        assert hf_fused.install_linears(m) == 4
        x = torch.randn(2, 3, 32).to(BF16)
        assert close(m(x), own(x))


def test_a_number_or_a_forward_that_changes_afterwards(stand_in):
    class Scaled(Mlp):
        def __init__(self):
            super().__init__()
            self.scale = 1.0

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x) * self.scale) * self.up_proj(x))
    torch.manual_seed(5)
    m, own = installed(Scaled())
    x = torch.randn(3, 32).to(BF16)
    assert close(m(x), own(x))
    first = m(x)
    stand_in.calls = 0
    assert torch.equal(copy.deepcopy(m)(x), first) and stand_in.calls == 3
    m.scale = own.scale = 3.0
    assert close(m(x), own(x)) and not close(m(x), first)
    m.scale = own.scale = 1.0
    Scaled.forward = lambda self, x: self.down_proj(self.act_fn(self.gate_proj(x)) + self.up_proj(x))
    assert close(m(x), own(x)) and not close(m(x), first)


def test_installation_changes_no_mode_and_no_generator(stand_in):
    torch.manual_seed(6)
    m = Mlp().to(BF16)
    m.act_fn.eval()
    state = torch.get_rng_state()
    stand_in.calls = 0
    assert hf_fused.install_linears(m) == 4 and stand_in.calls == 0
    assert m.training and m.gate_proj.training and not m.act_fn.training and torch.equal(state, torch.get_rng_state())


# ---- calls that torch's own machinery has to see ------------------------------------------------------------------
@pytest.fixture(params=[lambda: torch.nn.Linear(32, 32), lambda: Mlp(32, 48)], ids=["linear", "mlp"])
def pair(request, stand_in):
    torch.manual_seed(7)
    m, own = installed(request.param())
    x = torch.randn(3, 32).to(BF16)
    assert close(m(x), own(x)) and stand_in.calls > 0
    return m, own, x


def test_forward_mode_differentiation(pair):
    import torch.autograd.forward_ad as fw
    m, own, x = pair
    t = torch.randn(3, 32).to(BF16)
    with fw.dual_level():
        got, want = (fw.unpack_dual(f(fw.make_dual(x, t))) for f in (m, own))
        assert got.tangent is not None and close(got.tangent, want.tangent) and close(got.primal, want.primal)
        with torch.no_grad():
            assert close(fw.unpack_dual(m(x)).primal, own(x))
    for a, b in zip(torch.func.jvp(m, (x,), (t,)), torch.func.jvp(own, (x,), (t,))):
        assert close(a, b)


def test_transforms(pair):
    m, own, x = pair
    many = torch.randn(4, 3, 32).to(BF16)
    assert close(torch.func.vmap(m)(many), torch.func.vmap(own)(many))
    stacked = {k: torch.stack([v, 2 * v]) for k, v in own.state_dict().items()}
    got, want = (torch.func.vmap(lambda p, f=f: torch.func.functional_call(f, p, (x,)))(stacked) for f in (m, own))
    assert close(got, want)
    grad = [torch.func.grad(lambda v, f=f: f(v).float().square().sum())(x) for f in (m, own)]
    assert close(*grad)


def test_tracers_and_compilers(pair, stand_in):
    from torch.fx.experimental.proxy_tensor import make_fx
    m, own, x = pair
    other = torch.randn(3, 32).to(BF16)
    for recorded in (torch.jit.trace(m, x, check_trace=False), make_fx(m)(x), torch.compile(m, backend="eager", fullgraph=True)):
        recorded(x)
        stand_in.calls = 0
        assert close(recorded(other), own(other)) and stand_in.calls == 0


def test_modes_that_count_operations(pair, stand_in):
    from torch.utils.flop_counter import FlopCounterMode
    m, own, x = pair
    counts, stand_in.calls = [], 0
    for f in (m, own):
        with FlopCounterMode(display=False) as c:
            f(x)
        counts.append(c.get_total_flops())
    assert counts[0] == counts[1] > 0 and stand_in.calls == 0


class Marked(torch.Tensor):
    """A tensor of another class, which says what it was in."""
    seen = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        Marked.seen.append(getattr(func, "__name__", str(func)))
        return super().__torch_function__(func, types, args, kwargs or {})


def test_tensors_of_other_classes(pair):
    m, own, x = pair
    Marked.seen.clear()
    y = m(x.as_subclass(Marked))
    assert type(y) is Marked and "linear" in Marked.seen and close(y.as_subclass(torch.Tensor), own(x))
    layer = m if isinstance(m, torch.nn.Linear) else m.up_proj
    layer.weight = torch.nn.Parameter(layer.weight.detach().as_subclass(Marked), requires_grad=False)
    Marked.seen.clear()
    assert close(m(x).as_subclass(torch.Tensor), own(x)) and "linear" in Marked.seen


def test_autocast(pair, stand_in):
    m, own, x = pair
    stand_in.calls = 0
    with torch.autocast("cpu", dtype=torch.float16):
        assert m(x).dtype == own(x).dtype == torch.float16 and close(m(x), own(x))
    assert stand_in.calls == 0
    with torch.autocast("cpu", dtype=BF16):
        assert m(x.float()).dtype == own(x.float()).dtype == BF16 and close(m(x), own(x))


def test_inputs_that_do_not_fit_fail_as_ever(pair):
    m, own, x = pair
    for bad in (x[:, :-1], x.float(), torch.tensor(1.0, dtype=BF16)):
        for f in (m, own):
            with pytest.raises(RuntimeError):
                f(bad)


# ---- which calls take the product ------------------------------------------------------------------------------------
@pytest.mark.parametrize("K,N", [(32, 48), (32, 9472), (32, 9480), (32, 9473), (32, 50), (36, 48), (36, 50), (33, 50), (1, 8), (1, 1)])
def test_calls_that_torch_is_faster_for_keep_it(stand_in, K, N):
    m, own = installed(torch.nn.Linear(K, N))
    aligned, odd = K % 8 == 0, N % 8 != 0
    m(torch.zeros(1, K, dtype=BF16))
    for M in (1, 8, 16, 17, 64, 600):
        for x in (torch.randn(M, K).to(BF16), torch.randn(1, M, K).to(BF16)):
            stand_in.calls = 0
            assert close(m(x), own(x))
            assert stand_in.calls == ((odd or N <= 9472) if M <= 16 else (odd and aligned)), M


def test_weights_exchanged_for_others_of_another_size(stand_in):
    m, own = installed(torch.nn.Linear(32, 48))
    x = torch.randn(16, 32).to(BF16)
    m(x)
    for shape in ((24, 64), (24, 16), (9480, 8), (9472, 8), (5, 64)):
        for model in (m, own):
            model.weight, model.bias = (torch.nn.Parameter(t, requires_grad=False) for t in (torch.ones(shape).to(BF16), torch.ones(shape[0]).to(BF16)))
        for M in (1, 16, 40):
            x = torch.randn(M, shape[1]).to(BF16)
            assert close(m(x), own(x))
    m.weight.data = m.weight.data[:4]  # the same memory, fewer rows
    m.bias.data = m.bias.data[:4]
    assert m(x).shape == (40, 4) and m(x[:2]).shape == (2, 4)


def test_inputs_with_strides(stand_in):
    m, own = installed(torch.nn.Linear(32, 50))
    for x in (torch.randn(32, 9).to(BF16).t(), torch.randn(4, 64).to(BF16)[:, 1:33], torch.randn(1, 32).to(BF16).expand(7, 32),
              torch.randn(2, 3, 40).to(BF16)[..., 8:], torch.randn(700, 32).to(BF16)[::2], torch.randn(0, 32).to(BF16), torch.randn(32).to(BF16)):
        y = m(x)
        assert y.shape == own(x).shape and close(y, own(x))


def test_a_call_while_another_one_makes_the_product(stand_in, monkeypatch):
    """As a second thread would come in between."""
    m, own = installed(torch.nn.Linear(32, 48))
    x, begun, inside = torch.randn(3, 32).to(BF16), [], []

    class Slow(StandIn):
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            begun.append(self)
            if len(begun) == 1:
                inside.append(m(x))
    monkeypatch.setattr(hf_fused.ops, "Linear", Slow)
    assert close(m(x), own(x)) and close(inside[0], own(x))
    m.weight, own.weight = (torch.nn.Parameter(2 * own.weight.detach(), requires_grad=False) for _ in range(2))
    begun.clear()
    assert close(m(x), own(x)) and close(inside[1], own(x))


def test_a_bias_cut_short_in_place(stand_in):
    """The same address, fewer values: there is nothing to read behind them."""
    m, own = installed(torch.nn.Linear(32, 48))
    x = torch.randn(3, 32).to(BF16)
    m(x)
    for model in (m, own):
        model.bias.data = model.bias.data[:40]
        with pytest.raises(RuntimeError):
            model(x)


def test_an_up_projection_of_another_tensor_class(stand_in):
    torch.manual_seed(8)
    m, own = installed(Mlp())
    x = torch.randn(3, 32).to(BF16)
    m(x)
    for model in (m, own):
        model.up_proj.register_forward_hook(lambda mod, args, out: out.as_subclass(Marked))
    assert type(m(x)) is type(own(x)) is Marked and close(m(x).as_subclass(torch.Tensor), own(x).as_subclass(torch.Tensor))
