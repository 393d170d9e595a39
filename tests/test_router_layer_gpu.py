"""Layers whose router has a rule of its own (sigmoid scores, a correction bias, groups): the layer call, the expert-parallel
form, blocks of transformers models; and what an injected model offers beside its experts (install_linears, score_tokens)."""
import copy

import numpy as np
import pytest
import torch

from oracle import moe_math as om
from promoe_b200 import ops
from tests.helpers import TinyModel, dev, dev_bf16
from tests.test_operators_gpu import route_oracle

pytestmark = pytest.mark.gpu

RULES = {
    "sigmoid_bias_groups": dict(scoring="sigmoid", bias=True, n_group=4, topk_group=2, group_score="top2", norm=True, scale=2.5),
    "softmax_groups": dict(n_group=4, topk_group=2, scale=16.0),
    "sigmoid": dict(scoring="sigmoid", norm=True),
    "softmax_bias": dict(bias=True),
}


def make(rule, seed=3, E=24, k=4, shared=True, **kw):
    model = TinyModel(seed=seed, L=1, E=E, H=256, I=64, k=k, shared_I=128 if shared else 0, shared_gate=shared, gate_std=0.1, **kw)
    cache = model.make_cache(cache_rate=1.0)
    cache.set("keep_routing", 1)
    rule = dict(rule)
    rng = np.random.default_rng(seed)
    if rule.get("bias") is True:
        rule["bias"] = dev((0.1 * rng.standard_normal(E)).astype(np.float32))
    return model, cache, rule


def set_router(cache, model, rule):
    r = dict(rule)
    norm, scale = r.pop("norm", False), r.pop("scale", 1.0)
    cache.set_router(0, ops.Router(model.E, model.k, norm_topk=norm, routed_scale=scale, **r))


def expected(model, rule, x):
    """The layer in 64 bits, from the ids that the definition gives for the layer's own logits."""
    lg = om.gate_logits_canonical(x, model.gate_w[0], None if model.gate_bias is None else model.gate_bias[0])
    ids, w = route_oracle(torch.from_numpy(lg), model.k, **rule)
    y = np.zeros((x.shape[0], model.H))
    for e in range(model.E):
        tok, slot = np.nonzero(ids == e)
        if tok.size:
            y[tok] += w[tok, slot][:, None] * om.swiglu_mlp(x[tok], *model.experts[0][e], True)
    y[np.isnan(w).any(1)] = np.nan
    if model.shared is not None:
        s = om.swiglu_mlp(x, *model.shared[0], True)
        y = y + s * (1 / (1 + np.exp(-(x.astype(np.float64) @ model.shared_gate_w[0].astype(np.float64)))))[:, None]
    return ids, w, y


def check_layer(model, cache, rule, x):
    y = cache.forward(0, dev_bf16(x))
    torch.cuda.synchronize()
    ids, w = cache.last_routing(0, x.shape[0], model.k)
    ref_ids, ref_w, ref = expected(model, rule, x)
    assert np.array_equal(ids, ref_ids)
    np.testing.assert_allclose(w, ref_w, rtol=1.2e-5)
    got = y.float().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = ~np.isnan(ref)
    # bf16 intermediate rows and results, as for every layer call: half steps of 2^-8 each, relative to the row
    np.testing.assert_allclose(got[ok], ref[ok], rtol=2e-2, atol=5e-3 * np.abs(ref[ok]).max())


@pytest.mark.parametrize("T", [1, 3, 16, 17, 40, 297, 1801])
@pytest.mark.parametrize("name", list(RULES))
def test_layer_call(lib, T, name):
    model, cache, rule = make(RULES[name])
    set_router(cache, model, rule)
    x = model.hidden_stream(T, 1)[0]
    check_layer(model, cache, rule, x)
    check_layer(model, cache, rule, x)  # again, with the experts resident
    cache.close()


@pytest.mark.parametrize("T", [2, 20, 100])
def test_tokens_with_few_experts_none_and_nan(lib, T):
    model, cache, rule = make(dict(scoring="sigmoid", norm=True))
    bias = torch.zeros(model.E, device="cuda")
    bias[3:] = -float("inf")  # three experts can be chosen, k is four
    rule["bias"] = bias
    set_router(cache, model, rule)
    x = model.hidden_stream(T, 1)[0]
    check_layer(model, cache, rule, x)
    bias[:] = -float("inf")  # none
    check_layer(model, cache, rule, x)
    bias[:] = 0.0
    x[1, 5] = np.nan  # this token's logits are NaN, and so is its output; the others' are not
    xd = dev_bf16(x)
    y = cache.forward(0, xd).float()
    ids, w = cache.last_routing(0, T, model.k)
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isnan(y[[i for i in range(T) if i != 1]]).any())
    assert (ids[1] == -1).all() and np.isnan(w[1]).all() and (ids[[i for i in range(T) if i != 1]] >= 0).all()
    x[1, 5] = 0.0
    check_layer(model, cache, rule, x)  # nothing of it is left behind
    cache.close()


@pytest.mark.parametrize("T", [5, 50])
def test_a_router_taken_back_leaves_the_old_results(lib, T):
    model, cache, rule = make(RULES["sigmoid_bias_groups"])
    xd = dev_bf16(model.hidden_stream(T, 1)[0])
    want = cache.forward(0, xd).clone()
    set_router(cache, model, rule)
    assert not torch.equal(cache.forward(0, xd), want)
    cache.set_router(0, None)
    assert torch.equal(cache.forward(0, xd), want)
    cache.close()


def test_router_of_256_experts_and_large_hidden(lib):
    """The scratch of the choice shares shared memory with token rows: more of one than of the other, both ways."""
    for H, E, T in ((64, 256, 16), (64, 250, 9), (2048, 64, 16), (64, 256, 40)):
        model = TinyModel(seed=5, L=1, E=E, H=H, I=32, k=8, gate_std=0.2)
        cache = model.make_cache(cache_rate=1.0)
        cache.set("keep_routing", 1)
        bias = dev((0.1 * np.random.default_rng(1).standard_normal(E)).astype(np.float32))
        rule = dict(scoring="sigmoid", bias=bias, n_group=2, topk_group=1, group_score="top2")
        set_router(cache, model, rule)
        x = model.hidden_stream(T, 1)[0]
        cache.forward(0, dev_bf16(x))
        torch.cuda.synchronize()
        ids, w = cache.last_routing(0, T, 8)
        lg = om.gate_logits_canonical(x, model.gate_w[0], model.gate_bias[0])
        ref_ids, ref_w = route_oracle(torch.from_numpy(lg), 8, **rule)
        assert np.array_equal(ids, ref_ids)
        np.testing.assert_allclose(w, ref_w, rtol=1.2e-5)
        cache.close()


def test_expert_parallel_layer_with_a_router(lib):
    from tests.ep_common import build_rank
    model, _, ep, be, cache = build_rank(0, 1, with_pred=False, tokens=6)
    bias = dev((0.1 * np.random.default_rng(2).standard_normal(model.E)).astype(np.float32))
    bias[::2] = -float("inf")
    rule = dict(scoring="sigmoid", bias=bias, n_group=8, topk_group=3, group_score="top2", norm=True, scale=2.0)  # 3 experts for k = 4
    rule_args = {k: v for k, v in rule.items() if k not in ("norm", "scale")}
    for layer in be.layers:
        rule3 = dict(rule_args)
        layer["router"] = ops.Router(model.E, model.k, norm_topk=True, routed_scale=2.0, **rule3)
    x = model.hidden_stream(6, 1)[0]
    y = ep.forward(0, dev_bf16(x)).float().cpu().numpy()
    _, _, ref = expected(model, rule, x)
    np.testing.assert_allclose(y, ref, rtol=2e-2, atol=5e-3 * np.abs(ref).max())
    cache.close()


def rel_err(a, b):
    a, b = a.float(), b.float()
    return float((a - b).norm() / b.norm())


def test_group_limited_block_of_transformers(lib):
    from transformers.models.deepseek_v2.configuration_deepseek_v2 import DeepseekV2Config
    from transformers.models.deepseek_v2.modeling_deepseek_v2 import DeepseekV2Moe
    from promoe_b200.hf_fused import inject_hf_fused_model
    torch.manual_seed(2)
    cfg = DeepseekV2Config(hidden_size=128, moe_intermediate_size=64, n_routed_experts=16, num_experts_per_tok=3, n_shared_experts=2,
                           routed_scaling_factor=2.0, topk_method="group_limited_greedy", n_group=4, topk_group=2)

    class Wrapper(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = DeepseekV2Moe(cfg)

    w = Wrapper().to(torch.bfloat16).eval()
    with torch.no_grad():
        for p in w.parameters():
            p.normal_(0, 0.05)
        w.block.gate.weight.normal_(0, 0.5)
    ref = copy.deepcopy(w).cuda()
    ref.block.num_experts = 16  # transformers 5.5.0's own group-limited forward reads it without setting it
    cache = inject_hf_fused_model(w, cache_rate=0.5)
    w.cuda()
    for T in (7, 40):
        x = torch.randn(1, T, 128, device="cuda").to(torch.bfloat16)
        with torch.no_grad():
            assert rel_err(w.block(x), ref.block(x)) < 3e-2
    cache.close()


def test_block_with_a_correction_bias(lib):
    """A block as transformers lays them out whose gate holds `e_score_correction_bias`."""
    from promoe_b200.hf_fused import inject_hf_fused_model
    E, H, I, k = 16, 128, 64, 4

    class Gate(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.weight = torch.nn.Parameter(torch.randn(E, H) * 0.3)
            self.register_buffer("e_score_correction_bias", 0.2 * torch.randn(E))

    class Experts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_up_proj = torch.nn.Parameter(torch.randn(E, 2 * I, H) * 0.05)
            self.down_proj = torch.nn.Parameter(torch.randn(E, H, I) * 0.05)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate, self.experts = Gate(), Experts()
            self.n_group, self.topk_group, self.top_k, self.norm_topk_prob, self.routed_scaling_factor = 4, 2, k, True, 2.5

    class Wrapper(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = Block()

    torch.manual_seed(4)
    w = Wrapper()
    for p in w.parameters():
        p.data = p.data.to(torch.bfloat16)
    gate, gu, dn = (p.detach().double() for p in (w.block.gate.weight, w.block.experts.gate_up_proj, w.block.experts.down_proj))
    bias = w.block.gate.e_score_correction_bias.clone()
    cache = inject_hf_fused_model(w, cache_rate=0.5)
    x = torch.randn(1, 9, H).to(torch.bfloat16)
    got = w.block(x.cuda()).double().cpu()[0]
    xd = x[0].double()
    ids, wt = route_oracle(xd @ gate.T, k, "sigmoid", bias, 4, 2, "top2", True, 2.5)
    want = torch.zeros(9, H, dtype=torch.float64)
    for t in range(9):
        for e, p in zip(ids[t], wt[t]):
            h = gu[e] @ xd[t]
            want[t] += p * (dn[e] @ (torch.nn.functional.silu(h[:I]) * h[I:]))
    assert rel_err(got, want) < 1e-2  # three roundings to bf16 (2^-8 each at most) on the way
    cache.close()


def test_install_linears_and_score_tokens_of_an_injected_model(lib):
    from promoe_b200.hf_fused import inject_hf_fused_model, install_linears, score_tokens
    from tests.test_hf_fused_gpu import tiny_qwen
    model = tiny_qwen()
    ref = copy.deepcopy(model).cuda()
    cache = inject_hf_fused_model(model, cache_rate=0.5, num_predict_expert_per_layer=0)
    model.cuda()
    n = install_linears(model)
    assert n >= 9  # four projections of two layers' attention and the vocabulary's
    assert install_linears(model) == 0
    ids = torch.randint(0, 128, (2, 11), device="cuda")
    mask = torch.ones_like(ids)
    mask[1, 8:] = 0
    with torch.no_grad():
        assert rel_err(model(input_ids=ids, attention_mask=mask).logits, ref(input_ids=ids, attention_mask=mask).logits) < 3e-2
        mine = score_tokens(model, ids, mask, top_n=3)
        logits = model(input_ids=ids, attention_mask=mask).logits.double()[:, :-1]
    lp = torch.log_softmax(logits, -1)
    want = torch.gather(lp, 2, ids[:, 1:, None])[..., 0].masked_fill(mask[:, 1:] == 0, 0.0)
    # the model's own logits are rounded to bf16 (half a step of values up to 4), the scored ones are not
    assert float((mine["logp"].double() - want).abs().max()) < 4 * 2.0 ** -8 * 2
    assert float((mine["entropy"].double() + (lp.exp() * lp).sum(-1)).abs().max()) < 4 * 2.0 ** -8 * 4
    assert mine["top_ids"].shape == (2, 10, 3) and bool((mine["top_logp"][..., 0] >= mine["top_logp"][..., 1]).all())
    best = torch.gather(lp, 2, mine["top_ids"].long())
    assert float((best - mine["top_logp"].double()).abs().max()) < 4 * 2.0 ** -8 * 2
    none = score_tokens(model, ids[:, :1], top_n=2)                # a text of one token has nothing to predict
    assert none["logp"].shape == (2, 0) and none["top_ids"].shape == (2, 0, 2)
    model.config.final_logit_softcapping = 30.0
    with pytest.raises(ValueError):
        score_tokens(model, ids)
    cache.close()


def test_install_linears_fuses_a_gated_mlp_and_steps_aside_for_gradients(lib):
    from promoe_b200.hf_fused import install_linears

    class Mlp(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(96, 200, bias=False), torch.nn.Linear(96, 200, bias=False)
            self.down_proj, self.act_fn = torch.nn.Linear(200, 96), torch.nn.SiLU()

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))

    torch.manual_seed(0)
    m = Mlp().to(torch.bfloat16).cuda()
    ref = copy.deepcopy(m).double()
    assert install_linears(m) == 4
    x = torch.randn(3, 5, 96, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        assert rel_err(m(x), ref(x.double())) < 1e-2  # four roundings to bf16
    x.requires_grad_()
    m(x).sum().backward()
    assert x.grad is not None and float(x.grad.float().norm()) > 0


def test_installed_linears_follow_their_modules(lib):
    """Weights that are changed, exchanged or copied, inputs with strides, no rows at all, and parameters that learn."""
    from promoe_b200.hf_fused import install_linears
    torch.manual_seed(1)
    m = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.ReLU(), torch.nn.Linear(96, 40, bias=False)).to(torch.bfloat16).cuda()
    assert install_linears(m) == 2
    x = torch.randn(5, 64, device="cuda").to(torch.bfloat16)

    def same(model, y, rows=None):
        first, last = model[0], model[2]
        h = torch.nn.functional.linear((x if rows is None else rows).double(), first.weight.double(), first.bias.double()).relu()
        assert rel_err(y, torch.nn.functional.linear(h, last.weight.double())) < 1e-2  # two roundings to bf16
    with torch.no_grad():
        same(m, m(x))
        other = copy.deepcopy(m)
        for p in other.parameters():
            p.mul_(-2.0)
        same(other, other(x))                                     # the copy's weights
        same(m, m(x))
        m[0].weight.mul_(3.0)                                     # changed in place
        same(m, m(x))
        m[2].weight = torch.nn.Parameter(torch.randn(40, 96, device="cuda").to(torch.bfloat16))  # exchanged
        m[0].bias.data = torch.randn(96, device="cuda").to(torch.bfloat16)
        same(m, m(x))
        same(m, m(x[:1].expand(7, 64)), x[:1].expand(7, 64))      # rows over one another
        wide = torch.randn(64, 9, device="cuda").to(torch.bfloat16).t()
        same(m, m(wide), wide)                                    # rows that are not dense
        assert m(x[:0]).shape == (0, 40) and m(x[0]).shape == (40,)
    y = m(x)                                                      # the parameters require a gradient, the input does not
    y.sum().backward()
    assert float(m[0].weight.grad.float().norm()) > 0
    m.requires_grad_(False)
    same(m, m(x))
    with pytest.raises(ValueError):
        ops.Linear(torch.nn.Parameter(m[0].weight.data))(x)


def test_mlps_of_another_kind_stay_as_they_are(lib):
    from promoe_b200.hf_fused import install_linears

    class Mlp(torch.nn.Module):
        def __init__(self, scale):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(64, 72, bias=False), torch.nn.Linear(64, 72, bias=False)
            self.down_proj, self.act_fn, self.scale = torch.nn.Linear(72, 64), torch.nn.SiLU(), scale

        def forward(self, x):
            return self.down_proj(self.act_fn(self.gate_proj(x) * self.scale) * self.up_proj(x))

    state = torch.cuda.get_rng_state()
    plain, scaled = (Mlp(s).to(torch.bfloat16).cuda() for s in (1.0, 2.0))
    assert install_linears(plain) == 4 and install_linears(scaled) == 3
    assert torch.equal(state, torch.cuda.get_rng_state()) and plain.training and scaled.act_fn.training
    x = torch.randn(3, 64, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        assert plain.eval()(x[:0]).shape == (0, 64)
        for m in (plain, scaled):
            assert rel_err(m(x), copy.deepcopy(m).double()(x.double())) < 1e-2
