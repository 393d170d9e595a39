"""What a block's router is taken for, without a GPU."""
import types

import pytest
import torch

from promoe_b200.hf_fused import _describe
from promoe_b200.moe_block import describe_block, describe_router


def block(config=None, bias=None, gate=None, **attrs):
    b = torch.nn.Module()
    b.gate = torch.nn.Module()
    b.gate.weight = torch.nn.Parameter(torch.zeros(16, 8))
    if bias is not None:
        b.gate.register_buffer("e_score_correction_bias", bias)
    for k, v in (gate or {}).items():
        setattr(b.gate, k, v)
    for k, v in attrs.items():
        setattr(b, k, v)
    if config is not None:
        b.config = types.SimpleNamespace(**config)
    return b


@pytest.mark.parametrize("where", ["gate", "block", "config", "given config"])
@pytest.mark.parametrize("method", [None, "greedy", "group_limited_greedy"])
@pytest.mark.parametrize("scoring", [None, "softmax", "sigmoid"])
def test_scores_are_what_the_block_says(where, method, scoring):
    said = {} if scoring is None else {"scoring_func": scoring}
    kw, given = {}, None
    if where == "gate":
        kw["gate"] = said
    elif where == "block":
        kw = dict(said)
    elif where == "config":
        kw["config"] = said
    else:
        given = types.SimpleNamespace(**said)
    if method is not None:
        kw["topk_method"] = method
    if method == "group_limited_greedy":
        kw.update(n_group=4, topk_group=2)
    got = describe_router(block(**kw), given)
    if method == "group_limited_greedy":
        assert got == dict(scoring=scoring or "softmax", group_score="max", n_group=4, topk_group=2)
    elif scoring == "sigmoid":
        assert got == dict(scoring="sigmoid")
    else:
        assert got is None


@pytest.mark.parametrize("where", ["gate", "block", "config", "given config"])
def test_the_method_is_where_the_block_says(where):
    said, kw, given = {"topk_method": "group_limited_greedy"}, dict(n_group=4, topk_group=2), None
    if where == "gate":
        kw["gate"] = said
    elif where == "block":
        kw.update(said)
    elif where == "config":
        kw["config"] = said
    else:
        given = types.SimpleNamespace(**said)
    assert describe_router(block(**kw), given) == dict(scoring="softmax", group_score="max", n_group=4, topk_group=2)


@pytest.mark.parametrize("scoring", [None, "softmax", "sigmoid"])
def test_scores_beside_a_correction_bias(scoring):
    b = torch.randn(16)
    for place in ("gate", "config"):
        said = {} if scoring is None else {"scoring_func": scoring}
        got = describe_router(block(bias=b, n_group=4, topk_group=2, **{place: said}))
        assert torch.equal(got.pop("bias"), b)
        assert got == dict(scoring=scoring or "sigmoid", group_score="top2", n_group=4, topk_group=2)


@pytest.mark.parametrize("attrs", [dict(scoring_func="tanh"), dict(scoring_func="sqrtsoftplus", topk_method="greedy"),
                                   dict(topk_method="random")])
def test_other_rules_are_refused(attrs):
    with pytest.raises(ValueError):
        describe_router(block(**attrs))


# ---- blocks of the installed transformers: routed as the class does, or refused ----------------------------------
def installed(family, block_name, config_name, **config):
    import importlib
    m = importlib.import_module(f"transformers.models.{family}.modeling_{family}")
    c = importlib.import_module(f"transformers.models.{family}.configuration_{family}")
    b = getattr(m, block_name)(getattr(c, config_name)(hidden_size=64, num_attention_heads=4, num_key_value_heads=2, **config))
    with torch.no_grad():
        for p in b.parameters():
            p.normal_(0, 0.1)
    return b


V3 = dict(moe_intermediate_size=32, n_routed_experts=16, num_experts_per_tok=4, n_group=4, topk_group=2, n_shared_experts=1, norm_topk_prob=True)


@pytest.mark.parametrize("case,norm", [
    (("deepseek_v3", "DeepseekV3MoE", "DeepseekV3Config", V3), True),
    (("deepseek_v3", "DeepseekV3MoE", "DeepseekV3Config", V3 | dict(norm_topk_prob=False)), False),
    (("glm4_moe", "Glm4MoeMoE", "Glm4MoeConfig", V3), True),
    (("mixtral", "MixtralSparseMoeBlock", "MixtralConfig", dict(num_local_experts=8, num_experts_per_tok=2)), True),
    (("qwen2_moe", "Qwen2MoeSparseMoeBlock", "Qwen2MoeConfig", dict(num_experts=16, num_experts_per_tok=4, norm_topk_prob=False)), False),
    # no attribute says that these renormalise
    (("qwen3_vl_moe", "Qwen3VLMoeTextSparseMoeBlock", "Qwen3VLMoeTextConfig", dict(num_experts=16, num_experts_per_tok=4)), True),
    (("minimax", "MiniMaxSparseMoeBlock", "MiniMaxConfig", dict(num_local_experts=8, num_experts_per_tok=2)), True)],
    ids=lambda v: v[1] + str(v[3].get("norm_topk_prob", "")) if isinstance(v, tuple) else None)
def test_installed_blocks_are_described_as_they_route(case, norm):
    family, name, config, kw = case
    b = installed(family, name, config, **kw)
    before = {k: v.clone() for k, v in b.state_dict().items()}
    d = _describe(b)
    assert d["norm_topk"] is norm and d["top_k"] == kw["num_experts_per_tok"]
    assert all(torch.equal(v, before[k]) for k, v in b.state_dict().items()) and b.training


@pytest.mark.parametrize("case", [
    ("minimax_m2", "MiniMaxM2SparseMoeBlock", "MiniMaxM2Config", dict(num_local_experts=16, num_experts_per_tok=4)),
    ("ernie4_5_moe", "Ernie4_5_MoeSparseMoeBlock", "Ernie4_5_MoeConfig", dict(moe_num_experts=16, moe_k=4)),
    ("lfm2_moe", "Lfm2MoeSparseMoeBlock", "Lfm2MoeConfig", dict(num_experts=16, num_experts_per_tok=4))], ids=lambda c: c[1])
def test_installed_blocks_that_route_by_other_rules_are_refused(case):
    """Corrections held elsewhere than on the gate, or under another name."""
    family, name, config, kw = case
    with pytest.raises(ValueError, match=name):
        _describe(installed(family, name, config, **kw))


class OneByOne(torch.nn.Module):
    """A block with a module for each expert, as transformers 4.x has them."""

    def __init__(self, score, H=32, E=8, I=16, gate_bias=False):
        super().__init__()
        self.score, self.top_k, self.norm_topk_prob = score, 2, False
        self.gate = torch.nn.Linear(H, E, bias=gate_bias)

        class Expert(torch.nn.Module):
            def __init__(self):
                super().__init__()
                self.gate_proj, self.up_proj, self.down_proj = (torch.nn.Linear(*s, bias=False) for s in ((H, I), (H, I), (I, H)))

            def forward(self, x):
                return self.down_proj(torch.nn.functional.silu(self.gate_proj(x)) * self.up_proj(x))
        self.experts = torch.nn.ModuleList(Expert() for _ in range(E))
        self.shared_expert = Expert()

    def forward(self, hidden_states):
        x = hidden_states.reshape(-1, hidden_states.shape[-1])
        logits = self.gate(x)
        w, ids = self.score(logits).topk(self.top_k, -1)
        y = self.shared_expert(x)
        for e, expert in enumerate(self.experts):
            tok, slot = torch.where(ids == e)
            y = y.index_add(0, tok, expert(x[tok]) * w[tok, slot, None])
        return y.view(hidden_states.shape), logits


def softmax(l):
    return torch.softmax(l, -1)


def test_blocks_with_a_module_for_each_expert():
    assert describe_block(OneByOne(softmax))["norm_topk"] is False
    for other in (OneByOne(torch.sigmoid), OneByOne(softmax, gate_bias=True), OneByOne(lambda l: torch.softmax(l, -1).square())):
        with pytest.raises(ValueError, match="OneByOne"):
            describe_block(other)


def test_blocks_that_cannot_be_run_alone():
    class Needs(OneByOne):
        def forward(self, hidden_states, more):
            raise AssertionError
    assert describe_block(Needs(softmax))["router"] is None
    with pytest.raises(ValueError, match="bias"):
        describe_block(Needs(softmax, gate_bias=True))


def test_describing_a_block_runs_none_of_its_hooks():
    b = OneByOne(softmax)

    def never(*args):
        raise AssertionError
    for m in (b, b.gate, b.experts[0]):
        m.register_forward_hook(never)
        m.register_forward_pre_hook(never)
    b.gate.forward = never
    assert describe_block(b)["router"] is None
    with pytest.raises(ValueError):
        describe_block(OneByOne(torch.sigmoid))


@pytest.mark.parametrize("fill", [0.0, -float("inf")])
@pytest.mark.parametrize("bias", [0.3, -0.9])
def test_dropped_groups_are_treated_as_the_block_does(fill, bias):
    """Whatever its present correction is: with a positive one there is no difference."""
    b = installed("deepseek_v3", "DeepseekV3MoE", "DeepseekV3Config", **V3)
    b.gate.e_score_correction_bias.fill_(bias)
    if fill != 0.0:  # the installed class fills with 0
        class Out(type(b)):
            def route_tokens_to_experts(self, logits):
                s = logits.sigmoid()
                c = s + self.gate.e_score_correction_bias
                best = c.view(-1, self.n_group, 4).topk(2, -1)[0].sum(-1).topk(self.topk_group, -1)[1]
                keep = torch.zeros(len(c), self.n_group).scatter_(1, best, 1.0).repeat_interleave(4, 1).bool()
                ids = c.masked_fill(~keep, fill).topk(self.top_k, -1)[1]
                w = s.gather(1, ids)
                return ids, w / (w.sum(-1, keepdim=True) + 1e-20) * self.routed_scaling_factor
        b.__class__ = Out
    assert _describe(b)["router"].get("dropped", "out") == ("zero" if fill == 0.0 else "out")


def test_dropped_groups_as_zero_need_a_correction_bias(lib):
    from promoe_b200 import _lib
    from tests.test_operators_refusals import PTR, route
    for value in (16, 17):
        with pytest.raises(_lib.PromoeError):
            route(group_score=value, n_group=4, topk_group=2)
        route(group_score=value, n_group=4, topk_group=2, choice_bias=PTR)
    for value in (18, 32, 48, -16):
        with pytest.raises(_lib.PromoeError):
            route(group_score=value, n_group=4, topk_group=2, choice_bias=PTR)


@pytest.mark.parametrize("kw", [dict(num_expert=2 ** 32 + 64), dict(top_k=2 ** 32 + 6), dict(n_group=2 ** 32 + 1), dict(n_group=8, topk_group=2 ** 32 + 2),
                                dict(n_group=8, topk_group=2 - 2 ** 32)])
def test_numbers_beyond_32_bits_are_refused(lib, kw):
    from promoe_b200 import ops
    with pytest.raises(ValueError):
        ops.Router(**(dict(num_expert=64, top_k=6) | kw))


def test_a_layer_refuses_a_router_of_another_device(lib):
    import types
    from promoe_b200.engine import ExpertCache
    cache = ExpertCache(1, 16, num_expert_per_token=4)
    cache._device = 0  # as its weights would leave it
    with pytest.raises(ValueError, match="cuda:1"):
        cache.set_router(0, types.SimpleNamespace(device_index=1, rule=None, bias=None))
    cache.close()
