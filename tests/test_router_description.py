"""What a block's router is taken for, without a GPU."""
import types

import pytest
import torch

from promoe_b200.moe_block import describe_router


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
