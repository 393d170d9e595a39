"""Routers that count the choices of dropped groups as 0 (dropped="zero"): the operator against a 64-bit form, the layer against the
installed class."""
import copy
import math

import numpy as np
import pytest
import torch

from promoe_b200 import _lib, ops
from tests.test_operators_gpu import BF16, F16, F32, INF, gen, randn

pytestmark = pytest.mark.gpu


def oracle(logits, k, scoring, bias, n_group, topk_group, group_score, norm, scale):
    """Row by row in Python floats: experts whose logit or choice is -inf (or NaN by the bias) cannot be chosen at all."""
    T, E = logits.shape
    per = E // n_group
    l64, b = logits.double().cpu().numpy(), bias.double().cpu().numpy()
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t, row in enumerate(l64):
        if np.isnan(row).any() or (scoring == "softmax" and np.isposinf(row).any()):
            w[t] = np.nan
            continue
        live = [e for e in range(E) if row[e] != -INF]
        if scoring == "softmax":
            top = max((row[e] for e in live), default=0.0)
            z = math.fsum(math.exp(row[e] - top) for e in live)
            s = {e: math.exp(row[e] - top) / z for e in live}
        else:
            s = {e: 1.0 / (1.0 + math.exp(-row[e])) if row[e] > -700 else 0.0 for e in live}
        c = {e: s[e] + b[e] for e in live if s[e] + b[e] > -INF}
        groups = {}
        for e in c:
            groups.setdefault(e // per, []).append(c[e])
        worth = {g: sum(sorted(v, reverse=True)[:2 if group_score == "top2" else 1]) for g, v in groups.items()}
        kept = sorted(worth, key=lambda g: (-worth[g], g))[:topk_group]
        c = {e: v if e // per in kept else 0.0 for e, v in c.items()}
        best = sorted(c, key=lambda e: (-c[e], e))[:k]
        z = sum(s[e] for e in best) + 1e-20 if norm else 1.0
        for j, e in enumerate(best):
            ids[t, j], w[t, j] = e, s[e] / z * scale
    return ids, w


def check(logits, k, norm=False, scale=1.0, **rule):
    ids, w = ops.Router(logits.shape[1], k, norm_topk=norm, routed_scale=scale, dropped="zero", **rule)(logits)
    ref_ids, ref_w = oracle(logits, k, rule.get("scoring", "softmax"), rule["bias"], rule.get("n_group", 1), rule.get("topk_group", 1),
                            rule.get("group_score", "max"), norm, scale)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    # a weight is a quotient of float32 exponentials, whose arguments of at most 90 are off by half a step
    np.testing.assert_allclose(w.cpu().numpy(), ref_w, rtol=1.2e-5, atol=1e-30)


@pytest.mark.parametrize("T,E,k,dtype,G,kept", [(1, 32, 4, F32, 8, 2), (3, 60, 4, F32, 4, 2), (65, 64, 6, BF16, 8, 1), (130, 160, 6, F16, 8, 3),
                                                (33, 256, 8, F32, 8, 4), (17, 256, 32, F32, 32, 8), (9, 512, 10, BF16, 16, 2),
                                                (5, 1024, 32, F32, 4, 1), (7, 36, 9, F32, 3, 1), (4, 64, 6, F32, 4, 4), (2, 64, 6, F32, 1, 1)])
@pytest.mark.parametrize("mean", [0.2, -0.3, -0.6, -0.9, -1.5])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_matches_the_definition(lib, T, E, k, dtype, G, kept, mean, scoring, group_score):
    g = gen(T * 1000 + E)
    logits = (2 * randn(g, T, E) + randn(g, E)).to(dtype)
    check(logits, k, True, 2.5, scoring=scoring, bias=mean + 0.1 * randn(g, E), n_group=G, topk_group=kept, group_score=group_score)


def test_masks_ties_and_rows_without_experts(lib):
    g = gen(1)
    T, E = 12, 64
    logits = randn(g, T, E)
    logits[0] = -INF
    logits[1, 3:] = -INF
    logits[2, :60] = -INF
    logits[3] = torch.finfo(F32).min
    logits[4, 7] = float("nan")
    logits[5] = 0.0
    logits[6, ::2] = -INF
    for bias in (torch.full((E,), -0.5, device="cuda"), -0.5 + 0.3 * randn(g, E), torch.full((E,), -2.0, device="cuda")):
        for scoring in ("softmax", "sigmoid"):
            check(logits, 6, scoring=scoring, bias=bias, n_group=8, topk_group=2, group_score="top2", norm=True)
    bias = -0.5 + 0.3 * randn(g, E)
    bias[5], bias[6], bias[40:48] = -INF, float("nan"), -INF
    check(logits, 6, scoring="sigmoid", bias=bias, n_group=8, topk_group=2, group_score="top2")


@pytest.mark.parametrize("steps", [0.25, 1, 3])
def test_choices_near_zero_are_told_apart_exactly(lib, steps):
    """Scores + bias that lie some float32 steps about 0, beside dropped experts that are 0."""
    g = gen(int(steps * 4))
    T, E, k = 64, 64, 8
    logits = randn(g, T, E)
    logits[1:32] = logits[0] + 1e-7 * randn(g, 31, E)
    s = torch.sigmoid(logits.double())
    bias = ((torch.randperm(E, generator=torch.Generator().manual_seed(3)).cuda().double() - E / 2) * steps * 2.0 ** -24 - s[0]).float()
    check(logits, k, scoring="sigmoid", bias=bias, n_group=8, topk_group=4, group_score="top2")


def test_refusals(lib):
    bias = torch.zeros(64, device="cuda")
    with pytest.raises(_lib.PromoeError):
        ops.Router(64, 6, n_group=8, topk_group=2, dropped="zero")  # without a bias there is no negative choice
    with pytest.raises(ValueError):
        ops.Router(64, 6, bias=bias, n_group=8, topk_group=2, dropped="one")


@pytest.mark.parametrize("mean", [0.0, -0.3, -0.8])
@pytest.mark.parametrize("T", [5, 60])
def test_injected_block_of_the_installed_class(lib, T, mean):
    from promoe_b200.hf_fused import inject_hf_fused_model
    from transformers.models.deepseek_v3.configuration_deepseek_v3 import DeepseekV3Config
    from transformers.models.deepseek_v3.modeling_deepseek_v3 import DeepseekV3MoE
    torch.manual_seed(2)
    cfg = DeepseekV3Config(hidden_size=128, moe_intermediate_size=64, n_routed_experts=32, num_experts_per_tok=4, n_shared_experts=1,
                           n_group=8, topk_group=2, routed_scaling_factor=2.5, norm_topk_prob=True)

    class Wrapper(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = DeepseekV3MoE(cfg)

    w = Wrapper().to(torch.bfloat16).eval()
    with torch.no_grad():
        for p in w.parameters():
            p.normal_(0, 0.05)
        w.block.gate.weight.normal_(0, 0.2)
        w.block.gate.e_score_correction_bias = mean + 0.1 * torch.randn(32)
    ref = copy.deepcopy(w).cuda()
    cache = inject_hf_fused_model(w, cache_rate=1.0)
    cache.set("keep_routing", 1)
    w.cuda()
    x = torch.randn(1, T, 128, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        got, want = w.block(x).float(), ref.block(x).float()
        ids, _ = ref.block.route_tokens_to_experts(ref.block.gate(x))
    torch.cuda.synchronize()
    mine, _ = cache.last_routing(0, T, 4)
    # both take float32 logits of bf16 rows, summed in another order: choices that lie closer than that may differ, hardly ever
    same = (np.sort(mine, 1) == np.sort(ids.cpu().numpy(), 1)).all(1)
    assert same.mean() >= 0.95
    err = (got - want)[0].norm(dim=1) / want[0].norm(dim=1)
    assert float(err[torch.from_numpy(same).cuda()].max()) < 3e-2
    cache.close()
