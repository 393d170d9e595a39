"""The MoE-block replacement: swaps the forward of an HF 4.x style sparse MoE module for one call
into the fused B200 path (route -> permute -> cache bookkeeping and copies -> grouped SwiGLU
FFN by cache slot -> combine).

The reference ships this piece as a patch to the transformers modelling files (its fork:
install.md:23-27), whose forward computes the routing, calls `self.report_experts(ids)`
(src/sparse_llm_cache/utils/__init__.py:82-89) and loops over the expert modules. Here the
module keeps its structure (`gate`, `experts`, shared expert children, so the name patterns of
utils/common_metas.py still match) and only `forward` changes.
"""
from __future__ import annotations

import torch

from .ops import Router


def _first(module, names):
    for n in names:
        child = getattr(module, n, None)
        if child is not None:
            return child
    return None


def _bf16_dev(t: torch.Tensor, device) -> torch.Tensor:
    return t.detach().to(device=device, dtype=torch.bfloat16).contiguous()


def describe_router(block: torch.nn.Module, config=None) -> dict | None:
    """Arguments of the promoe_b200.ops.Router that the block's routing needs, besides num_expert, top_k, norm_topk and
    routed_scale; None for softmax with greedy top-k. Blocks whose gate carries a correction bias (`e_score_correction_bias`)
    rank scores + bias and value groups by their two best; `topk_method="group_limited_greedy"` values groups by their best.
    Scores are what `scoring_func` of the gate, the block or the configuration says, softmax or sigmoid; without it sigmoid where
    there is a correction bias and softmax elsewhere."""
    gate = block.gate
    cfg = config if config is not None else getattr(block, "config", None)

    def attr(*names):
        for obj in (gate, block, cfg):
            for n in names:
                v = getattr(obj, n, None)
                if v is not None:
                    return v
        return None
    groups = dict(n_group=int(attr("n_group", "num_group") or 1), topk_group=int(attr("topk_group") or 1))
    if groups["n_group"] == 1:
        groups["topk_group"] = 1
    bias = getattr(gate, "e_score_correction_bias", None)
    method = attr("topk_method")
    scoring = attr("scoring_func") or ("softmax" if bias is None else "sigmoid")
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"the router scores by softmax or sigmoid; this block uses {scoring!r}")
    if bias is not None and method in (None, "noaux_tc"):
        return dict(scoring=scoring, bias=bias, group_score="top2", **groups)
    if method == "group_limited_greedy":
        return dict(scoring=scoring, group_score="max", **groups)
    if method is None and groups["n_group"] > groups["topk_group"]:
        raise ValueError("the block has groups of experts, but does not say how they are valued")
    if method in (None, "greedy"):
        return None if scoring == "softmax" else dict(scoring=scoring)
    raise ValueError(f"the router selects greedily, by groups or with a correction bias; this block uses {method!r}")


class _NoExpert(torch.nn.Module):
    """Stands in for what a block computes besides its routed experts."""

    def forward(self, x, *args, **kwargs):
        return torch.zeros_like(x)


class _Expert(torch.nn.Module):
    """Stands in for expert e: a one in column e, so that a block's output shows the expert's weight there."""

    def __init__(self, e: int):
        super().__init__()
        self.e = e

    def forward(self, x, *args, **kwargs):
        y = torch.zeros_like(x)
        y[..., self.e] = 1
        return y


class _Experts(torch.nn.Module):
    """The same for all experts in one module, which is given hidden rows, ids and weights."""

    def __init__(self, num_expert: int):
        super().__init__()
        self.num_expert, self.weights = num_expert, None

    def forward(self, x, *args, **kwargs):
        given = [t for t in (*args, *kwargs.values()) if torch.is_tensor(t) and t.dim() == 2]
        ids = next(t for t in given if not t.is_floating_point())
        w = next(t for t in given if t.is_floating_point() and t.shape == ids.shape)
        self.weights = torch.zeros(ids.shape[0], self.num_expert, dtype=w.dtype).scatter_add_(1, ids.long(), w)
        return torch.zeros_like(x)


def _bare(m: torch.nn.Module, instead: dict) -> torch.nn.Module:
    """A float32 copy of m on the CPU, in eval mode, without hooks and forwards of its instances; instead[id(child)] takes a
    child's place."""
    if id(m) in instead:
        return instead[id(m)]
    b = object.__new__(type(m))
    b.__dict__.update({k: type(v)() if "hooks" in k and isinstance(v, dict) else v for k, v in vars(m).items() if k != "forward"})
    if "report_experts" in vars(b):  # what tells the cache of a block's experts
        b.__dict__["report_experts"] = lambda ids: ids
    plain = lambda t: t.detach().to("cpu", torch.float32 if t.is_floating_point() else t.dtype, copy=True)  # noqa: E731
    b.__dict__["_parameters"] = {n: None if t is None else torch.nn.Parameter(plain(t), requires_grad=False) for n, t in m._parameters.items()}
    b.__dict__["_buffers"] = {n: None if t is None else plain(t) for n, t in m._buffers.items()}
    b.__dict__["_modules"] = {n: None if c is None else _bare(c, instead) for n, c in m._modules.items()}
    b.__dict__["training"] = False
    return b


def _observe(block: torch.nn.Module, gate_w: torch.Tensor):
    """Routes some tokens through a copy of the block with random numbers in its gate: (logits [T, E] float64,
    the weight of every expert [T, E], the copy). None where the block cannot be run like that."""
    E, H = gate_w.shape
    try:
        experts = block.experts
        one_each = isinstance(experts, torch.nn.ModuleList)
        if one_each and E > H:
            return None
        instead = {id(c): _NoExpert() for c in block.children() if c is not block.gate and c is not experts}
        if one_each:
            instead.update({id(c): _Expert(e) for e, c in enumerate(experts)})
        else:
            instead[id(experts)] = _Experts(E)
        probe = _bare(block, instead)
        rng = torch.Generator().manual_seed(0)
        T = 64
        x = torch.randn(1, T, H, generator=rng)
        with torch.no_grad():
            for owner, deep in ((probe.gate, True), (probe, False)):
                for t in (*owner.parameters(deep), *owner.buffers(deep)):
                    if t.is_floating_point():  # corrections leave some choices negative
                        t.copy_(torch.randn(t.shape, generator=rng) * 2 / H ** 0.5 if t.dim() == 2 else
                                -0.3 - 0.7 * torch.rand(t.shape, generator=rng))
            y = probe(x)
        y = y[0] if isinstance(y, tuple) else y
        seen = y.reshape(T, H)[:, :E] if one_each else probe.experts.weights
        return x[0].double() @ probe.gate.weight.double().T, seen.double(), probe
    except Exception:  # noqa: BLE001 - whatever a block of unknown make says to being run here
        return None


def _weights_by_rule(logits: torch.Tensor, d: dict, bias: torch.Tensor | None) -> torch.Tensor:
    """The weight of every expert [T, E] as the layer will choose them, in 64 bits (logits float64)."""
    r = d["router"] or {}
    T, E = logits.shape
    s = torch.sigmoid(logits) if r.get("scoring") == "sigmoid" else torch.softmax(logits, 1)
    c = s if bias is None else s + bias.double()
    G, kept = r.get("n_group", 1), r.get("topk_group", 1)
    if G > kept:
        groups = c.view(T, G, E // G)
        best = groups.topk(2 if r.get("group_score") == "top2" and E // G > 1 else 1, 2).values.sum(2)
        out = torch.ones(T, G, dtype=torch.bool).scatter_(1, best.topk(kept, 1).indices, False)
        c = groups.masked_fill(out[..., None], 0.0 if r.get("dropped") == "zero" else -float("inf")).view(T, E)
    ids = c.topk(d["top_k"], 1).indices
    w = s.gather(1, ids)
    if d["norm_topk"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return torch.zeros_like(s).scatter_(1, ids, w * d["routed_scale"])


def confirm_router(block: torch.nn.Module, d: dict, gate_w: torch.Tensor) -> None:
    """Compares the description with how a copy of the block routes. Blocks that renormalise their weights without an attribute
    that says so, or the other way round, are followed (d["norm_topk"]), and so are those that count the choices of dropped groups as 0
    beside a correction bias (d["router"]["dropped"]); one that routes by another rule is refused (ValueError). Of a block that cannot
    be run like that, a gate that holds more than the description knows is refused."""
    what = f"{type(block).__name__} chooses or weighs its experts in a way that this library does not know"
    seen = _observe(block, gate_w)
    if seen is not None:
        logits, weights, probe = seen
        has_bias = d["router"] is not None and d["router"].get("bias") is not None
        bias = probe.gate.e_score_correction_bias if has_bias else None
        rules = [d["router"]]
        if has_bias and d["router"]["n_group"] > d["router"]["topk_group"]:
            rules.append({**d["router"], "dropped": "zero"})
        for norm, rule in ((n, r) for n in (d["norm_topk"], not d["norm_topk"]) for r in rules):
            want = _weights_by_rule(logits, {**d, "norm_topk": norm, "router": rule}, bias)
            same = ((weights - want).abs() <= 1e-4 * (weights.abs() + want.abs()) + 1e-6).all(1)
            if float(same.double().mean()) >= 0.95:  # a few rows for choices that float32 rounds into another order
                d["norm_topk"], d["router"] = norm, rule
                return
        raise ValueError(what)
    known = {"weight", "e_score_correction_bias"} if d["router"] is not None else {"weight"}
    held = {n for n, _ in (*block.gate.named_parameters(), *block.gate.named_buffers())}
    held |= {n for n, _ in (*block.named_parameters(recurse=False), *block.named_buffers(recurse=False))}
    if held - known:
        raise ValueError(f"{what} ({', '.join(sorted(held - known))})")


def set_router(cache, layer: int, d: dict, num_expert: int, device) -> None:
    """Gives the layer the router that describe_router found, if any."""
    if d["router"] is None:
        return
    kw = dict(d["router"])
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].detach().to(device=device, dtype=torch.float32).contiguous()
    cache.set_router(layer, Router(num_expert, d["top_k"], norm_topk=d["norm_topk"], routed_scale=d["routed_scale"], **kw))


def describe_block(block: torch.nn.Module, config=None) -> dict:
    """Extracts what the fused layer needs from an HF 4.x style MoE block:
    Qwen2-MoE (`gate`, `experts[i].{gate,up,down}_proj`, `shared_expert`, `shared_expert_gate`),
    DeepSeek-MoE / V2 (`gate.weight`, `shared_experts`, routed_scaling_factor; greedy or group-limited),
    Mixtral (`gate`, `experts[i].{w1,w3,w2}`, top-k renormalised)."""
    gate = block.gate
    gate_w = gate.weight
    first = block.experts[0]
    mixtral = hasattr(first, "w1")
    proj = first.w1 if mixtral else first.gate_proj
    # uint4 experts in this library's layout (promoe_b200.quant4.adapt_quantised_linear): packed rows
    quant4 = getattr(proj, "qweight", None) is not None and getattr(proj, "scale_zero", None) is not None
    inter = proj.qweight.shape[0] if quant4 else proj.weight.shape[0]
    router = describe_router(block, config)
    shared = _first(block, ("shared_expert", "shared_experts"))
    shared_gate = getattr(block, "shared_expert_gate", None)
    cfg = config if config is not None else getattr(block, "config", None)
    top_k = (getattr(block, "top_k", None) or getattr(gate, "top_k", None)
             or getattr(cfg, "num_experts_per_tok", None))
    if top_k is None:
        raise ValueError("cannot find the number of experts per token on the block or its config")
    if mixtral:
        norm = True
    else:
        norm = bool(getattr(block, "norm_topk_prob", getattr(gate, "norm_topk_prob", getattr(cfg, "norm_topk_prob", False))))
    scale = float(getattr(block, "routed_scaling_factor", getattr(gate, "routed_scaling_factor", 1.0)) or 1.0)
    d = dict(gate_w=gate_w, inter=inter, top_k=int(top_k), norm_topk=norm, routed_scale=scale,
             shared=shared, shared_gate=shared_gate, quant4=quant4, router=router)
    confirm_router(block, d, gate_w)
    return d


def install_fused_forward(block: torch.nn.Module, cache, layer_id: int, device="cuda", config=None,
                          returns_router_logits: bool = False):
    """Uploads the block's resident weights (router, shared expert) and replaces `block.forward`.
    `cache` is the promoe_b200.engine.ExpertCache that already holds the block's experts."""
    d = describe_block(block, config)
    dev = torch.device(device)
    shared = None
    if d["shared"] is not None:
        s = d["shared"]
        shared = [_bf16_dev(s.gate_proj.weight, dev), _bf16_dev(s.up_proj.weight, dev), _bf16_dev(s.down_proj.weight, dev)]
    sgw = None
    if d["shared_gate"] is not None:
        sgw = _bf16_dev(d["shared_gate"].weight.reshape(-1), dev)
    cache.set_layer_weights(layer_id, _bf16_dev(d["gate_w"], dev), d["inter"], d["top_k"], d["norm_topk"],
                            d["routed_scale"], shared=shared, shared_gate_w=sgw, quant4=d["quant4"])
    set_router(cache, layer_id, d, d["gate_w"].shape[0], dev)
    block._promoe_layer_id = layer_id
    block._promoe_cache = cache
    if not hasattr(block, "_unfused_forward"):
        block._unfused_forward = block.forward

    def fused_forward(hidden_states, *args, **kwargs):
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1])
        if x.dtype != torch.bfloat16:
            x = x.to(torch.bfloat16)
        x = x.contiguous()
        cache.set("seq_len", shape[1] if len(shape) == 3 else 1)
        y = cache.forward(layer_id, x).view(shape).to(hidden_states.dtype)
        return (y, None) if returns_router_logits else y

    block.forward = fused_forward
    return block
