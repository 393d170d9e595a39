"""Attaches the expert cache to a stock HuggingFace transformers 5.x MoE model.

The reference hooks into a transformers 4.x fork whose MoE blocks hold one module per expert
(`...mlp.experts.N`, src/sparse_llm_cache/utils/common_metas.py). Stock transformers 5.x keeps the
experts of a block in two 3-D parameters instead (`experts.gate_up_proj [E, 2I, H]`,
`experts.down_proj [E, H, I]`), so name-pattern injection finds nothing there. This module does the
same job for that layout: every expert's three matrices are sliced out of the fused tensors and
registered with the cache, the fused tensors are released, and the block's forward becomes one call
into the fused device path. Supported blocks: Qwen2-MoE (shared expert with sigmoid gate),
Mixtral (renormalised top-k), DeepSeek-V2 with greedy or group-limited top-k (shared experts, routed scaling), and blocks
whose gate ranks sigmoid scores with a correction bias.

`install_linears` hands the model's other matrix products to the library where it is faster, `score_tokens` says what a text's tokens were
worth to the model.
"""
from __future__ import annotations

import copy
import inspect
import operator
import types
import weakref

import torch
import torch.fx
from torch.autograd import forward_ad

from . import ops
from .engine import ExpertCache
from .moe_block import confirm_router, describe_router, set_router


def find_moe_blocks(model: torch.nn.Module) -> list[tuple[str, torch.nn.Module]]:
    """MoE blocks in forward order: modules that own `experts.gate_up_proj` and a `gate`."""
    out = []
    for name, mod in model.named_modules():
        experts = getattr(mod, "experts", None)
        if experts is not None and hasattr(experts, "gate_up_proj") and hasattr(mod, "gate"):
            out.append((name, mod))
    return out


def _describe(block) -> dict:
    gate = block.gate
    experts = block.experts
    E, two_i, H = experts.gate_up_proj.shape
    top_k = getattr(gate, "top_k", None) or getattr(block, "top_k", None)
    if top_k is None:
        raise ValueError("cannot find top_k on the MoE block")
    kind = type(block).__name__.lower()
    if "mixtral" in kind:
        norm = True
    else:
        norm = bool(getattr(gate, "norm_topk_prob", getattr(block, "norm_topk_prob", False)))
    d = dict(router=describe_router(block), E=E, H=H, I=two_i // 2, top_k=int(top_k), norm_topk=norm,
             routed_scale=float(getattr(block, "routed_scaling_factor", 1.0) or 1.0),
             shared=getattr(block, "shared_expert", None) or getattr(block, "shared_experts", None),
             shared_gate=getattr(block, "shared_expert_gate", None))
    confirm_router(block, d, gate.weight)
    return d


def inject_hf_fused_model(model: torch.nn.Module, cache_rate: float = 0.375, cache_policy: str = "lru",
                          num_predict_expert_per_layer: int = 0, device="cuda", **config) -> ExpertCache:
    """Moves every routed expert of `model` into a pinned host record + cache lines and replaces the
    MoE blocks' forwards. The rest of the model is left where it is (move it to `device` yourself).
    Returns the ExpertCache; it is also stored as `model._promoe_cache`."""
    blocks = find_moe_blocks(model)
    if not blocks:
        raise ValueError("no MoE block with fused expert tensors found")
    descs = [_describe(block) for _, block in blocks]  # what is refused is refused before anything is moved
    d0 = descs[0]
    model_id = getattr(getattr(model, "config", None), "_name_or_path", "") or type(model).__name__
    cache = ExpertCache(len(blocks), d0["E"], num_expert_per_token=d0["top_k"], cache_rate=repr(float(cache_rate)),
                        cache_policy=cache_policy, num_predict_expert_per_layer=num_predict_expert_per_layer,
                        model_arch_string=model_id, **config)
    cache.set_param_list(["gate_proj.weight", "up_proj.weight", "down_proj.weight"])
    for layer, ((name, block), d) in enumerate(zip(blocks, descs)):
        if (d["E"], d["H"], d["I"], d["top_k"]) != (d0["E"], d0["H"], d0["I"], d0["top_k"]):
            raise ValueError(f"MoE block {name} has a different shape than the first one")
        gu = block.experts.gate_up_proj.detach().to("cpu", torch.bfloat16)
        dn = block.experts.down_proj.detach().to("cpu", torch.bfloat16)
        for e in range(d["E"]):
            cache.register_expert(layer, e, [gu[e, : d["I"]].contiguous(), gu[e, d["I"]:].contiguous(), dn[e].contiguous()])
    cache.pin_all()
    cache.build_slab()
    dev = torch.device(device)
    to_dev = lambda t: t.detach().to(dev, torch.bfloat16).contiguous()  # noqa: E731
    for layer, ((name, block), d) in enumerate(zip(blocks, descs)):
        shared = None
        if d["shared"] is not None:
            s = d["shared"]
            shared = [to_dev(s.gate_proj.weight), to_dev(s.up_proj.weight), to_dev(s.down_proj.weight)]
        sgw = to_dev(d["shared_gate"].weight.reshape(-1)) if d["shared_gate"] is not None else None
        cache.set_layer_weights(layer, to_dev(block.gate.weight), d["I"], d["top_k"], d["norm_topk"], d["routed_scale"],
                                shared=shared, shared_gate_w=sgw)
        set_router(cache, layer, d, d["E"], dev)
        # the fused tensors are no longer needed: the experts live in the cache now
        block.experts.gate_up_proj = torch.nn.Parameter(torch.empty(0, dtype=torch.bfloat16), requires_grad=False)
        block.experts.down_proj = torch.nn.Parameter(torch.empty(0, dtype=torch.bfloat16), requires_grad=False)
        _replace_forward(block, cache, layer)
    model._promoe_cache = cache
    return cache


def _replace_forward(block, cache: ExpertCache, layer: int):
    block._unfused_forward = block.forward

    def fused_forward(hidden_states, *args, **kwargs):
        shape = hidden_states.shape
        x = hidden_states.reshape(-1, shape[-1])
        if x.dtype != torch.bfloat16:
            x = x.to(torch.bfloat16)
        cache.set("seq_len", shape[1] if len(shape) == 3 else 1)
        return cache.forward(layer, x.contiguous()).view(shape).to(hidden_states.dtype)

    block.forward = fused_forward


_PLAIN = (torch.Tensor, torch.nn.Parameter)
_tracing, _transforms, _modes = torch._C._get_tracing_state, torch._C._functorch.peek_interpreter_stack, torch._C._len_torch_dispatch_stack


def _watched() -> bool:
    """Whether something has to see torch's own operations: a compiler or a tracer, a transform (vmap, jvp), a dispatch mode, forward-mode
    differentiation."""
    return (torch.compiler.is_compiling() or _tracing() is not None or _transforms() is not None or _modes() > 0
            or forward_ad._current_level >= 0)


def _usable(m) -> bool:
    w, b = m.weight, m.bias
    return (isinstance(m, torch.nn.Linear) and w.is_cuda and w.dtype in (torch.bfloat16, torch.float16) and w.dim() == 2 and w.numel() > 0
            and w.stride(1) == 1 and w.stride(0) >= w.shape[1]
            and (b is None or (b.dtype == w.dtype and b.shape == w.shape[:1] and b.is_contiguous() and b.device == w.device)))


# Calls that the library's product is at least as fast for as torch's; others keep torch's. us in a CUDA graph with cold weights, bf16,
# torch's and this one's: up to 16 tokens 2048 -> 512 5.3 and 2.5-3.0, 2048 -> 2048 5.5-8.4 and 3.0-3.5, 4096 -> 4096 9.7-13.7 and 6.5-7.5,
# 3584 -> 4608 8.6-9.9 and 6.6-7.4, 2048 -> 9472 8.7-8.9 and 6.4-7.7; 17 tokens 5.3 and 5.4, 5.6 and 6.6, 9.8 and 10.9, 8.6 and 10.6; 512
# tokens 5.5 and 7.7, 7.2 and 11.8, 14.8 and 19.6, 14.7 and 18.3. More results of few tokens: 2048 -> 11008 9.4-10.6 and 9.7-11.6, -> 40000
# 26-30 and 32-33 (but -> 32000, at most 8 tokens, 25 and 22). Result rows off 16-byte boundaries slow torch's down at every number of
# tokens: 2048 -> 2050 6.2 and 3.0 for one, 20 and 7.4 for 64, 62 and 17 for 2048; 2048 -> 100003 97 and 65, 409 and 70. Rows of
# tokens or weights off them slow this one's down more from 17 on: 2050 -> 4096 21 and 27 for 64, 135 and 283 for 2048.
_FEW, _NARROW = 16, 9472


def _most(w: torch.Tensor) -> float:
    """The number of input values up to which a call takes the library's product with these weights."""
    N, K = w.shape
    if N % 8 and K % 8 == 0 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0:
        return float("inf")
    return _FEW * K if N % 8 or N <= _NARROW else 0


class _Product:
    """The library's product with a module's weights as they are now, remade where they have moved. It holds none of their memory."""

    def __init__(self, activation: str | None = None):
        self.activation, self.have, self.most = activation, (None, None), float("inf")

    def of(self, m: torch.nn.Linear, x: torch.Tensor) -> torch.Tensor | None:
        """x times m's weights; None where m's own forward has to do: it is faster, other types, kinds of tensors, devices or shapes, a
        gradient to record, operations that something has to see."""
        if _tracing() is not None or (n := x.numel()) > self.most:
            return None
        p = m._parameters
        w, b = p.get("weight"), p.get("bias")
        if type(x) not in _PLAIN or type(w) not in _PLAIN or not (b is None or type(b) in _PLAIN) or _watched():
            return None
        if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (b is not None and b.requires_grad)):
            return None
        device, dtype, shape = w.device, w.dtype, w.shape
        if x.dtype is not dtype or x.device != device or x.layout is not torch.strided or x.is_nested or x.shape[-1:] != shape[1:]:
            return None
        kind = device.type
        if torch.is_autocast_enabled(kind) and torch.get_autocast_dtype(kind) is not dtype:
            return None
        key = (w.data_ptr(), dtype, shape, w.stride(), None if b is None else (b.data_ptr(), b.dtype, b.shape, b.stride()))
        have, made = self.have  # in one step: other threads may be here too
        if have != key:
            if not _usable(m):
                return None
            made = ops.Linear(w.detach(), None if b is None else b.detach(), self.activation)._without_memory()
            self.have, self.most = (key, made), _most(w)
            if n > self.most:
                return None
        rows = n // shape[1]
        if rows > 1 << 30 or (rows > _FEW and x.data_ptr() % 16):
            return None
        return made._dense(x if x.is_contiguous() else x.contiguous(), rows, w, b)


class _Forward:
    """The forward of a replaced module. A copied or unpickled module gets one of its own, which makes its own product."""

    activation = None

    def __init__(self, m: torch.nn.Module, settings: dict | None = None):
        self.m, self.settings, self.product = m, settings, _Product(self.activation)

    def __deepcopy__(self, memo):
        return type(self)(copy.deepcopy(self.m, memo), self.settings)

    def __reduce__(self):
        return type(self), (self.m, self.settings)


class _LinearForward(_Forward):
    def __call__(self, input):  # noqa: A002 - torch.nn.Linear's own name for it
        y = self.product.of(self.m, input)
        return type(self.m).forward(self.m, input) if y is None else y


_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")
_EVERYWHERE = [getattr(torch.nn.modules.module, "_global" + h) for h in _HOOKS]


def _untouched(m: torch.nn.Module, kinds) -> bool:
    """Whether calling m is what its class does and nothing else; a torch.nn.Linear's forward may be the installed one."""
    own = vars(m)
    forward = own.get("forward")
    return (type(m) in kinds and not any(own[h] for h in _HOOKS) and not any(_EVERYWHERE)
            and (forward is None or (isinstance(forward, _LinearForward) and forward.m is m)))


def _silu(m: torch.nn.Module) -> bool:
    kind = type(m)
    return _untouched(m, (torch.nn.SiLU,) if kind.__name__ != "SiLUActivation" or not kind.__module__.startswith("transformers.") else (kind,))


class _Whole(torch.fx.Tracer):
    def is_leaf_module(self, m, qualified_name):
        return True


# Classes whose forward has been read, with that forward.
_READ: "weakref.WeakKeyDictionary[type, types.FunctionType]" = weakref.WeakKeyDictionary()


def _settings(m: torch.nn.Module):
    """The numbers that m's forward takes from m besides its parts gate_proj, up_proj, down_proj and act_fn; None where it takes anything
    else (or is wrapped), so that it is not known from m alone."""
    forward = type(m).forward
    code = getattr(forward, "__code__", None)
    if (code is None or code.co_freevars or forward.__defaults__ or forward.__kwdefaults__ or type(m).__getattr__ is not torch.nn.Module.__getattr__
            or any(isinstance(c, types.CodeType) for c in code.co_consts)):
        return None
    names = set(code.co_names) - {"gate_proj", "up_proj", "down_proj", "act_fn"}
    if any(hasattr(type(m), n) or type(vars(m).get(n, m)) not in (int, float, bool) for n in names):
        return None
    return {n: vars(m)[n] for n in names}


def _is_gated(m: torch.nn.Module) -> bool:
    """Whether m's forward is down_proj(act_fn(gate_proj(x)) * up_proj(x)) and nothing else: it is traced, not tried."""
    if _settings(m) is None:
        return False
    still = object.__new__(type(m))  # m in eval mode
    still.__dict__.update(vars(m), training=False)
    try:
        nodes = list(_Whole().trace(still).nodes)
    except Exception:  # noqa: BLE001 - a forward that looks at its input's values or sizes
        return False
    met = []

    def is_times(n):
        return n.op == "call_function" and n.target in (operator.mul, operator.imul, torch.mul) and len(n.args) == 2 and not n.kwargs

    def behind(n):  # n without factors of 1
        met.append(n)
        if is_times(n) and any(type(a) in (int, float) and a == 1 for a in n.args):
            return behind(next(a for a in n.args if isinstance(a, torch.fx.Node)))
        return n

    def part(n, name):  # the argument of this part's call
        n = behind(n) if isinstance(n, torch.fx.Node) else None
        return n.args[0] if n is not None and n.op == "call_module" and n.target == name and len(n.args) == 1 and not n.kwargs else None

    x, out = nodes[0], nodes[-1]
    met += [x, out]
    product = part(out.args[0], "down_proj")
    product = behind(product) if isinstance(product, torch.fx.Node) else None
    if x.op != "placeholder" or product is None or not is_times(product):
        return False
    for a, b in (product.args, product.args[::-1]):
        seen = len(met)
        gate = part(part(a, "act_fn"), "gate_proj")
        up = part(b, "up_proj")
        if gate is x and up is x:
            return set(met) == set(nodes)
        del met[seen:]
    return False


class _GatedForward(_Forward):
    """Three products, SiLU in the first one's epilogue. gate_proj and act_fn are passed by, so only while there is nothing else to them
    (hooks, adapters around them, another activation); the other two are called as ever."""

    activation = "silu"

    def __call__(self, x):
        m = self.m
        gate_proj, act_fn = m._modules.get("gate_proj"), m._modules.get("act_fn")
        learns = torch.is_grad_enabled() and any(p.requires_grad for p in m.parameters())
        y = None
        same = _READ.get(type(m)) is type(m).forward and all(vars(m).get(n) == v for n, v in self.settings.items())
        if same and not (m.training or learns) and gate_proj is not None and act_fn is not None:
            if _untouched(gate_proj, (torch.nn.Linear,)) and _silu(act_fn):
                y = self.product.of(gate_proj, x)
        if y is None:
            return type(m).forward(m, x)
        up = m.up_proj(x)
        return m.down_proj(y.mul_(up) if up.dtype == y.dtype and up.shape == y.shape else y * up)


def install_linears(model: torch.nn.Module) -> int:
    """Gives every torch.nn.Linear with bf16 or fp16 weights on a GPU a forward that takes promoe_b200.ops.Linear (bias in the
    product's epilogue) where that is faster: calls of at most 16 tokens (decoding), and any number of them where the rows of the
    result do not start on 16-byte boundaries; prompts keep torch's product. Gated MLPs (`gate_proj`, `up_proj`, `down_proj` around a
    SiLU and nothing else: dense layers between MoE blocks) get one with SiLU in the first product's epilogue. For inference, under
    torch.no_grad() or with parameters that require no gradient: calls that a gradient is to be recorded for keep the module's own forward, as
    do those that torch traces, compiles, transforms, casts or counts, and a gated MLP's in training mode or with hooks or adapters on
    gate_proj or act_fn. A token's result may differ in its last bits with the number of tokens of the call, as with torch's.
    Call it once the model is on its device. Weights are used in place; they may be changed or
    exchanged afterwards, and a copied model works on its own. Modules of other classes than torch.nn.Linear itself, or with a forward of
    their own (hooks of other libraries), stay as they are. MoE blocks that inject_hf_fused_model replaced do
    not call theirs any more. Returns the number of replaced modules."""
    replaced = 0
    for m in list(model.modules()):
        if type(m) is torch.nn.Linear and _usable(m) and "forward" not in vars(m):
            m.forward = _LinearForward(m)
            replaced += 1
    mine = lambda m: isinstance(vars(m).get("forward"), _LinearForward)  # noqa: E731
    for m in list(model.modules()):
        parts = dict(m.named_children())
        act = parts.pop("act_fn", None)
        if (sorted(parts) != ["down_proj", "gate_proj", "up_proj"] or not all(mine(p) for p in parts.values())
                or act is None or not _silu(act) or "forward" in vars(m)):
            continue
        if _is_gated(m):
            _READ[type(m)] = type(m).forward
            m.forward = _GatedForward(m, _settings(m))
            replaced += 1
    return replaced


def _compare_logits(lin, rows: torch.Tensor, own: torch.Tensor) -> None:
    """Raises where a model's logits are not what its vocabulary projection makes of these hidden rows. Its own are rounded to the
    projection's type, perhaps twice: a step of the value and of a usual one."""
    mine = lin(rows)
    if own.shape[-1] != mine.shape[-1] or own.numel() != mine.numel():
        raise ValueError("this model's logits have another shape than its vocabulary projection gives them")
    own = own.reshape(mine.shape).float()
    usual = mine.square().mean(1, keepdim=True).sqrt()
    off = (own - mine).abs() > torch.finfo(rows.dtype).eps * (mine.abs() + usual) + 1e-4 * usual
    off |= own.isnan() != mine.isnan()
    if bool((off & rows.isfinite().all(1, keepdim=True)).any()):
        raise ValueError("this model changes its logits behind the vocabulary projection")


@torch.no_grad()
def score_tokens(model: torch.nn.Module, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None, top_n: int = 0) -> dict:
    """What a causal LM thinks of a text: for every position but the last, the log probability of the token that follows, the
    entropy of the model's prediction there and its top_n favourites. input_ids [B, S] -> {"logp": [B, S - 1], "entropy": [B, S - 1],
    "top_ids", "top_logp": [B, S - 1, top_n]}. Only tokens inside attention_mask [B, S] that follow one inside it are scored, the others' logp
    is 0; positions count from a text's first token inside it, so that padding on either side changes nothing. The vocabulary
    projection (bf16 or fp16, on the GPU) runs with float32 logits, for as many positions at a time as 64 Mi logits hold,
    so a long text does not need all its logits at once. Models whose logits are something else than that projection (they cap or
    scale them, or have an adapter there) are refused: some of them are compared with the model's own."""
    for name in ("final_logit_softcapping", "logit_scale", "logits_scaling", "lm_head_multiplier"):
        if getattr(model.config, name, None) not in (None, 1.0):
            raise ValueError(f"this model changes its logits behind the vocabulary projection ({name})")
    head = model.get_output_embeddings()
    trunk = getattr(model, model.base_model_prefix)
    takes = inspect.signature(trunk.forward).parameters
    given = {"use_cache": False} if "use_cache" in takes else {}  # keys and values that nobody reads
    if attention_mask is not None:
        if attention_mask.shape != input_ids.shape:
            raise ValueError(f"attention_mask must have the shape of input_ids, {tuple(input_ids.shape)}")
        if "position_ids" in takes:
            given["position_ids"] = (attention_mask.long().cumsum(-1) - 1).clamp_min(0)
    B, S = input_ids.shape
    lin = ops.Linear(head.weight, getattr(head, "bias", None), out_dtype=torch.float32)
    own_takes = inspect.signature(model.forward).parameters
    seen = []  # what the trunk gives the model's own forward
    handle = trunk.register_forward_hook(lambda m, args, out: seen.append(out.last_hidden_state if hasattr(out, "last_hidden_state") else out[0]))
    try:
        def logits_of(ids, **kw):
            kw.update({k: v for k, v in (("use_cache", False), ("output_router_logits", False)) if k in own_takes})
            own = model(input_ids=ids, **kw).logits
            if len(seen) != 1:
                raise ValueError(f"this model's forward does not take its hidden rows from {model.base_model_prefix!r} once")
            return own, seen.pop()
        if "logits_to_keep" in own_takes:  # one pass for both, the logits of the last two positions
            last = min(2, S)
            own, hidden = logits_of(input_ids, attention_mask=attention_mask, logits_to_keep=last, **{k: v for k, v in given.items() if k in own_takes})
            rows = hidden[:, -last:]
        else:
            own, rows = logits_of(input_ids[:1, :4])
            hidden = trunk(input_ids=input_ids, attention_mask=attention_mask, **given).last_hidden_state
    finally:
        handle.remove()
    _compare_logits(lin, rows.reshape(-1, rows.shape[-1]).to(head.weight.dtype), own)
    x = hidden[:, :-1].reshape(B * (S - 1), hidden.shape[-1]).to(head.weight.dtype)
    targets = input_ids[:, 1:].to(torch.int64)
    if attention_mask is not None:
        targets = targets.masked_fill((attention_mask[:, 1:] == 0) | (attention_mask[:, :-1] == 0), -100)
    targets = targets.reshape(-1)
    T = x.shape[0]
    new = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=x.device)  # noqa: E731
    logp, entropy, ids, best = new(T), new(T), new(T, top_n, dtype=torch.int32), new(T, top_n)
    step = max(1, min(T, (1 << 26) // lin.N))
    logits = new(step, lin.N)
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        lin(x[t0:t1], out=logits[:t1 - t0])
        ops.token_logprobs(logits[:t1 - t0], targets[t0:t1], top_n, out=(logp[t0:t1], entropy[t0:t1], ids[t0:t1], best[t0:t1]))
    return {"logp": logp.view(B, S - 1), "entropy": entropy.view(B, S - 1), "top_ids": ids.view(B, S - 1, top_n),
            "top_logp": best.view(B, S - 1, top_n)}
