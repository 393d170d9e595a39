"""What the operators around the experts cost: routing, dense products and the scoring of answers.

Three operators that a mixture-of-experts model needs beside its expert layers, in their plain form (elementary torch
operations) and as the framework offers them (`promoe_b200.ops`):

  route   router logits -> the experts of every token and their weights
  linear  y = act(x W^T + bias) + residual
  logp    vocabulary logits -> log probability of the given token, entropy and the best alternatives, row by row
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _route(T, E, k, dtype="f32", scoring="softmax", bias=False, groups=1, keep=1, group_score="max", norm=False, scale=1.0,
           masked=0.0):
    return dict(op="route", T=T, E=E, k=k, dtype=dtype, scoring=scoring, bias=bias, groups=groups, keep=keep,
                group_score=group_score, norm=norm, scale=scale, masked=masked)


def _linear(M, K, N, dtype="bf16", out="same", bias="none", act="none", residual=False, pitch=0):
    return dict(op="linear", M=M, K=K, N=N, dtype=dtype, out=out, bias=bias, act=act, residual=residual, pitch=pitch)


def _logp(T, V, dtype="bf16", top=0, masked=0.0, skipped=0.0):
    return dict(op="logp", T=T, V=V, dtype=dtype, top=top, masked=masked, skipped=skipped)


def listed():
    def c(name, case):
        return dict(case, name=name)
    return [
        # one user typing: the router of a 64-expert layer for a single token
        c("route1_e64", _route(1, 64, 6)),
        # a decode batch through a router with sigmoid scores, a correction bias and groups scored by their two best
        c("route64_e256_sigmoid", _route(64, 256, 8, scoring="sigmoid", bias=True, groups=8, keep=4, group_score="top2",
                                         norm=True, scale=2.5)),
        # a short prompt of odd length, group-limited softmax routing on 16-bit logits, some experts masked out
        c("route777_e160_groups", _route(777, 160, 6, dtype="bf16", groups=8, keep=3, scale=16.0, masked=0.1)),
        # a batch of long prompts through the sigmoid router
        c("route16384_e256_sigmoid", _route(16384, 256, 8, scoring="sigmoid", bias=True, groups=8, keep=4,
                                            group_score="top2", norm=True, scale=2.5)),
        # first layer of the expert predictor, one sequence: bias and ReLU, float32 out
        c("linear1_relu", _linear(1, 2048, 512, out="f32", bias="f32", act="relu")),
        # attention projections with bias, a decode batch of 8 (hidden 3584)
        c("linear8_bias", _linear(8, 3584, 4608, bias="same")),
        # vocabulary projection of a decode batch, float32 logits, an odd vocabulary
        c("linear33_vocab", _linear(33, 2048, 100003, out="f32")),
        # projection back to the hidden size with residual, a short prompt of odd length, fp16
        c("linear777_residual", _linear(777, 5632, 2048, dtype="f16", residual=True)),
        # first product of a dense layer, batch of long prompts
        c("linear8192_silu", _linear(8192, 4096, 14336, act="silu")),
        # one generated token: log probability and the 20 best alternatives
        c("logp1_top20", _logp(1, 131072, dtype="f32", top=20)),
        # a decode batch under an allowed-token mask, odd vocabulary
        c("logp33_masked", _logp(33, 50001, dtype="bf16", top=5, masked=0.5)),
        # scoring of a long text: every token of 4096 positions, padding among them
        c("logp4096_top5", _logp(4096, 131072, dtype="bf16", top=5, skipped=0.02)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another call of these ranges."""
    op = rng.choice(["route", "linear", "linear", "logp"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * rng.randint(max(2, 8 // groups), 512 // groups)
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(12, keep * (E // groups)))
        scoring = rng.choice(["softmax", "sigmoid"])
        T = _log_int(rng, 1, max(1, min(16384, 16384 * 256 // E)))
        return _route(T, E, k, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), scoring=scoring,
                      bias=rng.random() < 0.5, groups=groups, keep=keep,
                      group_score=rng.choice(["max", "top2"]) if E // groups > 1 else "max", norm=rng.random() < 0.5,
                      scale=rng.choice([1.0, 2.5, 16.0]), masked=rng.choice([0.0, 0.0, 0.2]))
    if op == "linear":
        dtype = rng.choice(["bf16", "bf16", "f16"])
        # rows of most models start on 16-byte boundaries; some views and narrow layers do not
        step = rng.choice([64, 64, 8, 1])
        K = max(1, _log_int(rng, 64, 8192) // step) * step
        N = _log_int(rng, 64, 131072)
        most = min(8192, 8192 * 4096 * 14336 // (K * N), (1 << 28) // N)
        M = _log_int(rng, 1, max(1, most))
        out = rng.choice(["same", "same", "f32"])
        return _linear(M, K, N, dtype=dtype, out=out, bias=rng.choice(["none", "same", "f32"]),
                       act=rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh"]),
                       residual=rng.random() < 0.4, pitch=rng.choice([0, 0, 64]))
    V = _log_int(rng, 1000, 131072)
    T = _log_int(rng, 1, max(1, min(4096, 4096 * 65536 // V)))
    return _logp(T, V, dtype=rng.choice(["bf16", "bf16", "f32", "f16"]), top=rng.choice([0, 1, 5, 20]),
                 masked=rng.choice([0.0, 0.0, 0.5, 0.99]), skipped=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------------------------------------ inputs
def _gen(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + {"route": 1, "linear": 2, "logp": 3}[case["op"]])


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _inputs(case, seed):
    g = _gen(case, seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        # some experts are liked better than others; a token's logits spread around that
        logits = 1.5 * _randn(g, T, E) + 0.5 * _randn(g, E)
        if case["masked"]:
            logits.masked_fill_(torch.rand((T, E), generator=g, device="cuda") < case["masked"], float("-inf"))
            if T > 2:
                logits[T // 2] = float("-inf")  # a padding row
        bias = 0.1 * _randn(g, E) if case["bias"] else None
        return dict(logits=logits.to(dt), bias=bias)
    if case["op"] == "linear":
        M, K, N, p = case["M"], case["K"], case["N"], case["pitch"]
        x = _randn(g, M, K + p).to(dt)[:, :K]
        w = (_randn(g, N, K) * 0.02).to(dt)
        od = dt if case["out"] == "same" else torch.float32
        bias = None if case["bias"] == "none" else (_randn(g, N) * 0.1).to(dt if case["bias"] == "same" else torch.float32)
        res = _randn(g, M, N + p).to(od)[:, :N] if case["residual"] else None
        return dict(x=x, w=w, bias=bias, res=res, od=od)
    T, V = case["T"], case["V"]
    logits = torch.empty((T, V), dtype=dt, device="cuda")
    for t0 in range(0, T, 512):  # float32 only for a part at a time
        part = 2.5 * _randn(g, min(512, T - t0), V)
        if case["masked"]:
            part.masked_fill_(torch.rand(part.shape, generator=g, device="cuda") < case["masked"], float("-inf"))
        logits[t0:t0 + 512] = part.to(dt)
    if case["masked"] and T > 2:
        logits[T // 2] = float("-inf")  # a row whose mask leaves nothing
    targets = torch.randint(0, V, (T,), generator=g, device="cuda")
    if case["skipped"]:
        targets.masked_fill_(torch.rand((T,), generator=g, device="cuda") < case["skipped"], -100)
    return dict(logits=logits, targets=targets)


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        # what a program keeps between calls: the router, the layer's weights, the buffers of the results
        from promoe_b200 import ops
        s["ops"] = ops
        if case["op"] == "route":
            s["router"] = ops.Router(case["E"], case["k"], scoring=case["scoring"], bias=s["bias"], n_group=case["groups"],
                                     topk_group=case["keep"], group_score=case["group_score"], norm_topk=case["norm"],
                                     routed_scale=case["scale"])
            s["out"] = (torch.empty((case["T"], case["k"]), dtype=torch.int32, device="cuda"),
                        torch.empty((case["T"], case["k"]), dtype=torch.float32, device="cuda"))
        elif case["op"] == "linear":
            s["linear"] = ops.Linear(s["w"], s["bias"], activation=case["act"], out_dtype=s["od"])
            s["out"] = torch.empty((case["M"], case["N"]), dtype=s["od"], device="cuda")
        else:
            T, n = case["T"], case["top"]
            s["out"] = (torch.empty(T, dtype=torch.float32, device="cuda"), torch.empty(T, dtype=torch.float32, device="cuda"),
                        torch.empty((T, n), dtype=torch.int32, device="cuda"),
                        torch.empty((T, n), dtype=torch.float32, device="cuda"))
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_route(logits, bias, case):
    """Scores and choices in 64 bits: two choices may be neighbours in 32."""
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    ninf = float("-inf")
    l = logits.double()
    out = l == ninf
    if case["scoring"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        m = l.amax(1, keepdim=True)
        e = torch.exp(l - torch.where(m == ninf, torch.zeros_like(m), m))
        s = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    c = (s + bias.double() if bias is not None else s).masked_fill(out, ninf)
    if G > 1:
        best = c.view(T, G, E // G).sort(dim=2, descending=True).values
        value = best[:, :, 0]
        if case["group_score"] == "top2":
            second = best[:, :, 1]
            value = value + torch.where(second == ninf, torch.zeros_like(second), second)
        order = value.sort(dim=1, descending=True, stable=True).indices
        kept = torch.zeros((T, G), dtype=torch.bool, device=l.device).scatter_(1, order[:, :case["keep"]], True)
        c = c.masked_fill(~kept.repeat_interleave(E // G, dim=1), ninf)
    best, ids = c.sort(dim=1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    none = best == ninf
    w = torch.gather(s, 1, ids).masked_fill(none, 0.0)
    if case["norm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return ids.masked_fill(none, -1).to(torch.int32), (w * case["scale"]).float()


def _activate(v, act):
    if act == "relu":
        return torch.clamp_min(v, 0.0)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_linear(x, w, bias, res, od, act):
    v = x.float() @ w.float().T
    if bias is not None:
        v = v + bias.float()
    v = _activate(v, act)
    if res is not None:
        v = v + res.float()
    return v.to(od)


def _plain_logp(logits, targets, n):
    T, V = logits.shape
    l = logits.float()
    m = l.amax(1)
    d = l - m[:, None]
    e = torch.exp(d)
    s = e.sum(1)
    entropy = torch.log(s) - torch.where(e > 0, e * d, torch.where(torch.isnan(e), e, torch.zeros_like(e))).sum(1) / s
    at = torch.gather(d, 1, targets.clamp(0, V - 1)[:, None])[:, 0]
    logp = torch.where(targets < 0, torch.zeros_like(m), at - torch.log(s))
    # the largest, ties to the lower index: values as ordered integers above the reversed index
    bits = (l + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device=l.device))
    ids = V - 1 - (torch.topk(key, n, dim=1).values & 0xFFFFFFFF)
    best = torch.gather(d, 1, ids) - torch.log(s)[:, None]
    none = torch.isnan(s)[:, None] | (best == float("-inf"))
    return logp, entropy, ids.masked_fill(none, -1).to(torch.int32), best


def run(state):
    case = state["case"]
    if case["op"] == "route":
        if own:
            return state["router"](state["logits"], out=state["out"])
        return _plain_route(state["logits"], state["bias"], case)
    if case["op"] == "linear":
        if own:
            return state["linear"](state["x"], residual=state["res"], out=state["out"])
        return _plain_linear(state["x"], state["w"], state["bias"], state["res"], state["od"], case["act"])
    if own:
        return state["ops"].token_logprobs(state["logits"], state["targets"], top_n=case["top"], out=state["out"])
    return _plain_logp(state["logits"], state["targets"], case["top"])


# ------------------------------------------------------------------------------------------ from the definitions, 64 bits
def _exact_route(case, x):
    """Rank by counting, in numpy: a choice's place is the number of choices before it."""
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    ids, weights = np.full((T, k), -1, np.int32), np.zeros((T, k))
    bias = np.zeros(E) if x["bias"] is None else x["bias"].double().cpu().numpy()
    for t0 in range(0, T, 1024):
        row = x["logits"][t0:t0 + 1024].double().cpu().numpy()
        n = len(row)
        score = np.exp(-np.logaddexp(0.0, -row))
        if case["scoring"] == "softmax":
            score = np.exp(row - np.logaddexp.reduce(row, axis=1, keepdims=True, where=row > -np.inf, initial=-np.inf)
                           .clip(min=-1e300))
        choice = np.where(row > -np.inf, score + bias, -np.inf)
        if G > 1:
            parts = -np.sort(-choice.reshape(n, G, E // G), axis=2)[:, :, :2]
            value = parts[:, :, 0] + (np.maximum(parts[:, :, 1], -1e300) * (parts[:, :, 1] > -np.inf)
                                      if case["group_score"] == "top2" else 0.0)
            before = (value[:, None, :] > value[:, :, None]).sum(2)
            before += ((value[:, None, :] == value[:, :, None]) & np.tri(G, k=-1, dtype=bool)).sum(2)
            choice = np.where(np.repeat(before < case["keep"], E // G, axis=1), choice, -np.inf)
        order = np.lexsort((np.broadcast_to(np.arange(E), choice.shape), -choice), axis=1)[:, :k]
        there = np.take_along_axis(choice, order, 1) > -np.inf
        w = np.where(there, np.take_along_axis(score, order, 1), 0.0)
        if case["norm"]:
            w = w / (w.sum(1, keepdims=True) + 1e-20)
        ids[t0:t0 + n], weights[t0:t0 + n] = np.where(there, order, -1), w * case["scale"]
    return ids, weights


def _exact_linear(case, x):
    rows = []
    w = x["w"].double()
    for m0 in range(0, case["M"], 2048):
        v = torch.mm(x["x"][m0:m0 + 2048].double(), w.t())
        if x["bias"] is not None:
            v += x["bias"].double()
        if case["act"] == "relu":
            v = torch.where(v > 0, v, torch.zeros_like(v))
        elif case["act"] == "silu":
            v = v * torch.special.expit(v)
        elif case["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        elif case["act"] == "gelu_tanh":
            v = v * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
        if x["res"] is not None:
            v += x["res"][m0:m0 + 2048].double()
        rows.append(v)
    return torch.cat(rows)


def _exact_logp(case, x):
    got = [[], [], [], []]
    for t0 in range(0, case["T"], 256):
        l, t = x["logits"][t0:t0 + 256].double(), x["targets"][t0:t0 + 256]
        dead = torch.isneginf(l).all(1)
        lse = torch.logsumexp(l, 1)
        lse[dead] = float("nan")
        p = torch.exp(l - lse[:, None])
        got[0].append(torch.where(t < 0, torch.zeros_like(lse), l[torch.arange(len(t), device=t.device), t.clamp_min(0)] - lse))
        got[1].append(-torch.xlogy(p, p).sum(1))
        best, ids = torch.sort(l, dim=1, descending=True, stable=True)
        best, ids = best[:, :case["top"]], ids[:, :case["top"]]
        none = dead[:, None] | torch.isneginf(best)
        got[2].append(torch.where(none, -1, ids).to(torch.int32))
        got[3].append(best - lse[:, None])
    return tuple(torch.cat(g) for g in got)


def exact(case, seed):
    x = _inputs(case, seed)
    return {"route": _exact_route, "linear": _exact_linear, "logp": _exact_logp}[case["op"]](case, x)


def work(case):
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        return {"bytes": float(T * E * SIZES[case["dtype"]] + (4 * E if case["bias"] else 0) + 8 * T * case["k"]),
                "flops": 10.0 * T * E}
    if case["op"] == "linear":
        M, K, N, size = case["M"], case["K"], case["N"], SIZES[case["dtype"]]
        out = size if case["out"] == "same" else 4
        b = {"none": 0, "same": size, "f32": 4}[case["bias"]]
        return {"bytes": float((M * K + N * K) * size + N * b + M * N * out * (2 if case["residual"] else 1)),
                "flops": 2.0 * M * N * K}
    T, V = case["T"], case["V"]
    return {"bytes": float(T * V * SIZES[case["dtype"]] + T * (16 + 8 * case["top"])), "flops": 8.0 * T * V}
