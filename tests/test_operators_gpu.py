"""The operators around the experts (promoe_b200.ops: Router, Linear, token_logprobs) against plain 64-bit forms, at the sizes,
masks, strides and streams where they can go wrong. half_step(t) is the largest relative error of one rounding to t."""
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from promoe_b200 import _lib, ops

pytestmark = pytest.mark.gpu

INF = float("inf")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=F32)


# ------------------------------------------------------------------------------------------------ routing
def route_oracle(logits, k, scoring="softmax", bias=None, n_group=1, topk_group=1, group_score="max", norm=False, scale=1.0):
    """Row by row in Python floats (64 bits)."""
    T, E = logits.shape
    per = E // n_group
    l64 = logits.double().cpu().numpy()
    b = np.zeros(E) if bias is None else bias.double().cpu().numpy()
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t, row in enumerate(l64):
        if np.isnan(row).any() or (scoring == "softmax" and np.isposinf(row).any()):
            w[t] = np.nan
            continue
        alive = [e for e in range(E) if row[e] != -INF]
        if scoring == "softmax":
            top = max((row[e] for e in alive), default=0.0)
            z = math.fsum(math.exp(row[e] - top) for e in alive)
            s = {e: math.exp(row[e] - top) / z for e in alive}
        else:
            s = {e: 1.0 / (1.0 + math.exp(-row[e])) if row[e] > -700 else 0.0 for e in alive}
        c = {e: s[e] + b[e] for e in alive}
        alive = [e for e in alive if c[e] > -INF]  # not NaN either
        if bias is None:  # equal scores of unequal logits (saturated ones) are ranked as exact arithmetic would
            order = lambda e: (-row[e], e)  # noqa: E731
        else:
            order = lambda e: (-c[e], e)  # noqa: E731
        groups = {}
        for e in alive:
            groups.setdefault(e // per, []).append(e)
        if n_group > 1:
            def worth(g):
                best = sorted(groups[g], key=order)[:2 if group_score == "top2" else 1]
                if group_score == "top2" or bias is not None:
                    return (-sum(c[e] for e in best), g)
                return (-row[best[0]], g)
            kept = sorted(groups, key=worth)[:topk_group]
            alive = [e for g in kept for e in groups[g]]
        best = sorted(alive, key=order)[:k]
        z = sum(s[e] for e in best) + 1e-20 if norm else 1.0
        for j, e in enumerate(best):
            ids[t, j], w[t, j] = e, s[e] / z * scale
    return ids, w


def check_route(logits, k, **rule):
    kw = dict(rule)
    norm, scale = kw.pop("norm", False), kw.pop("scale", 1.0)
    ids, w = ops.Router(logits.shape[1], k, norm_topk=norm, routed_scale=scale, **kw)(logits)
    ref_ids, ref_w = route_oracle(logits, k, norm=norm, scale=scale, **kw)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    # a weight is a quotient of float32 exponentials: each argument is off by half a step of at most 90 (2^-24 * 90 = 5.4e-6),
    # and so is the sum's share; products and quotients add a few half steps
    np.testing.assert_allclose(w.cpu().numpy(), ref_w, rtol=1.2e-5, atol=1e-30)
    return ids, w


RULES = [dict(), dict(norm=True), dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=True, norm=True, scale=2.5),
         dict(bias=True), dict(n_group=4, topk_group=2), dict(n_group=4, topk_group=3, group_score="top2"),
         dict(scoring="sigmoid", bias=True, n_group=4, topk_group=2, group_score="top2", norm=True, scale=2.5),
         dict(scoring="sigmoid", n_group=4, topk_group=1), dict(n_group=4, topk_group=4, bias=True)]


@pytest.mark.parametrize("rule", RULES, ids=lambda r: "-".join(f"{k}={v}" for k, v in r.items()) or "plain")
@pytest.mark.parametrize("T,E,k,dtype", [(1, 8, 2, F32), (3, 60, 4, F32), (65, 64, 6, BF16), (130, 160, 6, F16), (33, 256, 8, F32),
                                         (17, 384, 8, F32), (9, 512, 10, BF16), (5, 1024, 32, F32), (7, 36, 9, F32)])
def test_route_matches_the_definition(lib, T, E, k, dtype, rule):
    rule = dict(rule)
    g = gen(T * 1000 + E)
    logits = (2 * randn(g, T, E) + randn(g, E)).to(dtype)
    if rule.get("bias"):
        rule["bias"] = 0.2 * randn(g, E)
    n_group = rule.get("n_group", 1)
    k = min(k, rule.get("topk_group", 1) * (E // n_group) if n_group > 1 else E)
    check_route(logits, k, **rule)


def test_route_masks_and_rows_without_experts(lib):
    g = gen(1)
    T, E = 12, 64
    logits = randn(g, T, E)
    logits[0] = -INF                                  # nothing
    logits[1, 3:] = -INF                              # fewer than k
    logits[2, :60] = -INF                             # only the last group
    logits[3] = torch.finfo(F32).min                  # lowest finite values: all equal
    logits[4, ::2] = torch.finfo(F32).min
    logits[5, 7] = float("nan")
    logits[6, 9] = INF
    logits[7] = 0.0
    logits[7, ::2] = -0.0                             # equal to 0.0: ties to the lower id
    logits[8] = 60.0 + torch.arange(E, device="cuda") / 64  # saturated sigmoid scores
    for rule in (dict(), dict(scoring="sigmoid"), dict(n_group=8, topk_group=2), dict(n_group=8, topk_group=2, group_score="top2"),
                 dict(norm=True, scale=2.0)):
        check_route(logits, 6, **rule)
    bias = 0.1 * randn(g, E)
    bias[5], bias[6] = -INF, float("nan")             # experts taken out by the bias
    keep = [0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11]        # row 8's scores tie in 64 bits, the bias decides there
    for rule in (dict(bias=bias), dict(scoring="sigmoid", bias=bias, n_group=8, topk_group=2, group_score="top2", norm=True)):
        check_route(logits[keep].contiguous(), 6, **rule)


def test_route_ties_go_to_the_lower_id_and_group(lib):
    logits = torch.zeros((3, 64), device="cuda")
    logits[1, 40:48] = 1.0
    bias = torch.zeros(64, device="cuda")
    for rule in (dict(), dict(scoring="sigmoid"), dict(bias=bias), dict(n_group=8, topk_group=2, group_score="top2"),
                 dict(scoring="sigmoid", bias=bias, n_group=8, topk_group=3, group_score="top2")):
        check_route(logits, 8, **rule)


@pytest.mark.parametrize("steps", [0.25, 1, 3, 20])
def test_route_decides_near_ties_exactly(lib, steps):
    """Choices that lie some float32 steps apart, too close for float32 arithmetic to rank."""
    g = gen(int(steps * 4))
    T, E, k = 64, 64, 8
    logits = randn(g, T, E)
    s = torch.sigmoid(logits.double())
    # bias of expert e brings its choice in row 0 to 1 + e * steps * 2^-24, the rows differ by chance
    bias = (1.0 + torch.randperm(E, generator=torch.Generator().manual_seed(3)).cuda().double() * steps * 2.0 ** -24 - s[0]).float()
    logits[1:32] = logits[0] + 1e-7 * randn(g, 31, E)
    check_route(logits, k, scoring="sigmoid", bias=bias)
    check_route(logits, k, scoring="sigmoid", bias=bias, n_group=8, topk_group=4, group_score="top2")
    p = torch.softmax(logits.double(), 1)
    bias = (1.0 + torch.randperm(E, generator=torch.Generator().manual_seed(4)).cuda().double() * steps * 2.0 ** -24 - p[0]).float()
    check_route(logits, k, bias=bias, norm=True)


def test_route_strided_rows_and_given_outputs(lib):
    g = gen(2)
    wide = randn(g, 21, 200)
    for view in (wide[:, :64], wide[:, 7:71], wide[::3, 8:72], wide[:, :64].to(BF16), torch.zeros((21, 70), dtype=F16, device="cuda")
                 [:, 3:67].copy_(wide[:, :64])):
        check_route(view, 5, norm=True)
    r = ops.Router(64, 5)
    out = (torch.full((24, 5), 77, dtype=torch.int32, device="cuda"), torch.full((24, 5), 7.0, device="cuda"))
    r(wide[:, :64], out=(out[0][:21], out[1][:21]))
    ref = route_oracle(wide[:, :64], 5)
    assert np.array_equal(out[0][:21].cpu().numpy(), ref[0]) and bool((out[0][21:] == 77).all()) and bool((out[1][21:] == 7.0).all())
    ids, w = r(wide[:0, :64])
    assert ids.shape == (0, 5) and w.shape == (0, 5)


# ------------------------------------------------------------------------------------------------ linear
def act64(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def check_linear(x, w, bias=None, act=None, residual=None, out_dtype=None, out=None):
    before = None if residual is None else residual.double().clone()
    y = ops.Linear(w, bias, act, out_dtype)(x, residual=residual, out=out)
    x64, w64 = x.double(), w.double()
    v = x64 @ w64.T
    size = x64.abs() @ w64.abs().T
    if bias is not None:
        v = v + bias.double()
        size = size + bias.double().abs()
    ref = act64(v, act)
    if residual is not None:
        ref = ref + before
    K = x.shape[1]
    # Sums: K additions, each off by at most a step (2^-23) of a partial sum, which never exceeds the sum of magnitudes. The
    # activations' slopes stay below 1.13, their exponentials' arguments are off by steps of |v|: 16 steps of 1 + |v|. The
    # residual's addition and the result's rounding: half a step each.
    tol = 1.13 * (K + 64) * 2.0 ** -23 * size + 16 * 2.0 ** -23 * (1 + v.abs())
    tol = tol + (half_step(F32) + half_step(y.dtype)) * (ref.abs() + tol) + torch.finfo(y.dtype).tiny * half_step(y.dtype) * 2
    bad = ((y.double() - ref).abs() > tol).sum()
    assert int(bad) == 0, f"{int(bad)} of {y.numel()} outputs out of tolerance, worst {float(((y.double() - ref).abs() / tol).max())}"
    # errors of single products average out: far inside the bound above
    assert float((y.double() - ref).norm()) <= (2e-6 + half_step(y.dtype)) * float(ref.norm() + size.norm() * 0.05) + 1e-30
    return y


@pytest.mark.parametrize("M,K,N", [(1, 64, 128), (1, 2048, 512), (1, 8, 1), (2, 72, 130), (7, 200, 257), (8, 3584, 320), (16, 512, 33),
                                   (17, 136, 1000), (33, 1024, 5003), (64, 4096, 256), (100, 64, 384), (129, 264, 129),
                                   (256, 128, 512), (257, 320, 513), (300, 2048, 640), (777, 704, 1408), (1030, 512, 2049)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_sizes(lib, M, K, N, dtype):
    g = gen(M + K + N)
    check_linear(randn(g, M, K).to(dtype), (randn(g, N, K) * 0.05).to(dtype))


@pytest.mark.parametrize("M", [1, 8, 9, 16])
@pytest.mark.parametrize("K,N", [(8, 16), (200, 15), (64, 2368), (1160, 2369), (72, 4737), (520, 9000), (64, 9473), (128, 37889)])
@pytest.mark.parametrize("out_dtype", [F16, F32])
def test_linear_few_tokens(lib, M, K, N, out_dtype):
    """Either side of where the kernels for few tokens take each other's place, with rows that end inside a step."""
    g = gen(M + K + N)
    x, w = randn(g, M, K).to(F16), (randn(g, N, K) * 0.05).to(F16)
    check_linear(x, w, randn(g, N).to(F16), "gelu_tanh", randn(g, M, N).to(out_dtype), out_dtype)


@pytest.mark.parametrize("M", [1, 8, 9, 16])
@pytest.mark.parametrize("K,N", [(1, 17), (77, 40), (130, 2369), (1001, 2368), (67, 7105)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_linear_few_tokens_off_16_byte_boundaries(lib, M, K, N, out_dtype):
    """Every offset of rows in a 16-byte word, with values around them that must not count."""
    g = gen(M + K + N)
    for lead, pitch in ((1, K + 1), (3, K + 12), (6, K + 7)):
        xb = torch.full((M * pitch + 16,), float("nan"), dtype=BF16, device="cuda")
        wb = torch.full((N * (pitch + 2) + 16,), float("nan"), dtype=BF16, device="cuda")
        x, w = xb.as_strided((M, K), (pitch, 1), lead), wb.as_strided((N, K), (pitch + 2, 1), lead + 1)
        x.copy_(randn(g, M, K))
        w.copy_(randn(g, N, K) * 0.1)
        check_linear(x, w, randn(g, N).to(BF16), "gelu", None, out_dtype)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,K,N", [(1, 512, 640), (5, 4096, 200), (40, 256, 300), (600, 192, 2304)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("bias_dtype", [None, BF16, F32])
def test_linear_epilogue(lib, act, M, K, N, out_dtype, bias_dtype):
    g = gen(M * 7 + K)
    x, w = randn(g, M, K).to(BF16), (randn(g, N, K) * (2.0 / math.sqrt(K))).to(BF16)
    bias = None if bias_dtype is None else randn(g, N).to(bias_dtype)
    res = randn(g, M, N).to(out_dtype)
    check_linear(x, w, bias, act, None, out_dtype)
    y = check_linear(x, w, bias, act, res, out_dtype)
    # over the residual itself
    again = ops.Linear(w, bias, act, out_dtype)(x, residual=res, out=res)
    assert again is res and torch.equal(again, y)


@pytest.mark.parametrize("M,K,N", [(1, 77, 40), (3, 1001, 130), (65, 99, 67), (200, 513, 300), (1, 1, 1), (5, 7, 3)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_rows_off_16_byte_boundaries(lib, M, K, N, dtype):
    g = gen(M + K)
    check_linear(randn(g, M, K).to(dtype), (randn(g, N, K) * 0.05).to(dtype), randn(g, N).to(dtype), "silu", randn(g, M, N).to(dtype))
    # rows of 8 k, but the first starts elsewhere
    x = torch.zeros((M, 88), dtype=dtype, device="cuda")[:, 1:73].copy_(randn(g, M, 72).to(dtype))
    check_linear(x, (randn(g, N, 72) * 0.05).to(dtype))


@pytest.mark.parametrize("M,N", [(3, 100), (70, 333), (515, 260)])
def test_linear_strides_and_rows_left_alone(lib, M, N):
    g = gen(M)
    K = 100  # rows of 100 values, 128 apart: the last step of 64 k ends inside the pitch, whose values must not count
    xb, wb = torch.full((M + 2, 128), float("nan"), dtype=BF16, device="cuda"), torch.full((N + 2, 128), float("nan"), dtype=BF16, device="cuda")
    x, w = xb[1:-1, 8:8 + K], wb[1:-1, 16:16 + K]
    x.copy_(randn(g, M, K))
    w.copy_(randn(g, N, K) * 0.1)
    res = randn(g, M, N + 3)[:, 1:N + 1]
    yb = torch.full((M + 2, N + 5), 7.0, device="cuda")
    y = yb[1:-1, 3:N + 3]
    check_linear(x, w, None, "relu", res, F32, out=y)
    mask = torch.ones_like(yb, dtype=torch.bool)
    mask[1:-1, 3:N + 3] = False
    assert bool((yb[mask] == 7.0).all())


def test_linear_infinities_and_nan_stay_in_their_rows_and_columns(lib):
    g = gen(9)
    M, K, N = 20, 128, 200
    x, w = randn(g, M, K).to(BF16), (randn(g, N, K) * 0.1).to(BF16)
    clean = ops.Linear(w)(x)
    x[3, 5], x[4, 6] = float("nan"), INF
    w[7, 9] = -INF
    y = ops.Linear(w)(x)
    ref = x.double() @ w.double().T
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isinf(y), torch.isinf(ref))
    rows = [i for i in range(M) if i not in (3, 4)]
    cols = [j for j in range(N) if j != 7]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])
    r = ops.Linear(w, None, "relu")(x)
    assert torch.equal(torch.isnan(r), torch.isnan(ref))


@pytest.mark.parametrize("M", [1, 12, 40])
def test_linear_weights_written_by_the_kernel_before(lib, M):
    """A call may begin before its predecessor in the stream ends; it reads weights and tokens only after that."""
    g = gen(M)
    K, N = 2048, 2304
    x = randn(g, M, K).to(BF16)
    w = torch.zeros((N, K), dtype=BF16, device="cuda")
    lin, new = ops.Linear(w, out_dtype=F32), [randn(g, N, K).to(BF16) for _ in range(6)]
    want = [x.double() @ n.double().T for n in new]
    got = []
    for n in new:
        w.copy_(n)
        got.append(lin(x))
    for a, b in zip(got, want):
        assert float((a.double() - b).norm()) <= 1.6e-6 * float(b.norm())
    # and tokens written by a product itself
    up, down = ops.Linear(new[0][:K].contiguous()), ops.Linear(new[1][:K].contiguous())
    h = up(x)
    y = down(h)
    assert float((y.double() - h.double() @ new[1][:K].double().T).norm()) <= 2.0 ** -8 * float(y.double().norm())


@pytest.mark.parametrize("M", [1, 12, 40, 300])
@pytest.mark.parametrize("K", [4160, 4099])
def test_linear_float32_results_keep_their_precision(lib, M, K):
    """Tensor cores cut running sums off (by up to 2^-23 of them, half of that on average): 32 additions of 16 k of
    terms with random signs, whose partial sums grow with the root of their number, shrink a sum by 2^-24 * 32 * 2/3 = 1.3e-6 of what it
    is like. Nine such sums are added and the result is rounded: 2^-24 * (sqrt(9) + 1) at most. 4099 k in one sum: 1e-5."""
    g = gen(M + K)
    x, w = randn(g, M, K).to(BF16), randn(g, 700, K).to(BF16)
    want = x.double() @ w.double().T
    y = ops.Linear(w, out_dtype=F32)(x)
    assert float((y.double() - want).norm()) <= 1.6e-6 * float(want.norm())


def test_linear_is_reproducible_and_independent_of_other_rows(lib):
    g = gen(10)
    for M, K, N in ((1, 4096, 256), (24, 8192, 512), (500, 1024, 1000)):
        x, w = randn(g, M, K).to(BF16), (randn(g, N, K) * 0.05).to(BF16)
        lin = ops.Linear(w, out_dtype=F32)
        y = lin(x).clone()
        for _ in range(3):
            assert torch.equal(lin(x), y)


# ------------------------------------------------------------------------------------------------ log probabilities
def logprob_oracle(logits, targets, n):
    l = logits.double()
    dead = torch.isnan(l).any(1) | torch.isposinf(l).any(1) | torch.isneginf(l).all(1)
    safe = torch.where(dead[:, None], torch.zeros_like(l), l)
    m = safe.amax(1, keepdim=True)
    z = torch.exp(safe - m)
    lse = m[:, 0] + torch.log(z.sum(1))
    p = z / z.sum(1, keepdim=True)
    nan = torch.full_like(lse, float("nan"))
    ent = torch.where(dead, nan, -torch.xlogy(p, p).sum(1))
    V = l.shape[1]
    at = torch.gather(safe, 1, targets.clamp(0, V - 1)[:, None])[:, 0] - lse
    logp = torch.where(targets < 0, torch.zeros_like(lse), torch.where(dead | (targets >= V), nan, at))
    best, ids = torch.sort(safe, dim=1, descending=True, stable=True)
    best, ids = best[:, :n], ids[:, :n]
    none = dead[:, None] | torch.isneginf(best)
    return logp, ent, torch.where(none, -1, ids).int(), torch.where(dead[:, None], nan[:, None], best - lse[:, None])


def check_logprobs(logits, targets, n, out=None):
    got = ops.token_logprobs(logits, targets, n, out=out)
    want = logprob_oracle(logits, targets, n)
    assert torch.equal(got[2], want[2])
    finite = logits.double()[torch.isfinite(logits)]
    span = min(float(finite.abs().max()) if finite.numel() else 0.0, 1e4)
    # A term's exponent is off by two half steps of the logits' size, the exponential by four steps: each term and so the sum by
    # (span * 2^-23 + 2^-21) relative, the logarithm by as much absolutely; the result is rounded once. The entropy weighs the
    # terms by their own logarithm (at most ln V below the maximum counts, 20 is generous).
    off = span * 2.0 ** -23 + 2.0 ** -21
    for i, scale in ((0, 1.0), (1, 40.0), (3, 1.0)):
        a, b = got[i].double(), want[i]
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(b)
        assert bool(((a - b).abs()[ok] <= off * scale + half_step(F32) * b.abs()[ok]).all()), (i, float((a - b).abs()[ok].max()))
    return got


@pytest.mark.parametrize("T,V,dtype,n", [(1, 1, F32, 1), (1, 5, BF16, 5), (2, 33, F16, 32), (3, 1000, F32, 20), (5, 4099, BF16, 5),
                                         (1, 131072, F32, 20), (1, 50001, BF16, 1), (4, 65537, F16, 7), (40, 30011, BF16, 20),
                                         (160, 32768, BF16, 5), (700, 2000, F32, 3), (301, 16385, F32, 0), (9, 131072, BF16, 32)])
def test_logprobs_sizes(lib, T, V, dtype, n):
    g = gen(T + V)
    logits = (3 * randn(g, T, V)).to(dtype)
    targets = torch.randint(0, V, (T,), generator=g, device="cuda")
    targets[0] = 0
    targets[-1] = V - 1
    check_logprobs(logits, targets, n)


@pytest.mark.parametrize("V", [7, 900, 5000, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_logprobs_masks_and_rows_without_a_distribution(lib, V, dtype):
    g = gen(V)
    n = min(V, 12)
    logits = (2 * randn(g, 14, V)).to(dtype)
    low = torch.finfo(dtype).min
    logits[0] = -INF
    logits[1, 1:] = -INF
    logits[2, torch.rand(V, generator=g, device="cuda") < 0.97] = -INF
    logits[3, torch.rand(V, generator=g, device="cuda") < 0.97] = low
    logits[4] = low
    logits[5, V // 2] = float("nan")
    logits[6, V // 3] = INF
    logits[7] = 0.0                                   # all equal
    logits[8] = torch.arange(V, device="cuda").to(dtype) / 64  # ascending: every value is a new best
    logits[9, V - 1] = 50.0
    logits[10, :-1] = -INF
    logits[10, -1] = float("nan")
    logits[11] = torch.finfo(dtype).max
    targets = torch.randint(0, V, (14,), generator=g, device="cuda")
    targets[1], targets[9], targets[12], targets[13] = min(1, V - 1), V - 1, -100, V
    check_logprobs(logits, targets, n)


@pytest.mark.parametrize("T,V", [(1, 131072), (9, 40000), (200, 3000)])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 24, 25, 32])
def test_logprobs_every_number_of_alternatives(lib, T, V, n):
    g = gen(T + n)
    for order in ("random", "ascending", "descending", "equal"):
        logits = 3 * randn(g, T, V)
        if order in ("ascending", "descending"):  # lists that overflow; the best of one part of the row alone
            logits = logits.sort(1, descending=order == "descending").values.contiguous()
        elif order == "equal":
            logits = logits.round()
        check_logprobs(logits.to(BF16), torch.randint(0, V, (T,), generator=g, device="cuda"), n)


@pytest.mark.parametrize("V", [5, 14, 33, 250, 5003, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_logprobs_lowest_values_as_alternatives(lib, V, dtype):
    """Fewer ordinary logits than alternatives: the lowest finite values take the remaining places, lower ids first, wherever the
    16-byte boundaries of a row lie."""
    g = gen(V)
    n = min(V, 20)
    for ordinary in (0, 1, n - 1):
        logits = torch.full((9, V), torch.finfo(dtype).min, device="cuda")
        for t in range(9):
            logits[t, torch.randperm(V, generator=g, device="cuda")[:ordinary]] = randn(g, ordinary)
        logits[4:, ::3] = -INF
        check_logprobs(logits.to(dtype), torch.zeros(9, dtype=torch.long, device="cuda"), n)


def test_logprobs_strided_rows_off_boundaries(lib):
    g = gen(4)
    wide = 2 * randn(g, 11, 9100)
    targets = torch.randint(0, 9000, (11,), generator=g, device="cuda")
    for dtype in (F32, BF16, F16):
        buf = wide.to(dtype)
        for first in (0, 1, 3, 8):
            check_logprobs(buf[:, first:first + 9000], targets, 6)
        check_logprobs(buf.reshape(-1)[5:5 + 11 * 9001].view(11, 9001)[:, 1:], targets, 6)
    got = ops.token_logprobs(wide[:0], targets[:0], 3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_logprobs_rows_far_beyond_32_bits(lib):
    """A row whose first element lies more than 2^31 elements into the buffer."""
    V = 65536
    rows = (1 << 31) // V + 3
    logits = torch.zeros((rows, V), dtype=BF16, device="cuda")
    g = gen(5)
    logits[-2:] = randn(g, 2, V).to(BF16)
    targets = torch.full((rows,), 17, dtype=torch.int64, device="cuda")
    got = ops.token_logprobs(logits, targets, 2)
    want = logprob_oracle(logits[-2:], targets[-2:], 2)
    assert torch.equal(got[2][-2:], want[2])
    assert bool(((got[0][-2:].double() - want[0]).abs() < 1e-5).all())
    assert bool(((got[0][:-2] + math.log(V)).abs() < 1e-5).all()) and got[2][:-2].unique(dim=0).tolist() == [[0, 1]]


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def build_run(seed, T=37, H=256, E=64, V=3001):
    g = gen(seed)
    x = randn(g, T, H).to(BF16)
    gate = ops.Linear((randn(g, E, H) * 0.1).to(BF16), out_dtype=F32)
    router = ops.Router(E, 6, scoring="sigmoid", bias=0.05 * randn(g, E), n_group=8, topk_group=3, group_score="top2",
                        norm_topk=True, routed_scale=2.5)
    up = ops.Linear((randn(g, 512, H) * 0.06).to(BF16), randn(g, 512).to(BF16), "silu")
    down = ops.Linear((randn(g, H, 512) * 0.06).to(BF16))
    head = ops.Linear((randn(g, V, H) * 0.1).to(BF16), out_dtype=F32)
    targets = torch.randint(0, V, (T,), generator=g, device="cuda")
    return x, gate, router, up, down, head, targets


def forward(x, gate, router, up, down, head, targets):
    ids, w = router(gate(x))
    y = down(up(x), residual=x)
    return ids, w, y, *ops.token_logprobs(head(y), targets, 4)


def test_a_run_of_them_together(lib):
    x, gate, router, up, down, head, targets = parts = build_run(1)
    ids, w, y, logp, ent, top, top_logp = forward(*parts)
    logits = gate(x)
    ref_ids, ref_w = route_oracle(logits, 6, "sigmoid", router.bias, 8, 3, "top2", True, 2.5)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    np.testing.assert_allclose(w.cpu().numpy(), ref_w, rtol=1.2e-5)
    ref_logits = x.double() @ gate.weight.double().T
    assert float((logits.double() - ref_logits).norm() / ref_logits.norm()) < 1e-6
    h = (lambda v: v * torch.sigmoid(v))(x.double() @ up.weight.double().T + up.bias.double())
    ref_y = h @ down.weight.double().T + x.double()
    assert float((y.double() - ref_y).norm() / ref_y.norm()) < 2 * half_step(BF16)
    want = logprob_oracle((y.double() @ head.weight.double().T), targets, 4)
    assert float((logp.double() - want[0]).abs().max()) < 1e-4 and float((ent.double() - want[1]).abs().max()) < 1e-4
    # the experts' products on the router's choice
    assert bool((ids >= 0).all()) and float((w.sum(1) - 2.5).abs().max()) < 1e-5


def test_captured_and_replayed_beside_an_eager_run(lib):
    parts, other = build_run(2), build_run(3, T=5)
    want, want_other = forward(*parts), forward(*other)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        forward(*parts)
    torch.cuda.current_stream().wait_stream(s)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = forward(*parts)
    with torch.cuda.graph(second):
        got_other = forward(*other)
    x = parts[0]
    keep = x.clone()
    for _ in range(3):
        graph.replay()
        second.replay()
        eager = forward(*other)
    torch.cuda.synchronize()
    for a, b in list(zip(got, want)) + list(zip(got_other, want_other)) + list(zip(eager, want_other)):
        assert torch.equal(a, b)
    x.copy_(torch.flip(keep, [0]))  # new inputs in the captured buffers
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(torch.flip(a, [0]), b)


FIRST_CALLS = """
import torch
from promoe_b200 import ops
torch.manual_seed(0)
rand = lambda *s: torch.randn(s, device="cuda")
l, b = rand(40, 64), rand(64)
w, wo = rand(300, 128).bfloat16(), rand(300, 77).bfloat16()
x, few, xo, v, t = rand(40, 128).bfloat16(), rand(3, 128).bfloat16(), rand(40, 77).bfloat16(), rand(2, 50000), torch.tensor([3, 4], device="cuda")
many = rand(600, 128).bfloat16()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = ops.Router(64, 6, "sigmoid", b, 8, 3, "top2")(l)
    y = [ops.Linear(w, out_dtype=torch.float32)(x), ops.Linear(w)(few), ops.Linear(wo)(xo), ops.Linear(w)(many)]
    p = ops.token_logprobs(v, t, 5)
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
assert torch.equal(r[0], ops.Router(64, 6, "sigmoid", b, 8, 3, "top2")(l)[0])
for have, rows, weight in zip(y, (x, few, xo, many), (w, w, wo, w)):
    want = rows.double() @ weight.double().T
    assert float((have.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
assert float((p[0].double() - torch.log_softmax(v.double(), -1)[torch.arange(2), t.cpu()]).abs().max()) < 1e-5
"""


def test_first_call_of_a_process_inside_a_capture(lib):
    root = Path(__file__).resolve().parent.parent
    subprocess.run([sys.executable, "-c", FIRST_CALLS], check=True, timeout=300, cwd=root)


def test_two_threads_on_two_streams(lib):
    import threading
    runs = [build_run(4), build_run(5, T=200)]
    want = [forward(*r) for r in runs]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        s = torch.cuda.Stream()
        try:
            with torch.cuda.stream(s):
                for _ in range(50):
                    got = forward(*runs[i])
            s.synchronize()
            for a, b in zip(got, want[i]):
                assert torch.equal(a, b)
        except Exception as e:  # noqa: BLE001 - reported by the test's thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


def test_calls_that_are_refused(lib):
    x, gate, router, up, down, head, targets = build_run(6, T=3)
    bad = [lambda: gate(x[:, :-1]), lambda: gate(x.float()), lambda: gate(x.cpu()), lambda: gate(x.T.contiguous().T),
           lambda: gate(x, residual=x), lambda: down(up(x), residual=x.float()), lambda: down(up(x), residual=x[:2]),
           lambda: gate(x[:1].expand(3, -1)), lambda: gate(x, out=torch.empty((3, 63), device="cuda")),
           lambda: up(x, out=torch.empty((1, 512), dtype=BF16, device="cuda").expand(3, -1)),
           lambda: gate(x.detach().requires_grad_()), lambda: ops.Linear(x, activation="tanh"), lambda: ops.Linear(x.float()),
           lambda: ops.Linear(x, out_dtype=F16), lambda: ops.Linear(x, bias=torch.zeros(4, device="cuda")),
           lambda: ops.Linear(x, bias=torch.zeros(3)),
           lambda: router(torch.zeros((3, 63), device="cuda")), lambda: router(torch.zeros((3, 64))),
           lambda: router(torch.zeros((3, 64), dtype=torch.float64, device="cuda")),
           lambda: router(torch.zeros((3, 64), device="cuda"), out=(torch.zeros((3, 6), device="cuda"),) * 2),
           lambda: ops.token_logprobs(head(x), targets.int(), 1), lambda: ops.token_logprobs(head(x), targets[:2], 1),
           lambda: ops.token_logprobs(head(x), targets.cpu(), 1),
           lambda: ops.token_logprobs(head(x), targets, 1, out=(torch.empty(2, device="cuda"), None, None, None)),
           lambda: ops.token_logprobs(head(x), targets, 1, out=(torch.empty(3, device="cuda"), None, None, None)),
           lambda: ops.token_logprobs(head(x), targets, -1),
           lambda: router(torch.zeros((3, 64), device="cuda"), out=(None, None)),
           lambda: router(torch.zeros((3, 64), device="cuda"), out=(torch.zeros((3, 6), dtype=torch.int32), torch.zeros((3, 6), device="cuda"))),
           lambda: ops.token_logprobs(torch.empty(1, device="cuda").expand(2 ** 32 + 1, 1), targets, 0)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(_lib.PromoeError):
        ops.token_logprobs(head(x), targets, 33)
