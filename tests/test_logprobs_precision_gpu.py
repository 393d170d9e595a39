"""Log probabilities at the edges of their arithmetic: rows far from zero, rows of one token, maxima of every size."""
import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import BF16, F16, F32, INF, gen, half_step, logprob_oracle, randn

pytestmark = pytest.mark.gpu


def tolerance(V, size):
    """Of a log probability `size`: an exponential is off by 2^-22 of itself and by what half a step of its argument (at most log2 V
    counts) and the float32 log2 e (1.4e-8 of the same) make of it; a thread adds at most V / 512 + 32 terms one after another, half a
    step each; the logarithm and the result are rounded once each."""
    return 2.0 ** -22 + V.bit_length() * (2.0 ** -24 + 1.4e-8) + (V / 512 + 32) * 2.0 ** -24 + 2 * half_step(F32) * (1 + size)


@pytest.mark.parametrize("V", [33, 4099, 131072])
@pytest.mark.parametrize("n", [0, 3])
def test_a_common_offset_changes_nothing(lib, V, n):
    """l - max - log sum has no term that grows with the maximum."""
    g = gen(V + n)
    base = 3 * randn(g, 4, V)
    targets = torch.randint(0, V, (4,), generator=g, device="cuda")
    for offset in (0.0, 100.0, 1000.0, 30000.0, -1000.0, -30000.0):
        logits = base + offset  # rounded to float32: these are the logits
        got, want = ops.token_logprobs(logits, targets, n), logprob_oracle(logits, targets, n)
        assert torch.equal(got[2], want[2])
        for i in (0, 3):
            assert bool(((got[i].double() - want[i]).abs() <= tolerance(V, want[i].abs())).all()), (offset, i)
        assert bool(((got[1].double() - want[1]).abs() <= 20 * tolerance(V, want[1].abs())).all()), offset


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 9, 5000, 131072])
def test_one_allowed_token_is_certain(lib, V, dtype):
    """Its log probability is 0: one exponential, off by 2^-22, and one logarithm of about 1."""
    levels = [20.0, 50.0, 100.0, 1000.0, 60000.0, -50.0, -1000.0]
    logits = torch.full((len(levels), V), -INF, dtype=dtype, device="cuda")
    logits[:, V // 2] = torch.tensor(levels, device="cuda").to(dtype)
    targets = torch.full((len(levels),), V // 2, dtype=torch.int64, device="cuda")
    logp, entropy, ids, best = ops.token_logprobs(logits, targets, 1)
    assert ids.flatten().tolist() == [V // 2] * len(levels)
    for r in (logp, entropy, best):
        assert float(r.abs().max()) <= 2.0 ** -21, r.tolist()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [9, 5000, 131072])
@pytest.mark.parametrize("rest", [0.0, -INF])
def test_one_logit_far_above_the_others(lib, V, dtype, rest):
    """Certain, whatever its size: log probability and entropy 0."""
    levels = torch.tensor([9e7, 1.1e8, 2e9, 1e10, 3e15, 1e20, 1e33, 1e34, 1e35, 9e36, 1.1e37, 3e38], device="cuda").to(dtype)
    logits = torch.full((len(levels), V), rest, dtype=dtype, device="cuda")
    logits[:, V - 2] = levels
    targets = torch.full((len(levels),), V - 2, dtype=torch.int64, device="cuda")
    logp, entropy, ids, best = ops.token_logprobs(logits, targets, 2)
    assert ids[:, 0].tolist() == [V - 2] * len(levels)
    for r in (logp, entropy, best[:, 0]):
        assert float(r.abs().max()) <= 2.0 ** -21, r.tolist()


@pytest.mark.parametrize("V", [33, 4099, 131072])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_large_logits_a_few_steps_apart(lib, V, sign):
    """Rows around a size at which neighbouring float32 numbers differ by 1/16 to thousands."""
    g = gen(V)
    sizes = [1e6, 9e6, 9e7, 1.1e8, 5e8, 2e9, 1e10, 1e12, 1e18, 1e19, 1e25]
    logits = torch.stack([sign * (s + float(2.0 ** -23 * 2.0 ** int(torch.tensor(s).log2().floor())) *
                                  torch.randint(0, 3, (V,), generator=g, device="cuda").float()) for s in sizes])
    targets = torch.randint(0, V, (len(sizes),), generator=g, device="cuda")
    got, want = ops.token_logprobs(logits, targets, 4), logprob_oracle(logits, targets, 4)
    assert torch.equal(got[2], want[2])
    for i in (0, 3):
        assert bool(((got[i].double() - want[i]).abs() <= tolerance(V, want[i].abs())).all()), i
    assert bool(((got[1].double() - want[1]).abs() <= 20 * tolerance(V, want[1].abs())).all())


@pytest.mark.parametrize("V", [700, 5000, 131072])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-1e9, -1e12, -1e17, -1e19, -3e38])
def test_ordinary_logits_among_very_low_ones(lib, V, dtype, low):
    """Threads that meet the low ones first, wherever the ordinary ones lie."""
    g = gen(V)
    logits = low * (1 + 0.01 * torch.rand(6, V, generator=g, device="cuda"))
    logits[0, -1] = 1.0
    logits[1, :V // 2] = randn(g, V // 2)
    logits[2, V // 2:] = randn(g, V - V // 2)
    logits[3, ::3] = -65504.0
    logits[4, torch.randperm(V, generator=g, device="cuda")[:V // 50]] = randn(g, V // 50)
    logits[5, 1] = -2.0
    logits[5, V - 2] = 3.0
    logits = logits.clamp(min=torch.finfo(dtype).min).to(dtype)
    targets = torch.tensor([V - 1, 0, V - 1, 3, 0, 1], device="cuda")
    got, want = ops.token_logprobs(logits, targets, 3), logprob_oracle(logits, targets, 3)
    assert torch.equal(got[2], want[2])
    for i in (0, 3):
        ok = want[i] > -3e38
        assert bool(((got[i].double() - want[i]).abs()[ok] <= tolerance(V, want[i].abs())[ok]).all()), i
    assert bool(((got[1].double() - want[1]).abs() <= 20 * tolerance(V, want[1].abs())).all())
