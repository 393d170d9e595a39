"""What a row of a dense product depends on: its own values, the weights, and the sizes of the call."""
import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import BF16, F32, INF, gen, half_step, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", [(2, 4096, 256), (16, 1000, 300), (16, 77, 40), (24, 8192, 512), (64, 4096, 4096), (100, 99, 200),
                                   (500, 1024, 1000), (600, 192, 8192)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_other_rows_change_nothing(lib, M, K, N, out):
    g = gen(M + K)
    x, w = randn(g, M, K).to(BF16), (randn(g, N, K) * 0.05).to(BF16)
    res = randn(g, M, N).to(out)
    lin = ops.Linear(w, randn(g, N).to(BF16), "silu", out)
    y = lin(x, residual=res)
    keep = [0, M // 2, M - 1]
    for other in (0.0, 3.0, float("nan"), INF):
        z, r = torch.full_like(x, other), torch.full_like(res, other)
        z[keep], r[keep] = x[keep], res[keep]
        assert torch.equal(lin(z, residual=r)[keep], y[keep])


@pytest.mark.parametrize("K,N", [(4096, 256), (1000, 3000)])
def test_the_number_of_rows_changes_last_bits_at_most(lib, K, N):
    g = gen(K)
    x, w = randn(g, 600, K).to(BF16), (randn(g, N, K) * 0.05).to(BF16)
    lin = ops.Linear(w, out_dtype=F32)
    want = x[:1].double() @ w.double().T
    size = x[:1].double().abs() @ w.double().abs().T
    for M in (1, 9, 17, 64, 200, 600):
        # every order of summation: K additions, each off by at most a step of the sum of magnitudes
        assert bool(((lin(x[:M])[:1].double() - want).abs() <= (K + 1) * 2 * half_step(F32) * size).all())
