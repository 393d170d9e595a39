"""Dense products whose sizes pass 32 bits somewhere."""
import pytest
import torch

from promoe_b200 import ops
from tests.test_operators_gpu import BF16, F32, gen, randn

pytestmark = pytest.mark.gpu


def check_rows(x, w, y, rows):
    want = x[rows].double() @ w.double().T
    assert float((y[rows].double() - want).norm()) <= 2.0 ** -8 * float(want.norm())


@pytest.mark.parametrize("M,K,N", [(70_000_000, 8, 32), (33_000, 64, 65_600), (17, 40, 130_000_000), (40_000_000, 7, 56)])
def test_results_beyond_2_to_the_31_elements(lib, M, K, N):
    """Many tokens, many of both, many weight rows, rows off 16-byte boundaries; the first and last rows and columns, and those about the
    element 2^31."""
    g = gen(K)
    x, w = torch.empty((M, K), dtype=BF16, device="cuda").normal_(generator=g), torch.empty((N, K), dtype=BF16, device="cuda").normal_(generator=g)
    y = ops.Linear(w)(x)
    assert M * N > 1 << 31
    at = (1 << 31) // N
    rows = sorted({0, 1, M // 2, max(0, at - 1), min(M - 1, at), min(M - 1, at + 1), M - 2, M - 1})
    cols = slice(None) if N < 1 << 20 else torch.tensor([0, 1, N // 2, N - 2, N - 1, (1 << 31) % N], device="cuda")
    check_rows(x, w[cols], y[:, cols] if N >= 1 << 20 else y, torch.tensor(rows, device="cuda"))


def test_pitches_beyond_32_bits(lib):
    """Rows of a result that lie more than 2^31 elements apart."""
    g = gen(4)
    x, w = randn(g, 2, 64).to(BF16), randn(g, 40, 64).to(BF16)
    buffer = torch.empty((1 << 31) + 200, dtype=BF16, device="cuda")
    out = buffer.as_strided((2, 40), ((1 << 31) + 64, 1), 8)
    ops.Linear(w)(x, out=out)
    check_rows(x, w, out, slice(None))
