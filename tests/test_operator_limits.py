"""Limits of the operators' sizes, without a GPU."""
import pytest

from promoe_b200 import _lib
from tests.test_operators_refusals import logprobs


@pytest.mark.parametrize("vocab", [0x7fff0001, 0x7fffffff])
def test_rows_whose_end_lies_too_near_the_end_of_32_bits(lib, vocab):
    with pytest.raises(_lib.PromoeError) as e:
        logprobs(vocab=vocab, ld=vocab, rows=0)
    assert e.value.code == 1
    logprobs(vocab=0x7fff0000, ld=0x7fff0000, rows=0)
