"""Options of reported log probabilities and of a cache of 8-bit codes that would fail late (host side)."""
import numpy as np
import pytest


@pytest.mark.parametrize("n", [5.5, 5.0, float("nan"), float("inf"), "5"])
def test_alternatives_are_a_whole_number(n):
    from kestrel_llm_b200.sampling import SamplingParams
    with pytest.raises(ValueError, match="whole number"):
        SamplingParams(logprobs=n)


def test_whole_numbers_of_any_type_are_alternatives():
    from kestrel_llm_b200.sampling import SamplingParams
    got = SamplingParams(logprobs=np.int64(5)).logprobs
    assert got == 5 and type(got) is int
