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


@pytest.mark.parametrize("head_dim,takes", [(16, True), (256, True), (264, False), (272, False), (512, False)])
def test_layers_whose_heads_the_operators_refuse_take_no_codes(head_dim, takes):
    import torch
    from kestrel_llm_b200.cache.manager import CacheError, CacheManager
    from kestrel_llm_b200.parts import GroupedQueryAttention
    spec = GroupedQueryAttention(64, 4, 2, head_dim, torch.float32, "cpu", "a.", None, None).cache_spec()
    assert spec.codes == takes
    if takes:
        CacheManager([spec], torch.float32, "cpu", 16, 2, 1, 64, codes=True)
    else:
        with pytest.raises(CacheError, match="layer 0"):
            CacheManager([spec], torch.float32, "cpu", 16, 2, 1, 64, codes=True)
