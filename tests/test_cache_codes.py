"""A cache of 8-bit codes: its planes and sizes, and what it refuses (host side)."""
import pytest


def test_planes_and_bytes_of_a_cache_of_codes():
    import torch
    from kestrel_llm_b200.cache.manager import CacheManager
    from kestrel_llm_b200.parts.base import FixedStateSpec, PagedKVSpec
    cm = CacheManager([PagedKVSpec(2, 64, codes=True), FixedStateSpec((5,)), PagedKVSpec(3, 32, 48, codes=True)], torch.bfloat16, "cpu", 32, 6, 2, 256, codes=True)
    assert cm.codes and [t is None for t in cm.k_scale] == [False, True, False] and cm.state[1].shape == (3, 5)
    for i, (heads, dim) in ((0, (2, 64)), (2, (3, 32))):
        lc = cm.layer(i)
        assert lc.k.dtype == lc.v.dtype == torch.int8 and lc.k.shape == lc.v.shape == (7, heads, 32, dim)
        assert lc.k_scale.dtype == lc.v_scale.dtype == torch.float32 and lc.k_scale.shape == lc.v_scale.shape == (7, heads, 2)
    # a code a number, and a float32 scale for every 16 tokens of a head, in both planes
    assert cm.bytes_per_token() == 2 * (2 * 64 + 2 * 4 / 16) + 2 * (3 * 32 + 3 * 4 / 16)
    plain = CacheManager([PagedKVSpec(2, 64, codes=True)], torch.bfloat16, "cpu", 32, 6, 2, 256)
    assert not plain.codes and plain.k_scale == [None] and plain.layer(0).k_scale is None and plain.k[0].dtype == torch.bfloat16
    assert plain.bytes_per_token() == 2 * 2 * 64 * 2


def test_layers_and_pages_that_hold_no_codes_are_refused():
    import torch
    from kestrel_llm_b200.cache.manager import CacheError, CacheManager
    from kestrel_llm_b200.parts.base import PagedKVSpec
    with pytest.raises(CacheError, match="layer 1"):
        CacheManager([PagedKVSpec(2, 64, codes=True), PagedKVSpec(2, 64)], torch.bfloat16, "cpu", 16, 6, 2, 256, codes=True)
    with pytest.raises(CacheError, match="whole blocks"):
        CacheManager([PagedKVSpec(2, 64, codes=True)], torch.bfloat16, "cpu", 8, 6, 2, 256, codes=True)


def test_options_say_what_a_cache_may_hold():
    from kestrel_llm_b200.config import EngineOptions
    assert not EngineOptions().cache_codes and EngineOptions(cache_dtype="int8").cache_codes
    with pytest.raises(ValueError):
        EngineOptions(cache_dtype="fp8").cache_codes


def test_the_number_of_reported_alternatives_is_bounded():
    from kestrel_llm_b200.sampling import SamplingParams
    assert SamplingParams().logprobs is None and SamplingParams(logprobs=0).logprobs == 0 and SamplingParams(logprobs=32).logprobs == 32
    for n in (-1, 33):
        with pytest.raises(ValueError):
            SamplingParams(logprobs=n)


def test_attention_layers_say_whether_they_take_codes():
    import torch
    from kestrel_llm_b200.parts import GroupedQueryAttention
    assert GroupedQueryAttention(64, 4, 2, 16, torch.float32, "cpu", "a.", None, None).cache_spec().codes
    assert not GroupedQueryAttention(64, 4, 2, 8, torch.float32, "cpu", "a.", None, None).cache_spec().codes
