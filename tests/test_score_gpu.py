"""Scored texts leave no trace in what is generated later (GPU)."""
import pytest

from test_engine_codes_gpu import _llm, _prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_dtype", ["", "int8"])
def test_requests_without_a_seed_sample_the_same_after_scoring(model_dirs, cache_dtype):
    from kestrel_llm_b200 import SamplingParams
    prompts = _prompts("B", (9, 33, 20))
    sampled = SamplingParams(temperature=1.0, max_tokens=16, ignore_eos=True)
    outs = []
    for texts in ([], prompts, prompts * 3):
        llm = _llm(model_dirs, "B", "float32", cache_dtype=cache_dtype)
        outs.append([])
        for _ in range(2):
            if texts:
                llm.score(texts)
            got = llm.generate(prompts, sampled)
            outs[-1].append([(o.request_id, o.token_ids) for o in got])
    assert outs[0] == outs[1] == outs[2]
    assert outs[0][0] != outs[0][1]                 # requests of other numbers have other seeds


def test_a_score_that_fails_gives_its_requests_back(model_dirs):
    llm = _llm(model_dirs, "B", "float32", max_tokens=64, max_model_len=128)
    good = _prompts("B", (40,))
    want = llm.score(good)
    with pytest.raises(Exception):
        llm.score([good[0], _prompts("B", (100,))[0]])          # no pages for the second
    assert llm.engine.cache.live_requests() == 0
    llm.engine.cache.check()
    assert llm.score(good) == want
