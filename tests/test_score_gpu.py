"""Scored texts: no trace in what is generated later, and what a cache of 8-bit codes does to the scores (GPU)."""
import numpy as np
import pytest

import plain_qwen3 as P
import replay_util as R
from q8_util import BLOCK, LOWEST
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


def _coded(x, mistake=""):
    """x [T, heads, hd] as a cache of 8-bit codes gives it back where the T tokens came in one step: the definition, in 64 bits."""
    T, heads, hd = x.shape
    blocks = np.zeros((-(-T // BLOCK), BLOCK, heads, hd))
    blocks.reshape(-1, heads, hd)[:T] = x
    scale = np.maximum(np.abs(blocks).max((1, 3), keepdims=True) / 127, LOWEST)
    codes = np.rint(blocks / scale)
    if mistake == "scales of the next block":
        scale = np.roll(scale, 1, 0)
    if mistake == "nothing":
        codes = codes * 0
    if mistake == "heads exchanged":
        codes, scale = codes[:, :, ::-1], scale[:, :, ::-1]
    if mistake == "codes cut":
        codes = np.floor(blocks / scale)
    return (codes * scale).reshape(-1, heads, hd)[:T].astype(np.float32)


@pytest.mark.parametrize("name", ["B", "D", "E", "F"])
def test_scores_from_codes_are_those_of_the_definition(model_dirs, monkeypatch, name):
    """Every log probability of a text under the 8-bit cache, against a plain forward pass over keys and values coded by the definition.  The
    two passes compute in float32, so numbers differ by at most 1e-5 (twice R.TOL) of the largest in their block, 1.3e-3 steps of its scale.  A code
    flips where x / scale is that near to a half, 2.6e-3 of all codes, and moves by one step; coding itself moves every number by
    1 / sqrt(12) steps on average.  The flips' part of what coding does to a score is then sqrt(12 * 2.6e-3) = 0.18 of it at most on
    average: a quarter is allowed, and what the logits' own rounding gives.  Mistakes, planted in the plain pass, lie beyond that."""
    texts = [_prompts(name, (n,))[0] for n in (100, 41)]
    llm = _llm(model_dirs, name, "float32", prefill_batch=128, max_step_tokens=128)
    got = np.concatenate([[s.logprob for s in llm.score([t])[0]] for t in texts])
    cfg, W = P.read_model(model_dirs[name]["float32"])
    attention, rounding = P.causal_attention, 0.0

    def scores(mistake):
        nonlocal rounding
        out = []
        with monkeypatch.context() as m:
            if mistake is not None:
                m.setattr(P, "causal_attention", lambda q, k, v, window=0: attention(
                    q, _coded(k, "" if mistake == "nothing" else mistake), _coded(v, mistake), window))
            for t in texts:
                x = P.forward_logits(cfg, W, t[:-1]).astype(np.float64)
                rounding = max(rounding, 2 * R.TOL["float32"] * np.abs(x).max())
                x -= x.max(1, keepdims=True)
                out.append((x - np.log(np.exp(x).sum(1, keepdims=True)))[np.arange(len(t) - 1), t[1:]])
        return np.concatenate(out)

    def rms(x):
        return np.sqrt(np.mean(x * x))
    want = scores("")
    coding = rms(scores(None) - want)
    allowed = 0.25 * coding + rounding
    assert rms(got - want) <= allowed
    for mistake in ("scales of the next block", "nothing", "heads exchanged", "codes cut"):
        if mistake == "heads exchanged" and cfg["num_key_value_heads"] == 1:
            continue
        assert rms(got - scores(mistake)) > 2 * allowed, mistake


@pytest.mark.parametrize("name", ["D", "E", "F"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_runner_and_the_walk_cut_steps_alike(model_dirs, name, dtype):
    """Heads of 64 and 128, windows, more than sixteen query heads a kv head: both plan by the requests' own lengths, so their bits agree."""
    from kestrel_llm_b200 import SamplingParams
    prompts = _prompts(name, (1, 33, 70, 129))
    outs = []
    for native in (True, False):
        llm = _llm(model_dirs, name, dtype, cuda_graphs=False, native_step=native)
        assert llm.engine.cache.codes and (llm.engine.runner is not None) == native
        got = llm.generate(prompts, SamplingParams(max_tokens=20, ignore_eos=True, logprobs=2))
        outs.append([(o.token_ids, [(s.logprob, s.entropy, s.top) for s in o.logprobs]) for o in got])
    assert outs[0] == outs[1]
