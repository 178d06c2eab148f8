"""Generation from a cache of 8-bit codes, reported log probabilities, and scored texts (GPU)."""
import math

import numpy as np
import pytest

import plain_qwen3 as P
import replay_util as R
import tiny_configs
from q8_util import BLOCK

pytestmark = pytest.mark.gpu


def _prompts(name, lengths, seed=3):
    return list(R.random_requests(tiny_configs.CONFIGS[name][0]["vocab_size"], lengths, seed=seed).values())


def _llm(model_dirs, name, dtype, **kw):
    from kestrel_llm_b200 import LLM
    options = dict(page_size=16, batch_max=4, max_tokens=1024, prefill_batch=24, max_step_tokens=64, cache_dtype="int8")
    return LLM(model_dirs[name][dtype], dtype=dtype, **{**options, **kw})


@pytest.mark.parametrize("window", [0, 40])
def test_a_layer_over_codes_against_float64(window):
    """The layer's queries, and its outputs over the values that its cache holds: float32 products of 96 numbers and sums, 2^-14 of the
    largest output in all."""
    import torch
    from kestrel_llm_b200.cache.manager import CacheManager
    from kestrel_llm_b200.engine import Entry, StepBatch
    from kestrel_llm_b200.parts import GroupedQueryAttention, RotaryHalf
    from q8_util import prepared64
    torch.manual_seed(5)
    W, H, G, D = 96, 6, 2, 32
    rot = RotaryHalf(D, 10000.0, "cuda:0")
    layer = GroupedQueryAttention(W, H, G, D, torch.float32, "cuda:0", "a.", rot, 1e-6, window=window)
    for slot in layer.weight_slots():
        slot.dest.normal_(1.0 if slot.init == "norm" else 0.0, 0.2)
    cache = CacheManager([layer.cache_spec()], torch.float32, "cuda:0", 32, 12, 2, 256, codes=True)
    cache.shuffle_free(2)
    lengths = [0, 0]
    for portions in ([(0, 50), (1, 7)], [(1, 20)], [(0, 1), (1, 1)], [(0, 1), (1, 30)]):
        entries = []
        for r, n in portions:
            if not cache.is_live(r):
                cache.admit(r)
            cache.reserve(r, n)
            entries.append(Entry(r, [1] * n))
        batch = StepBatch(entries, cache, "cuda:0")
        x = torch.randn(batch.num_tokens, W, device="cuda:0")
        got = layer.forward(x, batch, cache.layer(0)).reduce(torch.float32).double()
        w = layer.qkv.weight.double()
        q, _, _ = prepared64((x.double() @ w.T)[None], None, layer.q_norm, layer.k_norm, 1e-6, rot.rotary().inv_freq, D, batch.positions, H, G, D, False)
        want = torch.empty((batch.num_tokens, H, D), dtype=torch.float64, device="cuda:0")
        t = 0
        for r, n in portions:
            c = lengths[r]
            table = torch.tensor(cache.block_table(r, 0), device="cuda:0")
            pos = torch.arange(c + n, device="cuda:0")
            page, slot = table[pos // 32], pos % 32
            for i in range(n):
                lo = max(0, c + i - window + 1) if window else 0
                see = slice(lo, c + i + 1)
                for h in range(H):
                    g = h // (H // G)
                    k = cache.k[0][page[see], g, slot[see]].double() * cache.k_scale[0][page[see], g, slot[see] // BLOCK].double()[:, None]
                    v = cache.v[0][page[see], g, slot[see]].double() * cache.v_scale[0][page[see], g, slot[see] // BLOCK].double()[:, None]
                    want[t + i, h] = torch.softmax(k @ q[t + i, h] / math.sqrt(D), 0) @ v
            t += n
            lengths[r] += n
        want = want.reshape(batch.num_tokens, -1) @ layer.out.weight.double().T
        assert (got - want).abs().max() <= 2.0 ** -14 * want.abs().max()
        for r, n in portions:
            cache.commit(r, n)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_of_the_runner_the_walk_and_graphs_give_the_same_tokens(model_dirs, dtype):
    """The same kernels three ways: the native program, the parts' forward, and captured decode steps."""
    from kestrel_llm_b200 import SamplingParams
    prompts = _prompts("B", (1, 33, 70, 129))
    outs = []
    for kw in (dict(), dict(native_step=False), dict(cuda_graphs=False)):
        llm = _llm(model_dirs, "B", dtype, **kw)
        assert llm.engine.cache.codes and (llm.engine.runner is None) == (kw.get("native_step") is False)
        outs.append([o.token_ids for o in llm.generate(prompts, SamplingParams(max_tokens=20, ignore_eos=True))])
        assert llm.engine.cache.live_requests() == 0
    assert outs[0] == outs[1] == outs[2]


def test_codes_cost_little_of_the_scores(model_dirs):
    """What scoring from codes is for: the mean log probability of texts under both caches.  Both are proper distributions' and lie nearer to
    each other than a uniform guess lies to certainty."""
    vocab = tiny_configs.B["vocab_size"]
    texts = _prompts("B", (40, 7, 100))
    mean = []
    for cache_dtype in ("", "int8"):
        llm = _llm(model_dirs, "B", "float32", cache_dtype=cache_dtype)
        scores = llm.score(texts, top=2)
        assert [len(s) for s in scores] == [len(t) - 1 for t in texts] and llm.engine.cache.live_requests() == 0
        flat = [x for s in scores for x in s]
        assert all(math.isfinite(x.logprob) and 0 <= x.entropy <= math.log(vocab) + 1e-4 and len(x.top) == 2 for x in flat)
        mean.append(np.mean([x.logprob for x in flat]))
    assert abs(mean[0] - mean[1]) < math.log(vocab)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_reported_log_probabilities(model_dirs, dtype):
    """Of the tokens that were generated, beside requests that ask for none, against the plain implementation's logits: a log probability is
    off by at most twice what a logit is."""
    from kestrel_llm_b200 import SamplingParams
    prompts = _prompts("B", (9, 33, 20))
    params = [SamplingParams(max_tokens=10, ignore_eos=True, logprobs=n) for n in (3, None, 0)]
    llm = _llm(model_dirs, "B", dtype, cache_dtype="")
    plain = llm.generate(prompts, SamplingParams(max_tokens=10, ignore_eos=True))
    outs = llm.generate(prompts, params)
    assert [o.token_ids for o in outs] == [o.token_ids for o in plain]
    assert plain[0].logprobs is None and outs[1].logprobs is None
    cfg, W = P.read_model(model_dirs["B"]["float32"])
    for i, n in ((0, 3), (2, 0)):
        assert [s.token_id for s in outs[i].logprobs] == outs[i].token_ids
        toks = list(prompts[i])
        for s in outs[i].logprobs:
            logits = P.forward_logits(cfg, W, toks)[-1].astype(np.float64)
            off = 2 * R.TOL[dtype] * np.abs(logits).max() + 2.0 ** -18
            lp = logits - logits.max() - np.log(np.exp(logits - logits.max()).sum())
            assert abs(s.logprob - lp[s.token_id]) <= off
            assert len(s.top) == n and all(abs(v - lp[t]) <= off for t, v in s.top)
            assert [v for _, v in s.top] == sorted((v for _, v in s.top), reverse=True)
            toks.append(s.token_id)


def test_scores_of_a_text_are_those_of_its_generation(model_dirs):
    from kestrel_llm_b200 import SamplingParams
    prompts = _prompts("B", (9, 33, 20, 50, 3))
    llm = _llm(model_dirs, "B", "float32", cache_dtype="")
    outs = llm.generate(prompts, SamplingParams(max_tokens=12, ignore_eos=True, logprobs=5))
    texts = [p + o.token_ids for p, o in zip(prompts, outs)]
    scores = llm.score(texts + [[5], []], top=5)
    assert scores[-1] == scores[-2] == []
    for p, o, s in zip(prompts, outs, scores):
        assert [x.token_id for x in s] == (p + o.token_ids)[1:]
        for a, b in zip(o.logprobs, s[len(p) - 1:]):
            # the two computed their logits in steps cut differently: each is off by R.TOL of the largest, which is below 50 here
            assert abs(a.logprob - b.logprob) <= 1e-3 and abs(a.entropy - b.entropy) <= 1e-3
    assert llm.engine.cache.live_requests() == 0
    llm.engine.cache.check()
    # and the engine goes on
    again = llm.generate(prompts, SamplingParams(max_tokens=12, ignore_eos=True))
    assert [o.token_ids for o in again] == [o.token_ids for o in outs]


def test_score_refuses(model_dirs):
    from kestrel_llm_b200 import SamplingParams
    llm = _llm(model_dirs, "B", "float32", cache_dtype="", max_model_len=64)
    for texts, top in (([[1, 10 ** 6]], 0), ([[1] * 65], 0), ([[1, 2]], 33), ([[1, 2]], -1)):
        with pytest.raises(ValueError):
            llm.score(texts, top)
    llm.add_request([1, 2, 3], SamplingParams(max_tokens=4))
    with pytest.raises(RuntimeError):
        llm.score([[1, 2]])
    llm.run_until_done()
    assert len(llm.score([[1, 2]])[0]) == 1

