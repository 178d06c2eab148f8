"""Log probabilities, entropy and likeliest tokens, against float64."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _want(x, ids, top):
    import torch
    x = x.double()
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    given = lp.gather(1, ids.long()[:, None])[:, 0]
    return given, h, order.int(), lp.gather(1, order)


def _check(x, ids, top):
    """A difference of two numbers up to M from the maximum is off by 2^-23 M at most, a log of a sum of exponentials by their relative
    errors (2^-21 each: a base-2 exponential within two units, the sums' 2^-24 a level) and its own: 2^-20 + 2^-22 M in all.  The
    entropy's sum weighs the same distances by their probabilities: 2^-20 (1 + H) + 2^-19."""
    import torch
    from kestrel_llm_b200.csrc import ops
    got = ops.token_logprobs(x, ids, top)
    lp, h, order, tlp = _want(x, ids, top)
    for a, b in ((got.logprobs, lp), (got.top_logprobs, tlp)):
        inf = torch.isinf(b)
        assert torch.equal(torch.isinf(a) & (a < 0), inf)
        assert ((a.double() - b).abs()[~inf] <= (2.0 ** -20 + 2.0 ** -22 * b.abs())[~inf]).all()
    assert ((got.entropy.double() - h).abs() <= 2.0 ** -19 + 2.0 ** -20 * (1 + h)).all()
    assert torch.equal(got.top_ids, order)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 33), (3, 40), (2, 1000), (1, 8191), (2, 32768), (1, 151936), (7, 50257), (40, 32001), (300, 2051), (700, 3001)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_against_float64(rows, vocab, top):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = 3 * torch.randn((rows, vocab), generator=gen, device="cuda")
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    _check(x, ids, min(top, vocab))


@pytest.mark.parametrize("rows", [1, 5, 200])
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "masked", "few", "peaked", "steps", "shifted", "lowest"])
def test_hard_rows(rows, shape):
    import torch
    vocab, top = 9001, 20
    gen = torch.Generator(device="cuda").manual_seed(rows)
    i = torch.arange(vocab, device="cuda").float()
    x = torch.randn((rows, vocab), generator=gen, device="cuda")
    if shape == "equal":
        x = torch.full_like(x, -2.5)
    elif shape == "rising":
        x = (i / 1000).repeat(rows, 1)
    elif shape == "falling":
        x = (-i / 1000).repeat(rows, 1)
    elif shape == "masked":
        x[torch.rand(x.shape, generator=gen, device="cuda") < 0.99] = -math.inf
    elif shape == "few":                            # fewer tokens than are asked for
        keep = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        keep[[0, 4500, 9000]] = True
        x[:, ~keep] = -math.inf
    elif shape == "peaked":
        x[:, 77] = 90.0
    elif shape == "steps":                          # many ties, zeros of both signs
        x = torch.round(x * 2) / 2
        x[:, ::3] *= -1
    elif shape == "shifted":
        x = x + 1000.0
    else:                                           # masked by the type's lowest number
        x[torch.rand(x.shape, generator=gen, device="cuda") < 0.9] = torch.finfo(torch.float32).min
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if shape == "shifted":
        # a logit of 1,000 has steps of 2^-14: the rows' own numbers are what they are, differences are exact
        pass
    _check(x.contiguous(), ids, top)


def test_rows_further_apart_and_off_the_boundary():
    import torch
    big = torch.randn((6, 5003), device="cuda")
    for cut in (big[:, 1:4998], big[:, 3:], big[::2, 2:1003]):
        ids = torch.randint(0, cut.shape[1], (cut.shape[0],), device="cuda", dtype=torch.int32)
        _check(cut, ids, 7)


def test_rows_without_a_distribution():
    import torch
    from kestrel_llm_b200.csrc import ops
    x = torch.randn((5, 4000), device="cuda")
    x[1] = -math.inf
    x[2, 100] = float("nan")
    x[3, 200] = math.inf
    got = ops.token_logprobs(x, torch.tensor([3, 3, 3, 3, 3], dtype=torch.int32, device="cuda"), 4)
    bad = torch.tensor([False, True, True, True, False], device="cuda")
    assert torch.equal(torch.isnan(got.logprobs), bad) and torch.equal(torch.isnan(got.entropy), bad)
    assert torch.isnan(got.top_logprobs[bad]).all() and torch.isfinite(got.top_logprobs[~bad]).all()
    assert got.top_ids[1].tolist() == [0, 1, 2, 3] and int(got.top_ids[3, 0]) == 200
    assert ((got.top_ids >= 0) & (got.top_ids < 4000)).all()


def test_tokens_outside_the_vocabulary_and_no_tokens():
    import torch
    from kestrel_llm_b200.csrc import ops
    x = torch.randn((4, 3000), device="cuda")
    ids = torch.tensor([-1, 3000, 5, 2999], dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, ids)
    assert torch.isnan(got.logprobs).tolist() == [True, True, False, False] and got.top_ids.shape == (4, 0)
    none = ops.token_logprobs(x, None, 3)
    assert none.logprobs is None and torch.equal(none.entropy, got.entropy)
    one = ops.token_logprobs(x[2].clone()[:, None].t(), ids[2:3], 3)         # a row alone may have any stride
    assert torch.equal(one.logprobs, got.logprobs[2:3]) and torch.equal(one.top_ids, none.top_ids[2:3])
    empty = ops.token_logprobs(x[:0], ids[:0], 3)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_replay_with_other_rows():
    import torch
    from kestrel_llm_b200.csrc import ops
    x = torch.randn((3, 151936), device="cuda")
    ids = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    ops.token_logprobs(x, ids, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, ids, 5)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        now = ops.token_logprobs(x, ids, 5)
        for a, b in zip(got, now):
            assert torch.equal(a, b)


def test_refusals():
    import torch
    from kestrel_llm_b200.csrc import ops
    x = torch.randn((2, 100), device="cuda")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    for a in ((x.half(), ids, 1), (x.cpu(), ids, 1), (x[0], ids, 1), (x.t(), ids, 1), (x, ids.long(), 1), (x, ids[:1], 1), (x, ids.cpu(), 1),
              (x, ids, 33), (x, ids, -1), (x[:, :3], ids, 4), (x[:, :0], ids, 0)):
        with pytest.raises(ops.KernelError):
            ops.token_logprobs(*a)
