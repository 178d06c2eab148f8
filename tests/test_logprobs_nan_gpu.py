"""The likeliest tokens of rows with logits that are no numbers."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(1, 33), (3, 4001), (2, 151936), (300, 2051)])
@pytest.mark.parametrize("shape", ["few", "many", "negative", "all", "all negative", "among minus infinity"])
def test_order_with_nan_as_minus_infinity(rows, vocab, shape):
    """Whichever threads and runs of 16 the NaN fall into, and whatever their sign."""
    import torch
    from kestrel_llm_b200.csrc import ops
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn((rows, vocab), generator=gen, device="cuda")
    nan = torch.full((), float("nan"), device="cuda")
    if "negative" in shape:
        nan = torch.full((), -4194304, dtype=torch.int32, device="cuda").view(torch.float32)      # 0xffc00000
    if shape == "among minus infinity":
        x[torch.rand(x.shape, generator=gen, device="cuda") < 0.999] = -math.inf
    share = {"few": 2 / vocab, "negative": 0.3, "all": 2.0, "all negative": 2.0}.get(shape, 0.5)
    hit = torch.rand(x.shape, generator=gen, device="cuda") < share
    hit[:, x[0].argmax()] = True                                   # a thread's largest number's neighbourhood
    x = torch.where(hit, nan, x)
    assert torch.isnan(x).any(1).all()
    top = min(20, vocab)
    got = ops.token_logprobs(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), top)
    want = torch.sort(torch.where(torch.isnan(x), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids, want.int())
    for t in (got.logprobs, got.entropy, got.top_logprobs):
        assert torch.isnan(t).all()
