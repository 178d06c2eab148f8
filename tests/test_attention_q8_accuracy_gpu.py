"""How near attention over pages of 8-bit codes comes to 64 bits, over all outputs: what a loss of bits inside a kernel would show in first."""
import pytest

from q8_util import attend64, planes, step

pytestmark = pytest.mark.gpu

# single tokens in clusters and in stretches, a CTA a pair, portions, a portion beside single tokens
STEPS = [[(1, 500)] * 3, [(1, 9000)] * 5, [(1, 300)] * 64, [(130, 70), (1, 300)], [(300, 500)]]


def _errors(portions, nq, nkv, hd, dtype):
    import torch
    from kestrel_llm_b200.csrc import ops
    s = step(portions, 16)
    k, ks, v, vs = planes(s, nkv, hd)
    ks = ks.clamp(2.0 ** -7, 2.0 ** -6)             # scores of a few units
    gen = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn((s.num_tokens, nq * hd), generator=gen, device="cuda").to(getattr(torch, dtype))
    out = torch.full_like(q, float("nan"))
    ops.attention_q8(q, k, v, ks, vs, out, s, s.table, 16, nq, nkv, hd, 0, hd ** -0.5)
    ops.raise_on_kernel_error()
    want, _ = attend64(q, k, ks, v, vs, s, nq, nkv, hd, 0, hd ** -0.5)
    return out.view(want.shape).double() - want, want


@pytest.mark.parametrize("portions", STEPS)
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (8, 2, 64), (4, 1, 80)])
def test_float32_keeps_float32(portions, nq, nkv, hd):
    """A score is a sum of hd products, each of them, and each partial sum, off by 2^-23 at most of itself - two float16 parts of a query
    leave no more, nor does a sum that the matrix instructions cut off - and these errors are independent: 2^-23 / sqrt(3) of the products'
    root sum of squares for the parts, twice that for some ten partial sums, so 2^-22 of a score's size, which is below 4 nearly always: 2^-20
    of a weight.  Outputs average their keys' errors as they average their values, and add 2^-22 for weights' parts and sums: 2^-20 of the
    outputs' norm with room for both.  Operands of 16 bits would leave 2^-12."""
    error, want = _errors(portions, nq, nkv, hd, "float32")
    assert error.norm() <= 2.0 ** -20 * want.norm()


@pytest.mark.parametrize("portions", STEPS)
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (8, 2, 64), (4, 1, 80)])
def test_bfloat16_is_as_near_as_its_rounding(portions, nq, nkv, hd):
    """Weights in float16 are off by an eighth of what the output's rounding to bfloat16 is, and independently: sqrt(1 + 1 / 64) of the rounding
    alone, 1.008; scores in float32 and exponentials within 2^-21 add nothing to that."""
    error, want = _errors(portions, nq, nkv, hd, "bfloat16")
    assert error.norm() <= 1.02 * (want.bfloat16().double() - want).norm()
