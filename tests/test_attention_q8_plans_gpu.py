"""How a step of attention over pages of 8-bit codes is cut: by its requests' own lengths, and safely where these are not known."""
from types import SimpleNamespace

import pytest

from q8_util import attend64, planes, step
from test_attention_q8_gpu import _near

pytestmark = pytest.mark.gpu


def _inputs(s, nq, nkv, hd, dtype):
    import torch
    k, ks, v, vs = planes(s, nkv, hd)
    q = torch.randn((s.num_tokens, nq * hd), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(getattr(torch, dtype))
    return q, k, ks, v, vs


def _attend(s, nq, nkv, hd, q, k, ks, v, vs, out):
    """Kernels that the call launched."""
    from kestrel_llm_b200.csrc import ops
    before = ops.launches
    ops.attention_q8(q, k, v, ks, vs, out, s, s.table, s.page, nq, nkv, hd, 0, hd ** -0.5)
    return ops.launches - before


def _check(s, nq, nkv, hd, dtype, q, k, ks, v, vs, out):
    from kestrel_llm_b200.csrc import ops
    ops.raise_on_kernel_error()
    want, size = attend64(q, k, ks, v, vs, s, nq, nkv, hd, 0, hd ** -0.5)
    _near(s, out.view(s.num_tokens, nq, hd).double(), want, size, dtype)


@pytest.mark.parametrize("contexts,launches", [([16000] + [300] * 26, 2), ([300] * 26 + [16000], 2), ([4000] * 27, 1), ([16000] + [300] * 7, 2), ([1003], 1)])
def test_one_long_request_among_short_ones_is_shared_out(contexts, launches):
    """A cluster a pair (one kernel) would leave a long request to two CTAs while the others wait; stretches are two kernels."""
    import torch
    nq, nkv, hd = 32, 8, 128
    s = step([(1, c) for c in contexts], 64)
    x = _inputs(s, nq, nkv, hd, "bfloat16")
    out = torch.full_like(x[0], float("nan"))
    assert _attend(s, nq, nkv, hd, *x, out) == launches
    _check(s, nq, nkv, hd, "bfloat16", *x, out)


@pytest.mark.parametrize("nq,nkv", [(40, 1), (34, 2)])
@pytest.mark.parametrize("contexts", [[1000] * 10, [700, 3, 2000], [0]])
def test_more_than_sixteen_query_heads_a_kv_head(nq, nkv, contexts):
    """Single tokens of more rows than the kernel for few rows takes at once: no launch for requests of fewer rows, which there are none of."""
    import torch
    s = step([(1, c) for c in contexts], 16)
    x = _inputs(s, nq, nkv, 128, "bfloat16")
    out = torch.full_like(x[0], float("nan"))
    assert _attend(s, nq, nkv, 128, *x, out) == 1
    _check(s, nq, nkv, 128, "bfloat16", *x, out)


def test_host_lists_of_single_tokens_that_are_missing_or_longer():
    import torch
    nq, nkv, hd = 8, 2, 64
    s = step([(1, 90), (1, 4000), (1, 3)], 16)
    x = _inputs(s, nq, nkv, hd, "float32")
    outs = []
    for kw in (dict(), dict(cu_seqlens_host=[], kv_lens_host=[]), dict(cu_seqlens_host=s.cu_seqlens_host + [3], kv_lens_host=s.kv_lens_host + [9])):
        out = torch.full_like(x[0], float("nan"))
        _attend(SimpleNamespace(**{**vars(s), **kw}), nq, nkv, hd, *x, out)
        _check(s, nq, nkv, hd, "float32", *x, out)
        outs.append(out)
    assert torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("nq,nkv,bound,launches,replays", [
    (32, 8, 16384, 2, [[16000] + [300] * 7, [300] * 8, [0] * 7 + [16000], [16000] * 8]),       # shares of 42 tiles in clusters of 6: stretches
    (32, 8, 1024, 1, [[1000] + [20] * 7, [1000] * 8]),                                         # shares of three: clusters
    (40, 1, 1024, 2, [[1000] + [20] * 7, [1000] * 8, [0] * 8])])                               # the portions' kernel and its merge, nothing for fewer rows
def test_recorded_steps_are_cut_for_requests_of_any_length(nq, nkv, bound, launches, replays):
    import torch
    hd = 128
    held = step([(1, bound - 1)] * 8, 64)
    q, k, ks, v, vs = _inputs(held, nq, nkv, hd, "bfloat16")
    k.div_(4, rounding_mode="trunc")                # scores of a few units
    out = torch.empty_like(q)
    s = step([(1, bound - 1)] * 8, 64)
    s.table, s.captured, s.max_kv_len = held.table, True, bound
    assert _attend(s, nq, nkv, hd, q, k, ks, v, vs, out) == launches
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _attend(s, nq, nkv, hd, q, k, ks, v, vs, out)
    for contexts in replays:
        now = step([(1, c) for c in contexts], 64)
        now.table = held.table
        s.kv_lens.copy_(now.kv_lens)
        out.fill_(float("nan"))
        graph.replay()
        _check(now, nq, nkv, hd, "bfloat16", q, k, ks, v, vs, out)


def test_a_block_table_of_one_row_whatever_its_stride_says():
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd, page = 8, 2, 64, 16
    s = step([(1, 90)], page)
    inv_freq = torch.ones(hd // 2, device="cuda")
    qkv = torch.randn((1, 1, (nq + 2 * nkv) * hd), device="cuda")
    x = _inputs(s, nq, nkv, hd, "bfloat16")
    got = []
    for table in (s.table, s.table.reshape(-1, 1).clone().t()):
        assert table.shape == s.table.shape
        q, k, ks, v, vs = (t.clone() for t in x)
        out = torch.empty_like(q)
        ops.attn_prepare_q8(ops.Partials(qkv), None, None, 0.0, inv_freq, hd, s.positions, s.cu_seqlens, table, page, k, v, ks, vs, q, nq, nkv, hd)
        ops.attention_q8(q, k, v, ks, vs, out, s, table, page, nq, nkv, hd, 0, hd ** -0.5)
        got.append((k, v, q, out))
    assert all(torch.equal(a, b) for a, b in zip(*got))
