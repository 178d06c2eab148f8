"""Attention over pages of 8-bit codes, against float64."""
from types import SimpleNamespace

import pytest

from q8_util import BLOCK, attend64, planes, rows_of, step

pytestmark = pytest.mark.gpu


def _tolerance(out, size, dtype, keys):
    """float32: scores of up to 256 products and sums over up to 2^17 keys in a few partial sums, 2^-24 each, of numbers that are at most
    their keys' weighted magnitudes; exponentials within 2^-21: 2^-14 of these magnitudes.  A weight - a probability times its value's scale's
    power of two - is held in float16 parts that leave 2^-22 of it or 2^-39 of the row's largest, times a code of at most 127, where the key that
    holds the largest has codes of 64 and more: 2^-38 of the row's largest magnitude for every key.  bfloat16: the output is rounded by half a step,
    2^-8 of it; weights - a key's probability times its value's scale - are rounded to float16, 2^-11 of them each and at least 2^-25 of the
    row's largest, whose own magnitudes are the row's largest too; scores sum in float32: 2^-10 of the magnitudes, and 2^-24 of the row's
    largest for every key."""
    if dtype == "float32":
        return 2.0 ** -14 * size + keys * 2.0 ** -38 * size.amax(-1, keepdim=True)
    return 2.0 ** -8 * out.abs() + 2.0 ** -10 * size + keys * 2.0 ** -24 * size.amax(-1, keepdim=True)


def _run(s, nq, nkv, hd, window, dtype, scale=None, seed=3, q=None, planes_=None):
    import torch
    from kestrel_llm_b200.csrc import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, ks, v, vs = planes_ or planes(s, nkv, hd)
    if q is None:
        q = torch.randn((s.num_tokens, nq * hd), generator=gen, device="cuda").to(getattr(torch, dtype))
    out = torch.full_like(q, float("nan"))
    scale = scale or hd ** -0.5
    ops.attention_q8(q, k, v, ks, vs, out, s, s.table, s.page, nq, nkv, hd, window, scale)
    ops.raise_on_kernel_error()
    want, size = attend64(q, k, ks, v, vs, s, nq, nkv, hd, window, scale)
    return out.view(s.num_tokens, nq, hd).double(), want, size


def _near(s, got, want, size, dtype, more=0.0):
    import torch
    T = s.cu_seqlens_host[-1]
    assert torch.isnan(got[T:]).all()               # rows behind the last request
    assert torch.isfinite(got[:T]).all()
    worst = ((got[:T] - want[:T]).abs() / (_tolerance(want[:T], size[:T], dtype, s.max_kv_len) + (more[:T] if torch.is_tensor(more) else more))).max().item()
    assert worst <= 1, f"{worst} times the tolerance"


SMALL = [[(1, 0)], [(1, 15), (1, 16), (1, 200)], [(1, 1000)], [(2, 5), (0, 0), (1, 63), (3, 64)], [(1, 130)] * 40]
LARGE = [[(33, 0)], [(130, 70), (1, 300)], [(257, 0), (20, 111), (1, 0)], [(64, 1999)]]


@pytest.mark.parametrize("portions", SMALL + LARGE)
@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 2, 128, 16), (3, 1, 64, 32), (4, 4, 128, 64), (16, 1, 64, 16), (10, 2, 128, 128), (40, 1, 128, 16)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_bfloat16_against_float64(portions, nq, nkv, hd, page, window):
    s = step(portions, page, window=window, extra_tokens=2, spread=1)
    _near(s, *_run(s, nq, nkv, hd, window, "bfloat16"), "bfloat16")


@pytest.mark.parametrize("portions", [SMALL[1], SMALL[3], LARGE[1]])
@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 2, 128, 16), (3, 1, 64, 32), (2, 2, 256, 16), (4, 2, 80, 48), (2, 1, 16, 16)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_head_sizes_and_float32_against_float64(portions, nq, nkv, hd, page, window, dtype):
    s = step(portions, page, window=window, extra_tokens=2)
    _near(s, *_run(s, nq, nkv, hd, window, dtype), dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("portions", [[(1, 70000)], [(3, 20000), (1, 9)], [(40, 9000)], [(1, 5000)], [(2, 4500), (1, 300)], [(1, 6200)] * 3])
def test_long_contexts(portions, dtype):
    s = step(portions, 64)
    _near(s, *_run(s, 8, 2, 128, 0, dtype), dtype)


@pytest.mark.parametrize("portions", [[(1, 100)] * 3, [(150, 30)]])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_and_queries_of_every_size(portions, hd):
    """Values from 2^-60 to 2^60 beside one another, and queries whose rows differ as much: neither leaves a type's range on the way."""
    import torch
    s = step(portions, 16)
    nq, nkv = 8, 2
    k, ks, v, vs = planes(s, nkv, hd)
    gen = torch.Generator(device="cuda").manual_seed(9)
    powers = torch.randint(-60, 61, vs.shape, generator=gen, device="cuda")
    vs = torch.where(torch.isnan(vs), vs, 2.0 ** powers)
    q = torch.randn((s.num_tokens, nq * hd), generator=gen, device="cuda")
    q = (q.view(-1, nq, hd) * 2.0 ** torch.randint(-40, 41, (s.num_tokens, nq, 1), generator=gen, device="cuda")).view(q.shape).bfloat16()
    # Scores of thousands are off by 2^-24 of themselves and more: keys are small enough that the largest is about 1, whatever the query is
    ks = ks * 2.0 ** -44
    _near(s, *_run(s, nq, nkv, hd, 0, "bfloat16", q=q, planes_=(k, ks, v, vs)), "bfloat16")


@pytest.mark.parametrize("portions", [[(1, 40)] * 2, [(1, 1)], [(100, 5)], [(300, 20)]])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [0.1, 2.0 ** -100])
def test_keys_and_queries_of_nothing_leave_the_mask_alone(portions, hd, scale):
    """Scores that vanish - keys whose scale is zero or the least, queries of 2^-70, a factor of 2^-100 - weigh alike; a hidden key, whatever its scale, nothing."""
    import torch
    s = step(portions, 16)
    nq, nkv = 8, 2
    for keys in (0.0, 2.0 ** -64):
        k, ks, v, vs = planes(s, nkv, hd)
        ks = torch.where(torch.isnan(ks), ks, keys)
        q = (torch.randn((s.num_tokens, nq * hd), device="cuda") * 2.0 ** -70).bfloat16()
        _near(s, *_run(s, nq, nkv, hd, 0, "bfloat16", scale=scale, q=q, planes_=(k, ks, v, vs)), "bfloat16")
        got, _, _ = _run(s, nq, nkv, hd, 0, "bfloat16", scale=scale, q=q, planes_=(k, ks, v, torch.where(torch.isnan(vs), vs, 0.0)))
        assert (got.abs() <= 2.0 ** -57).all()


@pytest.mark.parametrize("portions,bad", [([(1, 40), (1, 40)], 0), ([(100, 0)], 60), ([(300, 20)], 130)])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 4, 128), (8, 1, 64), (2, 2, 80)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_it_alone(portions, bad, nq, nkv, hd, dtype):
    """The block of position ``bad`` of request 0 and of kv head 0 in V, and of the last kv head in K."""
    import torch
    from kestrel_llm_b200.csrc import ops
    s = step(portions, 16)
    k, ks, v, vs = planes(s, nkv, hd)
    p, slot = rows_of(s, 0, 0, s.kv_lens_host[0])
    vs[p[bad], 0, slot[bad] // BLOCK] = float("nan")
    ks[p[bad], nkv - 1, slot[bad] // BLOCK] = float("nan")
    q = torch.randn((s.num_tokens, nq * hd), device="cuda").to(getattr(torch, dtype))
    out = torch.zeros_like(q)
    ops.attention_q8(q, k, v, ks, vs, out, s, s.table, 16, nq, nkv, hd, 0, hd ** -0.5)
    got = torch.isnan(out.view(s.num_tokens, nkv, nq // nkv, hd).float())
    first = bad // BLOCK * BLOCK
    for r in range(s.num_seqs):
        for i in range(s.counts[r]):
            for h in range(nkv):
                sees = r == 0 and s.starts[r] + i >= first and h in (0, nkv - 1)
                assert bool(got[s.cu_seqlens_host[r] + i, h].all()) == sees and bool(got[s.cu_seqlens_host[r] + i, h].any()) == sees


@pytest.mark.parametrize("tokens", [1, 200])
def test_a_query_that_is_not_finite_stays_in_its_row(tokens):
    import torch
    s = step([(tokens, 90), (tokens, 7)], 16)
    nq, nkv, hd = 8, 2, 128
    q = torch.randn((s.num_tokens, nq * hd), device="cuda").bfloat16()
    q[0, 5] = float("inf")
    q[tokens, 3 * hd] = float("nan")
    got, want, size = _run(s, nq, nkv, hd, 0, "bfloat16", q=q)
    bad = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 0] = bad[tokens, 3] = True
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    assert ((got - want).abs() <= _tolerance(want, size, "bfloat16", s.max_kv_len))[~bad].all()


@pytest.mark.parametrize("portions", [[(1, 100)] * 3, [(150, 30)]])
@pytest.mark.parametrize("hd", [64, 128])
def test_float32_scales_and_queries_of_every_size(portions, hd):
    """Values from 2^-60 to 2^60 beside one another, and float32 queries whose rows differ as much and use all of their bits."""
    import torch
    s = step(portions, 16)
    nq, nkv = 8, 2
    k, ks, v, vs = planes(s, nkv, hd)
    gen = torch.Generator(device="cuda").manual_seed(9)
    powers = torch.randint(-60, 61, vs.shape, generator=gen, device="cuda")
    vs = torch.where(torch.isnan(vs), vs, 2.0 ** powers * (1 + torch.rand(vs.shape, generator=gen, device="cuda")))
    q = torch.randn((s.num_tokens, nq * hd), generator=gen, device="cuda")
    q = (q.view(-1, nq, hd) * 2.0 ** torch.randint(-40, 41, (s.num_tokens, nq, 1), generator=gen, device="cuda")).view(q.shape)
    ks = ks * 2.0 ** -44
    _near(s, *_run(s, nq, nkv, hd, 0, "float32", q=q, planes_=(k, ks, v, vs)), "float32")


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_a_float32_query_that_is_not_finite_stays_in_its_row(tokens, hd):
    import torch
    s = step([(tokens, 70), (tokens, 3)], 16)
    nq, nkv = 8, 2
    q = torch.randn((s.num_tokens, nq * hd), device="cuda")
    bad = torch.zeros((s.num_tokens, nq), dtype=torch.bool, device="cuda")
    for i, (t, h, x) in enumerate(((0, 1, "nan"), (s.num_tokens - 1, 4, "inf"), (s.num_tokens - 1, 7, "-inf"))):
        q.view(-1, nq, hd)[t, h, 3 + i] = float(x)
        bad[t, h] = True
    got, want, size = _run(s, nq, nkv, hd, 0, "float32", q=q)
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    assert ((got - want).abs() <= _tolerance(want, size, "float32", s.max_kv_len))[~bad].all()


@pytest.mark.parametrize("portions", [[(1, 100), (1, 500)], [(200, 300)]])
def test_pages_beyond_four_gigabytes(portions):
    """A plane of 2^32 codes and more: offsets of codes need more than 32 bits."""
    import torch
    nq, nkv, hd = 8, 8, 128
    s = step(portions, 16, extra_pages=280000)
    gen = torch.Generator(device="cuda").manual_seed(5)
    p = []
    for _ in range(2):
        p += [torch.zeros((s.pages, nkv, 16, hd), dtype=torch.int8, device="cuda"), torch.full((s.pages, nkv, 1), float("nan"), device="cuda")]
    assert p[0].numel() > 2 ** 32
    s.table[s.table >= 0] = (s.pages - 1 - torch.arange(int((s.table >= 0).sum()), device="cuda") * 2).int()
    used = s.table[s.table >= 0].long()
    for codes, scales in ((p[0], p[1]), (p[2], p[3])):
        codes[used] = torch.randint(-127, 128, (len(used), nkv, 16, hd), generator=gen, device="cuda", dtype=torch.int8)
        scales[used] = torch.exp(torch.randn((len(used), nkv, 1), generator=gen, device="cuda")) / 64
    for dtype in ("bfloat16", "float32"):
        got, want, size = _run(s, nq, nkv, hd, 0, dtype, scale=0.01, planes_=p)
        _near(s, got, want, size, dtype)


def test_append_then_attend_then_replay():
    """A prompt appended in portions and decoded on: attention over what the append wrote, eager and replayed from a graph with other contents."""
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd, page = 8, 2, 128, 16
    gen = torch.Generator(device="cuda").manual_seed(4)
    last = step([(1, 90), (1, 41)], page)
    k, ks, v, vs = planes(last, nkv, hd)
    ks.fill_(float("nan"))                          # whatever is not appended is no number
    vs.fill_(float("nan"))
    inv_freq = (1.0 / 10000.0 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().cuda()

    def run(s, qkv, q, out):
        ops.attn_prepare_q8(ops.Partials(qkv), None, None, 0.0, inv_freq, hd, s.positions, s.cu_seqlens, s.table, page, k, v, ks, vs, q, nq, nkv, hd)
        ops.attention_q8(q, k, v, ks, vs, out, s, s.table, page, nq, nkv, hd, 0, hd ** -0.5)

    def check(s, q, out):
        want, size = attend64(q, k, ks, v, vs, s, nq, nkv, hd, 0, hd ** -0.5)
        _near(s, out.view(-1, nq, hd).double(), want, size, "bfloat16")
    for portions in ([(30, 0), (5, 0)], [(59, 30), (1, 5)], [(1, 89), (35, 6)]):
        s = step(portions, page)
        s.table = last.table
        T = s.num_tokens
        qkv = torch.randn((1, T, (nq + 2 * nkv) * hd), generator=gen, device="cuda")
        q, out = torch.empty((T, nq * hd), dtype=torch.bfloat16, device="cuda"), torch.empty((T, nq * hd), dtype=torch.bfloat16, device="cuda")
        run(s, qkv, q, out)
        check(s, q, out)
    s = step([(1, 90), (1, 41)], page)
    s.table = last.table
    s.captured, s.max_kv_len = True, 4096           # recorded for contexts up to 4,096
    qkv = torch.randn((1, 2, (nq + 2 * nkv) * hd), generator=gen, device="cuda")
    q, out = torch.empty((2, nq * hd), dtype=torch.bfloat16, device="cuda"), torch.empty((2, nq * hd), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = [t.clone() for t in (k, ks, v, vs)]
    with torch.cuda.stream(side):
        run(s, qkv, q, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(s, qkv, q, out)
    for t, was in zip((k, ks, v, vs), state):
        t.copy_(was)
    out.fill_(float("nan"))
    graph.replay()
    check(s, q, out)
    first = out.clone()
    # the next tokens through the same graph
    s.positions.add_(1)
    s.kv_lens.add_(1)
    s.starts, s.kv_lens_host = [x + 1 for x in s.starts], [x + 1 for x in s.kv_lens_host]
    qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda"))
    graph.replay()
    check(s, q, out)
    assert not torch.equal(first, out)


def test_two_streams_at_once():
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd = 8, 2, 128
    jobs = []
    for i, portions in enumerate(([(1, 5000)], [(200, 300)], [(1, 3000)] * 4)):
        s = step(portions, 16, seed=i)
        k, ks, v, vs = planes(s, nkv, hd, seed=i)
        q = torch.randn((s.num_tokens, nq * hd), device="cuda").bfloat16()
        jobs.append((torch.cuda.Stream(), s, q, k, v, ks, vs, torch.empty_like(q)))
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, s, q, k, v, ks, vs, out in jobs:
            with torch.cuda.stream(stream):
                ops.attention_q8(q, k, v, ks, vs, out, s, s.table, 16, nq, nkv, hd, 0, hd ** -0.5)
    torch.cuda.synchronize()
    for _, s, q, k, v, ks, vs, out in jobs:
        want, size = attend64(q, k, ks, v, vs, s, nq, nkv, hd, 0, hd ** -0.5)
        _near(s, out.view(-1, nq, hd).double(), want, size, "bfloat16")


def test_a_description_that_kernels_write():
    """Lengths and tables that kernels in front of the call wrote count as they stand then, and copied ones give the same bits early."""
    import torch
    from kestrel_llm_b200.csrc import ops
    for portions in ([(1, 3000)] * 9, [(1, 40)], [(200, 300)], [(300, 0), (1, 9)]):
        for dtype in (torch.bfloat16, torch.float32):
            s = step(portions, 16)
            k, ks, v, vs = planes(s, 2, 128)
            q = torch.randn((s.num_tokens, 8 * 128), device="cuda").to(dtype)
            got = []
            for described in (True, False, False):
                out = torch.full_like(q, float("nan"))
                lens, table = s.kv_lens.clone(), s.table.clone()
                if not described:               # the smallest lengths and no pages, until a moment before the call
                    lens -= torch.tensor(s.starts, dtype=torch.int32, device="cuda")
                    table.fill_(-1)
                torch.cuda.synchronize()
                if not described:
                    torch.add(lens, torch.tensor(s.starts, dtype=torch.int32, device="cuda"), out=lens)
                    torch.maximum(table, s.table, out=table)
                here = SimpleNamespace(**{**vars(s), "kv_lens": lens})
                ops.attention_q8(q, k, v, ks, vs, out, here, table, 16, 8, 2, 128, 0, 0.1, described=described)
                got.append(out)
            assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
            assert torch.isfinite(got[0]).all()


@pytest.mark.parametrize("portions", [[(1, 900)] * 3, [(200, 300), (1, 70)], [(20, 40)]])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_window_of_every_size(portions, dtype):
    """Windows beyond the longest request hide nothing, up to the largest int32."""
    got = []
    for window in (0, 10000, 2 ** 31 - 1):
        out, want, size = _run(step(portions, 16), 8, 2, 128, window, dtype)
        _near(step(portions, 16), out, want, size, dtype)
        got.append(out)
    assert got[0].equal(got[1]) and got[0].equal(got[2])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_recorded_single_tokens_of_short_requests(dtype):
    """Recorded for contexts of up to 65,536, replayed with far shorter ones: less work than the launch was cut for."""
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd, n = 8, 2, 128, 40
    held = step([(1, 300)] * n, 16)
    k, ks, v, vs = planes(held, nkv, hd)
    k.div_(4, rounding_mode="trunc")                # scores of a few units
    q = torch.randn((n, nq * hd), device="cuda").to(getattr(torch, dtype))
    out = torch.empty_like(q)
    s = step([(1, 300)] * n, 16)
    s.table, s.captured, s.max_kv_len = held.table, True, 65536
    run = lambda: ops.attention_q8(q, k, v, ks, vs, out, s, s.table, 16, nq, nkv, hd, 0, 0.01)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for contexts in ([300] * n, [0] * n, [100] * n, list(range(3, 3 + 7 * n, 7)), [0] * (n - 1) + [300]):
        now = step([(1, c) for c in contexts], 16)
        now.table = held.table
        s.kv_lens.copy_(now.kv_lens)
        out.fill_(float("nan"))
        graph.replay()
        want, size = attend64(q, k, ks, v, vs, now, nq, nkv, hd, 0, 0.01)
        _near(now, out.view(-1, nq, hd).double(), want, size, dtype)


def test_recorded_portions_share_the_tokens():
    """A step recorded for eight requests of up to 300 tokens, 320 in all, and replayed with other cuts of them."""
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd = 8, 2, 128
    most = [(300, 0)] + [(0, 0)] * 7
    first = step([(300, 200)] + [(2, 498)] * 7, 16)
    for dtype in (torch.bfloat16, torch.float32):
        s = step(most, 16)
        s.table, s.pages, s.num_tokens, s.max_kv_len, s.captured = first.table, first.pages, 320, 500, True
        k, ks, v, vs = planes(first, nkv, hd)
        q = torch.randn((320, nq * hd), device="cuda").to(dtype)
        out = torch.empty_like(q)
        run = lambda: ops.attention_q8(q, k, v, ks, vs, out, s, s.table, 16, nq, nkv, hd, 0, hd ** -0.5)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for cuts in ([(300, 200)] + [(2, 498)] * 7, [(40, 100)] * 8, [(1, 499)] * 8, [(0, 0), (17, 3), (128, 0), (129, 371), (0, 0), (3, 400), (1, 0), (42, 42)]):
            now = step(cuts, 16)
            now.table, now.num_tokens = first.table, 320
            s.cu_seqlens.copy_(now.cu_seqlens)
            s.kv_lens.copy_(now.kv_lens)
            out.fill_(float("nan"))
            graph.replay()
            want, size = attend64(q, k, ks, v, vs, now, nq, nkv, hd, 0, hd ** -0.5)
            # Scores here reach 200 and more.  In float32 a score is a sum of hd products, each step off by 2^-24 of what the magnitudes add up
            # to, which is at most |q| |k| scale; so are a weight's logarithm and, over all keys, the sum's: twice that of the magnitudes.  A weight
            # below 2^-126 of the largest may vanish: where the seen keys' value is zero, that is all that an output is.
            more = 0.0
            if dtype is torch.float32:
                keys = (k.double() * ks.double().repeat_interleave(BLOCK, 2)[..., None]).norm(dim=-1).nan_to_num(0).max()
                reach = q.view(-1, nq, hd).double().norm(dim=-1, keepdim=True) * keys * hd ** -0.5
                more = 2 * (hd + 8) * 2.0 ** -24 * reach * size + 500 * 2.0 ** -126 * 127 * vs.nan_to_num(0).max().double()
            _near(now, out.view(-1, nq, hd).double(), want, size, "float32" if dtype is torch.float32 else "bfloat16", more)


def test_refusals():
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd, page = 4, 2, 64, 16
    s = step([(3, 20)], page)
    k, ks, v, vs = planes(s, nkv, hd)
    q = torch.randn((3, nq * hd), device="cuda").bfloat16()

    def call(**kw):
        a = dict(q=q, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, out=torch.empty_like(q), batch=s, block_table=s.table, page_size=page, nq=nq,
                 nkv=nkv, hd=hd, window=0, scale=0.125)
        a.update(kw)
        ops.attention_q8(**a)
    call()
    longer = SimpleNamespace(**{**vars(s), "num_tokens": 4})
    more = SimpleNamespace(**{**vars(s), "num_seqs": 2})
    beyond = SimpleNamespace(**{**vars(s), "max_kv_len": 33})
    short = SimpleNamespace(**{**vars(s), "cu_seqlens_host": [0]})
    padded = SimpleNamespace(**{**vars(s), "cu_seqlens_host": s.cu_seqlens_host + [3, 3], "kv_lens_host": s.kv_lens_host + [0, 0]})
    call(batch=padded)
    for kw in (dict(q=q.half()), dict(q=q.cpu()), dict(out=torch.empty_like(q).float()), dict(k_cache=k.float()), dict(k_cache=k[:, :1]),
               dict(v_scale=vs.half()), dict(k_scale=ks.cpu()), dict(page_size=24), dict(page_size=32), dict(nq=3), dict(hd=32), dict(window=-1),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(batch=longer), dict(batch=more), dict(batch=beyond), dict(batch=short), dict(block_table=s.table.long()),
               dict(block_table=s.table[:0]), dict(v_cache=v.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ops.KernelError):
            call(**kw)
