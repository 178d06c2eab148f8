"""Appending to pages of 8-bit codes, against float64 and the definition of the codes."""
import math

import pytest

from q8_util import BLOCK, LOWEST, planes, prepared64, rows_of, step

pytestmark = pytest.mark.gpu

# Numbers before they are coded: up to 8 slices and a bias summed, a norm (a sum, a square root, a division, two products) and a rotation
# (cosine and sine within 2 units, two products, a sum), all in float32 - fewer than 32 roundings of 2^-24, each relative to a number at
# most a few times the row's largest.
E = 2.0 ** -18


def _inputs(s, nq, nkv, hd, S, rot, norm, bias, seed=2):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    W = (nq + 2 * nkv) * hd
    qkv = rnd(S, s.num_tokens, W) / math.sqrt(S) * torch.exp(rnd(1, s.num_tokens, 1))
    inv_freq = (1.0 / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda() if rot else None
    return (qkv, 0.3 * rnd(W) if bias else None, 1 + 0.1 * rnd(hd) if norm else None, 1 + 0.1 * rnd(hd) if norm else None, inv_freq)


def _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, rot, interleaved=False, rot_scale=1.0, write_kv=True):
    from kestrel_llm_b200.csrc import ops
    qkv, bias, qw, kw, inv_freq = inputs
    ops.attn_prepare_q8(ops.Partials(qkv, bias), qw, kw, 1e-6, inv_freq, rot, s.positions, s.cu_seqlens, s.table, s.page, k, v, ks, vs, q, nq, nkv, hd,
                        write_kv=write_kv, rot_mode=int(interleaved), rot_scale=rot_scale)


def _check_plane(s, x, before, after, nkv):
    """x [T, nkv, hd] in 64 bits; before and after: (codes, scales).  The scales and codes of every block that the step touched follow from
    x and from what was there; all else has the same bits."""
    import torch
    codes0, scale0, codes1, scale1 = before[0].double(), before[1].double(), after[0].double(), after[1].double()
    touched = torch.zeros(codes0.shape, dtype=torch.bool, device="cuda")
    blocks = torch.zeros(scale0.shape, dtype=torch.bool, device="cuda")
    for r in range(s.num_seqs):
        c, n, t0 = s.starts[r], s.counts[r], s.cu_seqlens_host[r]
        for b in range(c // BLOCK, (c + n + BLOCK - 1) // BLOCK if n else c // BLOCK):
            lo, hi = max(c, b * BLOCK), min(c + n, (b + 1) * BLOCK)
            page, slot = (int(t) for t in (s.table[r, b * BLOCK // s.page], b * BLOCK % s.page))
            rows = x[t0 + lo - c:t0 + hi - c].transpose(0, 1)
            there = lo - b * BLOCK
            want = torch.clamp(rows.abs().amax((1, 2)) / 127, min=LOWEST)
            got = scale1[page, :, slot // BLOCK]
            blocks[page, :, slot // BLOCK] = True
            touched[page, :, slot:slot + there + hi - lo] = True
            if there:
                old = scale0[page, :, slot // BLOCK]
                want = torch.maximum(want, old)
            assert ((got - want).abs() <= E * want).all()
            new = codes1[page, :, slot + there:slot + there + hi - lo]
            assert new.abs().max() <= 127
            # half a step, and the errors of the number and of the scale, 127 steps at most
            assert ((new * got[:, None, None] - rows).abs() <= got[:, None, None] * (0.5 + 2 * 127 * E)).all()
            if there:
                kept, again = codes0[page, :, slot:slot + there], codes1[page, :, slot:slot + there]
                same = got == old
                assert torch.equal(kept[same], again[same])
                # the ratio and its product with a code: two roundings
                assert ((again - kept * (old / got)[:, None, None]).abs() <= 0.5 + 127 * 2.0 ** -22).all()
    assert torch.equal(before[0][~touched], after[0][~touched])
    assert torch.equal(before[1].view(torch.int32)[~blocks], after[1].view(torch.int32)[~blocks])


@pytest.mark.parametrize("portions", [[(1, 0)], [(1, 37)], [(1, 16), (1, 15), (1, 70001)], [(40, 0)], [(33, 5), (1, 90), (16, 32), (0, 8), (17, 47)]])
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 2, 128, 16), (6, 2, 64, 32), (2, 1, 256, 16), (3, 3, 48, 48), (40, 8, 128, 64)])
@pytest.mark.parametrize("dtype,S,rot_share,interleaved,norm,bias", [("bfloat16", 1, 1.0, False, True, False), ("float32", 5, 0.5, True, False, True),
                                                                   ("float32", 8, 0.5, False, True, True), ("bfloat16", 2, 0.0, False, False, False)])
def test_append_against_float64(portions, nq, nkv, hd, page, dtype, S, rot_share, interleaved, norm, bias):
    import torch
    s = step(portions, page, extra_tokens=3, spread=2)
    rot = int(hd * rot_share)
    k, ks, v, vs = planes(s, nkv, hd)
    before = [t.clone() for t in (k, ks, v, vs)]
    inputs = _inputs(s, nq, nkv, hd, S, rot, norm, bias)
    q = torch.full((s.num_tokens, nq * hd), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, rot, interleaved, 1.25)
    q64, k64, v64 = prepared64(*inputs[:4], 1e-6, inputs[4], rot, s.positions, nq, nkv, hd, interleaved, 1.25)
    T = s.cu_seqlens_host[-1]
    assert torch.isnan(q[T:]).all()                 # rows behind the last request
    got = q[:T].view(T, nq, hd).double()
    big = q64[:T].abs().amax(-1, keepdim=True) * 1.5
    half = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -24
    assert ((got - q64[:T]).abs() <= half * q64[:T].abs() + E * big).all()
    _check_plane(s, k64, (before[0], before[1]), (k, ks), nkv)
    _check_plane(s, v64, (before[2], before[3]), (v, vs), nkv)


def test_tokens_one_by_one_raise_a_block_scale():
    """Forty steps of one token, each twice as large as the one before for a while: every state follows from the one before it."""
    import torch
    nq, nkv, hd, page = 2, 2, 64, 32
    whole = step([(1, 40)], page)
    k, ks, v, vs = planes(whole, nkv, hd, stale=False)
    for t in range(41):
        s = step([(1, t)], page)
        s.table, s.pages = whole.table, whole.pages
        inputs = _inputs(s, nq, nkv, hd, 1, hd, False, False, seed=t)
        inputs[0].mul_(2.0 ** min(t % 16, 9) if t % 16 < 12 else 2.0 ** -20)
        before = [x.clone() for x in (k, ks, v, vs)]
        q = torch.empty((1, nq * hd), dtype=torch.float32, device="cuda")
        _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, hd)
        _, k64, v64 = prepared64(*inputs[:4], 1e-6, inputs[4], hd, s.positions, nq, nkv, hd, False)
        _check_plane(s, k64, (before[0], before[1]), (k, ks), nkv)
        _check_plane(s, v64, (before[2], before[3]), (v, vs), nkv)


def test_far_positions_keep_their_angles():
    """Positions up to 2^24 and beyond: the angle's error would be hundreds of times E in one float32 number."""
    import torch
    nq, nkv, hd = 2, 1, 128
    for at in (131071, (1 << 20) - 3, (1 << 24) + 1):
        s = step([(2, 0)], 16)
        s.starts, s.kv_lens_host = [at], [at + 2]
        s.positions = torch.tensor([at, at + 1], dtype=torch.int32, device="cuda")
        s.table = torch.zeros((1, at // 16 + 2), dtype=torch.int32, device="cuda")
        s.table[0, at // 16 + 1] = 1
        k, ks, v, vs = planes(step([(2, 0)], 16), nkv, hd, stale=False)
        inputs = _inputs(s, nq, nkv, hd, 1, hd, True, False)
        q = torch.empty((2, nq * hd), dtype=torch.float32, device="cuda")
        _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, hd)
        q64, _, _ = prepared64(*inputs[:4], 1e-6, inputs[4], hd, s.positions, nq, nkv, hd, False)
        assert ((q.view(2, nq, hd).double() - q64).abs() <= E * 1.5 * q64.abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_block(bad):
    import torch
    nq, nkv, hd, page = 2, 2, 64, 32
    s = step([(40, 3)], page)
    k, ks, v, vs = planes(s, nkv, hd, stale=False)
    inputs = _inputs(s, nq, nkv, hd, 2, hd, False, False)
    inputs[0][1, 20, (nq + 1) * hd + 5] = bad       # key head 1 of position 23
    inputs[0][0, 30, (nq + nkv) * hd + 9] = bad     # value head 0 of position 33
    q = torch.empty((40, nq * hd), dtype=torch.bfloat16, device="cuda")
    _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, hd)
    p, slot = rows_of(s, 0, 0, 43)
    for scales, head, block in ((ks, 1, 1), (vs, 0, 2)):
        got = torch.isnan(torch.stack([scales[p[16 * b], :, slot[16 * b] // BLOCK] for b in range(3)]))
        want = torch.zeros_like(got)
        want[block, head] = True
        assert torch.equal(got, want)
    assert not torch.isnan(q.float()).any()
    # a later token joins the block: it stays what it is; the same block begun anew is whole again
    s2 = step([(1, 43)], page)
    s2.table, s2.pages = s.table, s.pages
    clean = _inputs(s2, nq, nkv, hd, 1, hd, False, False)
    _append(s2, clean, k, ks, v, vs, q[:1], nq, nkv, hd, hd)
    assert torch.isnan(vs[p[40], 0, slot[40] // BLOCK])
    s3 = step([(40, 3)], page)
    s3.table, s3.pages = s.table, s.pages
    again = _inputs(s3, nq, nkv, hd, 1, hd, False, False)
    _append(s3, again, k, ks, v, vs, q, nq, nkv, hd, hd)
    assert not torch.isnan(ks[p[16], :, slot[16] // BLOCK]).any() and not torch.isnan(vs[p[32], :, slot[32] // BLOCK]).any()


def test_zeros_have_the_lowest_scale_and_absent_pages_are_left_out():
    import torch
    nq, nkv, hd, page = 2, 1, 64, 16
    s = step([(20, 0), (4, 10)], page)
    k, ks, v, vs = planes(s, nkv, hd)
    p, slot = rows_of(s, 0, 0, 20)
    inputs = _inputs(s, nq, nkv, hd, 1, hd, False, False)
    inputs[0].zero_()
    s.table[1] = -1                                 # request 1 has lost its page
    before = [t.clone() for t in (k, ks, v, vs)]
    q = torch.empty((24, nq * hd), dtype=torch.float32, device="cuda")
    _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, hd)
    assert (ks[p, :, slot // BLOCK] == LOWEST).all() and (k[p, :, slot] == 0).all() and (v[p, :, slot] == 0).all()
    keep = torch.ones(s.pages, dtype=torch.bool, device="cuda")
    keep[p] = False
    for was, now in zip(before, (k, ks, v, vs)):
        assert torch.equal(was[keep].view(torch.int8), now[keep].view(torch.int8))
    assert (q == 0).all()


def test_a_layer_that_reads_only_writes_nothing():
    import torch
    nq, nkv, hd, page = 2, 1, 128, 16
    s = step([(20, 7)], page)
    k, ks, v, vs = planes(s, nkv, hd)
    before = [t.clone() for t in (k, ks, v, vs)]
    inputs = _inputs(s, nq, nkv, hd, 1, hd, True, False)
    q = torch.empty((20, nq * hd), dtype=torch.float32, device="cuda")
    _append(s, inputs, k, ks, v, vs, q, nq, nkv, hd, hd, write_kv=False)
    for was, now in zip(before, (k, ks, v, vs)):
        assert torch.equal(was.view(torch.int8), now.view(torch.int8))
    q64, _, _ = prepared64(*inputs[:4], 1e-6, inputs[4], hd, s.positions, nq, nkv, hd, False)
    assert ((q.view(20, nq, hd).double() - q64).abs() <= E * 1.5 * q64.abs().amax(-1, keepdim=True)).all()


def test_pages_beyond_four_gigabytes():
    """A plane of 2^32 codes and more: what is written to its last pages is what is written to others."""
    import torch
    nq, nkv, hd = 4, 8, 128
    s = step([(40, 5), (3, 30)], 16)
    inputs = _inputs(s, nq, nkv, hd, 1, hd, True, False)
    small = [t.clone() for t in planes(s, nkv, hd)]
    pages = 280000
    large = [torch.zeros((pages,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in small]
    assert large[0].numel() > 2 ** 32
    for a, b in zip(large, small):
        a[-s.pages:] = b
    far = step([(40, 5), (3, 30)], 16)
    far.table[far.table >= 0] += pages - s.pages
    got = []
    for st, p in ((s, small), (far, large)):
        q = torch.empty((st.num_tokens, nq * hd), device="cuda")
        _append(st, inputs, *p, q, nq, nkv, hd, hd)
        got.append([t[-s.pages:] for t in p] + [q])
    for a, b in zip(*got):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert all(not t[:-s.pages].any() for t in large)


@pytest.mark.parametrize("hd", [64, 80])
def test_tokens_in_front_of_position_zero_are_left_out(hd):
    """A request from position -20 on: its queries are turned back, its keys and values begin at position 0."""
    import torch
    nq, nkv = 4, 2
    s = step([(10, 0), (3, 7)], 16)
    k, ks, v, vs = planes(s, nkv, hd)
    inputs = _inputs(s, nq, nkv, hd, 2, hd, True, True)
    early = step([(30, 0), (3, 7)], 16)
    early.positions[:30] = torch.arange(-20, 10, dtype=torch.int32)
    early.table = s.table
    longer = (torch.cat([torch.full((2, 20, inputs[0].shape[2]), 1e4, device="cuda"), inputs[0]], 1),) + inputs[1:]
    got = []
    for st, x in ((s, inputs), (early, longer)):
        p = [t.clone() for t in (k, ks, v, vs)]
        q = torch.full((st.num_tokens, nq * hd), float("nan"), device="cuda")
        _append(st, x, *p, q, nq, nkv, hd, hd)
        got.append(p + [q[-13:]])
        assert torch.isfinite(q).all()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.uint8), b.contiguous().view(torch.uint8))
    none = step([(5, 0)], 16)
    none.positions.copy_(torch.arange(-2 ** 31, -2 ** 31 + 5))
    q = torch.full((5, nq * hd), float("nan"), device="cuda")
    p = [t.clone() for t in (k, ks, v, vs)]
    _append(none, (inputs[0][:, :5].contiguous(),) + inputs[1:], *p, q, nq, nkv, hd, hd)
    assert torch.isfinite(q).all()
    for a, b in zip(p, (k, ks, v, vs)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals():
    import torch
    from kestrel_llm_b200.csrc import ops
    nq, nkv, hd, page = 2, 1, 64, 16
    s = step([(4, 0)], page)
    k, ks, v, vs = planes(s, nkv, hd)
    inputs = _inputs(s, nq, nkv, hd, 1, hd, True, False)
    q = torch.empty((4, nq * hd), dtype=torch.float32, device="cuda")

    def call(**kw):
        a = dict(qkv=ops.Partials(inputs[0]), q_norm_w=inputs[2], k_norm_w=inputs[3], norm_eps=1e-6, inv_freq=inputs[4], rotary_dim=hd,
                 positions=s.positions, cu_seqlens=s.cu_seqlens, block_table=s.table, page_size=page, k_cache=k, v_cache=v, k_scale=ks,
                 v_scale=vs, q_out=q, nq=nq, nkv=nkv, hd=hd)
        a.update(kw)
        ops.attn_prepare_q8(**a)
    call()
    for kw in (dict(page_size=8), dict(k_cache=k.float()), dict(k_scale=ks.double()), dict(v_scale=vs[:, :, :0]), dict(k_cache=k[:, :, :, ::2]),
               dict(positions=s.positions.long()), dict(cu_seqlens=s.cu_seqlens[:1]), dict(block_table=s.table.long()), dict(q_out=q.half()),
               dict(rotary_dim=hd + 2), dict(rotary_dim=7), dict(inv_freq=None), dict(inv_freq=inputs[4][:3]), dict(rot_mode=2), dict(hd=60),
               dict(q_norm_w=inputs[2][:9]), dict(positions=s.positions.cpu()), dict(block_table=s.table.cpu()), dict(k_cache=k.cpu()), dict(nkv=2),
               dict(block_table=s.table[:0])):
        with pytest.raises(ops.KernelError):
            call(**kw)
