"""Steps over pages of 8-bit codes, and their operators in 64 bits."""
import math
from types import SimpleNamespace

import torch

BLOCK = 16
LOWEST = 2.0 ** -64


def step(portions, page, device="cuda", window=0, extra_tokens=0, extra_pages=3, seed=0, spread=0):
    """A step of (tokens, context) per request: its description and a table of scattered pages; those that a window has given back, and
    those beyond a request's end, are -1.  ``extra_tokens`` rows stand behind the last request, ``spread`` columns behind the table's."""
    gen = torch.Generator().manual_seed(seed)
    counts, starts = [n for n, _ in portions], [c for _, c in portions]
    lens = [n + c for n, c in portions]
    width = max(1, max((x + page - 1) // page for x in lens))
    first = [max(0, c - window + 1) // page if window else 0 for c in starts]
    held = [(x + page - 1) // page - f for x, f in zip(lens, first)]
    order = torch.randperm(sum(held) + extra_pages, generator=gen).int()
    wide = torch.full((len(portions), width + spread), -1, dtype=torch.int32)
    at = 0
    for r, (f, h) in enumerate(zip(first, held)):
        wide[r, f:f + h] = order[at:at + h]
        at += h
    table = wide.to(device)[:, :width]
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    pos = [c + i for n, c in portions for i in range(n)] + [0] * extra_tokens
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return SimpleNamespace(num_tokens=cu[-1] + extra_tokens, num_seqs=len(portions), counts=counts, starts=starts, kv_lens_host=lens, cu_seqlens_host=cu,
                           cu_seqlens=ints(cu), kv_lens=ints(lens), positions=ints(pos), max_count=max(counts), max_kv_len=max(lens), captured=False,
                           table=table, pages=sum(held) + extra_pages, page=page)


def rows_of(s, r, lo, hi):
    """(page, slot) of positions [lo, hi) of request r."""
    pos = torch.arange(lo, hi, device=s.table.device)
    return s.table[r].long()[pos // s.page], pos % s.page


def planes(s, nkv, hd, seed=1, stale=True):
    """Codes and scales of random values; with ``stale`` every block that no request holds has a scale that is not a number."""
    gen = torch.Generator(device=s.table.device).manual_seed(seed)
    out = []
    for _ in range(2):
        codes = torch.randint(-127, 128, (s.pages, nkv, s.page, hd), generator=gen, device=s.table.device, dtype=torch.int8)
        scale = torch.exp(torch.randn((s.pages, nkv, s.page // BLOCK), generator=gen, device=s.table.device)) / 64
        if stale:
            live = torch.zeros((s.pages, s.page // BLOCK), dtype=torch.bool, device=s.table.device)
            for r, n in enumerate(s.kv_lens_host):
                at = (s.table[r] >= 0).nonzero().flatten()
                if at.numel():
                    p, slot = rows_of(s, r, int(at[0]) * s.page, n)
                    live[p, slot // BLOCK] = True
            scale = torch.where(live[:, None, :], scale, float("nan"))
        out += [codes, scale]
    return out


def attend64(q, k, ks, v, vs, s, nq, nkv, hd, window, scale):
    """Attention in 64 bits, and for every output the mean of the values' magnitudes under the row's weights."""
    G = nq // nkv
    out = torch.zeros((s.num_tokens, nq, hd), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    q = q.view(-1, nq, hd).double()
    for r in range(s.num_seqs):
        n, c, t0 = s.counts[r], s.starts[r], s.cu_seqlens_host[r]
        if n == 0:
            continue
        lo = max(0, c - window + 1) if window else 0
        p, slot = rows_of(s, r, lo, c + n)
        key = torch.arange(lo, c + n, device=q.device)
        pos = torch.arange(c, c + n, device=q.device)[:, None]
        hidden = (key > pos) | ((key <= pos - window) if window else (key < 0))
        for h in range(nkv):
            kk = k[p, h, slot].double() * ks[p, h, slot // BLOCK].double()[:, None]
            vv = v[p, h, slot].double() * vs[p, h, slot // BLOCK].double()[:, None]
            for g in range(G):
                w = (q[t0:t0 + n, h * G + g] @ kk.T * scale).masked_fill(hidden, -math.inf)
                w = torch.softmax(w, 1)
                # what a row may not see does not enter its sum, whatever it is
                out[t0:t0 + n, h * G + g] = torch.where(hidden, 0.0, w) @ torch.nan_to_num(vv) if not torch.isnan(vv).any() else \
                    torch.stack([w[i, ~hidden[i]] @ vv[~hidden[i]] for i in range(n)])
                size[t0:t0 + n, h * G + g] = torch.where(hidden, 0.0, w) @ vv.abs() if not torch.isnan(vv).any() else \
                    torch.stack([w[i, ~hidden[i]] @ vv[~hidden[i]].abs() for i in range(n)])
    return out, size


def turned64(x, pos, inv_freq, rot, interleaved, scale=1.0):
    """x [T, heads, hd] in 64 bits, rotated."""
    x = x.clone()
    if rot:
        ang = pos.double()[:, None] * inv_freq.double()
        c, sn = ang.cos()[:, None] * scale, ang.sin()[:, None] * scale
        a, b = (x[..., 0:rot:2].clone(), x[..., 1:rot:2].clone()) if interleaved else (x[..., :rot // 2].clone(), x[..., rot // 2:rot].clone())
        lo, hi = a * c - b * sn, b * c + a * sn
        if interleaved:
            x[..., 0:rot:2], x[..., 1:rot:2] = lo, hi
        else:
            x[..., :rot // 2], x[..., rot // 2:rot] = lo, hi
    return x


def prepared64(qkv, bias, qw, kw, eps, inv_freq, rot, pos, nq, nkv, hd, interleaved, rot_scale=1.0):
    """(q, k, v) [T, heads, hd] in 64 bits."""
    x = qkv.double().sum(0)
    if bias is not None:
        x = x + bias.double()
    x = x.view(x.shape[0], -1, hd)
    out = []
    for y, w in ((x[:, :nq], qw), (x[:, nq:nq + nkv], kw)):
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
        out.append(turned64(y, pos, inv_freq, rot, interleaved, rot_scale))
    return out[0], out[1], x[:, nq + nkv:]
