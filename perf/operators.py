"""The operators of an 8-bit key/value cache and of scored tokens, at the sizes a program that serves with this engine calls them.

`append`: bias, head norm, rotation; queries out, keys and values into pages of int8 codes with one float32 scale for every block of 16
tokens and head.  `attend`: causal grouped-query attention over such pages, for single tokens and for prompt portions.  `logprobs`: log
probabilities of given tokens, entropy and the likeliest alternatives from rows of logits.

A cache value is code * scale.  A block's scale is the largest magnitude it has met / 127 (at least 2^-64); codes are rounded to nearest,
ties to even; when a step's tokens raise the scale of a block that earlier steps began, the codes that are there are rounded again.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
BLOCK = 16              # tokens that share a scale
LOWEST = 2.0 ** -64     # the smallest scale
THETA = 1000000.0
VOCAB = 151936


def listed():
    return [
        # one user generating: the token of one request joins a block that earlier steps began; latency
        dict(name="append_one", kind="append", dtype="bfloat16", tokens=1, requests=1, context=1003, nq=32, nkv=8, hd=128, page=16, slices=8,
             norm=True, bias=False, rot=128, interleaved=False),
        # the true 32-bit path: ragged portions that begin inside blocks, half of the dimensions rotated in pairs, a bias
        dict(name="append_ragged", kind="append", dtype="float32", tokens=701, requests=5, context=3001, nq=16, nkv=4, hd=64, page=32, slices=1,
             norm=False, bias=True, rot=32, interleaved=True),
        # a whole prompt of the headline model's layer
        dict(name="append_prompt", kind="append", dtype="bfloat16", tokens=2048, requests=1, context=0, nq=32, nkv=8, hd=128, page=16, slices=1,
             norm=True, bias=False, rot=128, interleaved=False),
        # one user generating behind about a thousand tokens: latency
        dict(name="attend_one", kind="attend", dtype="bfloat16", tokens=1, requests=1, context=1003, nq=32, nkv=8, hd=128, page=16, window=0),
        # a serving batch at contexts up to 4,096: bound by the cache's bytes
        dict(name="attend_decode", kind="attend", dtype="bfloat16", tokens=64, requests=64, context=4095, nq=32, nkv=8, hd=128, page=16, window=0),
        # two requests far into long documents: few rows, many keys
        dict(name="attend_long", kind="attend", dtype="bfloat16", tokens=2, requests=2, context=65535, nq=32, nkv=8, hd=128, page=64, window=0),
        # a whole prompt: bound by the products
        dict(name="attend_prompt", kind="attend", dtype="bfloat16", tokens=2048, requests=1, context=0, nq=32, nkv=8, hd=128, page=16, window=0),
        # continuous batching on a windowed layer: a prompt portion beside requests that decode
        dict(name="attend_portions", kind="attend", dtype="bfloat16", tokens=512, requests=13, context=1500, nq=16, nkv=4, hd=64, page=16, window=1024),
        # the true 32-bit path, which replays and checks run on
        dict(name="attend_float32", kind="attend", dtype="float32", tokens=411, requests=2, context=0, nq=16, nkv=4, hd=128, page=16, window=0),
        # one user generating who asks for the twenty likeliest alternatives: latency
        dict(name="logprobs_one", kind="logprobs", rows=1, vocab=VOCAB, top=20, masked=0.0),
        # a serving batch with its answers' log probabilities, most of the vocabulary masked by a grammar
        dict(name="logprobs_decode", kind="logprobs", rows=64, vocab=VOCAB, top=5, masked=0.9),
        # scoring a prompt: every position's next token
        dict(name="logprobs_prompt", kind="logprobs", rows=1024, vocab=VOCAB, top=1, masked=0.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "logprobs", "logprobs"])
    if kind == "logprobs":
        rows = spread(1, 800)
        return dict(kind=kind, rows=rows, vocab=rng.choice([spread(1000, 150000), 32000, VOCAB]), top=rng.choice([0, 1, 5, 20]),
                    masked=rng.choice([0.0, 0.0, 0.9, 0.999]))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    nq, nkv = rng.choice([(32, 8), (16, 4), (16, 2), (12, 4), (8, 8), (40, 8)])
    hd, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    decode = rng.random() < 0.5
    requests = spread(1, 64) if decode else rng.randint(1, 6)
    tokens = requests if decode else max(requests, spread(1, 400 if dtype == "float32" else 1500))
    shape = dict(dtype=dtype, tokens=tokens, requests=requests, nq=nq, nkv=nkv, hd=hd, page=page)
    if kind == "append":
        return dict(kind=kind, context=rng.choice([0, spread(1, 100000)]), slices=rng.choice([1, 1, 2, 5, 8]) if tokens <= 64 else 1,
                    norm=rng.random() < 0.6, bias=rng.random() < 0.3, rot=rng.choice([hd, hd, hd // 2, 0]), interleaved=rng.random() < 0.3, **shape)
    context = spread(16, 4000) if decode else rng.choice([0, spread(1, 1500)])
    if dtype == "float32":
        context = min(context, 600)
    return dict(kind=kind, context=context, window=rng.choice([0, 0, spread(16, 2000)]), **shape)


# ---- the step that a program has in hand ----------------------------------------------------------

class Step:
    """One step's description, as the engine hands it from layer to layer: how many tokens every request brings, how long it is after
    them, and its pages."""

    captured = False

    def __init__(self, counts, starts, table):
        self.counts, self.starts = counts, starts
        self.kv_lens_host = [a + c for a, c in zip(starts, counts)]
        self.cu_seqlens_host = [0]
        for c in counts:
            self.cu_seqlens_host.append(self.cu_seqlens_host[-1] + c)
        self.num_tokens, self.num_seqs = sum(counts), len(counts)
        self.max_count, self.max_kv_len = max(counts), max(self.kv_lens_host)

        def ints(v):
            return torch.tensor(v, dtype=torch.int32, device=DEV)
        self.cu_seqlens, self.kv_lens = ints(self.cu_seqlens_host), ints(self.kv_lens_host)
        self.positions = ints([a + i for a, c in zip(starts, counts) for i in range(c)])
        self.seq_of_token = ints([r for r, c in enumerate(counts) for _ in range(c)])
        self.table = table

    def block_table(self, group):
        return self.table


def _portions(case):
    """(tokens, context) of every request.  A step of at most twice as many tokens as requests is shared out evenly; otherwise the first
    request brings what the others, one token each in a mixed step or unequal shares, leave.  Contexts are unequal, up to the case's."""
    n, T, ctx = case["requests"], case["tokens"], case["context"]
    if T >= 2 * n and n > 6:                        # a portion beside requests that decode
        counts = [T - (n - 1)] + [1] * (n - 1)
    else:
        edges = [T * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
        for i in range(1, n + 1):                   # every request has a token
            edges[i] = max(edges[i], edges[i - 1] + 1)
        for i in range(n, 0, -1):
            edges[i] = min(edges[i], T - (n - i))
        counts = [edges[i + 1] - edges[i] for i in range(n)]
    return counts, [ctx - (ctx * i) // (2 * n) for i in range(n)]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 11)


def _normal(gen, *shape):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(generator=gen)


def _table(gen, first, last):
    """Pages of every request in a scattered order; those before `first` have been given back by a window and are -1.  Returns the table and
    the number of pages."""
    width = max(last)
    held = [b - a for a, b in zip(first, last)]
    order = torch.randperm(sum(held) + 1, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(last), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, (a, b) in enumerate(zip(first, last)):
        table[r, a:b] = order[at:at + b - a]
        at += b - a
    return table, sum(held) + 1


def _pages(gen, pages, nkv, page, hd):
    """A plane of the cache as earlier steps left it: codes and scales of values whose size differs from head to head and token to token."""
    codes = torch.empty((pages, nkv, page, hd), dtype=torch.int8, device=DEV)
    scales = torch.empty((pages, nkv, page // BLOCK), dtype=torch.float32, device=DEV)
    size = torch.exp(0.5 * _normal(gen, 1, nkv, 1, 1))
    for a in range(0, pages, 4096):
        b = min(pages, a + 4096)
        x = _normal(gen, b - a, nkv, page, hd) * size * torch.exp(0.2 * _normal(gen, b - a, nkv, page, 1))
        s = x.view(b - a, nkv, page // BLOCK, BLOCK * hd).abs().amax(-1) / 127.0
        codes[a:b] = torch.round(x / s.repeat_interleave(BLOCK, 2).unsqueeze(-1)).to(torch.int8)
        scales[a:b] = s
    return codes, scales


class _State:
    pass


def prepare(case, seed):
    gen = _generator(seed)
    s = _State()
    s.case = case
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a few likely tokens far above the rest, as a trained model's rows have them
        s.logits = 2.5 * _normal(gen, rows, vocab)
        likely = torch.randint(0, vocab, (rows, 12), generator=gen, device=DEV)
        s.logits.scatter_add_(1, likely, 6.0 + 3.0 * _normal(gen, rows, 12))
        s.ids = likely[:, 0].to(torch.int32).contiguous()
        if case["masked"]:
            gone = torch.rand((rows, vocab), generator=gen, device=DEV) < case["masked"]
            gone.scatter_(1, likely[:, :6], False)
            s.logits.masked_fill_(gone, -math.inf)
        return s
    counts, starts = _portions(case)
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    dtype = getattr(torch, case["dtype"])
    last = [(a + c + page - 1) // page for a, c in zip(starts, counts)]
    if case["kind"] == "append":
        first = [a // page for a in starts]         # the pages before were given back: the layer has a window
    else:
        w = case["window"]
        first = [max(0, a - w + 1) // page if w else 0 for a in starts]
    table, pages = _table(gen, first, last)
    s.step = Step(counts, starts, table)
    s.k, s.k_scale = _pages(gen, pages, nkv, page, hd)
    s.v, s.v_scale = _pages(gen, pages, nkv, page, hd)
    T = s.step.num_tokens
    if case["kind"] == "attend":
        s.q = _normal(gen, T, nq * hd).to(dtype)
        s.out = torch.empty_like(s.q)
        return s
    width = (nq + 2 * nkv) * hd
    s.qkv = _normal(gen, case["slices"], T, width) / math.sqrt(case["slices"])
    s.bias = 0.2 * _normal(gen, width) if case["bias"] else None
    s.q_norm = 1.0 + 0.1 * _normal(gen, hd) if case["norm"] else None
    s.k_norm = 1.0 + 0.1 * _normal(gen, hd) if case["norm"] else None
    rot = case["rot"]
    s.inv_freq = (1.0 / THETA ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(DEV) if rot else None
    s.q = torch.empty((T, nq * hd), dtype=dtype, device=DEV)
    s.k_values = torch.empty(s.k.shape, dtype=torch.bfloat16, device=DEV)
    s.v_values = torch.empty(s.v.shape, dtype=torch.bfloat16, device=DEV)
    return s


def run(state):
    kind = state.case["kind"]
    if kind == "append":
        return _append(state)
    return _attend(state) if kind == "attend" else _logprobs(state)


def _values(codes, scales, out):
    """code * scale of a plane, rounded once to bfloat16."""
    n, h, p, d = codes.shape
    blocks = (n, h, p // BLOCK, BLOCK, d)
    torch.mul(codes.view(blocks), scales.view(n, h, p // BLOCK, 1, 1), out=out.view(blocks))
    return out


def _append(s):
    c, step = s.case, s.step
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    if own:
        from kestrel_llm_b200.csrc import ops
        ops.attn_prepare_q8(ops.Partials(s.qkv, s.bias), s.q_norm, s.k_norm, EPS, s.inv_freq, c["rot"], step.positions, step.cu_seqlens,
                            step.block_table(0), page, s.k, s.v, s.k_scale, s.v_scale, s.q, nq, nkv, hd, rot_mode=int(c["interleaved"]))
    else:
        T = step.num_tokens
        x = s.qkv.sum(0)
        if s.bias is not None:
            x = x + s.bias
        q, k, v = (t.view(T, -1, hd) for t in x.split([nq * hd, nkv * hd, nkv * hd], 1))
        q, k = _turn(s, _norm(q, s.q_norm)), _turn(s, _norm(k, s.k_norm))
        s.q.copy_(q.reshape(T, nq * hd))
        _write(s, k, s.k, s.k_scale)
        _write(s, v, s.v, s.v_scale)
    return {"q": s.q, "k": _values(s.k, s.k_scale, s.k_values), "v": _values(s.v, s.v_scale, s.v_values), "k_scale": s.k_scale,
            "v_scale": s.v_scale}


def _norm(x, weight):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _turn(s, x):
    rot = s.case["rot"]
    if not rot:
        return x
    angle = s.step.positions.double().unsqueeze(1) * s.inv_freq.double()        # far positions: 32 bits would lose the angle
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    if s.case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rot:]], -1)
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _write(s, x, plane, scales):
    """x [T, kv heads, hd] to the tokens' places in a plane of codes and scales."""
    step, page = s.step, s.case["page"]
    pages, nkv, _, hd = plane.shape
    per = page // BLOCK
    pos, seq = step.positions.long(), step.seq_of_token.long()
    at = step.table[seq, pos // page].long()
    slot = pos % page
    block = at * per + slot // BLOCK                                            # of every token, among all of the cache
    blocks = scales.transpose(1, 2).reshape(pages * per, nkv)                   # a copy
    largest = torch.zeros_like(blocks).scatter_reduce(0, block.unsqueeze(1).expand(-1, nkv), x.abs().amax(-1), "amax")
    head = step.cu_seqlens[:-1].long()                                          # every request's first token
    begun = (pos[head] % BLOCK > 0).unsqueeze(1)                                # ... joins a block that is there already
    before = blocks[block[head]]
    new = blocks.clone()
    new[block] = torch.clamp((largest / 127.0)[block], min=LOWEST)
    joined = torch.maximum(new[block[head]], before)
    new[block[head]] = torch.where(begun, joined, new[block[head]])
    # codes of a begun block under its new scale
    rows = (slot[head] // BLOCK * BLOCK).unsqueeze(1) + torch.arange(BLOCK, device=DEV)
    old = plane[at[head].unsqueeze(1), :, rows]                                 # [requests, BLOCK, kv heads, hd]
    again = torch.round(old.float() * (before / new[block[head]]).view(-1, 1, nkv, 1)).to(torch.int8)
    there = (rows < slot[head].unsqueeze(1)) & begun
    plane[at[head].unsqueeze(1), :, rows] = torch.where(there[..., None, None], again, old)
    plane[at, :, slot] = torch.clamp(torch.round(x / new[block].unsqueeze(-1)), -127, 127).to(torch.int8)
    scales.copy_(new.view(pages, per, nkv).transpose(1, 2))


def _attend(s):
    c, step = s.case, s.step
    nq, nkv, hd, page, window = c["nq"], c["nkv"], c["hd"], c["page"], c["window"]
    scale = 1.0 / math.sqrt(hd)
    if own:
        from kestrel_llm_b200.csrc import ops
        ops.attention_q8(s.q, s.k, s.v, s.k_scale, s.v_scale, s.out, step, step.block_table(0), page, nq, nkv, hd, window, scale)
        return s.out
    # padded to the longest request: queries [n, kv heads, rows of (token, head), hd], keys [n, kv heads, keys, hd]
    n, M, G = step.num_seqs, step.max_count, nq // nkv
    low = max(0, min(step.starts) - window + 1) // page if window else 0
    table = step.table[:, low:].long().clamp(min=0)
    keys = table.shape[1] * page

    def gather(plane, scales):
        x = plane[table].float() * scales[table].repeat_interleave(BLOCK, 3).unsqueeze(-1)      # [n, pages, kv heads, page, hd]
        return x.transpose(1, 2).reshape(n, nkv, keys, hd)
    counts = step.cu_seqlens[1:] - step.cu_seqlens[:-1]
    i = torch.arange(M, device=DEV)
    real = i < counts.unsqueeze(1)
    token = (step.cu_seqlens[:-1].unsqueeze(1) + i).clamp(max=step.num_tokens - 1).long()
    q = s.q.view(-1, nkv, G, hd)[token].float().permute(0, 2, 1, 3, 4).reshape(n, nkv, M * G, hd)
    pos = ((step.kv_lens - counts).unsqueeze(1) + i).repeat_interleave(G, 1).view(n, 1, M * G, 1)
    key = torch.arange(keys, device=DEV) + low * page
    seen = (key <= pos) & (key > pos - window if window else key >= 0)
    w = (torch.matmul(q, gather(s.k, s.k_scale).transpose(2, 3)) * scale).masked_fill(~seen, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    o = torch.matmul(w / w.sum(-1, keepdim=True), gather(s.v, s.v_scale))
    o = o.view(n, nkv, M, G, hd).transpose(1, 2).reshape(n, M, nq * hd)
    s.out.copy_(o[real])
    return s.out


def _logprobs(s):
    top = s.case["top"]
    if own:
        from kestrel_llm_b200.csrc import ops
        got = ops.token_logprobs(s.logits, s.ids, top)
        return {"logprobs": got.logprobs, "entropy": got.entropy, "top_ids": got.top_ids, "top_logprobs": got.top_logprobs}
    x = s.logits - s.logits.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lp = x - torch.log(total)
    entropy = -(torch.where(e > 0, lp, 0.0) * (e / total)).sum(1)
    given = lp.gather(1, s.ids.long().unsqueeze(1)).squeeze(1)
    if top:
        ids = torch.sort(s.logits, dim=1, descending=True, stable=True).indices[:, :top]
    else:
        ids = torch.empty((s.logits.shape[0], 0), dtype=torch.int64, device=DEV)
    return {"logprobs": given, "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprobs": lp.gather(1, ids)}


# ---- the same in 64 bits, from the definitions ------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    given, entropy, ids, likeliest = [], [], [], []
    for r in range(case["rows"]):
        x = s.logits[r].double()
        lse = torch.logsumexp(x, 0)
        p = torch.exp(x - lse)
        at = p > 0
        given.append(x[int(s.ids[r])] - lse)
        entropy.append(lse - (p[at] * x[at]).sum())
        # the top-th largest value, everything above it, and of its equals those with the lowest indices
        k = case["top"]
        if k:
            kth = torch.topk(x, k).values[-1]
            above, equal = (x > kth).nonzero().flatten(), (x == kth).nonzero().flatten()
            pick = torch.cat([above, equal[:k - above.numel()]])
            pick = pick[torch.argsort(-x[pick], stable=True)]
            ids.append(pick.to(torch.int32))
            likeliest.append(x[pick] - lse)
    none = torch.empty((case["rows"], 0), device=DEV)
    return {"logprobs": torch.stack(given), "entropy": torch.stack(entropy), "top_ids": torch.stack(ids) if ids else none.to(torch.int32),
            "top_logprobs": torch.stack(likeliest) if ids else none.double()}


def _exact_append(case, s):
    nq, nkv, hd, page, rot = case["nq"], case["nkv"], case["hd"], case["page"], case["rot"]
    T = s.step.num_tokens
    x = s.qkv.double().sum(0)
    if s.bias is not None:
        x = x + s.bias.double()
    x = x.view(T, nq + 2 * nkv, hd)
    parts = [x[:, :nq].clone(), x[:, nq:nq + nkv].clone()]
    for i, w in enumerate((s.q_norm, s.k_norm)):
        if w is not None:
            parts[i] = parts[i] / torch.sqrt((parts[i] ** 2).mean(-1, keepdim=True) + EPS) * w.double()
        for j in range(rot // 2):                  # a pair of dimensions as a complex number, turned
            a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + rot // 2)
            turn = torch.polar(torch.ones(T, dtype=torch.float64, device=DEV), s.step.positions.double() * s.inv_freq[j].double())
            z = torch.complex(parts[i][..., a], parts[i][..., b]) * turn.unsqueeze(1)
            parts[i][..., a], parts[i][..., b] = z.real, z.imag
    out = {"q": parts[0].reshape(T, nq * hd)}
    table = s.step.table.tolist()
    for name, new, codes, scales in (("k", parts[1], s.k, s.k_scale), ("v", x[:, nq + nkv:], s.v, s.v_scale)):
        codes, scales = codes.double(), scales.double()
        for r in range(s.step.num_seqs):
            t0, p0, p1 = s.step.cu_seqlens_host[r], s.step.starts[r], s.step.kv_lens_host[r]
            for b in range(p0 // BLOCK, (p1 + BLOCK - 1) // BLOCK):
                lo, hi = max(p0, b * BLOCK), min(p1, (b + 1) * BLOCK)
                at, first = table[r][b * BLOCK // page], b * BLOCK % page
                rows = new[t0 + lo - p0:t0 + hi - p0].transpose(0, 1)           # [kv heads, tokens, hd]
                scale = torch.clamp(rows.abs().amax((1, 2)) / 127.0, min=LOWEST)
                there = lo - b * BLOCK                                          # codes that are there already
                if there:
                    before = scales[at, :, first // BLOCK]
                    scale = torch.maximum(scale, before)
                    kept = codes[at, :, first:first + there] * (before / scale).view(-1, 1, 1)
                    codes[at, :, first:first + there] = torch.round(kept)
                codes[at, :, first + there:first + there + hi - lo] = torch.round(rows / scale.view(-1, 1, 1))
                scales[at, :, first // BLOCK] = scale
        out[name] = codes * scales.repeat_interleave(BLOCK, 2).unsqueeze(-1)
        out[name + "_scale"] = scales
    return out


def _exact_attend(case, s):
    nq, nkv, hd, page, window = case["nq"], case["nkv"], case["hd"], case["page"], case["window"]
    G = nq // nkv
    out = torch.empty((s.step.num_tokens, nq, hd), dtype=torch.float64, device=DEV)
    for r in range(s.step.num_seqs):
        t0, p0, p1 = s.step.cu_seqlens_host[r], s.step.starts[r], s.step.kv_lens_host[r]
        lo = max(0, p0 - window + 1) if window else 0
        key = torch.arange(lo, p1, device=DEV)
        at, slot = s.step.table[r].long()[key // page], key % page
        pos = torch.arange(p0, p1, device=DEV).unsqueeze(1)
        hidden = (key > pos) | ((pos - key >= window) if window else (key < 0))
        for h in range(nkv):
            k = s.k[at, h, slot].double() * s.k_scale[at, h, slot // BLOCK].double().unsqueeze(1)
            v = s.v[at, h, slot].double() * s.v_scale[at, h, slot // BLOCK].double().unsqueeze(1)
            for g in range(G):
                q = s.q[t0:t0 + p1 - p0].view(-1, nq, hd)[:, h * G + g].double()
                w = (q @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[t0:t0 + p1 - p0, h * G + g] = torch.softmax(w, 1) @ v
    return out.view(-1, nq * hd)


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    counts, starts = _portions(case)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    size = 4 if case["dtype"] == "float32" else 2
    T = sum(counts)
    if case["kind"] == "append":
        width = (nq + 2 * nkv) * hd
        blocks = sum((a + c + BLOCK - 1) // BLOCK - a // BLOCK for a, c in zip(starts, counts))
        # the product's slices and the queries; a new code a value, and a scale a block and head
        return {"bytes": 4 * case["slices"] * T * width + size * T * nq * hd + 2 * T * nkv * hd + 8 * blocks * nkv,
                "flops": T * width * (case["slices"] + 8)}
    keys = scores = 0
    for c, a in zip(counts, starts):
        w = case["window"] or a + c
        keys += a + c - max(0, a - w + 1)
        scores += sum(min(p + 1, w) for p in range(a, a + c))
    return {"bytes": 2 * keys * nkv * hd + 8 * keys * nkv // BLOCK + 2 * size * T * nq * hd, "flops": 4 * scores * nq * hd}
