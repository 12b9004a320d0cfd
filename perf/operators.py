"""Cases and plain forms of the operators for a batch of sequences that bring different numbers of new tokens.

One serving step over a paged cache runs three of them one after another:

  index      pages for the new tokens, their positions and slots, from the request lengths on the GPU; and the
             pages of tokens that are dropped again (drafts that were not accepted) given back
  rope       per-head RMSNorm + rotary embedding + append of the step's keys and values to their slots
  attention  causal attention of every sequence's new tokens over its pages

`listed` names the cases, `draw` makes more of the same ranges, `prepare` makes the inputs, `run` computes one pass
(`own` true: through the library; false: with elementary torch operations), `exact` the same in 64 bits.
"""
import math
import random

import torch

own = False

D = 128  # head_dim of the cache


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of the batch that the benchmark decodes: one token each
        dict(name="index decode 32", op="index", seqs=32, new_min=1, new_max=1, past_min=1023, past_max=16383, page=16, lengths=1),
        # drafts of one to nine tokens for a few hundred sequences, some without any
        dict(name="index drafts 300", op="index", seqs=300, new_min=0, new_max=9, past_min=0, past_max=8191, page=16, lengths=2),
        # prompts arriving at a large pool: every token opens or fills a page
        dict(name="index prompts 1000", op="index", seqs=1000, new_min=1, new_max=127, past_min=0, past_max=3000, page=32, lengths=3),
        # a single decode token: what counts is the latency
        dict(name="rope one token", op="rope", tokens=1, pad=0, dtype="f16", q_heads=48, kv_heads=8, rotary=64, norm=True, fused=False, page=16, past_max=16383),
        # a small step padded to the size of a captured graph, f32 projections
        dict(name="rope 77 of 96 f32", op="rope", tokens=77, pad=19, dtype="f32", q_heads=72, kv_heads=8, rotary=128, norm=True, fused=False, page=16, past_max=32767),
        # a full step of prompt chunks, q / k / v being parts of one projection's rows
        dict(name="rope chunk 8192", op="rope", tokens=8192, pad=0, dtype="f16", q_heads=48, kv_heads=8, rotary=64, norm=True, fused=True, page=16, past_max=30000),
        # one token after a short prompt: latency
        dict(name="attention one token", op="attention", decodes=1, draft=1, chunks=0, chunk=0, past_min=99, past_max=99, q_heads=48, kv_heads=8, page=16, window=0, gate=False, lengths=11),
        # the benchmark's decode batch, as a step that could also hold chunks
        dict(name="attention decode 32", op="attention", decodes=32, draft=1, chunks=0, chunk=0, past_min=1023, past_max=16383, q_heads=48, kv_heads=8, page=16, window=0, gate=True, lengths=12),
        # verification of drafts of up to six tokens
        dict(name="attention drafts 24x6", op="attention", decodes=24, draft=6, chunks=0, chunk=0, past_min=600, past_max=12000, q_heads=64, kv_heads=8, page=16, window=0, gate=False, lengths=13),
        # a sliding layer: the window hides most of the cache, a chunk of an odd length among the decodes
        dict(name="attention window 512", op="attention", decodes=40, draft=1, chunks=1, chunk=777, past_min=10, past_max=9000, q_heads=64, kv_heads=8, page=16, window=512, gate=True, lengths=14),
        # decodes and two prompt chunks in one step, as a scheduler packs them
        dict(name="attention mixed 2x1024", op="attention", decodes=46, draft=1, chunks=2, chunk=1024, past_min=500, past_max=8191, q_heads=48, kv_heads=8, page=16, window=0, gate=False, lengths=15),
        # a long prompt's next chunk over what is cached of it
        dict(name="attention chunk 4096", op="attention", decodes=0, draft=0, chunks=1, chunk=4096, past_min=8192, past_max=8192, q_heads=48, kv_heads=8, page=16, window=0, gate=False, lengths=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["index", "rope", "attention", "attention"])
    page = rng.choice([16, 16, 32, 48, 64])
    if op == "index":
        new_min = rng.choice([0, 1])
        return dict(op="index", seqs=_log_int(rng, 1, 1000), new_min=new_min, new_max=_log_int(rng, 1, 127),
                    past_min=rng.choice([0, 1, 15, 500]), past_max=_log_int(rng, 600, 16383), page=page, lengths=rng.randrange(1 << 30))
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 9, 12, 16])
    if op == "rope":
        q_heads = min(q_heads, 9 * kv_heads)
        return dict(op="rope", tokens=_log_int(rng, 1, 8000), pad=rng.choice([0, 0, 1, 13]), dtype=rng.choice(["f16", "f16", "f32"]),
                    q_heads=min(q_heads, 48), kv_heads=kv_heads if min(q_heads, 48) % kv_heads == 0 else 1, rotary=rng.choice([64, 128]),
                    norm=rng.random() < 0.7, fused=rng.random() < 0.5, page=page, past_max=_log_int(rng, 16, 60000))
    q_heads = q_heads if q_heads <= 72 else 6 * kv_heads
    shape = rng.choice(["decode", "drafts", "chunks", "mixed"])
    decodes = 0 if shape == "chunks" else _log_int(rng, 1, 48)
    chunks = rng.choice([1, 2, 3]) if shape in ("chunks", "mixed") else 0
    return dict(op="attention", decodes=decodes, draft=1 if shape in ("decode", "mixed") else rng.randint(2, 8), chunks=chunks,
                chunk=_log_int(rng, 9, 1100) if chunks else 0, past_min=rng.choice([0, 1, 40]), past_max=_log_int(rng, 60, 11000),
                q_heads=q_heads, kv_heads=kv_heads, page=page, window=rng.choice([0, 0, 0, 512, 100, 1]), gate=rng.random() < 0.3,
                lengths=rng.randrange(1 << 30))


def _lengths(case):
    """(cached, new) tokens of every sequence: set by the case alone. Lengths spread over their logarithm, chunks among the decodes."""
    rng = random.Random(case["lengths"])
    spread = lambda: _log_int(rng, case["past_min"] + 1, max(case["past_max"], case["past_min"]) + 1) - 1  # noqa: E731
    if case["op"] == "index":
        return [(spread(), rng.randint(case["new_min"], case["new_max"])) for _ in range(case["seqs"])]
    both = [(spread(), rng.randint(1, case["draft"])) for _ in range(case["decodes"])]
    for _ in range(case["chunks"]):
        both.insert(rng.randint(0, len(both)), (spread(), case["chunk"]))
    return both


def _cdiv(a, b):
    return (a + b - 1) // b


def work(case):
    if case["op"] == "index":
        both = _lengths(case)
        p = case["page"]
        fresh = sum(_cdiv(a + n, p) - _cdiv(a, p) for a, n in both)
        tokens = sum(n for _, n in both)
        return dict(bytes=4 * (7 * len(both) + 2 * tokens + 5 * fresh), flops=4 * tokens)
    if case["op"] == "rope":
        t, heads = case["tokens"], case["q_heads"] + 2 * case["kv_heads"]
        size = 2 if case["dtype"] == "f16" else 4
        return dict(bytes=t * heads * D * (size + 2) + 8 * (t + case["pad"]), flops=8 * t * heads * D)
    w, nbytes, pairs = case["window"], 0, 0
    for a, n in _lengths(case):
        seen = min(a + n, w + n - 1) if w else a + n
        nbytes += seen * case["kv_heads"] * D * 4 + n * case["q_heads"] * D * 4 + 4 * _cdiv(seen, case["page"])
        pairs += n * w - sum(max(0, w - (a + t + 1)) for t in range(n)) if w else n * a + n * (n + 1) // 2
    return dict(bytes=nbytes, flops=4 * D * case["q_heads"] * pairs)


# ------------------------------------------------------------------------------------------------ inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "index":
        return _prepare_index(case, g)
    if case["op"] == "rope":
        return _prepare_rope(case, g)
    return _prepare_attention(case, g)


def _table(both, page, pages):
    """Page table [seqs, widest] with `pages` (a tensor of distinct ids) dealt out to the cached tokens, -1 elsewhere."""
    used = torch.tensor([_cdiv(a, page) for a in both], device="cuda")
    width = max(1, max(_cdiv(a, page) for a in both))
    j = torch.arange(width, device="cuda")
    first = torch.cumsum(used, 0) - used
    at = (first[:, None] + j).clamp(max=max(0, pages.numel() - 1))
    return torch.where(j < used[:, None], pages[at], -1).to(torch.int32)


def _prepare_index(case, g):
    both, p = _lengths(case), case["page"]
    total = sum(_cdiv(a + n, p) for a, n in both)
    num_pages = total + 64
    ids = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    used = sum(_cdiv(a, p) for a, _ in both)
    width = max(1, max(_cdiv(a + n, p) for a, n in both))
    pages = torch.full((len(both), width), -1, dtype=torch.int32, device="cuda")
    t = _table([a for a, _ in both], p, ids[:max(1, used)])
    pages[:, :t.shape[1]] = t
    free = torch.zeros(num_pages, dtype=torch.int32, device="cuda")
    free[:num_pages - used] = ids[used:]
    tokens = sum(n for _, n in both)
    return dict(case=case, pages=pages, lens=_ints([a for a, _ in both]), free_pages=free, free_count=_ints([num_pages - used]),
                new=_ints([n for _, n in both]), max_tokens=max(1, tokens + tokens // 8), keep=_ints([a for a, _ in both]))


def _inv_freq(rotary, device="cuda"):
    return (1.0 / 500000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).to(torch.float32).to(device)


def _prepare_rope(case, g):
    t, n, hq, hkv, p = case["tokens"], case["tokens"] + case["pad"], case["q_heads"], case["kv_heads"], case["page"]
    dtype = torch.float16 if case["dtype"] == "f16" else torch.float32
    if case["fused"]:
        qkv = torch.randn((n, hq + 2 * hkv, D), generator=g, device="cuda", dtype=dtype)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        q, k, v = (torch.randn((n, h, D), generator=g, device="cuda", dtype=dtype) for h in (hq, hkv, hkv))
    num_pages = _cdiv(t, p) + 3
    slots = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    slots[:t] = torch.randperm(num_pages * p, generator=g, device="cuda")[:t].to(torch.int32)
    positions = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    positions[:t] = torch.randint(0, case["past_max"] + 1, (t,), generator=g, device="cuda", dtype=torch.int32)
    k_pool = torch.zeros((num_pages, hkv, p, D), dtype=torch.float16, device="cuda")
    norms = [1 + 0.2 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None for _ in range(2)]
    return dict(case=case, q=q, k=k, v=v, slots=slots, positions=positions, k_pool=k_pool, v_pool=torch.zeros_like(k_pool), q_norm=norms[0],
                k_norm=norms[1], eps=1e-6, inv_freq=_inv_freq(case["rotary"]), q_out=torch.zeros((n, hq, D), dtype=torch.float16, device="cuda"))


def _prepare_attention(case, g):
    both, p, hkv = _lengths(case), case["page"], case["kv_heads"]
    past, new = [a for a, _ in both], [n for _, n in both]
    num_pages = sum(_cdiv(a + n, p) for a, n in both) + 5
    ids = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    k_pool = torch.randn((num_pages, hkv, p, D), generator=g, device="cuda", dtype=torch.float16)
    v_pool = torch.randn((num_pages, hkv, p, D), generator=g, device="cuda", dtype=torch.float16)
    q = torch.randn((starts[-1], case["q_heads"], D), generator=g, device="cuda", dtype=torch.float16)
    gate = 2 * torch.randn((starts[-1], case["q_heads"]), generator=g, device="cuda") if case["gate"] else None
    return dict(case=case, past=past, new=new, starts=starts, pages=_table([a + n for a, n in both], p, ids), past_lens=_ints(past),
                q_starts=_ints(starts), k_pool=k_pool, v_pool=v_pool, q=q, gate=gate, out=torch.zeros_like(q))


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"index": _own_index, "rope": _own_rope, "attention": _own_attention}[op](s)
    return {"index": _plain_index, "rope": _plain_rope, "attention": _plain_attention}[op](s)


_be = None


def _backend():
    global _be
    if _be is None:
        from inferno_b200 import CudaBackend
        _be = CudaBackend(torch.cuda.current_device())
    return _be


def _own_index(s):
    be = _backend()
    if "index" not in s:
        s["index"] = be.device_index(s["pages"], s["lens"], s["free_pages"], s["free_count"], s["case"]["page"])
        s["batch"] = be.prepare_ragged_batch(s["lens"].numel(), s["max_tokens"])
    b = be.device_index_append(s["index"], s["new"], s["batch"])
    be.device_index_truncate(s["index"], s["keep"])
    return dict(past=b.past_lens, starts=b.q_starts, positions=b.positions, slots=b.slots, pages=s["pages"], lens=s["lens"],
                free_pages=s["free_pages"], free_count=s["free_count"])


def _own_rope(s):
    be = _backend()
    if "pool" not in s:
        s["pool"] = be.kv_pool(s["k_pool"], s["v_pool"])
        s["rope"] = be.prepare_rope_table(s["inv_freq"].cpu(), s["case"]["rotary"], 1.0)
    be.rope_append_gqa_ragged(s["q"], s["k"], s["v"], s["rope"], s["pool"], s["positions"], s["slots"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], eps=s["eps"], out=s["q_out"])
    return dict(q=s["q_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _own_attention(s):
    be = _backend()
    if "pool" not in s:
        s["pool"] = be.kv_pool(s["k_pool"], s["v_pool"])
        s["table"] = be.page_table(s["pages"], s["past_lens"], validate_on_host=False)
    return be.gqa_attention_ragged(s["q"], s["pool"], s["table"], s["q_starts"], sliding_window=s["case"]["window"], gate=s["gate"], out=s["out"])


def _plain_index(s):
    p, pages, lens, free, count = s["case"]["page"], s["pages"], s["lens"], s["free_pages"], s["free_count"]
    n, past, seqs = s["new"], s["lens"].clone(), s["lens"].numel()
    ends = torch.cumsum(n, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    mapped, after = (past + p - 1) // p, (past + n + p - 1) // p
    first = torch.cumsum(after - mapped, 0) - (after - mapped)  # fresh pages of the sequences before this one
    # the table: page j of a sequence that is not mapped yet is the next one from the top of the stack
    j = torch.arange(pages.shape[1], device=pages.device)
    fresh = (j >= mapped[:, None]) & (j < after[:, None])
    top = (count - 1 - (first[:, None] + j - mapped[:, None])).clamp(0, free.numel() - 1)
    pages.copy_(torch.where(fresh, free[top.long()], pages))
    # every token's sequence, position and slot; rows behind the last token hold -1
    t = torch.arange(s["max_tokens"], device=pages.device)
    seq = torch.searchsorted(ends, t, right=True).clamp(max=seqs - 1)
    live = t < ends[-1]
    pos = past[seq] + t - starts[seq]
    page = pages[seq, (pos // p).clamp(0, pages.shape[1] - 1)]
    positions = torch.where(live, pos, -1).to(torch.int32)
    slots = torch.where(live, page * p + pos % p, -1).to(torch.int32)
    lens.copy_(past + n)
    count.sub_((after - mapped).sum().to(torch.int32))
    # pages of the tokens beyond `keep` go back: the last sequence's last page first
    have, hold = (lens + p - 1) // p, (s["keep"] + p - 1) // p
    gone = have - hold
    behind = torch.flip(torch.cumsum(torch.flip(gone, [0]), 0), [0]) - gone
    drop = (j >= hold[:, None]) & (j < have[:, None])
    at = torch.where(drop, count + behind[:, None] + have[:, None] - 1 - j, free.numel())
    more = torch.cat([free, free[:1]])  # one place more, for the pages that stay
    more.scatter_(0, at.reshape(-1).long(), pages.reshape(-1))
    free.copy_(more[:-1])
    pages.masked_fill_(drop, -1)
    lens.copy_(s["keep"])
    count.add_(gone.sum().to(torch.int32))
    return dict(past=past, starts=starts, positions=positions, slots=slots, pages=pages, lens=lens, free_pages=free, free_count=count)


def _plain_rope(s):
    t, p, half = s["case"]["tokens"], s["case"]["page"], s["case"]["rotary"] // 2
    angle = s["positions"][:t].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x[:t].float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).half()

    s["q_out"][:t] = turned(s["q"], s["q_norm"])
    slot = s["slots"][:t].long()
    s["k_pool"][slot // p, :, slot % p] = turned(s["k"], s["k_norm"])
    s["v_pool"][slot // p, :, slot % p] = s["v"][:t].half()
    return dict(q=s["q_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_attention(s):
    c = s["case"]
    hq, hkv, w = c["q_heads"], c["kv_heads"], c["window"]
    g = hq // hkv
    for b, (past, n) in enumerate(zip(s["past"], s["new"])):
        rows = slice(s["starts"][b], s["starts"][b] + n)
        total = past + n
        ids = s["pages"][b, :_cdiv(total, c["page"])].long()
        k, v = (x[ids].permute(1, 0, 2, 3).reshape(hkv, -1, D)[:, :total].float() for x in (s["k_pool"], s["v_pool"]))
        q = s["q"][rows].float().view(n, hkv, g, D).permute(1, 0, 2, 3).reshape(hkv, n * g, D)
        score = (q @ k.transpose(1, 2)).mul_(D ** -0.5)
        key, row = torch.arange(total, device=q.device), past + torch.arange(n, device=q.device)
        hidden = key > row[:, None]
        if w:
            hidden |= key <= row[:, None] - w
        score.masked_fill_(hidden.repeat_interleave(g, 0), -math.inf)
        score.sub_(score.amax(-1, keepdim=True)).exp_()
        o = (score @ v) / score.sum(-1, keepdim=True)
        o = o.view(hkv, n, g, D).permute(1, 0, 2, 3).reshape(n, hq, D)
        if s["gate"] is not None:
            o = o * torch.log1p(torch.exp(s["gate"][rows]))[..., None]
        s["out"][rows] = o.half()
    return s["out"]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"index": _exact_index, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](s)


def _exact_index(s):
    """The step token by token, on the host."""
    p = s["case"]["page"]
    pages, lens, new = s["pages"].tolist(), s["lens"].tolist(), s["new"].tolist()
    stack = s["free_pages"].tolist()
    count = s["free_count"].item()
    positions, slots, starts = [], [], [0]
    for b, n in enumerate(new):
        for pos in range(lens[b], lens[b] + n):
            if pos % p == 0:
                count -= 1
                pages[b][pos // p] = stack[count]
            positions.append(pos)
            slots.append(pages[b][pos // p] * p + pos % p)
        starts.append(starts[-1] + n)
    for b in reversed(range(len(new))):
        for j in reversed(range(_cdiv(lens[b], p), _cdiv(lens[b] + new[b], p))):
            stack[count], pages[b][j] = pages[b][j], -1
            count += 1
    rest = [-1] * (s["max_tokens"] - len(slots))
    return dict(past=s["lens"].cpu(), starts=torch.tensor(starts), positions=torch.tensor(positions + rest), slots=torch.tensor(slots + rest),
                pages=torch.tensor(pages), lens=torch.tensor(lens), free_pages=torch.tensor(stack), free_count=torch.tensor([count]))


def _exact_rope(s):
    c = s["case"]
    n, half = c["tokens"], c["rotary"] // 2
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), s["positions"][:n, None].double() * s["inv_freq"].double())

    def rows(x, weight, rotate):
        x = x[:n].to(torch.float64)
        if rotate and weight is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + s["eps"]) * weight.double()
        if rotate:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn[:, None]
            x = torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
        return x

    q = torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda")
    q[:n] = rows(s["q"], s["q_norm"], True)
    pools = []
    for x, weight, rotate in ((s["k"], s["k_norm"], True), (s["v"], None, False)):
        num_pages, heads, p, _ = s["k_pool"].shape
        flat = torch.zeros((num_pages * p, heads, D), dtype=torch.float64, device="cuda")
        flat[s["slots"][:n].long()] = rows(x, weight, rotate)
        pools.append(flat.view(num_pages, p, heads, D).transpose(1, 2))
    return dict(q=q, k_pool=pools[0], v_pool=pools[1])


def _exact_attention(s):
    c = s["case"]
    g, p = c["q_heads"] // c["kv_heads"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["new"]):
        past, t0 = s["past"][b], s["starts"][b]
        at = torch.arange(past + n, device="cuda")
        page, slot = s["pages"][b].long()[at // p], at % p
        # how far back a key lies, seen from each new token; visible: 0 <= back, and back < window if there is one
        back = (past + torch.arange(n, device="cuda"))[:, None] - at
        seen = (back >= 0) & (back < c["window"]) if c["window"] else back >= 0
        for h in range(c["q_heads"]):
            k, v = (x[page, h // g, slot].double() for x in (s["k_pool"], s["v_pool"]))
            weight = torch.softmax(torch.where(seen, s["q"][t0:t0 + n, h].double() @ k.T / math.sqrt(D), -torch.inf), -1)
            out[t0:t0 + n, h] = weight @ v
    if s["gate"] is not None:
        out *= torch.nn.functional.softplus(s["gate"].double())[..., None]
    return out
