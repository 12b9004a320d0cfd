"""The ragged-batch operators against plain 64-bit statements: page bookkeeping on the GPU, RoPE + append by slot, and
attention of each sequence's new tokens over its pages."""
import random

import numpy as np
import pytest

from tests.ragged import Batch, assert_rows_close, rope_reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from inferno_b200 import CudaBackend
    b = CudaBackend(0)
    yield b
    b.device_flush()
    b.close()


def ints(be, v):
    return torch.tensor(v, dtype=torch.int32, device=be.device)


# ------------------------------------------------------------------------------------------------ index
@pytest.mark.parametrize("seqs,P,max_tokens", [(1, 16, 40), (7, 16, 900), (33, 48, 300), (1500, 1, 5000), (2100, 64, 70000), (16384, 16, 60000)])
def test_device_index_follows_the_host_index(be, seqs, P, max_tokens):
    """A random run of appends and cuts: table, lengths, order of the free list as the host's one-by-one bookkeeping."""
    from inferno_b200.paged import PagedIndex
    rng = random.Random(seqs * 100 + P)
    max_pages = 6
    num_pages = seqs * 4 + 5
    host = PagedIndex(num_pages, P, seqs, max_pages)
    index = be.prepare_device_index(num_pages, P, seqs, max_pages)
    batch = be.prepare_ragged_batch(seqs, max_tokens)
    for step in range(6):
        lens = [host.cached_tokens(b) for b in range(seqs)]
        new, left, free = [], max_tokens, host.free_pages()
        for b in range(seqs):
            n = min(rng.choice([0, 1, 1, rng.randint(0, 3 * P)]), max_pages * P - lens[b], left)
            if -(-(lens[b] + n) // P) - -(-lens[b] // P) > free:
                n = 0
            free -= -(-(lens[b] + n) // P) - -(-lens[b] // P)
            left -= n
            new.append(n)
        be.device_index_append(index, ints(be, new), batch)
        be.device_flush()
        positions, slots, starts = [], [], [0]
        for b, n in enumerate(new):
            if n:
                host.append(b, n)
            for t in range(lens[b], lens[b] + n):
                page, off = host.token_location(b, t)
                positions.append(t)
                slots.append(page * P + off)
            starts.append(starts[-1] + n)
        pages, hl = host.arrays()
        assert batch.past_lens.tolist() == lens and batch.q_starts.tolist() == starts
        assert batch.positions.tolist() == positions + [-1] * (max_tokens - len(positions))
        assert batch.slots.tolist() == slots + [-1] * (max_tokens - len(slots))
        assert np.array_equal(index.pages.cpu().numpy(), pages) and np.array_equal(index.lens.cpu().numpy(), hl)
        assert index.free_count.item() == host.free_pages()
        # cut some sequences, release some, leave the rest; the host goes through them from the last to the first
        keep = [rng.choice([-1, -1, 0, rng.randint(0, int(n))]) for n in hl]
        be.device_index_truncate(index, ints(be, keep))
        for b in reversed(range(seqs)):
            if keep[b] == 0:
                host.release(b)
            elif keep[b] > 0:
                _host_cut(host, b, keep[b])
        be.device_flush()
        pages, hl = host.arrays()
        assert np.array_equal(index.pages.cpu().numpy(), pages) and np.array_equal(index.lens.cpu().numpy(), hl)
        assert index.free_count.item() == host.free_pages()


def _host_cut(host, b, length):
    """A cut with the host index's calls: it gives back all pages, the last one first, and takes the ones that stay off the
    stack again, in their old order."""
    host.release(b)
    host.append(b, length)


def test_append_then_truncate_restores_the_index(be):
    rng = random.Random(5)
    index = be.prepare_device_index(400, 16, 40, 20)
    batch = be.prepare_ragged_batch(40, 4000)
    be.device_index_append(index, ints(be, [rng.randint(0, 60) for _ in range(40)]), batch)
    before = [t.clone() for t in (index.pages, index.lens, index.free_pages, index.free_count)]
    be.device_index_append(index, ints(be, [rng.randint(0, 60) for _ in range(40)]), batch)
    be.device_index_truncate(index, batch.past_lens)
    be.device_flush()
    for was, t in zip(before, (index.pages, index.lens, index.free_pages, index.free_count)):
        assert torch.equal(was, t)


@pytest.mark.parametrize("max_tokens", [50, 20001])
def test_index_outputs_at_any_word(be, max_tokens):
    """Layout buffers that start between 16-byte boundaries, as views of a larger one do; words around them stay."""
    index = be.prepare_device_index(3000, 16, 5, 2000)
    want = be.device_index_append(index, ints(be, [7, 0, max_tokens // 2, 3, 1]), be.prepare_ragged_batch(5, max_tokens))
    be.device_index_truncate(index, want.past_lens)
    arena = torch.full((2 * max_tokens + 64,), -7, dtype=torch.int32, device=be.device)
    sizes, at, views = (5, 6, max_tokens, max_tokens), 1, []
    for n in sizes:
        views.append(arena[at:at + n])
        at += n + 2
    got = be.device_index_append(index, ints(be, [7, 0, max_tokens // 2, 3, 1]), type(want)(*views))
    be.device_flush()
    for name in ("past_lens", "q_starts", "positions", "slots"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert int((arena == -7).sum()) == arena.numel() - sum(sizes)


@pytest.mark.parametrize("new,max_tokens,why", [
    ([10, 10, 10], 29, "length"),        # more rows than the buffers hold
    ([65, 0, 0], 100, "length"),         # beyond the table row of four pages
    ([1, -1, 1], 100, "length"),         # a negative length
    ([60, 60, 60], 200, "free list"),    # eleven pages in the pool, twelve needed
    ([2 ** 31 - 1, 2 ** 31 - 1, 2], 100, "length"),
])
def test_a_step_that_does_not_fit_changes_nothing(be, new, max_tokens, why):
    from inferno_b200 import InfernoError
    index = be.prepare_device_index(11, 16, 3, 4)
    batch = be.prepare_ragged_batch(3, max_tokens)
    be.device_index_append(index, ints(be, [3, 0, 1]), batch)
    be.device_flush()
    before = [t.clone() for t in (index.pages, index.lens, index.free_pages, index.free_count)]
    be.device_index_append(index, ints(be, new), batch)
    with pytest.raises(InfernoError, match=why):
        be.device_flush()
    be.device_index_truncate(index, ints(be, [4, 0, 0]))  # sequence 0 holds three tokens
    with pytest.raises(InfernoError, match="length"):
        be.device_flush()
    for was, t in zip(before, (index.pages, index.lens, index.free_pages, index.free_count)):
        assert torch.equal(was, t)
    assert batch.q_starts.tolist() == [0] * 4 and batch.past_lens.tolist() == [3, 0, 1]
    assert (batch.positions == -1).all() and (batch.slots == -1).all()


def _index_state(index):
    """What an index holds: the table, the lengths, the stack and its count."""
    return index.pages.clone(), index.lens.clone(), index.free_pages[:index.free_count.item()].clone(), index.free_count.clone()


@pytest.mark.parametrize("seqs", [3, 9000])
@pytest.mark.parametrize("bad", [-1, -2 ** 31, "pool", 2 ** 31 - 1])
def test_pages_outside_the_pool_refuse_the_call(be, seqs, bad):
    """A page id that is none, where a call takes, fills or gives back that page: it is reported and nothing changes.  The bad
    one stands with the last sequence, which another of the cluster's CTAs may hold than the first ones."""
    from inferno_b200 import InfernoError
    P, last = 16, seqs - 1
    num_pages = 3 * seqs + 4
    bad = num_pages if bad == "pool" else bad
    index = be.prepare_device_index(num_pages, P, seqs, 4)
    max_tokens = 40 * seqs
    batch = be.prepare_ragged_batch(seqs, max_tokens)
    be.device_index_append(index, ints(be, [20] * seqs), batch)  # two pages each, the second one partly filled
    be.device_flush()

    def refused(call):
        before = _index_state(index)
        call()
        with pytest.raises(InfernoError, match="page id"):
            be.device_flush()
        for was, now in zip(before, _index_state(index)):
            assert torch.equal(was, now)

    def refused_step(new):
        refused(lambda: be.device_index_append(index, new, batch))
        assert (batch.q_starts == 0).all() and (batch.positions == -1).all() and (batch.slots == -1).all()
        assert torch.equal(batch.past_lens, index.lens)

    step = ints(be, [1] * last + [30])  # two more pages for the last sequence, none for the others
    # a page that would be given back
    good = index.pages[last].clone()
    for slot in (0, 1):
        index.pages[last, slot] = bad
        refused(lambda: be.device_index_truncate(index, torch.zeros_like(index.lens)))
        index.pages[last] = good
    # a page that the step would go on filling
    index.pages[last, 1] = bad
    refused_step(step)
    index.pages[last] = good
    # a page that the step would take
    top = index.free_count.item() - 1
    for at in (top, top - 1):
        kept = index.free_pages[at].item()
        index.free_pages[at] = bad
        refused_step(step)
        index.free_pages[at] = kept
    # pages that no call touches may hold anything: a full one, a slot behind the length, an entry further down the stack
    index.pages[last, 0] = bad
    index.pages[0, 3] = bad
    index.free_pages[0] = bad
    be.device_index_append(index, step, batch)
    be.device_index_truncate(index, batch.past_lens)
    be.device_flush()
    index.pages[last, 0] = good[0]
    be.device_index_truncate(index, torch.zeros_like(index.lens))
    be.device_flush()
    assert index.free_count.item() == num_pages and (index.lens == 0).all()


def test_index_calls_refuse_an_index_elsewhere(be):
    """Tensors that are not on the context's GPU reach no kernel, whichever call gets the index first."""
    from inferno_b200 import InfernoError
    from inferno_b200.backend import DeviceIndex
    index = be.prepare_device_index(8, 16, 2, 4)
    away = DeviceIndex(index.pages.cpu(), index.lens.cpu(), index.free_pages.cpu(), index.free_count.cpu(), index.desc)
    for call in (lambda: be.device_index_reset(away), lambda: be.device_index_truncate(away, ints(be, [0, 0])),
                 lambda: be.device_index_append(away, ints(be, [1, 1]), be.prepare_ragged_batch(2, 4))):
        with pytest.raises(InfernoError) as e:
            call()
        assert e.value.kind == "Argument"


# ------------------------------------------------------------------------------------------------ rope + append
@pytest.mark.parametrize("T,pad,Hq,Hkv,rotary,norm,dtype,fused,P,far", [
    (1, 0, 48, 8, 64, True, torch.float16, False, 16, 100),
    (1, 0, 1, 1, 128, True, torch.float32, True, 16, 5),
    (5, 3, 6, 1, 128, False, torch.float32, False, 48, 30000),
    (77, 19, 72, 8, 64, True, torch.float32, True, 16, 1 << 20),
    (300, 0, 12, 4, 128, True, torch.float16, True, 32, 1 << 30),
    (33, 1, 7, 7, 64, True, torch.float16, False, 64, 2000),
    (9, 0, 128, 1, 64, True, torch.float16, False, 16, 2000),
    (700, 4, 48, 8, 64, True, torch.float16, True, 16, 16384),
])
def test_rope_append_ragged(be, T, pad, Hq, Hkv, rotary, norm, dtype, fused, P, far):
    g = torch.Generator(device=be.device).manual_seed(T * 31 + Hq)
    n, pages = T + pad, -(-T // P) + 2
    if fused:
        qkv = torch.randn((n, Hq + 2 * Hkv, 128), generator=g, device=be.device).to(dtype)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        q, k, v = (torch.randn((n, h, 128), generator=g, device=be.device).to(dtype) for h in (Hq, Hkv, Hkv))
    order = torch.randperm(n, generator=g, device=be.device)  # padding anywhere in the step
    live = order[:T]
    slots = torch.full((n,), -1, dtype=torch.int32, device=be.device)
    positions = slots.clone()
    slots[live] = torch.randperm(pages * P, generator=g, device=be.device)[:T].to(torch.int32)
    positions[live] = torch.randint(0, far, (T,), generator=g, device=be.device, dtype=torch.int32)
    qw, kw = ((1 + 0.2 * torch.randn(128, generator=g, device=be.device)) if norm else None for _ in range(2))
    inv = (1 / 500000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float()
    pool = be.prepare_kv_pool(pages, P, Hkv)
    pool.k.fill_(5.0)
    pool.v.fill_(6.0)
    out = torch.full((n, Hq, 128), 7.0, dtype=torch.float16, device=be.device)
    be.rope_append_gqa_ragged(q, k, v, be.prepare_rope_table(inv, rotary, 1.25), pool, positions, slots, q_norm=qw, k_norm=kw, out=out)
    be.device_flush()
    inv = inv.to(be.device)
    slot = slots[live].long()
    assert_rows_close(out[live], rope_reference(q[live], qw, 1e-6, positions[live], inv, rotary, 1.25), "q")
    assert_rows_close(pool.k[slot // P, :, slot % P], rope_reference(k[live], kw, 1e-6, positions[live], inv, rotary, 1.25), "k")
    assert torch.equal(pool.v[slot // P, :, slot % P], v[live].half())
    rest = torch.ones(n, dtype=torch.bool, device=be.device)
    rest[live] = False
    assert (out[rest] == 7).all()
    unused = torch.ones(pages * P, dtype=torch.bool, device=be.device)
    unused[slot] = False
    for p, filler in ((pool.k, 5), (pool.v, 6)):
        assert (p.transpose(1, 2).reshape(pages * P, Hkv, 128)[unused] == filler).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rotary,norm", [(0, ""), (64, "q"), (64, "k"), (128, "q"), (128, "k")])
def test_rope_append_ragged_without_a_table_or_with_one_norm(be, dtype, rotary, norm):
    """Without a table rows are stored as they are; a norm weight for one of the two leaves the other its size."""
    T, Hq, Hkv, P = 21, 12, 4, 16
    g = torch.Generator(device=be.device).manual_seed(44)
    q, k, v = (torch.randn((T, h, 128), generator=g, device=be.device).to(dtype) for h in (Hq, Hkv, Hkv))
    qw, kw = (1 + 0.2 * torch.randn(128, generator=g, device=be.device) if norm == x else None for x in "qk")
    slots = torch.randperm(3 * P, generator=g, device=be.device)[:T].to(torch.int32)
    positions = torch.randint(0, 5000, (T,), generator=g, device=be.device, dtype=torch.int32)
    pool = be.prepare_kv_pool(3, P, Hkv)
    inv = (1 / 10000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / max(1, rotary))).float()
    rope = be.prepare_rope_table(inv, rotary, 1.0) if rotary else None
    out = be.rope_append_gqa_ragged(q, k, v, rope, pool, positions, slots, q_norm=qw, k_norm=kw)
    be.device_flush()
    slot = slots.long()
    stored = pool.k[slot // P, :, slot % P]
    assert torch.equal(pool.v[slot // P, :, slot % P], v.half())
    if not rotary:
        assert torch.equal(out, q.half()) and torch.equal(stored, k.half())
        return
    inv = inv.to(be.device)
    assert_rows_close(out, rope_reference(q, qw, 1e-6, positions, inv, rotary), "q")
    assert_rows_close(stored, rope_reference(k, kw, 1e-6, positions, inv, rotary), "k")


def test_rope_append_ragged_agrees_with_the_uniform_call(be):
    """One token count for all sequences: the same rows as rope_append_gqa, the rotation aside, whose angle is taken in 64
    bits here: at positions below 2048 the two angles differ by 2^-14 at most, the rows by that times their size."""
    B, T, Hq, Hkv, P = 3, 20, 12, 2, 16
    g = torch.Generator(device=be.device).manual_seed(8)
    q, k, v = (torch.randn((B, T, h, 128), generator=g, device=be.device) for h in (Hq, Hkv, Hkv))
    past = [0, 13, 2000]
    index = be.prepare_device_index(200, P, B, 130)
    batch = be.prepare_ragged_batch(B, 3000)
    be.device_index_append(index, ints(be, past), batch)
    step = be.prepare_ragged_batch(B, B * T)
    be.device_index_append(index, ints(be, [T] * B), step)
    inv = (1 / 10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float()
    rope, w = be.prepare_rope_table(inv, 64, 1.0), torch.ones(128, device=be.device)
    one, two = be.prepare_kv_pool(200, P, Hkv), be.prepare_kv_pool(200, P, Hkv)
    a = be.rope_append_gqa(q, k, v, rope, one, be.page_table(index.pages, step.past_lens), q_norm=w, k_norm=w)
    b = be.rope_append_gqa_ragged(*(x.reshape(B * T, -1, 128) for x in (q, k, v)), rope, two, step.positions, step.slots, q_norm=w, k_norm=w)
    be.device_flush()
    assert torch.equal(one.v, two.v)
    tol = 2 * 2.0 ** -11 + 2.0 ** -14
    assert ((a.reshape(b.shape).double() - b.double()).abs() <= tol * b.double().abs().amax(-1, keepdim=True)).all()
    assert ((one.k.double() - two.k.double()).abs() <= tol * two.k.double().abs().amax(-1, keepdim=True)).all()


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("past,new,Hq,Hkv,P,window,gate", [
    ([0], [1], 6, 1, 16, 0, False),                        # one key
    ([15], [1], 48, 8, 16, 0, False),                      # the last slot of a page
    ([127, 128, 129], [1, 1, 1], 48, 8, 16, 0, True),      # around a key tile
    ([0, 0], [17, 1], 8, 8, 16, 0, False),                 # one head per KV head
    ([3, 0, 40], [0, 0, 5], 6, 2, 16, 0, False),           # sequences without new tokens
    ([5, 1, 300, 0], [21, 22, 43, 130], 48, 8, 16, 0, True),   # around a tile of 21 tokens x 6 heads
    ([1000], [257], 12, 2, 48, 0, False),                  # pages that end inside a tile
    ([2000, 9], [6, 3], 64, 8, 64, 0, False),              # drafts
    ([77, 200], [9, 33], 9, 1, 16, 0, False),              # nine heads per KV head
    ([50], [40], 128, 1, 32, 0, True),                     # 128 heads per KV head
    ([31], [9], 100, 1, 16, 0, False),                     # 100: one token per 128 rows
    ([500, 3], [300, 1], 16, 2, 16, 1, False),             # a window of one key
    ([700, 10, 0], [64, 1, 200], 16, 2, 16, 100, True),
    ([4000, 511, 512], [1, 3, 777], 64, 8, 16, 512, False),
    ([0], [1300], 24, 4, 128, 0, False),
    ([20000, 30], [2, 50], 6, 1, 16, 0, False),            # one long sequence for one KV head: split over its keys
    ([9000], [130], 12, 2, 16, 0, False),                  # a chunk split over its keys
])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_attention_ragged(be, past, new, Hq, Hkv, P, window, gate, out_dtype):
    Batch(be.device, past, new, Hq, Hkv, P, seed=sum(past) + Hq, window=window, spare_rows=3).check(be, gate, out_dtype)


@pytest.mark.parametrize("seed", range(12))
def test_attention_ragged_random_batches(be, seed):
    rng = random.Random(seed)
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 5, 6, 7, 8, 9, 11, 12, 16, 33])
    B = rng.choice([1, 2, 5, 40, 100])
    past = [rng.choice([0, 1, rng.randint(0, 300), rng.randint(0, 3000)]) for _ in range(B)]
    new = [rng.choice([0, 1, 1, 1, rng.randint(0, 9), rng.randint(0, 200) if B < 40 else 1]) for _ in range(B)]
    new[rng.randrange(B)] += 1
    Batch(be.device, past, new, Hkv * G, Hkv, rng.choice([16, 32, 48, 80]), seed=seed, window=rng.choice([0, 0, 1, 77, 512]),
          spare_rows=rng.choice([0, 5]), tight=rng.random() < 0.5).check(be, rng.random() < 0.5, scale=rng.choice([0.0, 0.05]))


def test_attention_ragged_more_sequences_than_threads(be):
    """Metadata of thousands of sequences, most of them idle."""
    B = 3000
    new = [1 if b % 7 == 3 else 0 for b in range(B)]
    new[B - 1] = 5
    Batch(be.device, [b % 61 for b in range(B)], new, 6, 1, 16, seed=1).check(be)


def test_attention_ragged_twice_gives_the_same_bits(be):
    b = Batch(be.device, [30000, 100, 5000], [1, 300, 7], 48, 8, 16, seed=3)
    assert torch.equal(b.check(be), b.check(be))


@pytest.mark.parametrize("past,new,Hq,Hkv", [
    ([30000, 7], [2, 90], 12, 2),  # one item cut many times, a light one; two streams
    ([9000], [130], 12, 2),
    ([30000], [5], 64, 8),
    ([100, 3], [20, 1], 12, 2),
])
def test_attention_ragged_keeps_nothing_of_the_call_before(be, past, new, Hq, Hkv):
    """Tiles, TMEM and scratch full of NaN from another call leave every bit of the next one alone."""
    b = Batch(be.device, past, new, Hq, Hkv, 16, seed=20)
    d = Batch(be.device, past, new, Hq, Hkv, 16, seed=20)
    d.q.fill_(float("nan"))

    def run(x):
        return be.gqa_attention_ragged(x.q, be.kv_pool(x.k, x.v), be.page_table(x.pages, x.past_lens, validate_on_host=False),
                                       x.q_starts, out_dtype=torch.float32)

    first = run(b)
    assert torch.isnan(run(d)).all()
    assert torch.equal(run(b), first)
    be.device_flush()


def test_attention_ragged_pages_below_the_window_given_back(be):
    """Host mirrors check the pages that a row can see and no others: the first row sees keys from past + 1 - window on."""
    from inferno_b200 import InfernoError
    b = Batch(be.device, [95, 200], [1, 3], 12, 2, 16, seed=22, window=64)  # lowest visible keys 32 and 137
    want = b.check(be)
    b.pages[0, :2] = -1
    b.pages[1, :8] = -1
    pool = be.kv_pool(b.k, b.v)
    got = be.gqa_attention_ragged(b.q, pool, be.page_table(b.pages, b.past_lens), b.q_starts, sliding_window=64)
    be.device_flush()
    assert torch.equal(got, want)
    b.pages[0, 2] = -1
    with pytest.raises(InfernoError, match="page"):
        be.gqa_attention_ragged(b.q, pool, be.page_table(b.pages, b.past_lens), b.q_starts, sliding_window=64)


@pytest.mark.parametrize("past,new,Hq,Hkv,window", [
    ([4150], [42], 6, 1, 0),       # 33 parts: the last two cuts move to the item's end, one in each 32 of them
    ([9000], [42], 6, 1, 4150),    # the same in a window
    ([8310], [42], 6, 1, 0),       # 65 parts
    ([12440, 3], [42, 1], 6, 1, 0),
])
def test_attention_ragged_items_of_many_pieces(be, past, new, Hq, Hkv, window):
    b = Batch(be.device, past, new, Hq, Hkv, 16, seed=24, window=window)
    assert torch.equal(b.check(be), b.check(be))


@pytest.mark.parametrize("past", list(range(4090, 4230, 10)) + list(range(8200, 8400, 20)))
def test_attention_ragged_around_whole_warps_of_cuts(be, past):
    Batch(be.device, [past, 20], [42, 2], 6, 1, 16, seed=past).check(be)


def test_a_pool_beyond_32_bits(be):
    """Pages whose rows lie more than 2^32 values into the pools: the same bits as in a pool of a few pages."""
    Hq, Hkv, P, past, new = 48, 8, 16, 70, 40
    far = 2 ** 32 // (Hkv * P * 128)  # pages below the first one used
    need = -(-(past + new) // P)
    if torch.cuda.mem_get_info(be.device)[0] < 2 * (far + need) * Hkv * P * 256 + 2 ** 31:
        pytest.skip("needs 18 GB of device memory")
    g = torch.Generator(device=be.device).manual_seed(2)
    cached = torch.randn((2, need, Hkv, P, 128), generator=g, device=be.device, dtype=torch.float16)
    q, k, v = (torch.randn((new, h, 128), generator=g, device=be.device) for h in (Hq, Hkv, Hkv))
    rope = be.prepare_rope_table(torch.ones(64) / (1 + torch.arange(64)), 128, 1.0)
    outs = []
    for first in (0, far):
        pools = [torch.empty((first + need, Hkv, P, 128), dtype=torch.float16, device=be.device) for _ in range(2)]
        for pool, rows in zip(pools, cached):
            pool[first:] = rows
        pool = be.kv_pool(*pools)
        positions = past + torch.arange(new, dtype=torch.int32, device=be.device)
        q16 = be.rope_append_gqa_ragged(q, k, v, rope, pool, positions, positions + first * P)
        table = be.page_table(first + torch.arange(need, dtype=torch.int32, device=be.device)[None], ints(be, [past]), validate_on_host=False)
        outs.append((be.gqa_attention_ragged(q16, pool, table, ints(be, [0, new])), pools[0][first:].clone(), pools[1][first:].clone()))
        be.device_flush()
        del pool, pools
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_attention_ragged_without_new_tokens(be):
    """A step in which no sequence has a token writes nothing, before and after one that cuts items over many CTAs."""
    b = Batch(be.device, [30000, 500], [1, 30], 12, 2, 16, seed=23)
    pool, table = be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens, validate_on_host=False)
    out = torch.full(b.q.shape, 7.0, dtype=torch.float16, device=be.device)
    for _ in range(2):
        be.gqa_attention_ragged(b.q, pool, table, ints(be, [0, 0, 0]), out=out)
        be.device_flush()
        assert (out == 7).all()
        b.check(be)


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_attention_ragged_rows_at_odd_sixteen_bytes(be, out_dtype):
    """Queries and output that begin 16 bytes into a 32-byte sector."""
    b = Batch(be.device, [300, 5000, 40], [90, 2, 30], 12, 2, 16, seed=21)
    pool, table = be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens, validate_on_host=False)
    want = be.gqa_attention_ragged(b.q, pool, table, b.q_starts, out_dtype=out_dtype)
    pad = 8 if out_dtype == torch.float16 else 4
    q = torch.empty(b.q.numel() + 8, dtype=torch.float16, device=be.device)[8:].view(b.q.shape).copy_(b.q)
    arena = torch.full((b.q.numel() + 2 * pad,), 7.0, dtype=out_dtype, device=be.device)
    got = be.gqa_attention_ragged(q, pool, table, b.q_starts, out=arena[pad:-pad].view(b.q.shape))
    be.device_flush()
    assert torch.equal(got, want) and (arena[:pad] == 7).all() and (arena[-pad:] == 7).all()


def test_attention_ragged_large_and_equal_scores(be):
    """Scores in the hundreds (the softmax is one key), and equal ones (the mean of the values)."""
    b = Batch(be.device, [300], [60], 12, 2, 16, seed=4, filler=0.0)
    b.q *= 40
    pool, table = be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens, validate_on_host=False)
    got = be.gqa_attention_ragged(b.q, pool, table, b.q_starts, out_dtype=torch.float32)
    be.device_flush()
    from tests.ragged import attention_reference
    want, size = attention_reference(b.q, b.k, b.v, b.pages, b.past, b.new)
    # 32-bit scores of size 40 * 12: off by 128 * 2^-24 * sum |q k| scale (about 300) at most, which a weight sees in its exponent
    tol = (2.0 ** -11 + 128 * 2.0 ** -24 * 300) * size + 2.0 ** -15
    assert ((got.double() - want).abs() <= tol).all()
    b.q.zero_()
    b.check(be)


@pytest.mark.parametrize("past,new,Hq,Hkv,window", [
    ([300, 0], [1, 2], 12, 2, 0),          # few rows
    ([700, 40], [9, 1], 6, 1, 0),          # a light item
    ([500], [20], 6, 1, 0),                # one stream of many rows
    ([700], [64], 12, 2, 100),             # two streams, tiles that hide every key from some row
    ([30000, 40], [2, 43], 6, 1, 0),       # items cut over many CTAs: the maxima meet in the join
    ([9000], [130], 12, 2, 0),
])
@pytest.mark.parametrize("size,scale", [(2.0 ** 13, 0.0), (2.0 ** 10, 0.0), (1.0, 1e15), (2.0 ** 13, 1e8), (1.0, 1e-20)])
@pytest.mark.parametrize("negative", [False, True])
def test_attention_ragged_scores_of_any_size(be, past, new, Hq, Hkv, window, size, scale, negative):
    """Queries and keys that are small whole numbers times a power of two: every sum of products is exact in 32 bits, so the
    weights are known however large the scores are.  Equal scores differ by nothing, others by at least size^2 * scale, which
    is rounded three times on its way into the exponent (3 * 2^-24 of it: below the tolerance where the weight is not 0)."""
    b = Batch(be.device, past, new, Hq, Hkv, 16, seed=40, window=window)
    b.q = (b.q * 1.2).round().clamp(-3, 3) * size
    b.k = (b.k * 1.2).round().clamp(-3, 3) * size  # slots that no row sees stay NaN
    if negative:
        b.q, b.k = b.q.abs(), -b.k.abs()
    for out_dtype in (torch.float16, torch.float32):
        b.check(be, out_dtype=out_dtype, scale=scale)


def test_attention_ragged_bad_page_and_bad_lengths_are_reported(be):
    from inferno_b200 import InfernoError
    b = Batch(be.device, [40, 100], [3, 2], 12, 2, 16, seed=6, filler=0.0)
    pool = be.kv_pool(b.k, b.v)

    def run(pages, lens, starts, rows=None):
        out = torch.full(b.q.shape, 7.0, dtype=torch.float16, device=be.device)
        table = be.page_table(pages, lens, validate_on_host=False)
        be.gqa_attention_ragged(b.q, pool, table, starts, out=out)
        with pytest.raises(InfernoError) as e:
            be.device_flush()
        return out, str(e.value)

    want = be.gqa_attention_ragged(b.q, pool, be.page_table(b.pages, b.past_lens), b.q_starts)
    be.device_flush()
    pages = b.pages.clone()
    pages[0, 1] = b.k.shape[0]
    out, why = run(pages, b.past_lens, b.q_starts)
    assert "page id" in why and torch.equal(out[3:], want[3:]) and torch.isfinite(out).all()
    for lens in ([40, 5000], [40, -1], [40, 2 ** 31 - 1]):
        out, why = run(b.pages, ints(be, lens), b.q_starts)
        assert "length" in why and torch.equal(out[:3], want[:3]) and (out[3:] == 7).all()
    for starts in ([0, 3, 6], [0, 3, 2], [0, 3, 2 ** 31 - 1]):
        out, why = run(b.pages, b.past_lens, ints(be, starts))
        assert "length" in why and torch.equal(out[:3], want[:3]) and (out[3:] == 7).all()
    assert torch.equal(be.gqa_attention_ragged(b.q, pool, be.page_table(b.pages, b.past_lens), b.q_starts), want)
    be.device_flush()


def test_attention_ragged_equals_the_uniform_prefill_and_decode(be):
    """Where the older calls offer the same thing the results agree: both are within one tolerance of the exact value."""
    B, T, Hq, Hkv, P = 2, 150, 12, 2, 16
    b = Batch(be.device, [37, 300], [T, T], Hq, Hkv, P, seed=9, filler=0.0)
    pool, table = be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens)
    got = be.gqa_attention_ragged(b.q, pool, table, b.q_starts, out_dtype=torch.float32)
    old = be.gqa_prefill_paged(b.q.view(B, T, Hq, 128), pool, table, out_dtype=torch.float32)
    be.device_flush()
    assert (got - old.view(got.shape)).abs().max() <= 2 * (2.0 ** -11 + 2.0 ** -14) * b.v.abs().max()


@pytest.mark.parametrize("past,Hq,Hkv,P,window", [
    ([0, 15, 127, 128, 700], 48, 8, 16, 0),
    ([3000, 1, 511], 12, 2, 64, 512),
    ([20000, 40], 64, 8, 16, 0),
    ([90, 5000], 8, 8, 32, 100),
])
@pytest.mark.parametrize("gate", [False, True])
def test_attention_ragged_of_one_token_each_equals_the_uniform_decode(be, past, Hq, Hkv, P, window, gate):
    """Both calls are within one tolerance of the exact value (assert_attention_close, 32-bit output), so within two of each
    other.  The uniform call takes the gate as log(1 + e^g), whose sum is off by 2^-24 and the logarithm by as much:
    2^-23 of the ungated row, and what is left of the two gates' roundings counts as often again."""
    from tests.ragged import attention_reference
    n = len(past)
    b = Batch(be.device, past, [1] * n, Hq, Hkv, P, seed=42, window=window, filler=0.0)
    pool, g = be.kv_pool(b.k, b.v), b.gate if gate else None
    got = be.gqa_attention_ragged(b.q, pool, be.page_table(b.pages, b.past_lens), b.q_starts, sliding_window=window, gate=g, out_dtype=torch.float32)
    old = be.gqa_decode_paged(b.q, pool, be.page_table(b.pages, b.past_lens + 1), max(past) + 1, sliding_window=window, gate=g, out_dtype=torch.float32)
    be.device_flush()
    _, size = attention_reference(b.q, b.k, b.v, b.pages, past, [1] * n, window, g)
    _, ungated = attention_reference(b.q, b.k, b.v, b.pages, past, [1] * n, window)
    tol = 2 * ((2.0 ** -11 + 2.0 ** -14 + 2.0 ** -24) * size + (b.keys * 2.0 ** -25 + 1e-7) * size.amax(-1, keepdim=True)) + 2.0 ** -22 * ungated
    err = (got.double() - old.double()).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("filler", [float("nan"), float("inf"), 6e4])
def test_attention_ragged_rows_behind_the_last_sequence_may_hold_anything(be, filler):
    """A batch padded to the size of a captured step: queries and gates of the padding enter tiles with real rows and
    change none of their bits."""
    for past, new, Hq, Hkv in (([300, 40], [1, 2], 12, 2), ([700], [9], 6, 1), ([500], [20], 6, 1), ([700, 9000], [64, 30], 12, 2)):
        b = Batch(be.device, past, new, Hq, Hkv, 16, seed=43, spare_rows=70)
        want = b.check(be, gate=True)
        b.q[b.rows:] = filler
        b.gate[b.rows:] = filler
        assert torch.equal(b.check(be, gate=True), want)


# ------------------------------------------------------------------------------------------------ the step
def _step_setup(be, seqs=6, P=16, Hq=12, Hkv=2, pages=300, width=40, max_tokens=160):
    s = dict(index=be.prepare_device_index(pages, P, seqs, width), batch=be.prepare_ragged_batch(seqs, max_tokens),
             pool=be.prepare_kv_pool(pages, P, Hkv), new=torch.zeros(seqs, dtype=torch.int32, device=be.device),
             q=torch.zeros((max_tokens, Hq, 128), device=be.device), k=torch.zeros((max_tokens, Hkv, 128), device=be.device),
             v=torch.zeros((max_tokens, Hkv, 128), device=be.device),
             q16=torch.zeros((max_tokens, Hq, 128), dtype=torch.float16, device=be.device),
             out=torch.zeros((max_tokens, Hq, 128), dtype=torch.float16, device=be.device))
    s["inv"] = (1 / 500000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float()
    s["rope"] = be.prepare_rope_table(s["inv"], 64, 1.0)
    s["table"] = be.page_table(s["index"].pages, s["batch"].past_lens, validate_on_host=False)
    assert s["table"].pages.data_ptr() == s["index"].pages.data_ptr()

    def step():
        b = be.device_index_append(s["index"], s["new"], s["batch"])
        be.rope_append_gqa_ragged(s["q"], s["k"], s["v"], s["rope"], s["pool"], b.positions, b.slots, out=s["q16"])
        be.gqa_attention_ragged(s["q16"], s["pool"], s["table"], b.q_starts, out=s["out"])

    return s, step


def _run_steps(be, s, step, seed):
    """Chunks, decodes, idle steps, cuts and releases; every output against the whole history in 64 bits."""
    rng = random.Random(seed)
    g = torch.Generator(device=be.device).manual_seed(seed)
    seqs, Hq, Hkv = s["new"].numel(), s["q"].shape[1], s["k"].shape[1]
    history = [[torch.zeros((0, Hkv, 128), device=be.device, dtype=torch.float16)] * 2 for _ in range(seqs)]
    for _ in range(9):
        new = [rng.choice([0, 1, 1, rng.randint(2, 6), rng.randint(0, 60)]) for _ in range(seqs)]
        while sum(new) > s["q"].shape[0]:
            new[rng.randrange(seqs)] = 0
        s["new"].copy_(ints(be, new))
        for x in (s["q"], s["k"], s["v"]):
            x.copy_(torch.randn(x.shape, generator=g, device=be.device))
        s["out"].fill_(7.0)
        step()
        be.device_flush()
        t0 = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            rows = slice(t0, t0 + n)
            past = history[b][0].shape[0]
            pos = past + torch.arange(n, device=be.device)
            k = rope_reference(s["k"][rows], None, 0, pos, s["inv"].to(be.device), 64)
            slots = s["batch"].slots[rows].long()
            P = s["pool"].k.shape[2]
            stored = s["pool"].k[slots // P, :, slots % P]
            assert_rows_close(stored, k, "k")
            assert_rows_close(s["q16"][rows], rope_reference(s["q"][rows], None, 0, pos, s["inv"].to(be.device), 64), "q")
            history[b] = [torch.cat([history[b][0], stored]), torch.cat([history[b][1], s["v"][rows].half()])]
            # the same rows over a cache laid out in one piece
            total = past + n
            kp, vp = (x[None].transpose(1, 2).contiguous() for x in history[b])
            from tests.ragged import assert_attention_close, attention_reference
            want, size = attention_reference(s["q16"][rows], kp, vp, torch.zeros((1, 1), dtype=torch.int32, device=be.device), [past], [n])
            assert_attention_close(s["out"][rows], want, size, total, f"sequence {b}")
            t0 += n
        assert (s["out"][t0:] == 7).all()
        keep = [rng.choice([-1, -1, 0, rng.randint(0, h[0].shape[0])]) for h in history]
        be.device_index_truncate(s["index"], ints(be, keep))
        history = [[x[:c] if c >= 0 else x for x in h] for h, c in zip(history, keep)]
    be.device_flush()


def test_steps_of_a_server(be):
    _run_steps(be, *_step_setup(be), seed=1)


def test_captured_steps_replay_with_other_lengths(be):
    """One captured step, replayed for every batch of _run_steps; the captured kernels read the lengths on the GPU."""
    s, step = _step_setup(be)
    graph = be.capture_graph(step)
    be.device_index_reset(s["index"])
    _run_steps(be, s, graph.replay, seed=2)


def test_a_first_call_without_tokens_is_enough_before_a_capture(be):
    """The context's first call allocates the scratch, whatever its step holds, so that the next one can be captured."""
    from inferno_b200 import CudaBackend
    b = Batch(be.device, [9000], [130], 12, 2, 16, seed=41)
    want = b.check(be)
    torch.cuda.synchronize()
    own = CudaBackend(0, stream=torch.cuda.Stream())
    pool, table, out = own.kv_pool(b.k, b.v), own.page_table(b.pages, b.past_lens, validate_on_host=False), torch.zeros_like(b.q)
    own.gqa_attention_ragged(b.q[:0], pool, table, ints(be, [0, 0]))
    graph = own.capture_graph(lambda: own.gqa_attention_ragged(b.q, pool, table, b.q_starts, out=out), warmup=0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:b.rows], want[:b.rows])
    own.close()


def test_two_graphs_of_one_context_share_its_scratch(be):
    """Two captured attentions, both with items cut over many CTAs, replayed in turn and twice in a row, with an eager call
    between: each gives the bits of its own eager call."""
    batches = [Batch(be.device, [30000, 7], [2, 90], 12, 2, 16, seed=30), Batch(be.device, [9000, 100, 5000], [130, 30, 1], 48, 8, 16, seed=31)]
    want = [b.check(be) for b in batches]
    outs = [torch.zeros_like(b.q) for b in batches]

    def call(i):
        b = batches[i]
        be.gqa_attention_ragged(b.q, be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens, validate_on_host=False), b.q_starts, out=outs[i])

    graphs = [be.capture_graph(lambda i=i: call(i)) for i in range(2)]
    for order in ((0, 1), (1, 0), (0, 0), (1, 1)):
        for o in outs:
            o.zero_()
        for i in order:
            graphs[i].replay()
        batches[0].check(be)
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(outs[i][:batches[i].rows], want[i][:batches[i].rows])
    be.device_flush()


def test_two_contexts_on_two_streams(be):
    """Split attention of two contexts at the same time: neither sees the other's partial results."""
    from inferno_b200 import CudaBackend
    streams = [torch.cuda.Stream() for _ in range(2)]
    backends = [CudaBackend(0, stream=s) for s in streams]
    batches = [Batch(be.device, [30000 + 1000 * i, 7], [2, 90], 12, 2, 16, seed=20 + i) for i in range(2)]
    want = [b.check(be) for b in batches]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, b in zip(backends, batches):
            got.append(x.gqa_attention_ragged(b.q, x.kv_pool(b.k, b.v), x.page_table(b.pages, b.past_lens, validate_on_host=False), b.q_starts))
    for x in backends:
        x.device_flush()
    for i, o in enumerate(got):
        assert torch.equal(o[:batches[i % 2].rows], want[i % 2][:batches[i % 2].rows])
    for x in backends:
        x.close()


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(be):
    from inferno_b200 import InfernoError
    b = Batch(be.device, [4, 0], [2, 3], 12, 2, 16, seed=1, filler=0.0)
    pool, table = be.kv_pool(b.k, b.v), be.page_table(b.pages, b.past_lens)

    def refuses(kind, call, *args, **kw):
        with pytest.raises(InfernoError) as e:
            call(*args, **kw)
        assert e.value.kind == kind, e.value

    att = be.gqa_attention_ragged
    refuses("DType", att, b.q.float(), pool, table, b.q_starts)
    refuses("DType", att, b.q, pool, table, b.q_starts.long())
    refuses("DType", att, b.q, pool, table, b.q_starts, out_dtype=torch.bfloat16)
    refuses("ShapeMismatch", att, b.q[..., :64].contiguous(), pool, table, b.q_starts)
    refuses("ShapeMismatch", att, b.q, pool, table, b.q_starts[:2])
    refuses("ShapeMismatch", att, b.q[:, :3].contiguous(), pool, table, b.q_starts)
    refuses("ShapeMismatch", att, b.q, pool, table, b.q_starts, gate=b.gate[:2].contiguous())
    refuses("ShapeMismatch", att, b.q, pool, table, b.q_starts, out=torch.empty_like(b.q[:2]))
    refuses("Config", att, b.q, pool, table, b.q_starts, sliding_window=-1)
    for scale in (float("nan"), float("inf"), 1e16):
        refuses("Config", att, b.q, pool, table, b.q_starts, scale=scale)
    refuses("Argument", att, b.q.transpose(0, 1), pool, table, b.q_starts)
    refuses("Argument", att, b.q.cpu(), pool, table, b.q_starts)
    assert att(torch.zeros((4, 258, 128), dtype=torch.float16, device=be.device), pool, table, b.q_starts) is None  # 129 heads per KV head
    assert att(b.q[:0], pool, table, ints(be, [0, 0, 0])).shape[0] == 0

    k = torch.randn((5, 2, 128), device=be.device)
    q = torch.randn((5, 12, 128), device=be.device)
    pos, slots = ints(be, [0, 1, 2, 3, 4]), ints(be, [0, 1, 2, 3, 4])
    rope = be.prepare_rope_table(torch.ones(32), 64, 1.0)
    app = be.rope_append_gqa_ragged
    refuses("DType", app, q, k.half(), k, rope, pool, pos, slots)
    refuses("DType", app, q.double(), k.double(), k.double(), rope, pool, pos, slots)
    refuses("DType", app, q, k, k, rope, pool, pos.long(), slots)
    refuses("ShapeMismatch", app, q, k[:4], k, rope, pool, pos, slots)
    refuses("ShapeMismatch", app, q, k, k, rope, pool, pos[:4].contiguous(), slots)
    refuses("ShapeMismatch", app, q[:, :5], k, k, rope, pool, pos, slots)
    refuses("ShapeMismatch", app, q, k, k, rope, pool, pos, slots, out=torch.empty((5, 11, 128), dtype=torch.float16, device=be.device))
    refuses("ShapeMismatch", app, q, k, k, rope, pool, pos, slots, q_norm=torch.ones(64, device=be.device))
    refuses("Argument", app, q, k, torch.randn((2, 5, 128), device=be.device).transpose(0, 1), rope, pool, pos, slots)
    refuses("Argument", app, torch.randn((5, 12 * 128 + 2), device=be.device)[:, :12 * 128].unflatten(1, (12, 128)), k, k, rope, pool, pos, slots)
    refuses("Argument", app, q, k, k, rope, pool, pos, slots, k_norm=torch.ones(129, device=be.device)[1:])
    refuses("Config", app, q, k, k, None, pool, pos, slots, q_norm=torch.ones(128, device=be.device))
    refuses("Config", app, q, k, k, rope, pool, pos, slots, eps=float("nan"))
    assert app(q[:0], k[:0], k[:0], rope, pool, pos[:0], slots[:0]).shape == (0, 12, 128)
    # a slot outside the pool: reported, dropped, the others stored
    pool.v.zero_()
    app(q, k, k, rope, pool, pos, ints(be, [0, 1 << 30, 2, -1, 4]))
    with pytest.raises(InfernoError, match="page id"):
        be.device_flush()
    assert torch.equal(pool.v[0, :, 4], k[4].half()) and (pool.v[0, :, 1] == 0).all()

    refuses("Cache", be.prepare_device_index, 0, 16, 1, 1)
    refuses("Cache", be.prepare_device_index, 8, 16, 16385, 1)
    index = be.prepare_device_index(8, 16, 2, 4)
    refuses("ShapeMismatch", be.prepare_ragged_batch, 2, 0)
    batch = be.prepare_ragged_batch(2, 10)
    refuses("ShapeMismatch", be.device_index_append, index, ints(be, [1]), batch)
    refuses("ShapeMismatch", be.device_index_append, index, ints(be, [1, 1]), be.prepare_ragged_batch(3, 10))
    parts = (batch.past_lens, batch.q_starts, batch.positions, batch.slots)
    refuses("ShapeMismatch", type(batch), *parts[:3], parts[3][:9])
    refuses("ShapeMismatch", type(batch), parts[0], parts[1][:2], *parts[2:])
    refuses("DType", type(batch), *parts[:3], parts[3].long())
    refuses("Argument", type(batch), *parts[:3], torch.zeros((10, 2), dtype=torch.int32, device=be.device)[:, 0])
    refuses("Argument", type(batch), *(t.cpu() for t in parts))
    refuses("DType", be.device_index_append, index, torch.ones(2, device=be.device), batch)
    refuses("ShapeMismatch", be.device_index_truncate, index, ints(be, [1, 1, 1]))
    wide = be.device_index(index.pages, index.lens, index.free_pages, index.free_count, 1 << 30)
    refuses("Cache", be.device_index_append, wide, ints(be, [1, 1]), batch)
    be.device_flush()
