"""GPU: calls of the paged ops at the edges of what their documentation allows,
against the float64 definition (tests/paged_ref.py)."""
from __future__ import annotations

import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(rows, H, D, dtype, dev, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)


@pytest.mark.parametrize("length", [0, -1, -2, -2 ** 31, -2 ** 31 + 1])
@pytest.mark.parametrize("tables", [False, True])
@pytest.mark.parametrize("rows", [None, [1, 1], [5, 2], [3, 700]], ids=str)
def test_appends_to_empty_sequences(llmik, cuda, length, tables, rows):
    """A sequence of a length <= 0 has no new tokens: a zero q, and nothing written."""
    H, Hkv, D, page = 4, 2, 64, 16
    k, v, table, _ = ref.make_cache([800, 800], Hkv, D, page, F16, cuda, 1)
    seq = torch.full((2,), length, dtype=torch.int32, device=cuda)
    n = 2 if rows is None else sum(rows)
    qkv = torch.ones(n, (H + 2 * Hkv) * D, dtype=F16, device=cuda)
    angles = torch.ones(900, D, dtype=F16, device=cuda) if tables else None
    k0, v0 = k.clone(), v.clone()
    q = llmik.rope_paged_append(qkv, angles, angles, k, v, table, seq,
                                None if rows is None else ref.offsets(rows, cuda))
    assert int(q.count_nonzero()) == 0
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_a_cache_stays_on_its_device(llmik, cuda):
    """Made on the current device, its batches go there whatever device is current later."""
    from llmik_cuda.kv_cache import PagedKVCache
    cache = PagedKVCache(4, 2, page_size=16, head_dim=64)
    assert cache.device == cache.k.device and cache.device.index is not None
    step = cache.batch([cache.add()], [3])
    assert step.page_table.device == step.seq_lens.device == cache.k.device


# ---------------------------------------------------------- graphs whose tables change

def _replays(graph, change, check, eager, turns=5):
    """Replays of one graph, with the program's own work and waits between them."""
    for turn in range(turns):
        change(turn)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(turn)
        eager()
    torch.cuda.synchronize()


def _captured(call):
    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call()
    return g, out


@pytest.mark.parametrize("dtype,D,window", [(F16, 128, 0), (BF16, 64, 700)], ids=str)
def test_a_replayed_prompt_follows_lengths_offsets_and_tables(llmik, cuda, dtype, D, window):
    """One graph of 64 rows: the sequences' rows, their contexts (and so the number of parts
    that a row tile's keys are cut into, 1 to several) and pages change between replays."""
    H, Hkv, page, B, rows = 16, 4, 16, 3, 64
    k, v, table, seq = ref.make_cache([5000] * B, Hkv, D, page, dtype, cuda, 1)
    q = _q(rows, H, D, dtype, cuda, 2)
    cu = ref.offsets([20, 20, 20], cuda)
    call = lambda: llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.1, window=window)   # noqa: E731
    g, out = _captured(call)
    turns = [([64, 0, 0], [4900, 0, 0]), ([1, 1, 1], [100, 3000, 0]), ([0, 30, 34], [10, 200, 2500]),
             ([0, 0, 0], [7, 0, 9]), ([10, 44, 5], [4000, 4956, 1])]

    def change(turn):
        new, ctx = turns[turn]
        cu.copy_(ref.offsets(new, cuda))
        seq.copy_(torch.tensor([a + b for a, b in zip(new, ctx)], dtype=torch.int32))
        table.copy_(table.roll(1, 0))

    def check(turn):
        new, ctx = turns[turn]
        want, bound = ref.attention(q, k, v, table, [a + b for a, b in zip(new, ctx)], new, 0.1, page, False,
                                    window=window)
        ref.check(out, want, bound)
        assert int(out[sum(new):].count_nonzero()) == 0

    _replays(g, change, check, call)


@pytest.mark.parametrize("dtype,D,window", [(F16, 128, 0), (BF16, 64, 900)], ids=str)
def test_a_replayed_shared_prefix_follows_lengths_and_pages(llmik, cuda, dtype, D, window):
    H, Hkv, page, B, P = 16, 4, 16, 5, 1000
    k, v, table, seq = ref.make_cache([1500] * (B + 1), Hkv, D, page, dtype, cuda, 3)
    pages, table, seq = table[-1, :-(-P // page)].contiguous(), table[:-1].contiguous(), seq[:-1].contiguous()
    q = _q(B, H, D, dtype, cuda, 4)
    call = lambda: llmik.paged_shared_prefix_attention(q, k, v, table, seq, pages, P, 0.1, window=window)   # noqa: E731
    g, out = _captured(call)
    turns = [[1001, 1500, 1200, 1003, 1016], [1, 0, 999, 1000, 1001], [1499] * B, [0] * B, [1030, 1001, 3, 1400, 1450]]

    def change(turn):
        seq.copy_(torch.tensor(turns[turn], dtype=torch.int32))
        table.copy_(table.roll(1, 0))
        pages.copy_(pages.roll(7))

    def check(turn):
        want, bound = ref.attention(q, k, v, table, turns[turn], [1] * B, 0.1, page, False, prefix_pages=pages,
                                    prefix_len=P, window=window)
        ref.check(out, want, bound)

    _replays(g, change, check, call)


def test_a_replayed_step_writes_and_reads_where_the_tables_say(llmik, cuda):
    """Append and decode of one step in a graph: a sequence grows by a token a replay, over
    page ends, one is replaced by another, one is empty."""
    H, Hkv, D, page, B = 8, 2, 128, 8, 3
    k, v, table, seq = ref.make_cache([60] * B, Hkv, D, page, F16, cuda, 5)
    qkv = torch.empty(B, (H + 2 * Hkv) * D, dtype=F16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(6)
    cos = torch.randn(64, D, generator=gen, device=cuda).half()
    sin = torch.randn(64, D, generator=gen, device=cuda).half()
    qkv.normal_(generator=gen)
    seq.copy_(torch.tensor([1, 1, 1], dtype=torch.int32))

    def call():
        q = llmik.rope_paged_append(qkv, cos, sin, k, v, table, seq)
        return q, llmik.paged_decode_attention(q, k, v, table, seq, 0.1)
    g, (q, out) = _captured(call)
    want_k, want_v = k.clone(), v.clone()
    for turn in range(6):
        lens = [7 + turn, 0 if turn % 2 else 30, 15 + 9 * turn]
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(table.roll(1, 0))
        qkv.normal_(generator=gen)
        want_k.copy_(k)
        want_v.copy_(v)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        x = qkv.view(B, H + 2 * Hkv, D)
        for b, n in enumerate(lens):
            if n == 0:
                assert int(q[b].count_nonzero()) == 0 and int(out[b].count_nonzero()) == 0
                continue
            at = int(table[b, (n - 1) // page]), slice(None), (n - 1) % page
            one = llmik.rope(x[b:b + 1, :H + Hkv].transpose(0, 1).reshape(1, H + Hkv, 1, D).contiguous(),
                             cos[n - 1:n], sin[n - 1:n])[0, :, 0]
            assert torch.equal(q[b], one[:H])
            want_k[at], want_v[at] = one[H:], x[b, H + Hkv:]
        assert torch.equal(k, want_k) and torch.equal(v, want_v)
        want, bound = ref.attention(q, k, v, table, lens, [1] * B, 0.1, page, True)
        ref.check(out, want, bound)


# --------------------------------------------------------------------- many sequences

@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)], ids=str)
def test_keys_in_parts_of_more_sequences_than_lanes(llmik, cuda, dtype, D):
    """100 sequences, so that a lane counts two, and contexts of several parts."""
    B, H, Hkv, page = 100, 2, 1, 16
    new = [(7 * b) % 4 for b in range(B)]
    lens = [n + (2500 + 9 * b if b % 9 == 0 else 3 * b) for b, n in enumerate(new)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 7, extra_columns=400)
    q = _q(sum(new) + 3, H, D, dtype, cuda, 8)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets(new, cuda), 0.1)
    want, bound = ref.attention(q, k, v, table, lens, new, 0.1, page, False)
    ref.check(got, want, bound)
    assert int(got[sum(new):].count_nonzero()) == 0


def test_more_than_4096_sequences(llmik, cuda):
    """A lane of the search counts more than 64 sequences: their ends are found in steps of 64."""
    B, H, Hkv, D, page = 4300, 4, 2, 64, 8
    lens = [(5 * b) % 23 if b % 50 else 0 for b in range(B)]
    lens[-1], lens[65], lens[130] = 21, 200, 90
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 9)
    q = _q(B, H, D, F16, cuda, 10)
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.1)
    some = sorted({*range(0, B, 41), *range(60, 140), B - 2, B - 1})

    def rows(out, b, r0, n, pair):
        kb, ok = ref.tokens_of(k, table[b], lens[b], page)
        vb, _ = ref.tokens_of(v, table[b], lens[b], page)
        pos = torch.arange(lens[b] - n, lens[b], device=cuda)
        up = (ref.PAIR if pair else ref.U)[F16]
        want, bound = ref.attend(q2[r0:r0 + n], kb, vb, ok, pos, 0.1, up=up)
        ref.check(out[r0:r0 + n], want, bound)
    q2 = q
    for b in some:
        rows(got, b, b, 1, True)
    empty = seq == 0
    assert int(got[empty].count_nonzero()) == 0 and bool((got[~empty].abs().amax((1, 2)) > 0).all())
    new = [min(n, b % 4) for b, n in enumerate(lens)]
    q2 = _q(sum(new) + 2, H, D, F16, cuda, 11)
    got = llmik.paged_prefill_attention(q2, k, v, table, seq, ref.offsets(new, cuda), 0.1)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    for b in some:
        if new[b]:
            rows(got, b, starts[b], new[b], False)
    assert int(got[sum(new):].count_nonzero()) == 0 and bool((got[:sum(new)].abs().amax((1, 2)) > 0).all())


# -------------------------------------------------- values that are no numbers, in parts

@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64)], ids=str)
@pytest.mark.parametrize("window", [0, 1200])
def test_values_that_are_no_numbers_where_keys_are_cut_into_parts(llmik, cuda, dtype, D, window):
    """A live NaN that some rows see, in the last part, and one that leaves the window of
    some, in the first: those rows are done again in their parts, the others stay numbers."""
    H, Hkv, page, ctx, new = 8, 2, 16, 3000, 60
    n = ctx + new
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, dtype, cuda, 12, extra_columns=100)
    q = _q(new, H, D, dtype, cuda, 13)
    cu = ref.offsets([new], cuda)
    bad = [ctx + 25] + ([ctx - window + 10] if window else [])
    for t in bad:
        v[int(table[0, t // page]), :, t % page] = 0.0
    want, bound = ref.attention(q, k, v, table, [n], [new], 0.1, page, False, window=window)
    for t in bad:
        v[int(table[0, t // page]), :, t % page] = math.nan
    got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.1, window=window)
    sees = torch.zeros(new, dtype=torch.bool, device=cuda)
    for t in bad:
        dist = torch.arange(ctx, n, device=cuda) - t
        sees |= (dist >= 0) & ((dist < window) if window else True)
    assert bool(got[sees].isnan().all())
    if bool((~sees).any()):
        ref.check(got[~sees], want[~sees], bound[~sees])
