"""GPU: attention of drafted token trees over a paged cache, against the float64
definition (tests/bounded_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(rows, H, D, dtype, dev, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)


def _slopes(H, dev):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev)


CASES = [
    # context, drafted, H, Hkv, D, page, dtype, options
    ([0], [1], 4, 1, 128, 16, F16, {}),
    ([1], [1], 1, 1, 64, 8, BF16, {}),
    ([0], [7], 8, 2, 64, 8, F16, {}),
    ([700], [8], 32, 8, 128, 16, F16, {}),
    ([63, 64, 65, 0], [5, 64, 63, 0], 8, 2, 128, 64, BF16, {}),
    ([1000, 0, 3], [65, 130, 1], 8, 2, 128, 16, F16, {}),              # three mask words
    ([5000], [64], 32, 8, 128, 64, BF16, {}),                          # several parts, several row tiles
    ([3000, 40, 1111], [24, 3, 17], 28, 4, 128, 24, F16, {}),
    ([2000, 100], [33, 12], 16, 16, 64, 32, BF16, {}),
    ([900], [40], 34, 1, 64, 40, F16, {}),
    ([1500, 70], [20, 9], 32, 8, 128, 16, F16, {"softcap": 20.0}),
    ([1500, 70], [20, 9], 16, 8, 64, 64, BF16, {"softcap": 300.0}),    # above the plain cap
    ([1500, 70], [20, 9], 32, 8, 128, 64, BF16, {"slopes": True}),
    ([1500, 70], [20, 9], 32, 8, 128, 32, F16, {"window": 100}),
    ([1500, 70], [20, 70], 8, 2, 64, 16, F16, {"window": 3}),          # hides drafted tokens too
    ([1500, 70], [20, 9], 12, 4, 128, 8, BF16, {"window": 1, "softcap": 30.0}),
    ([4100, 2000, 64], [30, 66, 5], 12, 4, 64, 32, BF16, {"window": 777, "slopes": True, "softcap": 30.0}),
    (ref.ragged(1, 70, 0, 600), ref.ragged(2, 70, 0, 9), 8, 2, 128, 64, F16, {}),   # two sequences a lane
    ([2500 if b % 9 == 0 else 3 * b for b in range(100)], [b % 5 for b in range(100)], 4, 1, 64, 16, BF16, {"slopes": True}),
]


def _id(case):
    return "-".join(str(x) if not isinstance(x, list) else "B%d_%d" % (len(x), max(x)) for x in case).replace("torch.", "")


def _run(llmik, dev, ctx, new, H, Hkv, D, page, dtype, opts, seed=0, pad=0, positions=True, mask=None, **cache):
    rng = random.Random(seed)
    lens = [a + b for a, b in zip(ctx, new)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, dev, seed, **cache)
    q = _q(sum(new) + pad, H, D, dtype, dev, seed + 1)
    grown, pos = bref.trees(rng, new, ctx)
    mask = (grown if mask is None else mask) + [0] * pad
    pos = pos + [0] * pad if positions else None
    opts = dict(opts)
    if opts.get("slopes") is True:
        opts["slopes"] = _slopes(H, dev)
    scale = 1.0 / math.sqrt(D)
    words = bref.words_of(mask, max(1, -(-max(new) // 64)), dev)
    at = None if pos is None else torch.tensor(pos, dtype=torch.int32, device=dev)
    call = lambda: llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets(new, dev), words, scale,   # noqa: E731
                                              positions=at, **opts)
    want, bound = bref.tree(q, k, v, table, lens, new, mask, pos, scale, page, **opts)
    return call(), want, bound, call


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_trees(llmik, cuda, case):
    got, want, bound, call = _run(llmik, cuda, *case)
    ref.check(got, want, bound)
    assert torch.equal(got, call())


@pytest.mark.parametrize("opts", [{}, {"slopes": True, "window": 40}], ids=str)
def test_positions_are_the_slots_by_default(llmik, cuda, opts):
    got, want, bound, _ = _run(llmik, cuda, [100, 900], [30, 5], 8, 2, 128, 16, F16, opts, positions=False)
    ref.check(got, want, bound)


def test_a_chain_is_a_prompt(llmik, cuda):
    """Where every drafted token hangs on the one before it, the tree is a prompt's chunk."""
    new = [40, 70]
    chain = [(1 << i + 1) - 1 for n in new for i in range(n)]
    got, want, bound, _ = _run(llmik, cuda, [300, 0], new, 16, 4, 64, 32, BF16, {"slopes": True, "window": 60},
                               positions=False, mask=chain)
    ref.check(got, want, bound)
    k, v, table, seq = ref.make_cache([340, 70], 4, 64, 32, BF16, cuda, 0)
    prompt = llmik.paged_prefill_attention(_q(110, 16, 64, BF16, cuda, 1), k, v, table, seq, ref.offsets(new, cuda),
                                           0.125, slopes=_slopes(16, cuda), window=60)
    ref.check(prompt, want, bound)


def test_masks_that_leave_rows_empty_and_rows_of_no_sequence(llmik, cuda):
    """Without cached tokens, a row without bits sees nothing: zeros. Bits of tokens that the
    sequence does not have, and a padded batch's rows, say nothing."""
    mask = [0, 1 << 1 | 1 << 40, 0, ~0 & (1 << 64) - 1, 1 << 3, 0, 0, 1]
    got, want, bound, _ = _run(llmik, cuda, [0, 50], [4, 4], 8, 2, 128, 16, F16, {}, pad=5, mask=mask)
    ref.check(got, want, bound)
    assert int(got[0].count_nonzero()) == 0 and int(got[2].count_nonzero()) == 0
    assert int(got[8:].count_nonzero()) == 0 and bool((got[[1, 3, 4, 5, 6, 7]].abs().amax((1, 2)) > 0).all())


def test_few_mask_words_hide_what_they_do_not_hold(llmik, cuda):
    new, ctx = [100], [70]
    mask = [(1 << 64) - 1] * 100
    k, v, table, seq = ref.make_cache([170], 2, 128, 16, F16, cuda, 3)
    q = _q(100, 4, 128, F16, cuda, 4)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets(new, cuda), bref.words_of(mask, 1, cuda), 0.1)
    want, bound = bref.tree(q, k, v, table, [170], new, mask, None, 0.1, 16)
    ref.check(got, want, bound)


@pytest.mark.parametrize("D", [64, 128])
def test_unmapped_pages_are_no_keys_and_dead_slots_are_not_read(llmik, cuda, D):
    """Pages missing from a table, in the context and among the drafted; slots behind the
    last token and pages of nobody hold NaN."""
    ctx, new, page = [300, 20], [30, 6], 16
    k, v, table, seq = ref.make_cache([330, 26], 2, D, page, F16, cuda, 5, fill=math.nan, gap=8)
    table[0, 3] = -1
    table[0, 19] = k.shape[0]
    rng = random.Random(5)
    mask, pos = bref.trees(rng, new, ctx)
    q = _q(36, 8, D, F16, cuda, 6)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets(new, cuda), bref.words_of(mask, 1, cuda), 0.1,
                                     positions=torch.tensor(pos, dtype=torch.int32, device=cuda))
    want, bound = bref.tree(q, k, v, table, [330, 26], new, mask, pos, 0.1, page)
    ref.check(got, want, bound)


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64)], ids=str)
@pytest.mark.parametrize("ctx", [70, 4000])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(llmik, cuda, dtype, D, ctx):
    """A drafted token whose V is NaN, or infinite: its descendants' rows have it, the others'
    are numbers and right."""
    new, page = 40, 16
    rng = random.Random(8)
    mask, pos = bref.trees(rng, [new], [ctx])
    k, v, table, seq = ref.make_cache([ctx + new], 2, D, page, dtype, cuda, 9)
    q = _q(new, 8, D, dtype, cuda, 10)
    bad = ctx + 5
    sees = torch.tensor([bool(m >> 5 & 1) for m in mask], device=cuda)
    assert 0 < int(sees.sum()) < new
    place = int(table[0, bad // page]), slice(None), bad % page
    v[place] = 0.0
    want, bound = bref.tree(q, k, v, table, [ctx + new], [new], mask, pos, 0.05, page)
    for value in (math.nan, math.inf):
        v[place] = value
        got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets([new], cuda), bref.words_of(mask, 1, cuda),
                                         0.05, positions=torch.tensor(pos, dtype=torch.int32, device=cuda))
        assert not bool(torch.isfinite(got[sees]).any())
        ref.check(got[~sees], want[~sees], bound[~sees])


@pytest.mark.parametrize("length", [0, -1, -2 ** 31])
def test_empty_and_short_sequences(llmik, cuda, length):
    """Rows of an empty sequence, and drafted tokens in front of a cache's first slot, are zero."""
    k, v, table, seq = ref.make_cache([40, 6], 2, 64, 16, F16, cuda, 11)
    seq.copy_(torch.tensor([length, 6], dtype=torch.int32))
    mask = [(1 << 10) - 1] * 12
    q = _q(12, 4, 64, F16, cuda, 12)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets([3, 9], cuda), bref.words_of(mask, 1, cuda), 0.1)
    assert int(got[:6].count_nonzero()) == 0        # the empty sequence's, and three rows before the other's first slot
    want, bound = bref.tree(q, k, v, table, [0, 6], [0, 9], mask[3:], None, 0.1, 16)
    want, bound = torch.zeros_like(want), torch.zeros_like(bound)
    live = ref.tokens_of(k, table[1], 6, 16)[0], ref.tokens_of(v, table[1], 6, 16)[0]
    ok = torch.ones(6, dtype=torch.bool, device=cuda)
    # rows 6 .. 11 are drafted tokens 3 .. 8; slot t is drafted token t + 3
    out, off = bref.attend(q[6:], *live, ok, torch.ones(6, 6, dtype=torch.bool, device=cuda),
                           torch.zeros(6, 6, dtype=torch.long, device=cuda), 0.1, ref.U[F16])
    ref.check(got[6:], out, off)


def test_a_replayed_tree_follows_lengths_offsets_masks_and_pages(llmik, cuda):
    """One graph of 48 rows: contexts (and so the number of parts), drafts and pages change."""
    H, Hkv, D, page, B, rows = 16, 4, 128, 16, 3, 48
    k, v, table, seq = ref.make_cache([5000] * B, Hkv, D, page, F16, cuda, 13)
    q = _q(rows, H, D, F16, cuda, 14)
    cu = ref.offsets([16, 16, 16], cuda)
    words = torch.zeros(rows, 1, dtype=torch.int64, device=cuda)
    at = torch.zeros(rows, dtype=torch.int32, device=cuda)
    call = lambda: llmik.paged_tree_attention(q, k, v, table, seq, cu, words, 0.1, positions=at, window=2000)   # noqa: E731
    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call()
    turns = [([48, 0, 0], [4900, 0, 0]), ([1, 1, 1], [100, 3000, 0]), ([0, 30, 18], [10, 200, 2500]),
             ([0, 0, 0], [7, 0, 9]), ([10, 24, 5], [4000, 4900, 1])]
    for turn, (new, ctx) in enumerate(turns):
        mask, pos = bref.trees(random.Random(turn), new, ctx)
        pad = rows - sum(new)
        words.copy_(bref.words_of(mask + [0] * pad, 1, cuda))
        at.copy_(torch.tensor(pos + [0] * pad, dtype=torch.int32))
        cu.copy_(ref.offsets(new, cuda))
        seq.copy_(torch.tensor([a + b for a, b in zip(new, ctx)], dtype=torch.int32))
        table.copy_(table.roll(1, 0))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, bound = bref.tree(q, k, v, table, [a + b for a, b in zip(new, ctx)], new, mask, pos, 0.1, page,
                                window=2000)
        ref.check(out, want, bound)
        assert int(out[sum(new):].count_nonzero()) == 0
        assert torch.equal(call(), out)
    torch.cuda.synchronize()


def test_another_stream_and_positions_of_any_size(llmik, cuda):
    """On a stream of its own; positions beyond 2^30 and below the context count as those."""
    ctx, new = [500], [6]
    k, v, table, seq = ref.make_cache([506], 2, 64, 16, F16, cuda, 15)
    q = _q(6, 4, 64, F16, cuda, 16)
    mask = [(1 << 6) - 1] * 6
    pos = [-5, 0, 600, 2 ** 31 - 1, 501, 499]
    args = (ref.offsets(new, cuda), bref.words_of(mask, 1, cuda), 0.1)
    at = torch.tensor(pos, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = llmik.paged_tree_attention(q, k, v, table, seq, *args, positions=at, window=120)
    s.synchronize()
    want, bound = bref.tree(q, k, v, table, [506], new, mask, pos, 0.1, 16, window=120)
    ref.check(got, want, bound)
