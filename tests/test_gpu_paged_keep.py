"""GPU: the selection of a sequence's tokens by weight and the moves that bring them
together, against plain restatements (tests/bounded_ref.py). Both are exact: slots
are whole numbers, and moved values keep their bits."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, I32 = torch.float16, torch.bfloat16, torch.int32


def _weights(R, Hkv, W, dev, seed, kind):
    gen = torch.Generator(device=dev).manual_seed(seed)
    w = torch.empty(R, Hkv, W, device=dev).exponential_(generator=gen)
    if kind == "ties":        # few values, and both zeros
        w = (w * 2).floor()
        w[w == 0] = torch.where(torch.rand(w[w == 0].shape, generator=gen, device=dev) < 0.5, 0.0, -0.0)
    elif kind == "equal":
        w.fill_(0.25)
    elif kind == "wide":      # all exponents, both signs
        w = torch.exp2(torch.empty_like(w).uniform_(-140, 120, generator=gen))
        w *= torch.where(torch.rand(w.shape, generator=gen, device=dev) < 0.3, -1.0, 1.0)
    elif kind == "not finite":
        r = torch.rand(w.shape, generator=gen, device=dev)
        w[r < 0.2], w[r > 0.9] = math.nan, math.inf
        w[(r > 0.5) & (r < 0.6)] = -math.inf
    return w


SELECT = [
    # lens, Hkv, weights' tokens, keep, first, recent, kind
    ([1], 1, 1, 1, 0, 0, "random"),
    ([5, 0, 1, -3, -2 ** 31], 2, 9, 2, 1, 0, "random"),
    ([100, 64, 65, 7], 8, 128, 64, 4, 16, "random"),
    ([100, 64, 65, 7], 4, 128, 64, 0, 0, "ties"),
    ([5000, 1200, 3000], 2, 5003, 1000, 3, 100, "wide"),
    ([5000, 1200, 3000], 2, 5003, 1000, 0, 100, "ties"),
    ([5000, 1500], 1, 5000, 1400, 1, 0, "equal"),
    ([3000, 1025, 1024], 2, 2000, 1024, 0, 1024, "random"),     # nothing to choose; longer than the weights
    ([3000, 1025, 1024], 2, 3000, 1023, 1000, 23, "random"),
    ([2000, 999], 3, 2000, 500, 2, 30, "not finite"),
    ([40000], 2, 40001, 3000, 4, 64, "random"),
    ([40000, 33000], 1, 40000, 32999, 4, 64, "ties"),
    (ref.ragged(1, 200, 0, 300), 3, 300, 77, 2, 5, "ties"),
]


def _id(case):
    return "-".join(str(x) if not isinstance(x, list) else "B%d_%d" % (len(x), max(x)) for x in case).replace("torch.", "")


@pytest.mark.parametrize("case", SELECT, ids=_id)
def test_select(llmik, cuda, case):
    lens, Hkv, W, keep, first, recent, kind = case
    w = _weights(len(lens), Hkv, W, cuda, 1, kind)
    before = w.clone()
    seq = torch.tensor(lens, dtype=I32, device=cuda)
    kept, new = llmik.paged_select_tokens(w, seq, keep, first, recent)
    want, out = bref.select(w, lens, keep, first, recent)
    assert kept.dtype == new.dtype == I32 and kept.shape == (len(lens), Hkv, keep)
    assert new.tolist() == out and kept.tolist() == want
    assert torch.equal(w.view(torch.int32), before.view(torch.int32))


def test_select_rows(llmik, cuda):
    """Rows in any order; a sequence without a row has weights 0: the lowest slots."""
    lens, rows = [90, 50, 60, 20], [4, 1, 9, -2 ** 31]
    w = _weights(5, 2, 100, cuda, 2, "random")
    kept, new = llmik.paged_select_tokens(w, torch.tensor(lens, dtype=I32, device=cuda), 40, 2, 8,
                                          torch.tensor(rows, dtype=I32, device=cuda))
    want, out = bref.select(w, lens, 40, 2, 8, rows)
    assert kept.tolist() == want and new.tolist() == out
    assert kept[2, 0].tolist() == [*range(32), *range(52, 60)]


def _kept(rng, n, start, count):
    """`count` slots of start .. n - 1 in order, none before its new one."""
    return sorted(rng.sample(range(start, n), min(count, n - start)))


COMPACT = [
    # lens, starts, entries, one list for all heads, Hkv, D, page, dtype
    ([1], None, 1, False, 1, 64, 8, F16),
    ([30, 0, 9], None, 7, False, 2, 128, 8, BF16),
    ([300, 17, 40], [290, 0, 39], 10, True, 8, 128, 16, F16),
    ([300, 17, 40], [250, 4, 40], 33, True, 4, 64, 24, BF16),
    ([700, 65, 1200], None, 512, False, 2, 128, 64, F16),
    ([5000], None, 3000, False, 2, 128, 16, BF16),
    ([5000, 4500], [10, 0], 4100, False, 1, 64, 256, F16),
    (ref.ragged(3, 60, 0, 200), None, 50, False, 3, 64, 16, F16),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("case", COMPACT, ids=_id)
def test_compact(llmik, cuda, case, weights):
    lens, starts, n, one, Hkv, D, page, dtype = case
    rng = random.Random(4)
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 5, gap=8 if n == 7 else 0)
    lists = [[_kept(rng, max(x, 0), 0 if starts is None else starts[b], rng.randint(0, n))
              for _ in range(1 if one else Hkv)] for b, x in enumerate(lens)]
    lists = [[row + [-1] * (n - len(row)) for row in heads] for heads in lists]
    kept = torch.tensor(lists, dtype=I32, device=cuda).view(len(lens), -1, n)
    if one:
        kept, lists = kept[:, 0].contiguous(), [heads[0] for heads in lists]
    w = _weights(len(lens) + 2, Hkv, max(lens) + 3, cuda, 6, "random") if weights else None
    rows = list(range(len(lens) + 1, 1, -1)) if weights and len(lens) % 2 else None
    want_k, want_v, want_w = bref.compact(k, v, table, lens, lists, starts, w, rows)
    llmik.paged_compact(k, v, table, seq, kept, None if starts is None else torch.tensor(starts, dtype=I32, device=cuda),
                        w, None if rows is None else torch.tensor(rows, dtype=I32, device=cuda))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    if weights:
        assert torch.equal(w, want_w)
    assert seq.tolist() == lens


def test_entries_that_move_nothing(llmik, cuda):
    """Negative ones, those at or behind the length or in front of their new slot, unmapped
    pages; entries out of order and slots that come twice."""
    lens, Hkv, D, page, n = [100, 90, 50, 20, 40], 2, 64, 16, 12
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 7)
    table[1, 0], table[1, 3] = -1, k.shape[0]
    lists = [[9, 8, 99, 100, 2 ** 31 - 1, 3, 50, 50, 20, -7, 60, -2 ** 31],
             [20, 3, 50, 18, 70, 60, 89, 33, 34, 35, 36, 37],
             [49] * 12, [19, 18, 17, 16, 15, 14, 13, 12, 11, 10, 9, 8], [-1] * 12]
    kept = torch.tensor(lists, dtype=I32, device=cuda)
    starts = [0, 0, 45, 0, -4]
    w = _weights(5, Hkv, 95, cuda, 8, "random")
    want_k, want_v, want_w = bref.compact(k, v, table, lens, lists, starts, w)
    llmik.paged_compact(k, v, table, seq, kept, torch.tensor(starts, dtype=I32, device=cuda), w)
    assert torch.equal(k, want_k) and torch.equal(v, want_v) and torch.equal(w, want_w)
    # no entries: the weights behind the starts become 0, the cache stays
    k0 = k.clone()
    llmik.paged_compact(k, v, table, seq, kept[:, :0].contiguous(), torch.tensor([10, 0, 50, 3, 39], dtype=I32, device=cuda), w)
    assert torch.equal(k, k0) and torch.equal(w[0, :, :10], want_w[0, :, :10])
    assert int(w[0, :, 10:].count_nonzero()) == 0 and int(w[1, :, :90].count_nonzero()) == 0
    assert torch.equal(w[2], want_w[2]) and torch.equal(w[3, :, 20:], want_w[3, :, 20:])


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_appends_at_positions(llmik, cuda, dtype, rotate):
    """Rows rotated by the positions that are given, written where their order says."""
    H, Hkv, D, page = 4, 2, 64, 16
    lens, new = [40, 7, 100], [10, 7, 1]
    pos = [500, 501, 501, 502, 30, 7, 0, 899, 900, -1, *range(90, 97), 555]
    gen = torch.Generator(device=cuda).manual_seed(9)
    qkv = torch.randn(18, (H + 2 * Hkv) * D, generator=gen, device=cuda).to(dtype)
    cos = torch.randn(900, D, generator=gen, device=cuda)
    sin = torch.randn(900, D, generator=gen, device=cuda)
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 10)
    want_k, want_v = k.double(), v.double()
    x = qkv.double().view(18, H + 2 * Hkv, D)
    at = torch.tensor(pos, device=cuda)
    ok = (at >= 0) & (at < 900) if rotate else torch.ones_like(at, dtype=torch.bool)
    turned = x[:, :H + Hkv]
    if rotate:
        turned = ref.rotate(turned, cos[at.clamp(0, 899)].double(), sin[at.clamp(0, 899)].double())
    turned = torch.where(ok[:, None, None], turned, torch.zeros_like(turned))
    for b, r0, n, first in ref.rows_of(lens, new):
        for i in range(n):
            if bool(ok[r0 + i]):
                place = int(table[b, (first + i) // page]), slice(None), (first + i) % page
                want_k[place], want_v[place] = turned[r0 + i, H:], x[r0 + i, H + Hkv:]
    q = llmik.rope_paged_append(qkv, cos if rotate else None, sin if rotate else None, k, v, table, seq,
                                ref.offsets(new, cuda), at.int())
    # one rounding to the type, and two products and a sum in fp32: 3 * 2^-24 of their sizes (|x| |cos| < 25)
    tol = lambda want: ref.U[dtype] * want.abs() + 3 * 25 * 2.0 ** -23   # noqa: E731
    for got, want in ((q, turned[:, :H]), (k, want_k), (v, want_v)):
        assert bool(((got.double() - want).abs() <= (tol(want) if rotate else 0 * want)).all())


def test_replays_follow_lengths_pages_and_lists(llmik, cuda):
    """A graph that selects and compacts, replayed with other lengths, weights and pages."""
    B, Hkv, D, page, keep = 3, 2, 128, 16, 100
    k, v, table, seq = ref.make_cache([400] * B, Hkv, D, page, F16, cuda, 11)
    w = _weights(B, Hkv, 400, cuda, 12, "random")
    seq.zero_()

    def call():
        kept, new = llmik.paged_select_tokens(w, seq, keep, 4, 20)
        llmik.paged_compact(k, v, table, seq, kept, None, w)
        return kept, new
    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        kept, new = call()
    for turn, lens in enumerate([[400, 101, 100], [0, 399, 250], [5, 300, 110], [222, 0, 400]]):
        seq.copy_(torch.tensor(lens, dtype=I32))
        table.copy_(table.roll(1, 0))
        w.copy_(_weights(B, Hkv, 400, cuda, 20 + turn, "ties"))
        want, out = bref.select(w, lens, keep, 4, 20)
        want_k, want_v, want_w = bref.compact(k, v, table, lens, want, None, w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert kept.tolist() == want and new.tolist() == out
        assert torch.equal(k, want_k) and torch.equal(v, want_v) and torch.equal(w, want_w)
        llmik.paged_select_tokens(w, seq, keep)
    torch.cuda.synchronize()
