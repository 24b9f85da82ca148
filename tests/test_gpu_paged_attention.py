"""GPU: decode, prompt and shared-prefix attention over a paged cache, against
the float64 definition (tests/paged_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(rows, H, D, dtype, dev, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)


def _slopes(H, dev):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev)


DECODE = [
    # lens, H, Hkv, D, page, dtype, options
    ([1], 4, 1, 128, 16, F16, {}),
    ([1], 1, 1, 64, 8, BF16, {}),
    ([31], 8, 2, 128, 32, F16, {}),
    ([32], 8, 2, 128, 32, BF16, {}),
    ([33, 0, 64, 65], 8, 2, 128, 16, F16, {}),
    ([700], 32, 8, 128, 16, F16, {}),
    ([1500, 3, 129, 0, 0, 777], 32, 8, 128, 64, BF16, {}),
    ([4097] * 3, 28, 4, 128, 24, F16, {}),
    ([1023, 40, 513], 40, 8, 64, 8, BF16, {}),
    ([9000], 64, 8, 64, 128, F16, {}),
    ([20000], 16, 16, 128, 256, F16, {}),
    ([300, 200], 34, 1, 128, 32, BF16, {}),          # 34 heads of a KV head: three chunks
    ([300, 200], 17, 1, 64, 40, F16, {}),
    ([100, 2000, 31], 32, 8, 128, 16, F16, {"softcap": 20.0}),
    ([100, 2000, 31], 32, 8, 128, 64, BF16, {"slopes": True}),
    ([100, 2000, 31], 32, 8, 128, 64, F16, {"window": 100}),
    ([100, 2000, 31], 32, 8, 128, 24, F16, {"window": 1}),
    ([5000, 2000, 4096], 12, 4, 64, 32, BF16, {"window": 777, "slopes": True, "softcap": 30.0}),
    ([20000, 20011] * 4, 8, 8, 64, 64, F16, {}),                      # many tiles a wave
    ([20000, 20011] * 4, 8, 8, 128, 16, BF16, {"window": 19000}),
    (ref.ragged(1, 70, 0, 900), 16, 8, 128, 64, F16, {}),             # more slabs than workgroups; two lengths a lane
    (ref.ragged(2, 130, 0, 700), 28, 4, 64, 16, BF16, {"softcap": 30.0, "slopes": True}),
    (ref.ragged(3, 300, 1, 60), 8, 2, 128, 8, F16, {}),
    (ref.ragged(4, 64, 300, 1500), 10, 10, 64, 32, BF16, {"window": 500}),
]


def _decode(llmik, dev, lens, H, Hkv, D, page, dtype, opts, seed=0, **cache):
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, dev, seed, **cache)
    q = _q(len(lens), H, D, dtype, dev, seed + 1)
    opts = dict(opts)
    if opts.get("slopes") is True:
        opts["slopes"] = _slopes(H, dev)
    scale = 1.0 / math.sqrt(D)
    got = llmik.paged_decode_attention(q, k, v, table, seq, scale, **opts)
    want, bound = ref.attention(q, k, v, table, lens, [1] * len(lens), scale, page, True, **opts)
    return got, want, bound


def _id(case):
    return "-".join(str(x) if not isinstance(x, list) else "B%d_%d" % (len(x), max(x)) for x in case).replace("torch.", "")


@pytest.mark.parametrize("case", DECODE, ids=_id)
def test_decode(llmik, cuda, case):
    got, want, bound = _decode(llmik, cuda, *case)
    ref.check(got, want, bound)
    for b, n in enumerate(case[0]):
        if n == 0:
            assert int(got[b].count_nonzero()) == 0


PREFILL = [
    # context, new, H, Hkv, D, page, dtype, options
    ([0], [1], 4, 1, 128, 16, F16, {}),
    ([0], [5], 8, 2, 64, 8, BF16, {}),
    ([0, 0, 0], [17, 150, 64], 32, 8, 128, 16, F16, {}),
    ([0, 63, 1000, 0], [64, 1, 3, 0], 32, 8, 128, 64, BF16, {}),
    ([0, 500], [700, 129], 28, 4, 128, 24, F16, {}),
    ([3, 0], [1000, 33], 8, 8, 64, 32, F16, {}),
    ([2000], [513], 16, 2, 128, 128, BF16, {}),
    ([10, 300], [200, 77], 32, 8, 128, 16, F16, {"softcap": 20.0}),
    ([10, 300], [200, 77], 24, 8, 64, 64, BF16, {"slopes": True}),
    ([10, 300], [200, 577], 32, 8, 128, 32, F16, {"window": 50}),
    ([10, 300], [20, 77], 8, 1, 128, 40, F16, {"window": 1}),
    ([1010, 300], [200, 577], 12, 4, 128, 32, BF16, {"window": 333, "slopes": True, "softcap": 30.0}),
    # keys in parts, several row tiles each
    ([715, 1136, 360], [106, 114, 87], 16, 8, 64, 16, F16, {"slopes": True}),
    ([3000, 0, 1500], [333, 65, 1], 8, 2, 64, 64, BF16, {}),
    ([3000, 0, 1500], [333, 65, 1], 8, 2, 128, 64, BF16, {"softcap": 40.0}),
]


def _prefill(llmik, dev, ctx, new, H, Hkv, D, page, dtype, opts, seed=0, pad=0, **cache):
    lens = [a + b for a, b in zip(ctx, new)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, dev, seed, **cache)
    q = _q(sum(new) + pad, H, D, dtype, dev, seed + 1)
    opts = dict(opts)
    if opts.get("slopes") is True:
        opts["slopes"] = _slopes(H, dev)
    scale = 1.0 / math.sqrt(D)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets(new, dev), scale, **opts)
    want, bound = ref.attention(q, k, v, table, lens, new, scale, page, False, **opts)
    return got, want, bound


@pytest.mark.parametrize("case", PREFILL, ids=_id)
def test_prefill(llmik, cuda, case):
    got, want, bound = _prefill(llmik, cuda, *case)
    ref.check(got, want, bound)


def test_prefill_rows_behind_the_last_sequence_are_zero(llmik, cuda):
    got, want, bound = _prefill(llmik, cuda, [0, 40], [30, 9], 8, 2, 128, 16, F16, {}, pad=7)
    ref.check(got, want, bound)
    assert int(got[39:].count_nonzero()) == 0


PREFIX = [
    # prefix, own tokens, H, Hkv, D, page, dtype, options
    (64, [1, 2], 8, 2, 128, 16, F16, {}),
    (1, [1], 4, 4, 64, 8, BF16, {}),
    (1500, [3, 200, 77, 1], 40, 8, 128, 16, BF16, {}),
    (4096, [10, 600] * 9, 32, 8, 128, 64, F16, {}),
    (777, [64] * 40, 28, 4, 64, 24, F16, {}),
    (1000, [5, 100, 33], 32, 8, 128, 32, F16, {"softcap": 20.0}),
    (1000, [5, 100, 33], 32, 8, 128, 32, BF16, {"slopes": True}),
    (1000, [5, 100, 33], 32, 8, 128, 32, F16, {"window": 64}),
    (1000, [5, 100, 700], 16, 8, 64, 40, BF16, {"window": 600, "slopes": True, "softcap": 50.0}),
    (700, ref.ragged(5, 70, 1, 300), 16, 8, 128, 64, F16, {}),
    (700, ref.ragged(6, 130, 1, 100), 32, 4, 64, 16, BF16, {"slopes": True}),
]


def _prefix(llmik, dev, P, own, H, Hkv, D, page, dtype, opts, seed=0, lens=None):
    lens = [P + n for n in own] if lens is None else lens
    k, v, table, seq = ref.make_cache(lens + [P], Hkv, D, page, dtype, dev, seed)
    prefix_pages = table[-1, :-(-P // page)].contiguous()
    table, seq = table[:-1].contiguous(), seq[:-1].contiguous()
    table[:, :P // page] = -1                      # the rows' own entries of the prefix are not read
    q = _q(len(lens), H, D, dtype, dev, seed + 1)
    opts = dict(opts)
    if opts.get("slopes") is True:
        opts["slopes"] = _slopes(H, dev)
    scale = 1.0 / math.sqrt(D)
    got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, prefix_pages, P, scale, **opts)
    want, bound = ref.attention(q, k, v, table, lens, [1] * len(lens), scale, page, False, prefix_pages=prefix_pages,
                                prefix_len=P, **opts)
    return got, want, bound


@pytest.mark.parametrize("case", PREFIX, ids=_id)
def test_shared_prefix(llmik, cuda, case):
    got, want, bound = _prefix(llmik, cuda, *case)
    ref.check(got, want, bound)


def test_shared_prefix_with_rows_shorter_than_it(llmik, cuda):
    got, want, bound = _prefix(llmik, cuda, 500, None, 32, 8, 128, 16, F16, {}, lens=[0, 1, 300, 500, 501, 900])
    ref.check(got, want, bound)
    assert int(got[0].count_nonzero()) == 0


# ---------------------------------------------------------- what no row may see

def _plant(cache, table_row, page, tokens, value):
    for t in tokens:
        cache[int(table_row[t // page]), :, t % page] = value


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_slots_without_a_live_token_are_never_used(llmik, cuda, fill, dtype):
    """Unwritten slots of used pages and pages that nobody owns hold values that
    are no numbers; decode, prompts and a prefix that end inside pages and tiles."""
    got, want, bound = _decode(llmik, cuda, [1, 33, 0, 700, 95], 8, 2, 128, 16, dtype, {}, fill=fill)
    ref.check(got, want, bound)
    got, want, bound = _prefill(llmik, cuda, [5, 0, 100], [33, 70, 1], 8, 2, 64, 24, dtype, {}, fill=fill)
    ref.check(got, want, bound)
    P, lens = 203, [210, 204, 150, 0]
    k, v, table, seq = ref.make_cache(lens + [P], 2, 128, 16, dtype, cuda, 7, fill=fill)
    pages, table, seq = table[-1, :13].contiguous(), table[:-1].contiguous(), seq[:-1].contiguous()
    q = _q(4, 8, 128, dtype, cuda, 8)
    got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, pages, P, 0.09)
    want, bound = ref.attention(q, k, v, table, lens, [1] * 4, 0.09, 16, False, prefix_pages=pages, prefix_len=P)
    ref.check(got, want, bound)


@pytest.mark.parametrize("value", [math.nan, math.inf], ids=str)
@pytest.mark.parametrize("where", ["k", "v", "both"])
@pytest.mark.parametrize("G", [1, 4])
def test_later_and_older_tokens_that_are_no_numbers(llmik, cuda, value, where, G):
    """A live token whose K or V is no number reaches the rows that see it and no
    other: a later token of the same prompt, and one that left the window."""
    H, Hkv, D, page, n, window = 2 * G, 2, 128, 16, 150, 40
    bad = [20, 90, 91]
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, F16, cuda, 3)
    for c, name in ((k, "k"), (v, "v")):
        if where in (name, "both"):
            _plant(c, table[0], page, bad, value)
    q = _q(n, H, D, F16, cuda, 4)
    cu = ref.offsets([n], cuda)
    pos = torch.arange(n, device=cuda)
    for w in (0, window):
        got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.09, window=w)
        dist = pos[:, None] - torch.tensor(bad, device=cuda)
        sees = (dist >= 0) & ((dist < w) if w else True)
        clean = ~sees.any(-1)
        # the rows that see none of them, from a cache without them
        k2, v2 = k.clone(), v.clone()
        _plant(k2, table[0], page, bad, 0.0)
        _plant(v2, table[0], page, bad, 0.0)
        want, bound = ref.attention(q, k2, v2, table, [n], [n], 0.09, page, False, window=w)
        ref.check(got[clean], want[clean], bound[clean])
        assert not bool(torch.isfinite(got[~clean]).all(-1).any())


def test_decode_and_prefix_windows_leave_out_tokens_that_are_no_numbers(llmik, cuda):
    H, Hkv, D, page, P = 8, 2, 128, 32, 300
    lens = [310, 420, 350]
    k, v, table, seq = ref.make_cache(lens + [P], Hkv, D, page, BF16, cuda, 5)
    pages, table, seq = table[-1, :10].contiguous(), table[:-1].contiguous(), seq[:-1].contiguous()
    q = _q(3, H, D, BF16, cuda, 6)
    # positions 200 .. 249 of the prefix: with a window of 100 only row 0 (210 .. 309) sees some
    _plant(v, pages, page, range(200, 250), math.nan)
    got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, pages, P, 0.09, window=100)
    assert bool(got[0].isnan().all())
    v2 = v.clone()
    _plant(v2, pages, page, range(200, 250), 0.0)
    want, bound = ref.attention(q, k, v2, table, lens, [1] * 3, 0.09, page, False, prefix_pages=pages, prefix_len=P,
                                window=100)
    ref.check(got[1:], want[1:], bound[1:])
    for b in range(3):
        _plant(v, table[b], page, range(lens[b] - 101), math.inf)   # all but the last 101: a window of 100 sees none
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.09, window=100)
    want, bound = ref.attention(q, k, v, table, lens, [1] * 3, 0.09, page, True, window=100)
    # the reference multiplies masked values by 0: from a cache without them
    v3 = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    want, bound = ref.attention(q, k, v3, table, lens, [1] * 3, 0.09, page, True, window=100)
    ref.check(got, want, bound)


def test_unmapped_pages_are_no_keys(llmik, cuda):
    H, Hkv, D, page, lens = 8, 2, 128, 16, [200, 77]
    for bad in (-1, 10 ** 6, -2 ** 31):
        k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 9)
        table[0, 3] = bad                   # tokens 48 .. 63
        table[0, 11] = bad                  # 176 .. 191
        table[1, :] = bad                   # the whole sequence
        q = _q(2, H, D, F16, cuda, 10)
        got = llmik.paged_decode_attention(q, k, v, table, seq, 0.09)
        want, bound = ref.attention(q, k, v, table, lens, [1, 1], 0.09, page, True)
        ref.check(got, want, bound)
        assert int(got[1].count_nonzero()) == 0
        new = [100, 77]
        q = _q(177, H, D, F16, cuda, 11)
        got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets(new, cuda), 0.09)
        want, bound = ref.attention(q, k, v, table, lens, new, 0.09, page, False)
        ref.check(got, want, bound)
        prefix = table[0, :7].contiguous()
        q = _q(2, H, D, F16, cuda, 12)
        got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, prefix, 100, 0.09)
        want, bound = ref.attention(q, k, v, table, lens, [1, 1], 0.09, page, False, prefix_pages=prefix,
                                    prefix_len=100)
        ref.check(got, want, bound)


def test_lengths_past_the_table_and_below_zero(llmik, cuda):
    """Tokens behind the table's columns do not exist, negative lengths are empty,
    and positions near 2^31 read nothing."""
    H, Hkv, D, page = 4, 2, 128, 16
    k, v, table, _ = ref.make_cache([64, 64, 64, 64], Hkv, D, page, F16, cuda, 13, extra_columns=0)
    lens = [100, -5, 2 ** 31 - 1, 64]
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = _q(4, H, D, F16, cuda, 14)
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.09)
    want, bound = ref.attention(q, k, v, table, [64] * 4, [1] * 4, 0.09, page, True)
    ref.check(got[[0, 2, 3]], want[[0, 2, 3]], bound[[0, 2, 3]])
    assert int(got[1].count_nonzero()) == 0
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.09, window=10)
    assert int(got[:3].count_nonzero()) == 0      # the newest 10 positions of 100 and of 2^31 - 1 lie behind the table
    want, bound = ref.attention(q, k, v, table, [64] * 4, [1] * 4, 0.09, page, True, window=10)
    ref.check(got[3:], want[3:], bound[3:])
    # prompts: a sequence shorter than its new rows (positions below zero see nothing)
    q = _q(20, H, D, F16, cuda, 15)
    cu = torch.tensor([0, 12, 20, 20, 20], dtype=torch.int32, device=cuda)
    seq = torch.tensor([5, 2 ** 31 - 1, 0, 0], dtype=torch.int32, device=cuda)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.09)
    assert int(got[:7].count_nonzero()) == 0
    want, bound = ref.attention(q[7:12], k, v, table, [5], [5], 0.09, page, False)
    ref.check(got[7:12], want, bound)
    kb, ok = ref.tokens_of(k, table[1], 64, page)
    vb, _ = ref.tokens_of(v, table[1], 64, page)
    want, bound = ref.attend(q[12:], kb, vb, ok, torch.full((8,), 10 ** 6, device=cuda), 0.09, up=2.0 ** -11)
    ref.check(got[12:], want, bound)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.09, window=5)
    assert int(got[12:].count_nonzero()) == 0


@pytest.mark.parametrize("length", [-1, -2 ** 31])
def test_negative_lengths_are_empty(llmik, cuda, length):
    H, Hkv, D, page = 4, 2, 64, 16
    k, v, table, _ = ref.make_cache([200, 200], Hkv, D, page, F16, cuda, 13)
    seq = torch.full((2,), length, dtype=torch.int32, device=cuda)
    q = _q(2, H, D, F16, cuda, 14)
    for window in (0, 5):
        assert int(llmik.paged_decode_attention(q, k, v, table, seq, 0.1, window=window).count_nonzero()) == 0
        assert int(llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([1, 1], cuda), 0.1,
                                                 window=window).count_nonzero()) == 0
        assert int(llmik.paged_shared_prefix_attention(q, k, v, table, seq, table[0].contiguous(), 150, 0.1,
                                                       window=window).count_nonzero()) == 0


def test_nan_queries_stay_nan(llmik, cuda):
    k, v, table, seq = ref.make_cache([50, 60], 2, 64, 16, F16, cuda, 16)
    q = _q(2, 4, 64, F16, cuda, 17)
    q[1, 2] = math.nan
    for got in (llmik.paged_decode_attention(q, k, v, table, seq, 0.1),
                llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([1, 1], cuda), 0.1),
                llmik.paged_shared_prefix_attention(q, k, v, table, seq, table[0].contiguous(), 40, 0.1)):
        assert bool(got[1, 2].isnan().all()) and bool(torch.isfinite(got[0]).all())
        assert bool(torch.isfinite(got[1, [0, 1, 3]]).all())


def test_a_wide_range_of_scores(llmik, cuda):
    """One key far above the rest, and rows whose largest score grows from tile to
    tile, in both types: the reference of the exponents moves many times."""
    for dtype in (F16, BF16):
        n, H, Hkv, D, page = 1000, 8, 2, 128, 16
        k, v, table, seq = ref.make_cache([n], Hkv, D, page, dtype, cuda, 18)
        q = _q(n, H, D, dtype, cuda, 19, spread=1.0)
        for t in range(n):
            k[int(table[0, t // page]), :, t % page] *= 0.05 + 4.0 * t / n
        k[int(table[0, 500 // page]), 0, 500 % page] *= 8.0
        cu = ref.offsets([n], cuda)
        got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.3)
        want, bound = ref.attention(q, k, v, table, [n], [n], 0.3, page, False)
        ref.check(got, want, bound)
        got = llmik.paged_decode_attention(q[-1:], k, v, table, seq, 0.3)
        want, bound = ref.attention(q[-1:], k, v, table, [n], [1], 0.3, page, True)
        ref.check(got, want, bound)
        got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, -0.3)
        want, bound = ref.attention(q, k, v, table, [n], [n], -0.3, page, False)
        ref.check(got, want, bound)


# ------------------------------------------------------ offsets, streams, graphs

def test_offsets_past_32_bits(llmik, cuda):
    """Pages beyond 4 GiB (and 2^31 elements) of a cache with a wide page stride."""
    H, Hkv, D, page, lens = 8, 2, 128, 16, [100, 70]
    stride = 1 << 28                                # elements between pages: page 11 lies 5.5 GiB in
    n_pages = 12
    pool_k = torch.empty(n_pages, stride, dtype=F16, device=cuda)
    pool_v = torch.empty(n_pages, stride, dtype=F16, device=cuda)
    shape = (n_pages, Hkv, page, D)
    k = pool_k[:, :Hkv * page * D].unflatten(1, shape[1:])
    v = pool_v[:, :Hkv * page * D].unflatten(1, shape[1:])
    gen = torch.Generator(device=cuda).manual_seed(1)
    k.copy_(torch.randn(shape, generator=gen, device=cuda))
    v.copy_(torch.randn(shape, generator=gen, device=cuda))
    table = torch.tensor([[11, 0, 9, 10, 3, 8, 5], [1, 7, 6, 2, 4, -1, -1]], dtype=torch.int32, device=cuda)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = _q(2, H, D, F16, cuda, 2)
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.09)
    want, bound = ref.attention(q, k, v, table, lens, [1, 1], 0.09, page, True)
    ref.check(got, want, bound)
    q = _q(60, H, D, F16, cuda, 3)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([40, 20], cuda), 0.09)
    want, bound = ref.attention(q, k, v, table, lens, [40, 20], 0.09, page, False)
    ref.check(got, want, bound)
    qkv = torch.randn(2, (H + 2 * Hkv) * D, generator=gen, device=cuda).half()
    llmik.rope_paged_append(qkv, None, None, k, v, table, seq)
    x = qkv.view(2, H + 2 * Hkv, D)
    assert torch.equal(k[5, :, 3], x[0, H:H + Hkv]) and torch.equal(v[4, :, 5], x[1, H + Hkv:])


def _calls(llmik, dev, seed=0):
    """The three attentions at sizes that hand parts over."""
    H, Hkv, D, page = 32, 8, 128, 16
    lens = [5000, 1300, 2900]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, dev, seed)
    q1, q2 = _q(3, H, D, F16, dev, seed + 1), _q(48, H, D, F16, dev, seed + 2)
    cu, pages = ref.offsets([16, 16, 16], dev), table[0, :80].contiguous()
    return [lambda: llmik.paged_decode_attention(q1, k, v, table, seq, 0.09),
            lambda: llmik.paged_prefill_attention(q2, k, v, table, seq, cu, 0.09),
            lambda: llmik.paged_shared_prefix_attention(q1, k, v, table, seq, pages, 1280, 0.09)]


def test_repeated_calls_give_the_same_bits(llmik, cuda):
    for call in _calls(llmik, cuda):
        first = call()
        outs = [call() for _ in range(30)]
        assert all(torch.equal(first, o) for o in outs)


def test_two_streams_at_once(llmik, cuda):
    calls = _calls(llmik, cuda)
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([c() for c in calls])
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_graphs_captured_on_one_stream_replay_on_two(llmik, cuda):
    """Two graphs share nothing, also where they were captured on one stream whose
    eager workspace exists; replays with eager calls and table changes between."""
    calls = _calls(llmik, cuda)
    want = [c() for c in calls]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for c in calls:
            c()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append([c() for c in calls])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(8):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        eager = [c() for c in calls]
        torch.cuda.synchronize()
        for o in outs + [eager]:
            assert all(torch.equal(a, b) for a, b in zip(o, want))
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()


def test_a_replayed_graph_follows_lengths_and_tables(llmik, cuda):
    """A decode step is captured once; its tables and lengths change between replays."""
    H, Hkv, D, page, B = 16, 4, 64, 16, 5
    lens = [900, 3, 77, 0, 400]
    k, v, table, seq = ref.make_cache([1000] * B, Hkv, D, page, BF16, cuda, 30)
    q = _q(B, H, D, BF16, cuda, 31)
    seq.copy_(torch.tensor(lens, dtype=torch.int32))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = llmik.paged_decode_attention(q, k, v, table, seq, 0.1, window=600)
    for turn in range(4):
        lens = [(n * 7 + 13 * turn) % 1000 for n in lens]
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(table.roll(1, 0))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, bound = ref.attention(q, k, v, table, lens, [1] * B, 0.1, page, True, window=600)
        ref.check(out, want, bound)


def test_empty_batches(llmik, cuda):
    k, v, table, seq = ref.make_cache([10], 2, 128, 16, F16, cuda, 32)
    none, t0 = seq[:0], table[:0]
    q0 = torch.zeros(0, 4, 128, dtype=F16, device=cuda)
    assert llmik.paged_decode_attention(q0, k, v, t0, none, 0.1).shape == (0, 4, 128)
    assert llmik.paged_shared_prefix_attention(q0, k, v, t0, none, table[0].contiguous(), 5, 0.1).shape == (0, 4, 128)
    cu = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = torch.ones(3, 4, 128, dtype=F16, device=cuda)
    assert int(llmik.paged_prefill_attention(q, k, v, t0, none, cu, 0.1).count_nonzero()) == 0
    cu = torch.zeros(2, dtype=torch.int32, device=cuda)
    assert int(llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.1).count_nonzero()) == 0
    q = torch.ones(1, 4, 128, dtype=F16, device=cuda)
    want = llmik.paged_decode_attention(q, k, v, table, seq, 0.1)
    got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, table[0, :0].contiguous(), 0, 0.1)
    assert torch.equal(got, want)


def test_a_long_table_of_many_sequences(llmik, cuda):
    """More sequences than lanes times lanes' share: 300 of 0 .. 40 tokens, most empty
    rows of a wide table, prompts and decode."""
    lens = ref.ragged(40, 300, -20, 40)
    lens = [max(n, 0) for n in lens]
    got, want, bound = _decode(llmik, cuda, lens, 4, 2, 64, 8, F16, {}, extra_columns=50)
    ref.check(got, want, bound)
    new = [min(n, 1 + i % 7) for i, n in enumerate(lens)]
    got, want, bound = _prefill(llmik, cuda, [n - m for n, m in zip(lens, new)], new, 4, 2, 64, 8, F16, {},
                                extra_columns=50)
    ref.check(got, want, bound)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_scales_of_zero_and_below(llmik, cuda, scale, softcap):
    lens, H, Hkv, D, page = [300, 65], 8, 2, 128, 16
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 3)
    for new in ([1, 1], [130, 65]):
        q = _q(sum(new), H, D, F16, cuda, 4)
        if new == [1, 1]:
            got = llmik.paged_decode_attention(q, k, v, table, seq, scale, softcap)
        else:
            got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets(new, cuda), scale, softcap)
        want, bound = ref.attention(q, k, v, table, lens, new, scale, page, new == [1, 1], softcap=softcap)
        ref.check(got, want, bound)


# ----------------------------------------------------------------- drawn shapes

def _drawn(seed):
    rng = random.Random(seed)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))   # noqa: E731
    Hkv = rng.choice([1, 2, 3, 4, 8])
    shape = (Hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 17]), Hkv, rng.choice([64, 128]),
             8 * rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([F16, BF16]))
    opts = {}
    if rng.random() < 0.3:
        opts["softcap"] = rng.choice([5.0, 30.0])
    if rng.random() < 0.3:
        opts["slopes"] = True
    if rng.random() < 0.3:
        opts["window"] = log(1, 3000)
    return rng, log, shape, opts


@pytest.mark.parametrize("seed", range(16))
def test_drawn_decodes(llmik, cuda, seed):
    rng, log, shape, opts = _drawn(100 + seed)
    hi = log(1, 6000)
    lens = [rng.randint(0, hi) for _ in range(log(1, 90))]
    got, want, bound = _decode(llmik, cuda, lens, *shape, opts, seed=seed)
    ref.check(got, want, bound)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_prompts(llmik, cuda, seed):
    rng, log, shape, opts = _drawn(200 + seed)
    B = rng.randint(1, 6)
    ctx = [rng.choice([0, log(1, 4000)]) for _ in range(B)]
    new = [rng.choice([0, log(1, 400)]) for _ in range(B)]
    got, want, bound = _prefill(llmik, cuda, ctx, new, *shape, opts, seed=seed, pad=rng.randint(0, 3))
    ref.check(got, want, bound)


@pytest.mark.parametrize("seed", range(16))
def test_drawn_prefixes(llmik, cuda, seed):
    rng, log, shape, opts = _drawn(300 + seed)
    P = log(1, 5000)
    own = [rng.randint(1, 300) for _ in range(log(1, 60))]
    got, want, bound = _prefix(llmik, cuda, P, own, *shape, opts, seed=seed)
    ref.check(got, want, bound)
