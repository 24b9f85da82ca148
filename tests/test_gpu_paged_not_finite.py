"""GPU: infinities and NaN in live values of a paged cache. A channel of a row is
sum_j p_j v_j with every p_j > 0: inf where the keys that the row sees hold inf,
-inf where they hold -inf, NaN where both or a NaN. All other channels are as if
those values were zeros (tests/paged_ref.py, where their tolerances are derived)."""
from __future__ import annotations

import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
INF = math.inf


def _plant(cache, table_row, page, token, channel, value):
    cache[int(table_row[token // page]), :, token % page, channel] = value


def _check(got, want, bound, marks):
    """marks: channel -> what it has to be, for rows [n, H, D]."""
    got = got.clone()
    for channel, value in marks.items():
        x = got[..., channel]
        same = x.isnan() if math.isnan(value) else x == value
        assert bool(same.all()), (channel, value, x[~same][:4].tolist())
        got[..., channel] = want[..., channel].to(got.dtype)
    keep = [c for c in range(got.shape[-1]) if c not in marks]
    ref.check(got[..., keep], want[..., keep], bound[..., keep])


MARKS = {3: INF, 10: -INF, 17: math.nan, 40: math.nan, 63: INF}


def _mark(v, table_row, page, first, second):
    """Values at two tokens that give MARKS: channel 40 has infinities of both signs."""
    for channel, value in ((3, INF), (10, -INF), (17, math.nan), (40, INF)):
        _plant(v, table_row, page, first, channel, value)
    for channel, value in ((3, INF), (40, -INF), (63, INF)):
        _plant(v, table_row, page, second, channel, value)


@pytest.mark.parametrize("n", [2, 33, 700, 20000])   # a tile, two, a piece per wave, many tiles a wave in parts
@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 128), (F16, 64), (BF16, 64)], ids=str)
def test_decode_keeps_infinities(llmik, cuda, n, dtype, D):
    H, Hkv, page = 8, 2, 16
    k, v, table, seq = ref.make_cache([n, 90], Hkv, D, page, dtype, cuda, 1)
    gen = torch.Generator(device=cuda).manual_seed(2)
    q = (2.0 * torch.randn(2, H, D, generator=gen, device=cuda)).to(dtype)
    # the largest key of a head (its p is exact, the second part is zero) and an early token
    kb, _ = ref.tokens_of(k, table[0], n, page)
    top = int((kb[0] @ q[0, 0].double()).argmax())
    other = 0 if top else 1
    clean = v.clone()
    for channel in MARKS:
        for t in (top, other):
            _plant(clean, table[0], page, t, channel, 0.0)
    want, bound = ref.attention(q, k, clean, table, [n, 90], [1, 1], 0.09, page, True)
    _mark(clean, table[0], page, top, other)
    got = llmik.paged_decode_attention(q, k, clean, table, seq, 0.09)
    _check(got[:1], want[:1], bound[:1], MARKS)
    ref.check(got[1:], want[1:], bound[1:])


@pytest.mark.parametrize("n", [100, 9000])
def test_decode_keeps_infinities_of_small_probabilities(llmik, cuda, n):
    """The first token's probability is below what 16 bits hold (2^-33 of the largest's),
    and below what 32 bits hold: a distance bias of 1 and of 2 a token."""
    H, Hkv, D, page = 4, 2, 64, 32
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, F16, cuda, 3)
    gen = torch.Generator(device=cuda).manual_seed(4)
    q = torch.randn(1, H, D, generator=gen, device=cuda).half()
    slopes = torch.tensor([0.3, 1.0, 2.0, 0.01], device=cuda)
    for channel in (5, 6):
        for t in (0, n // 2):
            _plant(v, table[0], page, t, channel, 0.0)
    want, bound = ref.attention(q, k, v, table, [n], [1], 0.1, page, True, slopes=slopes)
    _plant(v, table[0], page, 0, 5, INF)
    _plant(v, table[0], page, n // 2, 6, -INF)
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.1, slopes=slopes)
    _check(got, want, bound, {5: INF, 6: -INF})


def test_decode_leaves_out_infinities_that_no_row_sees(llmik, cuda):
    """Beside a live infinity, masked tokens of the same tile that are no numbers."""
    H, Hkv, D, page, n, window = 4, 2, 128, 64, 150, 40
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, BF16, cuda, 5, fill=math.nan)
    gen = torch.Generator(device=cuda).manual_seed(6)
    q = torch.randn(1, H, D, generator=gen, device=cuda).to(BF16)
    _plant(v, table[0], page, 120, 9, 0.0)
    want, bound = ref.attention(q, k, v, table, [n], [1], 0.1, page, True, window=window)
    _plant(v, table[0], page, 120, 9, INF)
    for t in (n - window - 1, n - window - 5):
        _plant(v, table[0], page, t, slice(None), math.nan)
        _plant(k, table[0], page, t, slice(None), -INF)
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.1, window=window)
    _check(got, want, bound, {9: INF})


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64)], ids=str)
def test_own_tokens_behind_a_prefix_keep_infinities(llmik, cuda, dtype, D):
    H, Hkv, page, P, lens = 8, 2, 16, 300, [310, 700, 301]
    k, v, table, seq = ref.make_cache(lens + [P], Hkv, D, page, dtype, cuda, 7)
    pages, table, seq = table[-1, :-(-P // page)].contiguous(), table[:-1].contiguous(), seq[:-1].contiguous()
    gen = torch.Generator(device=cuda).manual_seed(8)
    q = (2.0 * torch.randn(3, H, D, generator=gen, device=cuda)).to(dtype)
    spots = [(0, 305, 309), (1, 300, 650)]
    for b, s, t in spots:
        for channel in MARKS:
            _plant(v, table[b], page, s, channel, 0.0)
            _plant(v, table[b], page, t, channel, 0.0)
    want, bound = ref.attention(q, k, v, table, lens, [1] * 3, 0.09, page, False, prefix_pages=pages, prefix_len=P)
    for b, s, t in spots:
        _mark(v, table[b], page, s, t)
    got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, pages, P, 0.09)
    _check(got[:2], want[:2], bound[:2], MARKS)
    ref.check(got[2:], want[2:], bound[2:])


@pytest.mark.parametrize("ctx,new", [(0, 150), (3000, 40)])   # one part, keys in parts
def test_prompts_keep_infinities(llmik, cuda, ctx, new):
    """Scores of one size, so that every probability is one of 16 bits."""
    H, Hkv, D, page, n = 4, 2, 128, 16, ctx + new
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, F16, cuda, 9)
    gen = torch.Generator(device=cuda).manual_seed(10)
    q = (0.3 * torch.randn(new, H, D, generator=gen, device=cuda)).half()
    cu = ref.offsets([new], cuda)
    first, second = ctx // 2, ctx + new // 2
    for channel in MARKS:
        for t in (first, second):
            _plant(v, table[0], page, t, channel, 0.0)
    want, bound = ref.attention(q, k, v, table, [n], [new], 0.09, page, False)
    _mark(v, table[0], page, first, second)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, cu, 0.09)
    _check(got[second - ctx:], want[second - ctx:], bound[second - ctx:], MARKS)
    one = {3: INF, 10: -INF, 17: math.nan, 40: INF}
    _check(got[:second - ctx], want[:second - ctx], bound[:second - ctx], one)


def test_prompts_keep_infinities_of_small_probabilities(llmik, cuda):
    """A distance bias of 4 a token: from 30 tokens on a probability is 0 in 32 bits. The
    rows that see the infinity are no numbers all the same, those of its own tile inf."""
    H, Hkv, D, page, n = 4, 2, 64, 16, 150
    k, v, table, seq = ref.make_cache([n], Hkv, D, page, F16, cuda, 11)
    gen = torch.Generator(device=cuda).manual_seed(12)
    q = torch.randn(n, H, D, generator=gen, device=cuda).half()
    slopes = torch.full((H,), 4.0, device=cuda)
    _plant(v, table[0], page, 20, 7, 0.0)
    want, bound = ref.attention(q, k, v, table, [n], [n], 0.1, page, False, slopes=slopes)
    _plant(v, table[0], page, 20, 7, INF)
    got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([n], cuda), 0.1, slopes=slopes)
    ref.check(got[:20], want[:20], bound[:20])
    _check(got[20:64], want[20:64], bound[20:64], {7: INF})
    assert not bool(torch.isfinite(got[20:, :, 7]).any())
    keep = [c for c in range(D) if c != 7]
    ref.check(got[20:, :, keep], want[20:, :, keep], bound[20:, :, keep])
