"""GPU: a drafted tree's probabilities are as exact as a decode step's: they enter the
products with V as a pair of 16-bit values, so that ref.PAIR is left of each, not ref.U
(tests/bounded_ref.py, tests/paged_ref.py: where the bounds are derived)."""
from __future__ import annotations

import math
import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

CASES = [
    # context, drafted, H, Hkv, D, page, dtype, options
    (700, 8, 32, 8, 128, 16, F16, {}),
    (700, 8, 32, 8, 128, 16, BF16, {}),
    (8192, 64, 32, 8, 128, 64, BF16, {}),        # several parts, two row tiles
    (3000, 20, 8, 2, 64, 32, F16, {"softcap": 30.0}),
    (500, 70, 12, 4, 64, 16, BF16, {"window": 333}),
    (0, 5, 4, 1, 128, 8, F16, {}),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_probabilities_are_pairs(llmik, cuda, case):
    ctx, new, H, Hkv, D, page, dtype, opts = case
    k, v, table, seq = ref.make_cache([ctx + new], Hkv, D, page, dtype, cuda, 1)
    # scores of about 0.5: their own error is far below the probabilities' rounding
    q = (0.5 * torch.randn(new, H, D, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda)).to(dtype)
    mask, pos = bref.trees(random.Random(3), [new], [ctx])
    scale = 1.0 / math.sqrt(D)
    at = torch.tensor(pos, dtype=torch.int32, device=cuda)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets([new], cuda),
                                     bref.words_of(mask, -(-new // 64), cuda), scale, positions=at, **opts)
    n = ctx + new
    kb, ok = ref.tokens_of(k, table[0], n, page)
    vb, _ = ref.tokens_of(v, table[0], n, page)
    seen = torch.tensor([[True] * ctx + [bool(m >> j & 1) for j in range(new)] for m in mask], device=cuda)
    pos_k = torch.cat([torch.arange(ctx, device=cuda), at.long()])
    want, bound = bref.attend(q, kb, vb, ok, seen, at.long()[:, None] - pos_k, scale, ref.PAIR[dtype], **opts)
    ref.check(got, want, bound)


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)], ids=str)
@pytest.mark.parametrize("ctx", [40, 4000])
def test_infinities_that_all_rows_see_stay_infinities(llmik, cuda, dtype, D, ctx):
    """A cached token's value of both infinities and NaN, by channel: every row has them, of any
    probability, and the other channels are numbers and right."""
    new, page, bad = 9, 16, ctx // 2
    k, v, table, seq = ref.make_cache([ctx + new], 2, D, page, dtype, cuda, 4)
    q = (2.0 * torch.randn(new, 8, D, generator=torch.Generator(device=cuda).manual_seed(5), device=cuda)).to(dtype)
    mask, pos = bref.trees(random.Random(6), [new], [ctx])
    place = int(table[0, bad // page]), slice(None), bad % page
    v[place] = 0.0
    want, bound = bref.tree(q, k, v, table, [ctx + new], [new], mask, None, 0.2, page)
    v[place][:, :3] = torch.tensor([math.inf, -math.inf, math.nan], device=cuda)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets([new], cuda), bref.words_of(mask, 1, cuda), 0.2)
    assert bool((got[..., 0] == math.inf).all()) and bool((got[..., 1] == -math.inf).all())
    assert bool(got[..., 2].isnan().all())
    ref.check(got[..., 3:], want[..., 3:], bound[..., 3:])
