"""GPU: drafted trees over batches whose sequences nearly all have parts to join: the number
of their records, counted over the lanes' sequences, is the last lane's (float64 definitions
and tolerances: tests/bounded_ref.py)."""
from __future__ import annotations

import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1, 63, 64, 65, 130])
def test_every_cut_sequence_is_joined(llmik, cuda, B):
    H, Hkv, D, page, dtype = 4, 1, 64, 32, torch.float16
    rng = random.Random(B)
    new = [rng.randint(1, 3) for _ in range(B)]
    ctx = [rng.randint(900, 1100) for _ in range(B)]
    ctx[-1] = 3000
    lens = [a + b for a, b in zip(ctx, new)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 1)
    gen = torch.Generator(device=cuda).manual_seed(2)
    q = torch.randn(sum(new), H, D, generator=gen, device=cuda).to(dtype)
    mask, pos = bref.trees(rng, new, ctx)
    got = llmik.paged_tree_attention(q, k, v, table, seq, ref.offsets(new, cuda), bref.words_of(mask, 1, cuda), 0.125,
                                     positions=torch.tensor(pos, dtype=torch.int32, device=cuda))
    want, bound = bref.tree(q, k, v, table, lens, new, mask, pos, 0.125, page)
    ref.check(got, want, bound)
