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
