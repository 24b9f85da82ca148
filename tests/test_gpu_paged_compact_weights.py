"""GPU: what paged_compact does to weights where tokens stay: weights go by the entries' slots
alone, and end at the first negative entry. All values are exact."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _cache(dev, table):
    """Two heads; the K of the token in page p, slot s is 100 p + s, V its negative."""
    k = (100 * torch.arange(4.0)[:, None, None, None] + torch.arange(8.0)[None, None, :, None]).expand(4, 2, 8, 64)
    k = k.contiguous().half().to(dev)
    w = torch.arange(1.0, 25.0).repeat(1, 2, 1).to(dev)      # slot t: t + 1
    return k, -k, torch.tensor([table], dtype=I32, device=dev), torch.tensor([24], dtype=I32, device=dev), w


def _tokens(k, page):
    return k[page, 0, :, 0].tolist()


@pytest.mark.parametrize("table,moved", [([0, 1, 2], True), ([-1, 1, 2], False), ([0, 1, 4], False)], ids=str)
def test_weights_go_by_slots_whatever_the_pages(llmik, cuda, table, moved):
    """Slots 17 and 20 go to slots 0 and 1: the tokens where both pages are mapped, the weights always."""
    k, v, tab, lens, w = _cache(cuda, table)
    k0 = k.clone()
    llmik.paged_compact(k, v, tab, lens, torch.tensor([[17, 20]], dtype=I32, device=cuda), None, w)
    if moved:
        assert _tokens(k, 0)[:3] == [201.0, 204.0, 2.0] and _tokens(v, 0)[:3] == [-201.0, -204.0, -2.0]
    else:
        assert torch.equal(k, k0) and torch.equal(v, -k0)
    assert w.tolist() == [[[18.0, 21.0] + [0.0] * 22] * 2]


def test_weights_end_at_the_first_negative_entry(llmik, cuda):
    """The token behind it moves, its weight does not: it becomes 0 as all behind."""
    k, v, tab, lens, w = _cache(cuda, [0, 1, 2])
    llmik.paged_compact(k, v, tab, lens, torch.tensor([[9, -1, 20]], dtype=I32, device=cuda), None, w)
    assert _tokens(k, 0)[:4] == [101.0, 1.0, 204.0, 3.0]
    assert w.tolist() == [[[10.0] + [0.0] * 23] * 2]
