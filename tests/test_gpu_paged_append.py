"""GPU: new tokens into a paged cache with the rotary embedding on the way,
against the float64 definition and, for fp16, against `rope` bit for bit."""
from __future__ import annotations

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _tables(n, D, dtype, dev):
    ang = torch.arange(n, device=dev, dtype=torch.float64)[:, None] / (
        10000.0 ** (torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))[None]
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


CASES = [
    # context, new (None: a decode step of seq lens), H, Hkv, D, page, dtype, table dtype, pad rows
    ([0], [1], 4, 1, 128, 16, F16, F16, 0),
    ([0, 5, 100], [3, 1, 60], 32, 8, 128, 16, F16, F16, 0),
    ([0, 5, 100], [3, 0, 60], 32, 8, 128, 24, BF16, F32, 4),
    ([7, 0, 30], [200, 9, 1], 28, 4, 64, 8, BF16, BF16, 1),
    ([7, 0, 30], [200, 9, 1], 1, 1, 64, 32, F16, F32, 0),
    ([0] * 70, [2] * 70, 8, 8, 128, 16, F16, F16, 3),       # more than one wave of sequence ends
    ([100, 3], [500, 700], 64, 8, 128, 64, F16, F16, 0),
    ([699, 0, 15, 16, 1], None, 32, 8, 128, 16, F16, F16, 0),
    ([5] * 9, None, 40, 8, 64, 64, BF16, F32, 0),
    ([3, 4], [2, 5], 16, 2, 128, 16, BF16, None, 0),        # no rotation
]


def _run(llmik, dev, ctx, new, H, Hkv, D, page, dtype, tdtype, pad, seed=3, gap=0):
    step = new is None
    counts = [1] * len(ctx) if step else new
    lens = [a + b for a, b in zip(ctx, counts)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, dev, seed, gap=gap)
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows = sum(counts) + pad
    qkv = torch.randn(rows, (H + 2 * Hkv) * D, generator=gen, device=dev).to(dtype)
    cos, sin = (None, None) if tdtype is None else _tables(max(lens) + 2, D, tdtype, dev)
    k0, v0 = k.clone(), v.clone()
    q = llmik.rope_paged_append(qkv, cos, sin, k, v, table, seq, None if step else ref.offsets(counts, dev))
    # the definition
    wk, wv = k0.double(), v0.double()
    wq = torch.zeros(rows, H, D, dtype=torch.float64, device=dev)
    written = torch.zeros(k0.shape[0], page, dtype=torch.bool, device=dev)
    for b, r0, n, pos in ref.rows_of(lens, counts):
        x = qkv[r0:r0 + n].double().view(n, H + 2 * Hkv, D)
        p = torch.arange(pos, pos + n, device=dev)
        turned = x if cos is None else ref.rotate(x, cos[p].double(), sin[p].double())
        wq[r0:r0 + n] = turned[:, :H]
        pages = table[b][p // page].long()
        wk[pages, :, p % page] = turned[:, H:H + Hkv]
        wv[pages, :, p % page] = x[:, H + Hkv:]
        written[pages, p % page] = True
    return qkv, cos, sin, q, k, v, wq, wk, wv, written, k0, v0, lens, counts


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B%d-%s" % (len(c[0]), "-".join(str(x) for x in c[2:]).replace("torch.", "")))
def test_append(llmik, cuda, case):
    dtype = case[6]
    qkv, cos, sin, q, k, v, wq, wk, wv, written, k0, v0, _, _ = _run(llmik, cuda, *case)
    # Two fp32 products and their sum: 2^-24 of each product and of the sum, then
    # half a step of the result's type. |x cos| + |x' sin| <= 2 max|x|.
    top = qkv.abs().max().double()
    for got, want in ((q, wq), (k, wk)):
        bound = ref.U[dtype] * want.abs() + 2.0 ** -24 * 4 * top + (2.0 ** -25 if dtype == F16 else 0.0)
        assert bool(((got.double() - want).abs() <= bound * (1 + 2.0 ** -10)).all())
    assert torch.equal(v.double(), wv)                       # moved, not computed
    left = (~written)[:, None, :, None].expand_as(k0)
    assert torch.equal(k[left], k0[left])


def test_append_equals_rope_bit_for_bit(llmik, cuda):
    """fp16 q and k with fp16 tables: the rows that `rope` gives."""
    H, Hkv, D = 32, 8, 128
    qkv, cos, sin, q, k, v, *_, lens, counts = _run(llmik, cuda, [0, 5], [70, 41], H, Hkv, D, 16, F16, F16, 0)
    for b, r0, n, pos in ref.rows_of(lens, counts):
        x = qkv[r0:r0 + n].view(1, n, H + 2 * Hkv, D).transpose(1, 2).contiguous()
        want = llmik.rope(x[:, :H].contiguous(), cos[pos:pos + n], sin[pos:pos + n])
        assert torch.equal(q[r0:r0 + n], want[0].transpose(0, 1))


def test_append_into_views_of_one_allocation(llmik, cuda):
    """K and V pages side by side in one allocation: a page stride of two pages."""
    H, Hkv, D, page, n = 8, 2, 128, 16, 5
    both = torch.zeros(n, 2, Hkv, page, D, device=cuda, dtype=F16)
    apart = torch.zeros(2, n, Hkv, page, D, device=cuda, dtype=F16)
    table = torch.tensor([[3, 1, 4]], dtype=torch.int32, device=cuda)
    seq = torch.tensor([40], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 40], dtype=torch.int32, device=cuda)
    qkv = torch.randn(40, (H + 2 * Hkv) * D, device=cuda).half()
    cos, sin = _tables(64, D, F16, cuda)
    q = llmik.rope_paged_append(qkv, cos, sin, both[:, 0], both[:, 1], table, seq, cu)
    llmik.rope_paged_append(qkv, cos, sin, apart[0], apart[1], table, seq, cu)
    assert torch.equal(both.transpose(0, 1), apart)
    one = llmik.paged_prefill_attention(q, both[:, 0], both[:, 1], table, seq, cu, 0.1)
    two = llmik.paged_prefill_attention(q, apart[0], apart[1], table, seq, cu, 0.1)
    assert torch.equal(one, two)
