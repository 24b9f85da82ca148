"""GPU: capped scores over the whole range of caps, against the definition in 64 bits.

Score errors that are absolute in the cap show where a row has few keys and their
values cancel: two keys with v = +c, -c give tanh((s0 - s1) / 2) c, so an error e of a
score is one of e / 2 c of the output, whatever the output's size. The bound:

* the output's rounding, u |out|, and 2^-25 where fp16 is subnormal;
* a probability's: 2^-22 of it (2^-16 in bf16), in prompts u; the fp32 sums 2^-24 (16 + keys / 8);
* a score's e = (D + 8) 2^-24 sum |q k| scale (products, as in tests/paged_ref.py) + 2^-22
  (exp2) + 2^-20 |s| (the cap: 2^-21 of the score above a cap of 64, and four fp32 roundings
  of the score times log2(e)), or up to a cap of 64 instead of 2^-21 |s| 2^-20 cap; each changes p by
  a factor within 1 +- 2 e, and the sum of all p by as much: 4 e sum p |v|."""
from __future__ import annotations

import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _attend(q, k, v, pos, scale, cap, up, slopes=None):
    """q [L, H, D] at pos [L] over k, v [Hkv, n, D] in float64: (out, bound)."""
    L, H, D = q.shape
    n = k.shape[1]
    out = torch.zeros(L, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    seen = pos[:, None] >= torch.arange(n, device=q.device)
    for h in range(H):
        kh, vh, qh = k[h // (H // k.shape[0])], v[h // (H // k.shape[0])], q[:, h].double()
        s = cap * torch.tanh(qh @ kh.t().contiguous() * scale / cap)
        e = ((D + 8) * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().t().contiguous()) + 2.0 ** -22
             + 2.0 ** -20 * s.abs() + (2.0 ** -20 * cap if cap <= 64 else 0.0))
        if slopes is not None:
            bias = slopes[h].double() * (pos[:, None] - torch.arange(n, device=q.device))
            s, e = s - bias, e + 2.0 ** -22 * bias.abs()
        p = torch.softmax(s.masked_fill(~seen, -math.inf), dim=-1)
        worst = torch.where(seen, e, torch.zeros_like(e)).amax(-1, keepdim=True)
        out[:, h] = p @ vh
        bound[:, h] = (ref.U[q.dtype] * out[:, h].abs()
                       + (up + 4 * worst + 2.0 ** -24 * (16 + seen.sum(-1, keepdim=True) / 8.0)) * (p @ vh.abs())
                       + 2.0 ** -32 * n * vh.abs().amax() + (2.0 ** -25 if q.dtype == F16 else 0.0))
    return out, bound


def _inputs(dev, dtype, lens, rows, H, Hkv, D, page, seed, spread):
    """spread [H]: the size of a head's queries."""
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, dev, seed)
    gen = torch.Generator(device=dev).manual_seed(seed + 1)
    q = (spread[:, None] * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)
    return q, k, v, table, seq


CAPS = [0.5, 50.0, 64.0, 65.0, 200.0, 1000.0, 4096.0]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("D", [64, 128])
def test_two_keys(llmik, cuda, cap, D):
    """Scores from 1e-3 to thousands (a factor of ten a head), keys 0 and 1 of opposite values."""
    H, Hkv, page, B = 8, 1, 8, 64
    spread = torch.tensor([10.0 ** (0.9 * (h - 4)) for h in range(H)], device=cuda)
    q, k, v, table, seq = _inputs(cuda, F16, [2] * B, B, H, Hkv, D, page, 1, spread)
    v[:, :, 1] = -v[:, :, 0]
    got = llmik.paged_decode_attention(q, k, v, table, seq, 0.3, softcap=cap)
    for b in range(B):
        kb, _ = ref.tokens_of(k, table[b], 2, page)
        vb, _ = ref.tokens_of(v, table[b], 2, page)
        want, bound = _attend(q[b:b + 1], kb, vb, torch.tensor([1], device=cuda), 0.3, cap, 2.0 ** -22)
        ref.check(got[b:b + 1], want, bound)


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,D,scale,bias", [(F16, 128, 0.5, False), (BF16, 64, 0.5, True), (F16, 64, -0.5, True),
                                                (BF16, 128, 40.0, False)], ids=str)
def test_every_form(llmik, cuda, cap, dtype, D, scale, bias):
    """Decode, prompts (one part and many) and a shared prefix, scores on both sides of
    half the cap, with and without a bias, negative scales."""
    H, Hkv, page = 8, 2, 16
    spread = torch.tensor([0.05, 0.3, 1.0, 4.0] * 2, device=cuda)
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=cuda) if bias else None
    for n, new in ((300, 1), (300, 130), (3000, 40)):
        q, k, v, table, seq = _inputs(cuda, dtype, [n], new, H, Hkv, D, page, n + new, spread)
        kb, _ = ref.tokens_of(k, table[0], n, page)
        vb, _ = ref.tokens_of(v, table[0], n, page)
        pos = torch.arange(n - new, n, device=cuda)
        opts = dict(softcap=cap, slopes=slopes)
        if new == 1:
            want, bound = _attend(q, kb, vb, pos, scale, cap, ref.PAIR[dtype], slopes)
            ref.check(llmik.paged_decode_attention(q, k, v, table, seq, scale, **opts), want, bound)
            want, bound = _attend(q, kb, vb, pos, scale, cap, ref.U[dtype], slopes)
            got = llmik.paged_shared_prefix_attention(q, k, v, table, seq, table[0].contiguous(), 200, scale, **opts)
        else:
            want, bound = _attend(q, kb, vb, pos, scale, cap, ref.U[dtype], slopes)
            got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([new], cuda), scale, **opts)
        ref.check(got, want, bound)


def test_a_cap_beside_values_that_are_no_numbers(llmik, cuda):
    """The rows that are done again one by one use the same capped scores."""
    H, Hkv, D, page, n, cap = 8, 2, 128, 16, 150, 4096.0
    spread = torch.tensor([0.05, 0.3, 1.0, 4.0] * 2, device=cuda)
    q, k, v, table, seq = _inputs(cuda, F16, [n], n, H, Hkv, D, page, 5, spread)
    kb, _ = ref.tokens_of(k, table[0], n, page)
    vb, _ = ref.tokens_of(v, table[0], n, page)
    want, bound = _attend(q, kb, vb, torch.arange(n, device=cuda), 0.5, cap, ref.U[F16])
    for t in (70, 130):
        v[int(table[0, t // page]), :, t % page] = math.nan
    got = llmik.paged_prefill_attention(q, k, v, table, seq, ref.offsets([n], cuda), 0.5, softcap=cap)
    ref.check(got[:70], want[:70], bound[:70])
    assert bool(got[70:].isnan().all())
