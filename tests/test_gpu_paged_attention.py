"""GPU: decode, prompt and shared-prefix attention over a paged cache, against
the float64 definition (tests/paged_ref.py, where the tolerances are derived)."""
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
