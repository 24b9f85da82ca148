"""GPU: decode attention and prompts that record each token's attention weight, against
the float64 definition (tests/bounded_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import math

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(rows, H, D, dtype, dev, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)


def _slopes(H, dev):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=dev)


def _opts(opts, H, dev):
    return {**opts, "slopes": _slopes(H, dev)} if opts.get("slopes") else dict(opts)


def _id(case):
    return "-".join(str(x) if not isinstance(x, list) else "B%d_%d" % (len(x), max(x)) for x in case).replace("torch.", "")


DECODE = [
    # lens, H, Hkv, D, page, dtype, weights' tokens, options
    ([1], 1, 1, 64, 8, BF16, 5, {}),
    ([33, 0, 64, 65], 8, 2, 128, 16, F16, 70, {}),
    ([900], 32, 8, 128, 16, F16, 960, {}),
    ([1500, 3, 129, 0, 777], 28, 4, 128, 24, BF16, 1501, {}),
    ([1500, 3, 129], 16, 16, 64, 64, F16, 700, {}),              # longer than the weights
    ([9000], 40, 8, 128, 128, BF16, 9100, {}),
    ([300, 200], 34, 1, 128, 32, BF16, 333, {}),                 # three chunks of heads
    ([100, 2000, 31], 32, 8, 128, 16, F16, 2048, {"softcap": 20.0}),
    ([100, 2000, 31], 8, 4, 64, 16, F16, 2048, {"softcap": 500.0}),
    ([100, 2000, 31], 32, 8, 128, 64, BF16, 2001, {"slopes": True}),
    ([100, 2000, 31], 32, 8, 128, 64, F16, 2001, {"window": 77}),
    ([5000, 2000, 4096], 12, 4, 64, 32, BF16, 5000, {"window": 777, "slopes": True, "softcap": 30.0}),
    (ref.ragged(1, 70, 0, 900), 16, 8, 128, 64, F16, 901, {}),
    (ref.ragged(2, 130, 0, 700), 4, 2, 64, 8, BF16, 640, {"softcap": 30.0}),
]


@pytest.mark.parametrize("start", [0.0, 3.0])
@pytest.mark.parametrize("case", DECODE, ids=_id)
def test_decode(llmik, cuda, case, start):
    lens, H, Hkv, D, page, dtype, width, opts = case
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 0)
    q = _q(len(lens), H, D, dtype, cuda, 1)
    opts = _opts(opts, H, cuda)
    scale = 1.0 / math.sqrt(D)
    w = torch.rand(len(lens), Hkv, width, device=cuda) * start
    want, bound = bref.weights(w, None, q, k, table, lens, [1] * len(lens), scale, page, **opts)
    out = llmik.paged_decode_attention_weights(q, k, v, table, seq, w, scale, **opts)
    assert torch.equal(out, llmik.paged_decode_attention(q, k, v, table, seq, scale, **opts))
    ref.check(w, want, bound)


PROMPT = [
    # context, new, H, Hkv, D, page, dtype, weights' tokens, observe, options
    ([0], [1], 4, 1, 128, 16, F16, 4, 0, {}),
    ([0, 9], [5, 1], 8, 2, 64, 8, BF16, 10, 0, {}),
    ([0, 0, 0], [17, 150, 64], 32, 8, 128, 16, F16, 150, 0, {}),
    ([0, 63, 1000, 0], [64, 1, 3, 0], 32, 8, 128, 64, BF16, 1010, 0, {}),
    ([0, 500], [700, 129], 28, 4, 128, 24, F16, 701, 0, {}),
    ([2000], [513], 16, 2, 128, 128, BF16, 2000, 0, {}),          # longer than the weights
    ([3000, 0, 1500], [333, 65, 1], 8, 2, 64, 64, BF16, 3400, 0, {}),
    ([0, 0], [4000, 900], 32, 8, 128, 32, F16, 4000, 32, {}),
    ([100, 0], [700, 20], 8, 8, 64, 16, BF16, 800, 1, {}),
    ([0, 10], [30, 600], 16, 4, 128, 16, F16, 640, 100, {"softcap": 20.0}),
    ([10, 300], [200, 77], 8, 4, 64, 16, F16, 400, 0, {"softcap": 400.0}),
    ([10, 300], [200, 77], 24, 8, 64, 64, BF16, 400, 0, {"slopes": True}),
    ([10, 300], [200, 577], 32, 8, 128, 32, F16, 877, 0, {"window": 50}),
    ([10, 300], [20, 77], 8, 1, 128, 40, F16, 377, 0, {"window": 1}),
    ([1010, 300], [200, 577], 12, 4, 128, 32, BF16, 1300, 90, {"window": 333, "slopes": True, "softcap": 30.0}),
    ([2500 if b % 9 == 0 else 3 * b for b in range(100)], [b % 5 for b in range(100)], 4, 1, 64, 16, BF16, 2510, 2, {}),
    (ref.ragged(5, 70, 0, 50), ref.ragged(6, 70, 0, 200), 8, 2, 128, 64, F16, 256, 0, {"window": 100}),
]


@pytest.mark.parametrize("case", PROMPT, ids=_id)
def test_prompts(llmik, cuda, case):
    ctx, new, H, Hkv, D, page, dtype, width, observe, opts = case
    lens = [a + b for a, b in zip(ctx, new)]
    k, _, table, seq = ref.make_cache(lens, Hkv, D, page, dtype, cuda, 2)
    q = _q(sum(new), H, D, dtype, cuda, 3)
    opts = _opts(opts, H, cuda)
    scale = 1.0 / math.sqrt(D)
    w = torch.zeros(len(lens), Hkv, width, device=cuda)
    want, bound = bref.weights(w, None, q, k, table, lens, new, scale, page, observe, **opts)
    again = w.clone()
    call = lambda w: llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(new, cuda), w, scale,   # noqa: E731
                                                 observe=observe, **opts)
    assert call(w) is w or call is None
    ref.check(w, want, bound)
    call(again)
    assert torch.equal(again, w)
    call(w)   # and what was there is kept
    ref.check(w, 2 * want, 2 * bound + 2.0 ** -24 * 2 * want)


def test_every_row_gives_its_heads_as_much_as_one(llmik, cuda):
    """The weights of a step sum to the query heads of a KV head, a prompt's to that times its rows."""
    lens, H, Hkv, D, page = [400, 70], 8, 2, 128, 16
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 4)
    w = torch.zeros(2, Hkv, 400, device=cuda)
    llmik.paged_decode_attention_weights(_q(2, H, D, F16, cuda, 5), k, v, table, seq, w, 0.1)
    # 4 (1 + 2^-18): 470 fp32 terms of relative 2^-21 at most each
    assert float((w.sum(-1) - 4).abs().max()) < 4 * 2.0 ** -18
    w.zero_()
    llmik.paged_prefill_weights(_q(90, H, D, F16, cuda, 6), k, table, seq, ref.offsets([60, 30], cuda), w, 0.1)
    assert float((w.sum(-1) - torch.tensor([[240.0], [120.0]], device=cuda)).abs().max()) < 240 * 2.0 ** -18


@pytest.mark.parametrize("prompt", [False, True])
def test_rows_of_the_weights(llmik, cuda, prompt):
    """Sequences' rows in any order among others; a row outside the tensor is not recorded."""
    lens, H, Hkv, D, page = [300, 20, 111, 64], 8, 2, 64, 16
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, BF16, cuda, 7)
    rows = [5, -1, 0, 6]
    at = torch.tensor(rows, dtype=torch.int32, device=cuda)
    new = [30, 5, 1, 64] if prompt else [1] * 4
    q = _q(sum(new), H, D, BF16, cuda, 8)
    w = torch.rand(6, Hkv, 310, device=cuda)
    want, bound = bref.weights(w, rows, q, k, table, lens, new, 0.1, page)
    before = w.clone()
    if prompt:
        llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(new, cuda), w, 0.1, weight_rows=at)
    else:
        llmik.paged_decode_attention_weights(q, k, v, table, seq, w, 0.1, weight_rows=at)
    ref.check(w, want, bound)
    assert torch.equal(w[1:5], before[1:5])
    for row, n in ((5, 300), (0, 111)):
        assert torch.equal(w[row, :, n:], before[row, :, n:])


@pytest.mark.parametrize("prompt", [False, True])
def test_unmapped_pages_dead_slots_and_empty_sequences(llmik, cuda, prompt):
    """Tokens of unmapped pages get nothing, slots that hold NaN behind the length are not
    read, sequences of length <= 0 change nothing."""
    H, Hkv, D, page = 8, 2, 128, 16
    k, v, table, seq = ref.make_cache([300, 40, 33], Hkv, D, page, F16, cuda, 9, fill=math.nan)
    table[0, 2], table[0, 18] = -1, k.shape[0] + 4
    seq[1], lens = -2 ** 31, [300, 0, 33]
    new = [20, 0, 33] if prompt else [1] * 3
    q = _q(sum(new), H, D, F16, cuda, 10)
    w = torch.zeros(3, Hkv, 320, device=cuda)
    if prompt:
        want, bound = bref.weights(w, None, q, k, table, lens, new, 0.1, page)
        llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(new, cuda), w, 0.1)
    else:
        want, bound = bref.weights(w, None, q[[0, 2]], k, table, lens, [1, 0, 1], 0.1, page)
        llmik.paged_decode_attention_weights(q, k, v, table, seq, w, 0.1)
    ref.check(w, want, bound)
    assert int(w[1].count_nonzero()) == 0 and int(w[0, :, 32:48].count_nonzero()) == 0


@pytest.mark.parametrize("parts", [False, True])
def test_a_key_that_is_no_number_reaches_only_its_rows_keys(llmik, cuda, parts):
    """K of a new token is NaN: rows that see it give NaN to all keys that they see, and the
    keys that only other rows see stay right."""
    H, Hkv, D, page, ctx, new = 4, 1, 64, 16, 3000 if parts else 30, 40
    n = ctx + new
    k, _, table, seq = ref.make_cache([n, 50], Hkv, D, page, F16, cuda, 11)
    q = _q(new + 10, H, D, F16, cuda, 12)
    lens, rows = [n, 50], [new, 10]
    w = torch.zeros(2, Hkv, n, device=cuda)
    bad = n - 1
    place = int(table[0, bad // page]), slice(None), bad % page
    k[place] = 0.0
    want, bound = bref.weights(w, None, q, k, table, lens, rows, 0.1, page)
    k[place] = math.nan
    llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(rows, cuda), w, 0.1)
    assert bool(w[0].isnan().all())           # the last row sees all keys
    ref.check(w[1], want[1], bound[1])
    # with a window the last row leaves the first keys alone
    w.zero_()
    k[place] = 0.0
    want, bound = bref.weights(w, None, q, k, table, lens, rows, 0.1, page, window=20)
    k[place] = math.nan
    llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(rows, cuda), w, 0.1, window=20)
    assert bool(w[0, :, n - 20:].isnan().all())
    ref.check(w[0, :, :n - 20], want[0, :, :n - 20], bound[0, :, :n - 20])


def test_replays_follow_lengths_and_pages(llmik, cuda):
    """A graph of a step and a prompt's recording, replayed with other lengths, tables and rows."""
    H, Hkv, D, page, B = 16, 4, 128, 16, 3
    k, v, table, seq = ref.make_cache([4000] * B, Hkv, D, page, BF16, cuda, 13)
    q1, q2 = _q(B, H, D, BF16, cuda, 14), _q(40, H, D, BF16, cuda, 15)
    cu = ref.offsets([20, 10, 10], cuda)
    w = torch.zeros(4, Hkv, 4000, device=cuda)
    at = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)

    def call():
        out = llmik.paged_decode_attention_weights(q1, k, v, table, seq, w, 0.1, weight_rows=at)
        llmik.paged_prefill_weights(q2, k, table, seq, cu, w, 0.1, observe=15, weight_rows=at)
        return out
    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call()
    for turn, (new, lens) in enumerate([([20, 10, 10], [4000, 3000, 100]), ([40, 0, 0], [40, 0, 7]),
                                        ([0, 1, 30], [4, 2500, 3999]), ([1, 1, 1], [1, 2, 3])]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        cu.copy_(ref.offsets(new, cuda))
        table.copy_(table.roll(1, 0))
        at.copy_(at.roll(1))
        w.fill_(0.5)
        w0 = w.clone()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        rows = at.tolist()
        one = [min(n, 1) for n in lens]
        live = [b for b in range(B) if lens[b] > 0]
        want, bound = bref.weights(w0, rows, q1[live], k, table, lens, one, 0.1, page)
        more, off = bref.weights(torch.zeros_like(w0), rows, q2[:sum(new)], k, table, lens, new, 0.1, page, 15)
        ref.check(w, want + more, bound + off + 2.0 ** -23 * (want + more))
        got = w.clone()
        w.copy_(w0)
        assert torch.equal(call(), out) and torch.equal(w, got)
    torch.cuda.synchronize()
