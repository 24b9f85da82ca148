"""GPU: drafted trees, recorded weights, selections and moves where calls meet: streams,
graphs, offsets that decrease, very many KV heads, row groups of odd sizes; against the
float64 definitions (tests/bounded_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _q(rows, H, D, dtype, dev, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(rows, H, D, generator=gen, device=dev)).to(dtype)


def _calls(llmik, dev):
    """One of each operator, with tiles that are cut into parts; every call has its own weights."""
    lens, H, Hkv, D, page = [3000, 200, 1500], 16, 4, 128, 16
    k, v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, dev, 0)
    new = [30, 5, 20]
    mask, pos = bref.trees(random.Random(1), new, [n - m for n, m in zip(lens, new)])
    words, at = bref.words_of(mask, 1, dev), torch.tensor(pos, dtype=torch.int32, device=dev)
    q, q1 = _q(sum(new), H, D, F16, dev, 2), _q(3, H, D, F16, dev, 3)
    many = [900, 200, 400]
    qn, cu, cu_many = _q(sum(many), H, D, F16, dev, 4), ref.offsets(new, dev), ref.offsets(many, dev)
    some = torch.rand(3, Hkv, 3000, generator=torch.Generator(device=dev).manual_seed(5), device=dev)

    def decode():
        w = torch.zeros(3, Hkv, 3000, device=dev)
        return torch.cat([llmik.paged_decode_attention_weights(q1, k, v, table, seq, w, 0.1).float().flatten(), w.flatten()])

    def moved():
        kept, n = llmik.paged_select_tokens(some, seq, 700, 3, 50)
        k2, v2, w2 = k.clone(), v.clone(), some.clone()
        llmik.paged_compact(k2, v2, table, seq, kept, None, w2)
        return torch.cat([k2.float().flatten(), v2.float().flatten(), w2.flatten(), n.float()])

    return [
        lambda: llmik.paged_tree_attention(q, k, v, table, seq, cu, words, 0.1, positions=at),
        decode,
        lambda: llmik.paged_prefill_weights(qn, k, table, seq, cu_many, torch.zeros(3, Hkv, 3000, device=dev), 0.1),
        lambda: llmik.paged_prefill_weights(q, k, table, seq, cu, torch.zeros(3, Hkv, 3000, device=dev), 0.1, observe=8),
        moved,
    ]


def test_two_streams_at_once(llmik, cuda):
    calls = _calls(llmik, cuda)
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([c() for c in calls])
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_graphs_captured_on_one_stream_replay_on_two(llmik, cuda):
    """Two graphs share nothing, also where they were captured on one stream whose eager
    workspace exists; replays with eager calls between."""
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
    for _ in range(6):
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


def test_offsets_that_decrease_end_and_leave_the_workspace_usable(llmik, cuda):
    """Such offsets have no defined rows; the call ends, writes only its outputs, and the next
    calls, whose tiles are cut, are what they were before it."""
    calls = _calls(llmik, cuda)
    want = [c() for c in calls]
    lens, H, Hkv, D = [3000, 200, 1500], 16, 4, 128
    k, v, table, seq = ref.make_cache(lens, Hkv, D, 16, F16, cuda, 6)
    q = _q(60, H, D, F16, cuda, 7)
    words = torch.full((60, 1), -1, dtype=torch.int64, device=cuda)
    k0, v0 = k.clone(), v.clone()
    for cu in ([0, 60, 0, 60], [60, 0, 60, 10], [0, -7, 2 ** 31 - 1, 40], [5, 70, -2 ** 31, 60]):
        at = torch.tensor(cu, dtype=torch.int32, device=cuda)
        wide = torch.zeros(4, Hkv, 3000, device=cuda)
        llmik.paged_tree_attention(q, k, v, table, seq, at, words, 0.1)
        llmik.paged_prefill_weights(q, k, table, seq, at, wide[:3], 0.1)
        llmik.paged_prefill_weights(q, k, table, seq, at, wide[:3], 0.1, observe=4)
        torch.cuda.synchronize()
        assert int(wide[3].count_nonzero()) == 0
        for c, w in zip(calls, want):
            assert torch.equal(c(), w)
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_thousands_of_kv_heads(llmik, cuda):
    """More KV heads than a workspace has counters: nothing is cut."""
    lens, new, H, D, page = [90, 30], [9, 30], 4100, 64, 32
    ctx = [81, 0]
    k, v, table, seq = ref.make_cache(lens, H, D, page, F16, cuda, 8)
    q, cu = _q(39, H, D, F16, cuda, 9), ref.offsets(new, cuda)
    mask, pos = bref.trees(random.Random(9), new, ctx)
    got = llmik.paged_tree_attention(q, k, v, table, seq, cu, bref.words_of(mask, 1, cuda), 0.1,
                                     positions=torch.tensor(pos, dtype=torch.int32, device=cuda))
    ref.check(got, *bref.tree(q, k, v, table, lens, new, mask, pos, 0.1, page))
    for rows in (39, 200):   # one row tile of a KV head, several
        new = [9, 30] if rows == 39 else [70, 130]
        lens = [90, 30] if rows == 39 else [90, 130]
        k, v, table, seq = ref.make_cache(lens, H, D, page, F16, cuda, 10)
        q, cu = _q(sum(new), H, D, F16, cuda, 11), ref.offsets(new, cuda)
        w = torch.zeros(2, H, 130, device=cuda)
        want, bound = bref.weights(w, None, q, k, table, lens, new, 0.1, page)
        llmik.paged_prefill_weights(q, k, table, seq, cu, w, 0.1)
        ref.check(w, want, bound)


PROMPT = [
    # context, new, H, Hkv, D, dtype, weights' tokens, observe, options
    ([0, 700], [150, 90], 34, 1, 128, F16, 800, 0, {}),                    # 64 rows end inside a token
    ([2500], [300], 7, 1, 64, BF16, 2800, 0, {"window": 500}),             # the first keys are nobody's
    ([2500, 0], [300, 129], 10, 2, 128, F16, 2800, 0, {"window": 1}),
    ([2500], [700], 12, 4, 64, F16, 2600, 0, {"window": 130, "softcap": 15.0}),   # ends inside the rows
    ([4000, 40, 0], [40, 500, 0], 48, 2, 64, BF16, 4040, 0, {}),
    ([63, 64, 65, 127, 128, 129], [65, 64, 63, 1, 129, 128], 32, 2, 64, F16, 257, 0, {}),
    ([0], [2000], 4, 4, 128, BF16, 100, 0, {}),                            # most keys are not recorded
    ([100] * 90, [b % 70 for b in range(90)], 8, 2, 64, F16, 170, 0, {}),  # two sequences a lane
]


@pytest.mark.parametrize("case", PROMPT, ids=lambda c: "%dx%d-%s-%s" % (len(c[0]), max(c[1]), c[2:6], c[7:]))
def test_prompt_weights(llmik, cuda, case):
    ctx, new, H, Hkv, D, dtype, width, observe, opts = case
    lens = [a + b for a, b in zip(ctx, new)]
    k, _, table, seq = ref.make_cache(lens, Hkv, D, 16, dtype, cuda, 12)
    q = _q(sum(new) + 3, H, D, dtype, cuda, 13)   # (and a padded batch's rows)
    w = torch.rand(len(lens), Hkv, width, device=cuda)
    want, bound = bref.weights(w, None, q[:sum(new)], k, table, lens, new, 0.1, 16, observe, **opts)
    llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(new, cuda), w, 0.1, observe=observe, **opts)
    ref.check(w, want, bound)


def test_rows_that_are_not_recorded_cost_the_others_nothing(llmik, cuda):
    """Sequences without a row of the weights between others that have one, in both forms."""
    lens, new, H, Hkv, D = [600, 900, 100, 1200], [300, 900, 100, 200], 16, 4, 128
    k, _, table, seq = ref.make_cache(lens, Hkv, D, 64, BF16, cuda, 14)
    rows = [-1, 1, 7, 0]
    at = torch.tensor(rows, dtype=torch.int32, device=cuda)
    q = _q(sum(new), H, D, BF16, cuda, 15)
    for observe in (0, 20):
        w = torch.rand(2, Hkv, 1200, device=cuda)
        want, bound = bref.weights(w, rows, q, k, table, lens, new, 0.1, 64, observe)
        llmik.paged_prefill_weights(q, k, table, seq, ref.offsets(new, cuda), w, 0.1, observe=observe, weight_rows=at)
        ref.check(w, want, bound)


@pytest.mark.parametrize("window", [0, 40])
def test_a_query_that_is_no_number_reaches_only_the_keys_that_it_sees(llmik, cuda, window):
    """Q of one row is NaN: the keys that it sees have NaN, the others' weights are right."""
    ctx, new, H, Hkv, D = 500, 400, 8, 2, 64
    k, _, table, seq = ref.make_cache([ctx + new], Hkv, D, 16, F16, cuda, 16)
    q = _q(new, H, D, F16, cuda, 17)
    bad, head = 250, 5                       # of KV head 1
    q[bad, head] = 0.0
    w = torch.zeros(1, Hkv, ctx + new, device=cuda)
    want, bound = bref.weights(w, None, q, k, table, [ctx + new], [new], 0.1, 16, window=window)
    q[bad, head] = float("nan")
    llmik.paged_prefill_weights(q, k, table, seq, ref.offsets([new], cuda), w, 0.1, window=window)
    t = torch.arange(ctx + new, device=cuda)
    sees = (t <= ctx + bad) & ((t > ctx + bad - window) if window else (t >= 0))
    assert bool(w[0, 1, sees].isnan().all())
    ref.check(w[0, 0], want[0, 0], bound[0, 0])
    ref.check(w[0, 1, ~sees], want[0, 1, ~sees], bound[0, 1, ~sees])


@pytest.mark.parametrize("opts", [{"softcap": 5.0}, {}, {"window": 60}], ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_are_not_positive(llmik, cuda, scale, opts):
    ctx, new, H, Hkv, D = [300, 20], [40, 130], 8, 2, 128
    lens = [a + b for a, b in zip(ctx, new)]
    k, v, table, seq = ref.make_cache(lens, Hkv, D, 16, BF16, cuda, 20)
    q, cu = _q(sum(new), H, D, BF16, cuda, 21), ref.offsets(new, cuda)
    mask, pos = bref.trees(random.Random(22), new, ctx)
    at = torch.tensor(pos, dtype=torch.int32, device=cuda)
    got = llmik.paged_tree_attention(q, k, v, table, seq, cu, bref.words_of(mask, 3, cuda), scale, positions=at, **opts)
    ref.check(got, *bref.tree(q, k, v, table, lens, new, mask, pos, scale, 16, **opts))
    for observe in (0, 7):
        w = torch.zeros(2, Hkv, 340, device=cuda)
        want, bound = bref.weights(w, None, q, k, table, lens, new, scale, 16, observe, **opts)
        llmik.paged_prefill_weights(q, k, table, seq, cu, w, scale, observe=observe, **opts)
        ref.check(w, want, bound)
    w = torch.zeros(2, Hkv, 340, device=cuda)
    want, bound = bref.weights(w, None, q[:2], k, table, lens, [1, 1], scale, 16, **opts)
    llmik.paged_decode_attention_weights(q[:2], k, v, table, seq, w, scale, **opts)
    ref.check(w, want, bound)


def test_a_drafted_key_that_is_no_number_is_its_descendants_own(llmik, cuda):
    """K of a drafted token is NaN: the rows that see it are NaN, the others are right."""
    ctx, new, H, Hkv, D = 200, 40, 8, 2, 64
    mask, pos = bref.trees(random.Random(8), [new], [ctx])
    k, v, table, seq = ref.make_cache([ctx + new], Hkv, D, 16, F16, cuda, 23)
    q, cu = _q(new, H, D, F16, cuda, 24), ref.offsets([new], cuda)
    place = int(table[0, (ctx + 5) // 16]), slice(None), (ctx + 5) % 16
    sees = torch.tensor([bool(m >> 5 & 1) for m in mask], device=cuda)
    assert 0 < int(sees.sum()) < new
    k[place] = 0.0
    want, bound = bref.tree(q, k, v, table, [ctx + new], [new], mask, pos, 0.05, 16)
    k[place] = float("nan")
    got = llmik.paged_tree_attention(q, k, v, table, seq, cu, bref.words_of(mask, 1, cuda), 0.05,
                                     positions=torch.tensor(pos, dtype=torch.int32, device=cuda))
    assert bool(got[sees].isnan().all())
    ref.check(got[~sees], want[~sees], bound[~sees])


def test_pools_of_more_than_2_to_the_31_elements(llmik, cuda):
    """The same tokens on a large pool's last pages: the same bits."""
    lens, new, H, Hkv, D, page = [500, 90], [40, 9], 8, 2, 128, 64
    small_k, small_v, table, seq = ref.make_cache(lens, Hkv, D, page, F16, cuda, 25)
    n = small_k.shape[0]
    more = 2 ** 31 // (Hkv * page * D) + 3
    k = torch.zeros(more + n, Hkv, page, D, dtype=F16, device=cuda)
    v = torch.zeros_like(k)
    k[more:], v[more:] = small_k, small_v
    far = torch.where((table >= 0) & (table < n), table + more, -1).to(torch.int32)
    q, cu = _q(sum(new), H, D, F16, cuda, 26), ref.offsets(new, cuda)
    words = torch.full((sum(new), 1), 1023, dtype=torch.int64, device=cuda)
    kept = torch.tensor([list(range(30, 490, 2)) + [-1] * 5, list(range(5, 90)) + [-1] * 150], dtype=torch.int32, device=cuda)

    def all_of(k, v, table):
        out = [llmik.paged_tree_attention(q, k, v, table, seq, cu, words, 0.1)]
        for observe in (0, 9):
            out.append(llmik.paged_prefill_weights(q, k, table, seq, cu, torch.zeros(2, Hkv, 500, device=cuda), 0.1,
                                                   observe=observe))
        w = torch.zeros(2, Hkv, 500, device=cuda)
        out += [llmik.paged_decode_attention_weights(q[:2], k, v, table, seq, w, 0.1), w]
        llmik.paged_compact(k, v, table, seq, kept, torch.tensor([0, 4], dtype=torch.int32, device=cuda))
        return out
    for a, b in zip(all_of(k, v, far), all_of(small_k, small_v, table)):
        assert torch.equal(a, b)
    assert torch.equal(k[more:], small_k) and torch.equal(v[more:], small_v)
    assert int(k[:more].count_nonzero()) == 0 and int(v[:more].count_nonzero()) == 0


REFUSED = [
    ("tree", {"mask": lambda m: m.to(torch.int32)}, "int64"), ("tree", {"mask": lambda m: m[:4]}, "int64"),
    ("tree", {"mask": lambda m: m[:, :0]}, "at least one word"), ("tree", {"mask": lambda m: m[:, 0]}, "int64"),
    ("tree", {"mask": lambda m: m.expand(-1, 2)}, "contiguous"), ("tree", {"mask": lambda m: m.cpu()}, "CUDA"),
    ("tree", {"at": lambda t: t[:3]}, "positions"), ("tree", {"at": lambda t: t.long()}, "positions"),
    ("tree", {"at": lambda t: t.cpu()}, "CUDA"), ("append", {"at": lambda t: t[:3]}, "positions"),
    ("tree", {"q": lambda t: t.transpose(0, 1)}, "contiguous"),
    ("decode", {"w": lambda t: t.half()}, "fp32"), ("decode", {"w": lambda t: t[:, :1]}, "n_kv_heads"),
    ("decode", {"w": lambda t: t[:1]}, "row per sequence"), ("prompt", {"w": lambda t: t[..., ::2]}, "contiguous"),
    ("prompt", {"w": lambda t: t[..., :0].contiguous()}, "tokens per row"), ("prompt", {"w": lambda t: t.cpu()}, "CUDA"),
    ("prompt", {"rows": lambda t: t[:1]}, "weight_rows"), ("decode", {"rows": lambda t: t.long()}, "weight_rows"),
    ("select", {"rows": lambda t: t.cpu()}, "CUDA"), ("select", {"w": lambda t: t[0]}, "weights"),
    ("select", {"keep": lambda n: 0}, "keep"), ("select", {"first": lambda n: -1}, "first and recent"),
    ("select", {"recent": lambda n: 8}, "first and recent"), ("select", {"lens": lambda t: t.long()}, "seq_lens"),
    ("compact", {"kept": lambda t: t.long()}, "kept"), ("compact", {"kept": lambda t: t[:1]}, "kept"),
    ("compact", {"kept": lambda t: t[:, :1]}, "kept"), ("compact", {"kept": lambda t: t.transpose(0, 1)}, "kept"),
    ("compact", {"starts": lambda t: t[:1]}, "starts"), ("compact", {"starts": lambda t: t.long()}, "starts"),
    ("compact", {"w": lambda t: None}, "weight_rows come with weights"),
]


@pytest.mark.parametrize("name,change,msg", REFUSED, ids=["%s-%s-%d" % (n, *c, i) for i, (n, c, _) in enumerate(REFUSED)])
def test_refusals(llmik, cuda, name, change, msg):
    """Nothing is launched: k, v and weights keep their bits."""
    H, Hkv, D = 8, 2, 64
    k, v, table, seq = ref.make_cache([40, 20], Hkv, D, 16, F16, cuda, 18)
    a = dict(q=_q(5, H, D, F16, cuda, 19), cu=ref.offsets([3, 2], cuda), mask=torch.ones(5, 1, dtype=torch.int64, device=cuda),
             at=torch.full((5,), 40, dtype=torch.int32, device=cuda), w=torch.rand(2, Hkv, 40, device=cuda),
             rows=torch.tensor([0, 1], dtype=torch.int32, device=cuda), keep=8, first=1, recent=1, lens=seq,
             kept=torch.zeros(2, Hkv, 5, dtype=torch.int32, device=cuda), starts=torch.zeros(2, dtype=torch.int32, device=cuda))
    weights, kept = a["w"], [t.clone() for t in (k, v, a["w"])]
    for key, f in change.items():
        a[key] = f(a[key])
    if name == "decode" and change.keys() == {"w"}:
        a["rows"] = None
    calls = {
        "tree": lambda: llmik.paged_tree_attention(a["q"], k, v, table, seq, a["cu"], a["mask"], 0.1, positions=a["at"]),
        "append": lambda: llmik.rope_paged_append(torch.zeros(5, (H + 2 * Hkv) * D, dtype=F16, device=cuda), None, None, k, v,
                                                  table, seq, a["cu"], a["at"]),
        "decode": lambda: llmik.paged_decode_attention_weights(a["q"][:2], k, v, table, seq, a["w"], 0.1,
                                                               weight_rows=a["rows"]),
        "prompt": lambda: llmik.paged_prefill_weights(a["q"], k, table, seq, a["cu"], a["w"], 0.1, weight_rows=a["rows"]),
        "select": lambda: llmik.paged_select_tokens(a["w"], a["lens"], a["keep"], a["first"], a["recent"], a["rows"]),
        "compact": lambda: llmik.paged_compact(k, v, table, seq, a["kept"], a["starts"], a["w"], a["rows"]),
    }
    with pytest.raises(RuntimeError, match=msg):
        calls[name]()
    assert all(torch.equal(x, y) for x, y in zip((k, v, weights), kept))
