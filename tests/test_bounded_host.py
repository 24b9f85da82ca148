"""CPU: the refusals of drafted trees and of caches bounded by attention weight, in the C
layer and the Python ops. No compute entry point is called with valid arguments here."""
from __future__ import annotations

import pytest
import torch

from tests.test_paged_host import (ALIGNMENT, BF, CACHES, I32, INVALID, UNSUPPORTED, WORKSPACE, _args, _at, _cache,
                                   _options, _t, as_device, lib, mod)  # noqa: F401

F32 = torch.float32


def _weights(**more):
    from llmik_cuda._lib import TokenWeights
    c = dict(weights=16, rows=16, n_rows=4, max_len=100)
    c.update(more)
    return TokenWeights(**c)


def _c_calls(lib, c, o, w, ws=16, n=1 << 60):
    return [lambda: lib.llmik_paged_tree_attention(_at(c), 16, 16, 16, 1, 16, 16, 2, 4, _at(o), ws, n, None),
            lambda: lib.llmik_paged_decode_attention_weights(_at(c), 16, 16, 4, _at(o), _at(w), 16, n, ws, n, None),
            lambda: lib.llmik_paged_prefill_weights(_at(c), 16, 16, 2, 4, _at(o), 0, _at(w), ws, n, None)]


@pytest.mark.parametrize("case", CACHES, ids=lambda c: str(c[0]))
def test_c_layer_refuses_caches(lib, case):   # noqa: F811
    more, code, msg = case
    c, o, w = _cache(**more), _options(), _weights()
    calls = _c_calls(lib, c, o, w)
    if "n_kv_heads" not in more or more["n_kv_heads"] != 3:   # (compaction has no query heads)
        calls.append(lambda: lib.llmik_paged_compact(_at(c), 16, 1, 3, 16, _at(w), None))
    if "v" in more:
        calls.pop(2)   # (prompt weights read no V)
    for call in calls:
        assert call() == code and msg in lib.llmik_last_error().decode()


def test_c_layer_refuses_options_and_weights(lib):   # noqa: F811
    err = lambda: lib.llmik_last_error().decode()   # noqa: E731
    c, o, w = _cache(), _options(), _weights()
    for more, msg in [(dict(softcap=-1.0), "softcap"), (dict(softcap=4097.0), "softcap"),
                      (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(window=-1), "window"),
                      (dict(softcap=1e-38, softmax_scale=100.0), "softcap too small")]:
        for call in _c_calls(lib, c, _options(**more), w):
            assert call() == INVALID and msg in err()
    for call in _c_calls(lib, c, _options(slopes=18), w):
        assert call() == ALIGNMENT and "slopes" in err()
    for more, code, msg in [(dict(n_rows=-1), INVALID, "n_rows"), (dict(max_len=0), INVALID, "max_len"),
                            (dict(max_len=(1 << 30) + 1), INVALID, "max_len"),
                            (dict(rows=None, n_rows=1), INVALID, "one row per sequence"),
                            (dict(weights=None), INVALID, "null weights"), (dict(weights=18), ALIGNMENT, "4-byte"),
                            (dict(rows=18), ALIGNMENT, "4-byte")]:
        bad = _weights(**more)
        for call in [*_c_calls(lib, c, o, bad)[1:],
                     lambda: lib.llmik_paged_select_tokens(_at(bad), 16, 2, 2, 8, 0, 0, 16, 16, None),
                     lambda: lib.llmik_paged_compact(_at(c), 16, 1, 3, 16, _at(bad), None)]:
            assert call() == code and msg in err(), more
        assert lib.llmik_paged_decode_weights_scratch_size(_at(c), 4, _at(bad)) == 0


def test_c_layer_refuses_arguments(lib):   # noqa: F811
    err = lambda: lib.llmik_last_error().decode()   # noqa: E731
    c, o, w = _cache(), _options(), _weights()

    def tree(**a):
        return lib.llmik_paged_tree_attention(*{**dict(c=_at(c), q=16, cu=16, mask=16, words=1, pos=16, out=16, rows=2,
                                                       heads=4, o=_at(o), ws=16, n=1 << 60, s=None), **a}.values())
    for a, code, msg in [(dict(c=None), INVALID, "null cache"), (dict(q=None), INVALID, "null q"),
                         (dict(q=24), ALIGNMENT, "16-byte"), (dict(out=8), ALIGNMENT, "16-byte"),
                         (dict(cu=None), INVALID, "null cu_tokens"), (dict(cu=18), ALIGNMENT, "4-byte"),
                         (dict(pos=18), ALIGNMENT, "4-byte"), (dict(mask=None), INVALID, "tree_mask"),
                         (dict(mask=20), ALIGNMENT, "8-byte"), (dict(words=0), INVALID, "one word"),
                         (dict(words=(1 << 24) + 1), UNSUPPORTED, "words"), (dict(rows=-1), INVALID, "rows must be"),
                         (dict(rows=1 << 30), UNSUPPORTED, "too many rows"), (dict(heads=5), INVALID, "multiple"),
                         (dict(o=None), INVALID, "null score options")]:
        assert tree(**a) == code and msg in err(), a
    long = _cache(max_pages=1000)
    need = lib.llmik_paged_tree_workspace_size(_at(long), 4, 2)
    assert need > 16384
    assert tree(c=_at(long), n=need - 1) == WORKSPACE and tree(c=_at(long), ws=None, n=need) == WORKSPACE
    assert lib.llmik_paged_tree_workspace_size(_at(c), 4, 2) == 0          # too few tokens to cut
    for bad in (_cache(head_dim=96), _cache(page_size=12), _cache(batch=-1)):
        assert lib.llmik_paged_tree_workspace_size(_at(bad), 4, 2) == 0
        assert lib.llmik_paged_prefill_weights_workspace_size(_at(bad), 4, 2, 0) == 0
    many = _cache(batch=1, max_pages=1 << 22, page_size=256)               # 2^30 tokens: 2^24 key tiles
    assert tree(c=_at(many), rows=1 << 14) == UNSUPPORTED and "capacity" in err()
    assert lib.llmik_paged_tree_workspace_size(_at(many), 4, 1 << 14) == 0

    scratch, need = lib.llmik_paged_decode_weights_scratch_size(_at(c), 4, _at(w)), lib.llmik_paged_workspace_size(_at(c), 4, 0)
    assert scratch == 2 * 4 * 64 * 4 + 256        # 32 tokens in two pages, in 64s; two numbers a head
    decode = lambda q=16, out=16, sc=16, m=scratch, ws=16, n=need: lib.llmik_paged_decode_attention_weights(   # noqa: E731
        _at(c), q, out, 4, _at(o), _at(w), sc, m, ws, n, None)
    assert decode(n=need - 1) == WORKSPACE and decode(ws=None) == WORKSPACE
    assert decode(m=scratch - 1) == WORKSPACE and decode(sc=None) == WORKSPACE and "scratch too small" in err()
    assert decode(q=None) == INVALID and decode(out=24) == ALIGNMENT and decode(sc=24) == ALIGNMENT
    assert lib.llmik_paged_decode_attention_weights(_at(c), 16, 16, 4, _at(o), None, 16, scratch, 16, need, None) == INVALID

    def prompt(**a):
        return lib.llmik_paged_prefill_weights(*{**dict(c=_at(c), q=16, cu=16, rows=2, heads=4, o=_at(o), observe=0,
                                                        w=_at(w), ws=16, n=1 << 60, s=None), **a}.values())
    need = lib.llmik_paged_prefill_weights_workspace_size(_at(c), 4, 2, 0)
    assert need > 16384 and lib.llmik_paged_prefill_weights_workspace_size(_at(c), 4, 2, -1) == 0
    for a, code, msg in [(dict(q=None), INVALID, "null q"), (dict(q=24), ALIGNMENT, "16-byte"),
                         (dict(cu=None), INVALID, "null cu"), (dict(cu=18), ALIGNMENT, "4-byte"),
                         (dict(rows=-1), INVALID, "rows must"), (dict(observe=-1), INVALID, "observe"),
                         (dict(w=None), INVALID, "null token weights"), (dict(n=need - 1), WORKSPACE, "workspace"),
                         (dict(ws=None), WORKSPACE, "workspace")]:
        assert prompt(**a) == code and msg in err(), a

    wide = _weights(n_rows=1 << 20)

    def select(**a):
        return lib.llmik_paged_select_tokens(*{**dict(w=_at(w), lens=16, batch=2, hkv=2, keep=8, first=2, recent=2,
                                                      kept=16, new=16, s=None), **a}.values())
    for a, code, msg in [(dict(batch=-1), INVALID, "batch"), (dict(hkv=0), INVALID, "head counts"),
                         (dict(keep=0), INVALID, "keep"), (dict(first=-1), INVALID, "first and recent"),
                         (dict(recent=7), INVALID, "first and recent"), (dict(recent=2 ** 31 - 1), INVALID, "first and"),
                         (dict(lens=None), INVALID, "null seq_lens"), (dict(kept=18), ALIGNMENT, "4-byte"),
                         (dict(batch=1 << 20, hkv=8), UNSUPPORTED, "too large")]:
        if a.get("batch", 0) > 4:
            a["w"] = _at(wide)
        assert select(**a) == code and msg in err(), a

    def compact(**a):
        return lib.llmik_paged_compact(*{**dict(c=_at(c), kept=16, heads=2, n=3, starts=16, w=_at(w), s=None),
                                         **a}.values())
    for a, code, msg in [(dict(c=None), INVALID, "null cache"), (dict(heads=3), INVALID, "kept_heads"),
                         (dict(n=-1), INVALID, "n must"), (dict(n=2 ** 31 - 1), UNSUPPORTED, "n too large"),
                         (dict(kept=None), INVALID, "null kept"), (dict(kept=18), ALIGNMENT, "4-byte"),
                         (dict(starts=18), ALIGNMENT, "4-byte")]:
        assert compact(**a) == code and msg in err(), a
    append = lambda pos: lib.llmik_rope_paged_append_at(_at(c), 16, 16, 16, 8, 0, 16, pos, 16, 2, 4, None)  # noqa: E731
    assert append(18) == ALIGNMENT and "positions" in err()


# ---------------------------------------------------------------- the Python ops

def _more(**more):
    return {**_args(mask=_t(2, 1, dtype=torch.int64), pos=_t(2, dtype=I32), w=_t(2, 2, 50, dtype=F32),
                    rows=_t(2, dtype=I32), observe=0, kept=_t(2, 2, 5, dtype=I32), starts=_t(2, dtype=I32), keep=8,
                    first=1, recent=1), **more}


def _calls(m, a):
    opts = (a["scale"], a["softcap"], a["slopes"], a["window"])
    base = (a["q"], a["k"], a["v"], a["table"], a["lens"])
    return {"tree": lambda: m.paged_tree_attention(*base, a["cu"], a["mask"], *opts, a["pos"]),
            "decode": lambda: m.paged_decode_attention_weights(*base, a["w"], *opts, a["rows"]),
            "prompt": lambda: m.paged_prefill_weights(a["q"], a["k"], a["table"], a["lens"], a["cu"], a["w"], *opts,
                                                      a["observe"], a["rows"]),
            "select": lambda: m.paged_select_tokens(a["w"], a["lens"], a["keep"], a["first"], a["recent"], a["rows"]),
            "compact": lambda: m.paged_compact(a["k"], a["v"], a["table"], a["lens"], a["kept"], a["starts"], a["w"],
                                               a["rows"])}


ATTENTION, CACHE, WEIGHTS = ("tree", "decode", "prompt"), ("tree", "decode", "compact"), ("decode", "prompt", "compact")


@pytest.mark.parametrize("names,more,msg", [
    (ATTENTION, dict(q=_t(2, 4, 128, dtype=F32)), "q must be fp16 or bf16"),
    (ATTENTION, dict(q=_t(2, 4, 128, dtype=BF)), "must have q's dtype"),
    (CACHE, dict(v=_t(3, 2, 16, 128, dtype=BF)), "must have"),
    (CACHE, dict(k=_t(3, 2, 16, 64)), "of one shape"),
    (CACHE, dict(table=_t(2, 2, dtype=torch.int64)), "must be int32"),
    (CACHE, dict(table=_t(2, 0, dtype=I32)), "at least one column"),
    (("compact",), dict(k=_t(3, 2, 16, 128, dtype=F32), v=_t(3, 2, 16, 128, dtype=F32)), "k_cache must be fp16 or bf16"),
    (ATTENTION, dict(softcap=1e-50), "softcap too small"), (ATTENTION, dict(scale=1e39), "softmax_scale"),
    (ATTENTION, dict(window=-1), "window"), (("prompt",), dict(observe=-1), "observe"),
    (("prompt",), dict(observe=1 << 31), "observe"),
    (tuple(_calls(None, _more())), dict(), "CUDA tensors of one device"),
], ids=lambda x: x if isinstance(x, str) else "-".join(x))
def test_python_refuses(as_device, names, more, msg):   # noqa: F811
    calls = _calls(as_device, _more(**more))
    for name in names:
        with pytest.raises(RuntimeError, match=msg):
            calls[name]()


def test_python_checks_devices_first(mod):   # noqa: F811
    for call in _calls(mod, _more()).values():
        with pytest.raises(RuntimeError, match="all inputs must be CUDA tensors"):
            call()


# ------------------------------------------------------------ PagedKVCache, on the host

@pytest.fixture
def kv(mod, monkeypatch):   # noqa: F811
    """The cache's module, with the GPU's part of evictions and acceptances noted down."""
    import llmik_cuda.kv_cache as kv
    kv.calls = []
    monkeypatch.setattr(kv, "paged_compact", lambda *a: kv.calls.append(("compact", a)))
    monkeypatch.setattr(kv, "paged_select_tokens", lambda *a: kv.calls.append(("select", a)) or ("lists", None))
    return kv


def test_drafts_describe_their_trees(kv):
    cache = kv.PagedKVCache(20, 2, page_size=8, head_dim=64, device="cpu")
    a, b, c = cache.add(), cache.add(), cache.add()
    cache.batch([a, b, c], [17, 3, 8])
    long = [-1] + [max(-1, j - 3) for j in range(1, 70)]
    step = cache.draft([a, b, c], [[-1, 0, 0, 2, -1], long, []])
    assert step.seq_lens.tolist() == [22, 73, 8] and step.cu_tokens.tolist() == [0, 5, 75, 75] and step.rows == 75
    assert step.tree_mask.dtype == torch.int64 and step.tree_mask.shape == (75, 2)
    assert step.tree_mask[:5].tolist() == [[1, 0], [3, 0], [5, 0], [13, 0], [16, 0]]
    assert step.positions[:5].tolist() == [17, 18, 18, 19, 17]
    seen, deep = [], []
    for j, p in enumerate(long):
        seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        deep.append(deep[p] + 1 if p >= 0 else 3)
    got = [[w + (1 << 64) if w < 0 else w for w in row] for row in step.tree_mask[5:].tolist()]
    assert got == [[m & (1 << 64) - 1, m >> 64] for m in seen] and step.positions[5:].tolist() == deep
    assert step.prefix_pages is None and not step.shortened and step.weight_rows is None
    empty = cache.draft([], [])
    assert empty.rows == 0 and empty.tree_mask.shape == (0, 1)


def test_acceptance_moves_paths_and_frees_pages(kv):
    cache = kv.PagedKVCache(20, 2, page_size=8, head_dim=64, device="cpu", n_layers=3)
    a, b, c = cache.add(), cache.add(), cache.add()
    cache.batch([a, b, c], [17, 3, 8])
    cache.draft([a, b, c], [[-1, 0, 0, 2, -1], [-1] * 30, [-1, 0]])
    assert cache.free_pages() == 20 - 3 - 5 - 2
    with pytest.raises(RuntimeError, match="draft that is not accepted"):
        cache.batch([a])
    with pytest.raises(RuntimeError, match="draft that is not accepted"):
        cache.add(share=b, tokens=1)
    for bad, msg in [(([a], [[1, 1]]), "ascending"), (([a], [[0, 5]]), "ascending"), (([a], [[-1]]), "ascending"),
                     (([a, a], [[0], [0]]), "twice"), (([a], []), "one path"), (([77], [[0]]), "no draft")]:
        with pytest.raises(RuntimeError, match=msg):
            cache.accept(*bad)
    assert cache.length(a) == 22 and kv.calls == []
    tables = {s: list(cache._pages[s]) for s in (a, b)}
    cache.accept([a, b, c], [[0, 2, 3], [29], [0, 1]])
    assert [cache.length(s) for s in (a, b, c)] == [20, 4, 10] and [cache.position(s) for s in (a, b, c)] == [20, 4, 10]
    assert cache.free_pages() == 20 - 3 - 1 - 2
    (name, (k, v, table, lens, lists, starts)), = kv.calls    # c's path is where it belongs already
    assert name == "compact" and k.shape == (60, 2, 8, 64) and k.data_ptr() == cache.k.data_ptr()
    assert lens.tolist() == [22, 33] * 3 and starts.tolist() == [17, 3] * 3
    assert lists.tolist() == [[17, 19, 20], [32, -1, -1]] * 3
    for layer in range(3):
        for i, s in enumerate((a, b)):
            row = table[2 * layer + i].tolist()
            assert row[:len(tables[s])] == [p + 20 * layer for p in tables[s]] and set(row[len(tables[s]):]) <= {-1}
    with pytest.raises(RuntimeError, match="no draft"):
        cache.accept([a], [[0]])
    cache.draft([a], [[-1, 0]])
    cache.accept([a], [[]])
    assert cache.length(a) == 20 and len(kv.calls) == 1
    cache.draft([b], [[-1] * 9])
    cache.remove(b)
    assert cache.free_pages() == 20 - 3 - 2
    for bad, msg in [([[0]], "follows an earlier"), ([[-1, 1]], "follows an earlier"), ([[-2]], "follows an earlier"),
                     ([], "one tree")]:
        with pytest.raises(RuntimeError, match=msg):
            cache.draft([a], bad)
    with pytest.raises(RuntimeError, match="no free page"):
        cache.draft([a], [[-1] * 300])
    assert cache.length(a) == 20 and cache.batch([a]).seq_lens.tolist() == [21]


def test_evictions_shorten_and_unshare(kv):
    cache = kv.PagedKVCache(30, 2, page_size=8, head_dim=64, device="cpu", n_layers=2, track_rows=3, track_tokens=64)
    assert cache.weights.shape == (2, 3, 2, 64)
    a = cache.add()
    cache.batch([a], [50])
    cache.weights[:, cache._rows[a], :, :50] = 2.0
    b = cache.add(share=a, tokens=44)                      # five shared pages and a copy
    assert bool((cache.weights[:, cache._rows[b], :, :44] == 2.0).all())
    assert int(cache.weights[:, cache._rows[b], :, 44:].count_nonzero()) == 0
    c = cache.add()
    with pytest.raises(RuntimeError, match="no free row"):
        cache.add()
    step = cache.batch([b, c], [3, 5])
    assert step.weight_rows.tolist() == [cache._rows[b], cache._rows[c]] and step.positions is None
    cache.k.normal_()
    before, pages_a = cache.k.clone(), list(cache._pages[a])
    pages_b = list(cache._pages[b])
    free = cache.free_pages()
    cache.evict([b, c], keep=20, first=2, recent=4)        # b: 47 -> 20 (three pages, all shared); c stays
    assert cache.length(b) == 20 and cache.length(c) == 5 and cache.position(b) == 47 and cache.position(c) == 5
    assert cache._pages[a] == pages_a and not set(cache._pages[b]) & set(pages_a) and len(cache._pages[b]) == 3
    assert cache.free_pages() == free - 3 + 1              # three copies, its own sixth page back
    for i in range(3):
        assert torch.equal(cache.k[:, cache._pages[b][i]], before[:, pages_b[i]])
    (n1, select), (n2, compact) = kv.calls
    assert (n1, n2) == ("select", "compact") and select[2:5] == (20, 2, 4)
    assert select[0].shape == (6, 2, 64) and select[1].tolist() == [47, 47]
    assert select[5].tolist() == [cache._rows[b], cache._rows[b] + 3] and compact[7] is select[5]
    assert compact[2].tolist() == [[*cache._pages[b], *pages_b[3:]], [p + 30 for p in [*cache._pages[b], *pages_b[3:]]]]
    assert compact[4] == "lists" and compact[5] is None and compact[6] is select[0]
    # what comes after: positions go on, window and slopes are refused, forks are whole
    step = cache.batch([c, b], [1, 3])
    assert step.shortened and step.positions.tolist() == [5, 47, 48, 49] and step.seq_lens.tolist() == [6, 23]
    assert cache.draft([b], [[-1, 0]]).positions.tolist() == [50, 51]
    cache.accept([b], [[]])
    for opts in (dict(window=5), dict(slopes=torch.ones(2))):
        with pytest.raises(RuntimeError, match="lost no tokens"):
            cache.attention(step, None, 0.1, **opts)
    cache.remove(a)
    with pytest.raises(RuntimeError, match="shared whole"):
        cache.add(share=b, tokens=7)
    d = cache.add(share=b, tokens=23)
    assert cache.position(d) == cache.position(b) == 50
    for bad, msg in [(dict(keep=0), "first and recent"), (dict(keep=5, first=3, recent=3), "first and recent"),
                     (dict(keep=5, first=-1), "first and recent")]:
        with pytest.raises(RuntimeError, match=msg):
            cache.evict([b], **bad)
    cache.batch([c], [60])
    with pytest.raises(RuntimeError, match="more tokens than weights"):
        cache.evict([c], keep=10)
    plain = kv.PagedKVCache(4, 1, page_size=8, head_dim=64, device="cpu")
    with pytest.raises(RuntimeError, match="records no weights"):
        plain.evict([plain.add()], keep=3)


def test_evictions_of_two_that_share_and_without_pages(kv):
    cache = kv.PagedKVCache(9, 1, page_size=8, head_dim=64, device="cpu", track_rows=4, track_tokens=64)
    a = cache.add()
    cache.batch([a], [32])
    b = cache.add(share=a, tokens=32)
    c = cache.add(share=a, tokens=32)
    cache.batch([a, b, c], [1, 1, 1])                      # four shared pages, one each: two are free
    pages = {s: list(cache._pages[s]) for s in (a, b, c)}
    with pytest.raises(RuntimeError, match="no free page"):
        cache.evict([a, b, c], keep=16)                    # four copies: of each page one sequence keeps it
    assert {s: cache._pages[s] for s in (a, b, c)} == pages and kv.calls == [] and cache.length(a) == 33
    cache.evict([a, b, c], keep=8)                         # two copies
    assert cache._pages[c] == pages[c][:1] and len({p for s in (a, b, c) for p in cache._pages[s]}) == 3
    held = [p for s in (a, b, c) for p in cache._pages[s]]
    assert cache.free_pages() == 6 and all(cache._users[p] == 1 for p in held)


def test_pages_and_rows_are_never_lost(kv):
    """Random batches, drafts, acceptances, evictions, forks and removals."""
    import random
    rng = random.Random(6)
    cache = kv.PagedKVCache(60, 1, page_size=8, head_dim=64, device="cpu", track_rows=8, track_tokens=200)
    live, drafted = [], set()
    for _ in range(1500):
        what, free = rng.random(), [s for s in live if s not in drafted]
        try:
            if what < 0.15:
                live.append(cache.add())
            elif what < 0.3 and free:
                s = rng.choice(free)
                n = cache.length(s) if cache._lost[s] else rng.randint(0, cache.length(s))
                live.append(cache.add(share=s, tokens=n))
            elif what < 0.45 and live:
                s = live.pop(rng.randrange(len(live)))
                drafted.discard(s)
                cache.remove(s)
            elif what < 0.6 and free:
                some = rng.sample(free, rng.randint(1, len(free)))
                cache.draft(some, [[rng.randrange(-1, j) for j in range(rng.randint(0, 12))] for _ in some])
                drafted |= set(some)
            elif what < 0.75 and drafted:
                some = rng.sample(sorted(drafted), rng.randint(1, len(drafted)))
                cache.accept(some, [sorted(rng.sample(range(cache._drafts[s][1]), rng.randint(0, cache._drafts[s][1])))
                                    for s in some])
                drafted -= set(some)
            elif what < 0.85 and free:
                cache.evict(rng.sample(free, rng.randint(1, len(free))), keep=rng.randint(1, 60))
            elif free:
                some = rng.sample(free, rng.randint(1, len(free)))
                cache.batch(some, [rng.randint(0, 20) for _ in some])
        except RuntimeError as e:
            assert "no free" in str(e) or "more tokens than weights" in str(e), e
        held = [p for s in live for p in cache._pages[s]]
        assert len(set(held)) + cache.free_pages() == 60 and not set(held) & set(cache._free)
        assert all(held.count(p) == cache._users[p] for p in set(held))
        assert all(len(cache._pages[s]) == -(-cache.length(s) // 8) for s in live)
        assert sorted([*cache._rows.values(), *cache._free_rows]) == list(range(8)) and set(cache._rows) == set(live)
        # the page that a sequence writes next is its own
        assert all(cache.length(s) % 8 == 0 or cache._users[cache._pages[s][-1]] == 1 for s in live)


def test_a_tracked_cache_takes_the_paths_that_record(kv, monkeypatch):
    taken = []
    for name in ("paged_decode_attention", "paged_decode_attention_weights", "paged_prefill_attention",
                 "paged_prefill_weights", "paged_tree_attention", "paged_shared_prefix_attention"):
        monkeypatch.setattr(kv, name, lambda *a, name=name: taken.append((name, a)))
    cache = kv.PagedKVCache(600, 8, page_size=64, head_dim=64, device="cpu", track_rows=64, track_tokens=100, observe=7,
                            n_layers=2)
    a = cache.add()
    cache.attention(cache.batch([a], [8192]), None, 0.1, window=9, layer=1)
    assert [n for n, _ in taken] == ["paged_prefill_weights", "paged_prefill_attention"]
    args = taken[0][1]
    assert args[5].data_ptr() == cache.weights[1].data_ptr() and args[6:10] == (0.1, 0.0, None, 9) and args[10] == 7
    assert args[11].tolist() == [cache._rows[a]]
    seqs = [a] + [cache.add(share=a, tokens=8192) for _ in range(31)]
    taken.clear()
    step = cache.batch(seqs)
    cache.attention(step, None, 0.1)
    (name, args), = taken
    assert name == "paged_decode_attention_weights" and args[5].data_ptr() == cache.weights[0].data_ptr()
    assert args[-1].tolist() == [cache._rows[s] for s in seqs]
    taken.clear()
    step = cache.draft([a], [[-1, 0]])
    cache.attention(step, None, 0.1, window=3)
    (name, args), = taken
    assert name == "paged_tree_attention" and args[6] is step.tree_mask and args[-1] is step.positions
