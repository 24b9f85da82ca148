"""CPU: what PagedKVCache.accept says of lists that are no paths of their drafts."""
from __future__ import annotations

import random
import warnings

import pytest

from tests.test_bounded_host import kv, mod   # noqa: F401


def _cache(kv):
    cache = kv.PagedKVCache(60, 2, page_size=8, head_dim=64, device="cpu")
    seqs = [cache.add(), cache.add()]
    cache.batch(seqs, [17, 3])
    return cache, seqs


TREE = [-1, 0, 0, 2, -1, 4, 3]


@pytest.mark.parametrize("path", [[1], [0, 3], [0, 1, 2], [4, 6], [0, 4], [0, 2, 6], [2, 3]], ids=str)
def test_lists_that_are_no_paths_give_a_warning(kv, path):   # noqa: F811
    """A token without its parent, siblings, a node behind another branch."""
    cache, (a, b) = _cache(kv)
    cache.draft([a, b], [TREE, [-1]])
    with pytest.warns(UserWarning, match=rf"sequences \[{a}\] is no path"):
        cache.accept([b, a], [[0], path])
    assert cache.length(a) == 17 + len(path) and cache.length(b) == 4


@pytest.mark.parametrize("path", [[], [0], [4], [0, 1], [0, 2], [4, 5], [0, 2, 3, 6]], ids=str)
def test_paths_give_none(kv, path):   # noqa: F811
    cache, (a, b) = _cache(kv)
    cache.draft([b, a], [[-1, 0, 1], TREE])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.accept([a, b], [path, [0, 1, 2]])
    assert cache.length(a) == 17 + len(path) and cache.length(b) == 6


def test_random_paths_are_paths(kv):   # noqa: F811
    """Every node's path of random trees, and every other ascending list of a small one."""
    rng = random.Random(1)
    cache, (a, _) = _cache(kv)
    for _ in range(60):
        tree = [rng.randrange(-1, j) for j in range(rng.randint(1, 9))]
        paths = {()}
        for j in range(len(tree)):
            path, at = [], j
            while at >= 0:
                path.append(at)
                at = tree[at]
            paths.add(tuple(path[::-1]))
        some = sorted(rng.sample(range(len(tree)), rng.randint(0, len(tree))))
        cache.draft([a], [tree])
        with warnings.catch_warnings(record=True) as said:
            warnings.simplefilter("always")
            cache.accept([a], [some])
        assert (len(said) == 0) == (tuple(some) in paths)
        cache.remove(a)
        a = cache.add()


def _tracked(kv, **more):
    cache = kv.PagedKVCache(60, 2, page_size=8, head_dim=64, device="cpu", n_layers=2, track_rows=4, track_tokens=200, **more)
    seqs = [cache.add(), cache.add()]
    cache.batch(seqs, [60, 50])
    return cache, seqs


def test_evictions_that_meet_unrecorded_drafts_give_a_warning(kv):   # noqa: F811
    cache, (a, b) = _tracked(kv)
    cache.draft([a, b], [[-1, 0], [-1]])
    cache.accept([a, b], [[0, 1], []])
    c = cache.add(share=a, tokens=62)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.evict([b], keep=40)                   # b accepted nothing
        cache.evict([a, c], keep=70)                # nothing is cut
    with pytest.warns(UserWarning, match=rf"sequences \[{a}, {c}\] hold nothing of drafted"):
        cache.evict([a, b, c], keep=30)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.evict([a, b, c], keep=20)             # said once, until more are accepted
    cache.draft([a], [[-1]])
    cache.accept([a], [[0]])
    cache.remove(c)
    with pytest.warns(UserWarning, match=rf"sequences \[{a}\] hold nothing"):
        cache.evict([a], keep=10)
    with pytest.raises(RuntimeError, match="track_drafts needs track_rows"):
        kv.PagedKVCache(4, 1, page_size=8, head_dim=64, device="cpu", track_drafts=True)


def test_accepted_tokens_are_recorded_as_a_prompt(kv, monkeypatch):   # noqa: F811
    """The calls' arguments: rows of the path in the step's q, the sequences as they are after it."""
    import torch
    recorded = []
    monkeypatch.setattr(kv, "paged_prefill_weights", lambda *args: recorded.append(args))
    monkeypatch.setattr(kv, "paged_tree_attention", lambda *args: None)
    cache, (a, b) = _tracked(kv, track_drafts=True)
    c = cache.add()
    cache.batch([c], [9])
    first = cache.draft([a, b], [[-1, 0, 0, 2], [-1] * 3])
    second = cache.draft([c], [[-1, 0]])
    slopes = torch.ones(2)
    q = torch.arange(7.0)[:, None, None].expand(7, 2, 64).contiguous()
    for layer in range(2):
        cache.attention(first, q + 10 * layer, 0.5, softcap=3.0, slopes=slopes, window=7, layer=layer)
    cache.attention(first, q + 100, 0.25, layer=1)   # the layer's last call counts
    kept = q.clone()
    q.zero_()                                        # a copy is kept
    cache.attention(second, kept[:2], 0.5)           # one layer of two
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        cache.accept([c, b, a], [[0], [2], [0, 2]])
    assert len(recorded) == 3
    for args, layer, rows, seqs, counts, opts in (
            (recorded[0], 0, kept[:1], [c], [1], (0.5, 0.0, None, 0)),
            (recorded[1], 0, kept[[6, 0, 2]], [b, a], [1, 2], (0.5, 3.0, slopes, 7)),
            (recorded[2], 1, kept[[6, 0, 2]] + 100, [b, a], [1, 2], (0.25, 0.0, None, 0))):
        got_q, k, table, lens, cu, w, *options, observe, weight_rows = args
        assert torch.equal(got_q, rows) and k.data_ptr() == cache.k[layer].data_ptr()
        assert w.data_ptr() == cache.weights[layer].data_ptr() and observe == 0
        assert options[:2] == list(opts[:2]) and options[2] is opts[2] and options[3] == opts[3]
        assert lens.tolist() == [cache.length(s) for s in seqs]
        assert cu.tolist() == [0, *(sum(counts[:i + 1]) for i in range(len(counts)))]
        assert weight_rows.tolist() == [cache._rows[s] for s in seqs]
        assert [[p for p in row if p >= 0] for row in table.tolist()] == [cache._pages[s] for s in seqs]
    assert cache._unrecorded == {c}
    recorded.clear()
    cache.draft([a], [[-1]])
    cache.accept([a], [[]])                          # nothing is accepted, nothing recorded
    assert recorded == [] and cache._unrecorded == {c}
