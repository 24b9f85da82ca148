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
