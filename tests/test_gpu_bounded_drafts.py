"""GPU: a bounded cache that decodes by drafts alone (track_drafts): what accepted tokens give
is recorded as decode steps of the same tokens would record it, against the float64 definition
(tests/bounded_ref.py, where the tolerances are derived)."""
from __future__ import annotations

import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Model:
    """A cache of two layers, its steps over random rows."""

    def __init__(self, dev, dtype, H, Hkv, D, page, opts, **more):
        from llmik_cuda.kv_cache import PagedKVCache
        self.dev, self.dtype, self.H, self.Hkv, self.D, self.page, self.opts = dev, dtype, H, Hkv, D, page, opts
        self.cache = PagedKVCache(100, Hkv, page_size=page, head_dim=D, dtype=dtype, n_layers=2, track_rows=4,
                                  track_tokens=400, track_drafts=True, **more)
        self.gen = torch.Generator(device=dev).manual_seed(1)
        self.scale = D ** -0.5

    def run(self, step):
        """q of every layer."""
        out = []
        for layer in range(2):
            qkv = torch.randn(step.rows, (self.H + 2 * self.Hkv) * self.D, generator=self.gen, device=self.dev).to(self.dtype)
            q = self.cache.append(step, qkv, None, None, layer=layer)
            self.cache.attention(step, q, self.scale, layer=layer, **self.opts)
            out.append(q)
        return out

    def check(self, before, seqs, q, counts):
        """The weights: those of `before` and what the sequences' last tokens give, whose rows q has by layer."""
        rows = [self.cache._rows[s] for s in seqs]
        lens = [self.cache.length(s) for s in seqs]
        width = max(len(self.cache._pages[s]) for s in seqs)
        table = torch.tensor([self.cache._pages[s] + [-1] * (width - len(self.cache._pages[s])) for s in seqs],
                             dtype=torch.int32, device=self.dev)
        for layer in range(2):
            want, bound = bref.weights(before[layer], rows, q[layer], self.cache.k[layer], table, lens, counts, self.scale,
                                       self.page, **self.opts)
            ref.check(self.cache.weights[layer], want, bound)


@pytest.mark.parametrize("dtype,H,Hkv,D,page,opts,lost", [
    (F16, 8, 2, 64, 16, {}, False),
    (BF16, 12, 4, 128, 8, {"softcap": 30.0}, True),
    (F16, 4, 4, 64, 32, {"slopes": True, "window": 60}, False),
], ids=str)
def test_accepted_tokens_record_what_they_give(llmik, cuda, dtype, H, Hkv, D, page, opts, lost):
    rng = random.Random(2)
    if opts.get("slopes"):
        opts = {**opts, "slopes": torch.tensor([0.5 ** (h + 1) for h in range(H)], device=cuda)}
    m = Model(cuda, dtype, H, Hkv, D, page, opts)
    cache = m.cache
    seqs = [cache.add() for _ in range(3)]
    m.run(cache.batch(seqs, [150, 40, 97]))
    if lost:
        cache.evict(seqs, keep=90, first=2, recent=9)
    for turn in range(3):
        trees = [[rng.randrange(-1, j) for j in range(n)] for n in (11, 1, 70)]
        before = cache.weights.clone()
        step = cache.draft(seqs, trees)
        q = m.run(step)
        assert torch.equal(cache.weights, before)          # the tree itself adds nothing
        paths = []
        for tree in trees:
            at, path = rng.randrange(len(tree)), []
            while at >= 0:
                path.append(at)
                at = tree[at]
            paths.append(path[::-1])
        if turn == 1:
            paths[1] = []
        starts, order = [0, len(trees[0]), len(trees[0]) + len(trees[1])], [2, 0, 1]
        rows = torch.tensor([starts[i] + j for i in order for j in paths[i]], device=cuda)
        cache.accept([seqs[i] for i in order], [paths[i] for i in order])
        m.check(before, [seqs[i] for i in order], [x[rows] for x in q], [len(paths[i]) for i in order])
    assert not cache._unrecorded
    if not opts.get("window"):
        cache.evict(seqs, keep=50, first=2, recent=9)
        assert [cache.length(s) for s in seqs] == [50 if cache.position(s) > 50 else cache.position(s) for s in seqs]


def test_drafts_and_decode_steps_record_alike(llmik, cuda):
    """A chain that is drafted and accepted gives the weights that decode steps of its tokens give."""
    H, Hkv, D, n = 8, 2, 64, 6
    m = Model(cuda, F16, H, Hkv, D, 16, {})
    cache = m.cache
    a = cache.add()
    m.run(cache.batch([a], [120]))
    b = cache.add(share=a, tokens=120)
    qkv = [torch.randn(n, (H + 2 * Hkv) * D, generator=m.gen, device=cuda).to(F16) for _ in range(2)]
    step = cache.draft([a], [[j - 1 for j in range(n)] + [0, 2]])      # and two that are dropped
    for layer in range(2):
        rows = torch.cat([qkv[layer], qkv[layer][:2]])
        cache.attention(step, cache.append(step, rows, None, None, layer=layer), m.scale, layer=layer)
    cache.accept([a], [list(range(n))])
    for j in range(n):
        step = cache.batch([b])
        for layer in range(2):
            cache.attention(step, cache.append(step, qkv[layer][j:j + 1], None, None, layer=layer), m.scale, layer=layer)
    got, want = (cache.weights[:, cache._rows[s], :, :120 + n].double() for s in (a, b))
    # each is off by at most the bound of bounded_ref.weights; of probabilities of all rows together: 4 e of
    # scores below 8, (D + 24) 2^-24 8, and their sums, 2^-24 (16 + 126 / 8), 2^-22
    rel = 4 * ((D + 24) * 2.0 ** -24 * 8 + 2.0 ** -22) + 2.0 ** -22 + 2.0 ** -24 * (32 + 4 * n * 4)
    assert bool(((got - want).abs() <= 2 * rel * want.abs() + 1e-37).all()) and bool((got > 0).all())
