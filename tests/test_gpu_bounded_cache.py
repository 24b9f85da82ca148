"""GPU: PagedKVCache with drafted trees and evictions, run together as a decoding loop
does, against lists of tokens that the test keeps (tests/bounded_ref.py)."""
from __future__ import annotations

import random

import pytest
import torch

from tests import bounded_ref as bref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Loop:
    """The cache and, for every (layer, sequence), the tokens that it should hold: k, v
    [Hkv, n, D] as they were written and w [Hkv, n] as they were recorded."""

    def __init__(self, dev, dtype, H=8, Hkv=2, D=64, page=16, layers=2, observe=0, track=True):
        from llmik_cuda.kv_cache import PagedKVCache
        self.H, self.Hkv, self.D, self.page, self.layers, self.dtype, self.dev = H, Hkv, D, page, layers, dtype, dev
        more = dict(track_rows=4, track_tokens=512, observe=observe) if track else {}
        self.cache = PagedKVCache(120, Hkv, page_size=page, head_dim=D, dtype=dtype, n_layers=layers, **more)
        self.gen = torch.Generator(device=dev).manual_seed(3)
        self.observe, self.scale = observe, D ** -0.5
        ang = torch.arange(1000, device=dev)[:, None] / 100.0 ** (torch.arange(0, D, 2, device=dev) / D)
        self.cos, self.sin = (torch.cat([f(ang), f(ang)], 1).float() for f in (torch.cos, torch.sin))
        self.kept = {}     # (layer, sequence) -> [k, v, w]
        self.text = {}     # sequence -> tokens of its text

    def add(self, share=None, tokens=0):
        s = self.cache.add(share, tokens)
        for layer in range(self.layers):
            if share is None:
                zero = torch.zeros(self.Hkv, 0, self.D, dtype=self.dtype, device=self.dev)
                self.kept[layer, s] = [zero, zero, torch.zeros(self.Hkv, 0, device=self.dev)]
            else:
                self.kept[layer, s] = [x[:, :tokens].clone() for x in self.kept[layer, share]]
        lost = 0 if share is None else self.text[share] - self.kept[0, share][0].shape[1]
        self.text[s] = tokens + (lost if tokens else 0)
        return s

    def slots(self, layer, table_row, n):
        """What the cache holds in a sequence's first n slots."""
        t = torch.arange(n, device=self.dev)
        at = table_row[t // self.page].long(), slice(None), t % self.page
        return [c[layer][at].transpose(0, 1) for c in (self.cache.k, self.cache.v)]

    def run(self, seqs, new, trees=None):
        """One step of all layers, its q, k and v checked against the rope of random rows, its
        attention against the lists. trees: parents of drafted tokens."""
        step = self.cache.batch(seqs, new) if trees is None else self.cache.draft(seqs, trees)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        for layer in range(self.layers):
            qkv = torch.randn(step.rows, (self.H + 2 * self.Hkv) * self.D, generator=self.gen, device=self.dev).to(self.dtype)
            q = self.cache.append(step, qkv, self.cos, self.sin, layer=layer)
            out = self.cache.attention(step, q, self.scale, softcap=30.0, layer=layer)
            x = qkv.double().view(step.rows, -1, self.D)
            for i, (s, n) in enumerate(zip(seqs, new)):
                if n == 0:
                    continue
                rows = slice(starts[i], starts[i + 1])
                held = self.kept[layer, s]
                have = held[0].shape[1]
                depth = list(range(n))
                seen = [(1 << j + 1) - 1 for j in range(n)]
                if trees is not None:
                    depth, seen = [], []
                    for j, p in enumerate(trees[i]):
                        depth.append(depth[p] + 1 if p >= 0 else 0)
                        seen.append((seen[p] if p >= 0 else 0) | 1 << j)
                pos = torch.tensor(depth, device=self.dev) + self.text[s]
                turned = ref.rotate(x[rows, :self.H + self.Hkv], self.cos[pos].double(), self.sin[pos].double())
                k, v = self.slots(layer, step.page_table[i], have + n)
                assert torch.equal(k[:, :have], held[0]) and torch.equal(v[:, :have], held[1])
                assert torch.equal(v[:, have:], qkv.view(step.rows, -1, self.D)[rows, self.H + self.Hkv:].transpose(0, 1))
                # one rounding, two products and a sum in fp32 of values below 6
                tol = lambda want: ref.U[self.dtype] * want.abs() + 18 * 2.0 ** -23   # noqa: E731
                for got, want in ((q[rows], turned[:, :self.H]), (k[:, have:].transpose(0, 1), turned[:, self.H:])):
                    assert bool(((got.double() - want).abs() <= tol(want)).all())
                mask = torch.tensor([[True] * have + [bool(m >> j & 1) for j in range(n)] for m in seen], device=self.dev)
                dist = torch.zeros(n, have + n, dtype=torch.long, device=self.dev)
                ok = torch.ones(have + n, dtype=torch.bool, device=self.dev)
                want, bound = bref.attend(q[rows], k.double(), v.double(), ok, mask, dist, self.scale,
                                          (ref.PAIR if step.cu_tokens is None else ref.U)[self.dtype], softcap=30.0)
                ref.check(out[rows], want, bound)
                if trees is not None:
                    self.drafted[layer, s] = [k[:, have:].clone(), v[:, have:].clone()]
                    continue
                w = torch.cat([held[2], torch.zeros(self.Hkv, n, device=self.dev)], 1)
                if self.cache.weights is not None:
                    first = max(0, n - self.observe) if self.observe and step.cu_tokens is not None else 0
                    p, rel, _ = bref.probabilities(q[rows][first:], k.double(), mask[first:], dist[first:], self.scale,
                                                   softcap=30.0)
                    G = self.H // self.Hkv
                    add, off = (y.sum(1).view(self.Hkv, G, -1).sum(1) for y in (p, p * rel))
                    got = self.cache.weights[layer, self.cache._rows[s], :, :have + n]
                    ref.check(got, w + add, off + (G * n + 4) * 2.0 ** -24 * (w + add))
                    assert int(self.cache.weights[layer, self.cache._rows[s], :, have + n:].count_nonzero()) == 0
                    w = got.clone()
                self.kept[layer, s] = [k.clone(), v.clone(), w]
        if trees is None:
            for s, n in zip(seqs, new):
                self.text[s] += n

    drafted: dict = {}

    def draft(self, seqs, trees):
        self.drafted = {}
        self.run(seqs, [len(t) for t in trees], trees)

    def accept(self, seqs, paths):
        self.cache.accept(seqs, paths)
        for s, path in zip(seqs, paths):
            for layer in range(self.layers):
                held = self.kept[layer, s]
                if (layer, s) in self.drafted:
                    for i in range(2):
                        held[i] = torch.cat([held[i], self.drafted[layer, s][i][:, path]], 1)
                    held[2] = torch.cat([held[2], torch.zeros(self.Hkv, len(path), device=self.dev)], 1)
            self.text[s] += len(path)

    def evict(self, seqs, keep, first, recent):
        for s in seqs:
            for layer in range(self.layers):
                held = self.kept[layer, s]
                lists, _ = bref.select(held[2][None], [held[2].shape[1]], keep, first, recent)
                for i in range(3):
                    held[i] = torch.stack([x[[t for t in pick if t >= 0]] for x, pick in zip(held[i], lists[0])])
        self.cache.evict(seqs, keep, first, recent)

    def check_kept(self):
        """Every sequence's slots and weights, read back."""
        for s in self.text:
            n = self.cache.length(s)
            row = torch.tensor(self.cache._pages[s], device=self.dev)
            for layer in range(self.layers):
                held = self.kept[layer, s]
                k, v = self.slots(layer, row, n)
                assert held[0].shape[1] == n and torch.equal(k, held[0]) and torch.equal(v, held[1])
                if self.cache.weights is not None:
                    w = self.cache.weights[layer, self.cache._rows[s]]
                    assert torch.equal(w[:, :n], held[2]) and int(w[:, n:].count_nonzero()) == 0
            assert self.cache.position(s) == self.text[s]


def _tree(rng, n):
    return [rng.randrange(-1, j) for j in range(n)]


def _path(rng, tree):
    if not tree:
        return []
    at, path = rng.randrange(len(tree)), []
    while at >= 0:
        path.append(at)
        at = tree[at]
    return path[::-1]


@pytest.mark.parametrize("dtype,observe", [(F16, 0), (BF16, 20)], ids=str)
def test_a_bounded_cache_that_drafts(llmik, cuda, dtype, observe):
    rng = random.Random(4)
    loop = Loop(cuda, dtype, observe=observe)
    a, b = loop.add(), loop.add()
    loop.run([a, b], [150, 40])
    c = loop.add(share=a, tokens=100)
    loop.run([c, b], [30, 3])
    loop.check_kept()
    loop.evict([a, c, b], keep=60, first=3, recent=10)      # a and c share pages; b stays
    loop.check_kept()
    for turn in range(3):
        loop.run([a, b, c], [1, 1, 1])
        trees = [_tree(rng, n) for n in (9, 0, 20)]
        loop.draft([a, b, c], trees)
        loop.accept([a, b, c], [_path(rng, t) for t in trees])
        loop.check_kept()
    d = loop.add(share=c, tokens=loop.cache.length(c))       # a fork of a sequence that lost tokens
    loop.run([d, a], [70, 1])                                # a chunk behind it
    loop.evict([a, b, c, d], keep=40, first=0, recent=40)    # the last ones alone
    loop.check_kept()
    loop.run([d, c, b, a], [1, 2, 0, 1])
    loop.check_kept()


def test_drafts_without_weights(llmik, cuda):
    rng = random.Random(5)
    loop = Loop(cuda, F16, Hkv=4, D=128, page=8, layers=3, track=False)
    a, b = loop.add(), loop.add()
    loop.run([a, b], [33, 8])
    for n in (1, 70, 5):
        trees = [_tree(rng, n), _tree(rng, 2 * n)]
        loop.draft([b, a], trees)
        loop.accept([a, b], [_path(rng, trees[1]), []])
        loop.run([a, b], [1, 1])
        loop.check_kept()
