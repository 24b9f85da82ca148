"""GPU: PagedKVCache as a serving loop uses it: prompts in chunks, decode steps of
changing batches, sequences that fork, end and reuse pages. Every output is
compared with attention over the tokens that the test itself kept."""
from __future__ import annotations

import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


def _tables(n, D, dev):
    ang = torch.arange(n, device=dev, dtype=torch.float64)[:, None] / (
        10000.0 ** (torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))[None]
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().float(), ang.sin().float()


@pytest.mark.parametrize("dtype,D,page,opts", [
    (torch.float16, 128, 16, {}),
    (torch.bfloat16, 64, 24, {"softcap": 25.0}),
    (torch.bfloat16, 128, 64, {"window": 90}),
], ids=str)
def test_a_serving_loop(llmik, cuda, dtype, D, page, opts):
    from llmik_cuda.kv_cache import PagedKVCache
    H, Hkv, scale = 8, 2, D ** -0.5
    rng = random.Random(11)
    gen = torch.Generator(device=cuda).manual_seed(12)
    cache = PagedKVCache(200, Hkv, page_size=page, head_dim=D, dtype=dtype)
    cache.SHARED_TOKENS, cache.SHARED_ROWS = 16, 400
    cos, sin = _tables(2000, D, cuda)
    kept = {}            # sequence -> (k, v) rows [n, Hkv, D] as the cache stores them
    shared_steps = 0

    def step(seqs, new):
        nonlocal shared_steps
        had = [cache.length(s) for s in seqs]
        batch = cache.batch(seqs, new)
        counts = new or [1] * len(seqs)
        qkv = torch.randn(sum(counts), (H + 2 * Hkv) * D, generator=gen, device=cuda).to(dtype)
        q = cache.append(batch, qkv, cos, sin)
        out = cache.attention(batch, q, scale, **opts)
        shared_steps += batch.prefix_pages is not None
        at = 0
        for s, n, h in zip(seqs, counts, had):
            x = qkv[at:at + n].double().view(n, H + 2 * Hkv, D)
            p = torch.arange(h, h + n, device=cuda)
            turned = ref.rotate(x[:, :H + Hkv], cos[p].double(), sin[p].double())
            # q and the cache hold roundings of these; take the stored k for what follows
            assert bool(((q[at:at + n].double() - turned[:, :H]).abs() <= 2 * ref.U[dtype] * turned[:, :H].abs()
                         + 2.0 ** -20).all())
            row = batch.page_table[seqs.index(s)]
            k, ok = ref.tokens_of(cache.k[0], row, h + n, page)
            v, _ = ref.tokens_of(cache.v[0], row, h + n, page)
            assert bool(ok.all())
            k, v = k.transpose(0, 1), v.transpose(0, 1)
            old_k, old_v = kept[s]
            assert torch.equal(k[:h], old_k) and torch.equal(v[:h], old_v)        # nothing that was there changed
            assert torch.equal(v[h:], x[:, H + Hkv:])
            assert bool(((k[h:] - turned[:, H:]).abs() <= 2 * ref.U[dtype] * turned[:, H:].abs() + 2.0 ** -20).all())
            kept[s] = (k, v)
            want, bound = ref.attend(q[at:at + n], k.transpose(0, 1), v.transpose(0, 1),
                                     torch.ones(h + n, dtype=torch.bool, device=cuda), p, scale, up=ref.U[dtype], **opts)
            ref.check(out[at:at + n], want, bound)
            at += n

    def add(**share):
        s = cache.add(**share)
        none = torch.zeros(0, Hkv, D, dtype=torch.float64, device=cuda)
        kept[s] = tuple(t[:share["tokens"]] for t in kept[share["share"]]) if share else (none, none)
        return s

    seqs = [add() for _ in range(3)]
    step(seqs, [150, 7, 40])                  # prompts
    step(seqs[1:], [100, 1])                  # a chunk of one, a token of another
    for _ in range(3):
        step(seqs, None)
    forks = [add(share=seqs[0], tokens=n) for n in (150, 140, 153)]
    step([seqs[0]] + forks, None)             # behind a shared prefix
    step(forks, [3, 20, 1])
    cache.remove(seqs.pop(1))
    seqs += forks + [add()]
    step(seqs[-1:], [60])
    for _ in range(3):
        some = rng.sample(seqs, rng.randint(1, len(seqs)))
        step(some, None)
        step(some, [rng.randint(0, 9) for _ in some])
    step([seqs[0]] + forks, None)
    assert shared_steps >= 2
    free = cache.free_pages()
    for s in seqs:
        cache.remove(s)
    assert cache.free_pages() == 200 > free


def test_layers_share_a_batch(llmik, cuda):
    """One batch serves two layers, and a fork's tokens are there in both."""
    from llmik_cuda.kv_cache import PagedKVCache
    H, Hkv, D = 8, 2, 128
    cache = PagedKVCache(20, Hkv, page_size=16, n_layers=2)
    a, b = cache.add(), cache.add()
    batch = cache.batch([a, b], [33, 5])
    x = torch.randn(38, (H + 2 * Hkv) * D, device=cuda).half()
    q1 = cache.append(batch, x, None, None)
    q2 = cache.append(batch, x, None, None, layer=1)
    assert torch.equal(q1, q2) and torch.equal(cache.k[0], cache.k[1]) and torch.equal(cache.v[0], cache.v[1])
    assert torch.equal(cache.attention(batch, q1, 0.1), cache.attention(batch, q2, 0.1, layer=1))
    batch = cache.batch([a, cache.add(share=a, tokens=33)])
    x = torch.randn(1, (H + 2 * Hkv) * D, device=cuda).half().expand(2, -1)
    for layer in range(2):
        q = cache.append(batch, x, None, None, layer=layer)
        out = cache.attention(batch, q, 0.1, layer=layer)
        assert torch.equal(out[0], out[1])      # the same tokens, the same query
