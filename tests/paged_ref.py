"""Plain float64 restatement of the paged cache's operators, and their error bounds.

Everything loops over sequences and reads the page table token by token, as the
definition does. `attend` returns the result and a bound on a kernel's error,
from what the kernels round:

* the output once, to its type: half a step, u |out| (u: fp16 2^-11, bf16 2^-8);
* each probability p_j before the product with V, by a relative up: 2^-22 /
  2^-16 where it is carried as a pair of 16-bit values (decode), u where it is
  one (prompts, prefix), and below 2^-22 of the row's largest an fp16 value
  loses steps (at most 2^-33 of the largest each, 2^-25 / 2^8): up * sum_j p_j
  |v_j| + 2^-32 max|v| * keys;
* the score, in fp32: a product of D terms and its scaling, (D + 8) 2^-24 sum_d
  |q_d k_d| scale; the cap, cap 2^-20 (exp2, a reciprocal and a fma of values up
  to 2 cap, log2(e) included); the bias, 2^-23 |bias|; exp2 itself 2^-22. A score error e
  changes p by a factor within 1 +- 2 e, and the sum of all p by as much: 4 e
  sum_j p_j |v_j|;
* fp32 sums over the keys in any order: (keys) 2^-24 at most, and sqrt(keys) in
  all but contrived inputs; 2^-24 (16 + keys / 8) is used, as a lane adds at
  most keys / 8 values one after the other before partial sums join.
"""
from __future__ import annotations

import math
import random

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
PAIR = {torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def make_cache(lens, Hkv, D, page, dtype, dev, seed, spare=3, extra_columns=1, gap=0, fill=None):
    """(k, v, table, seq_lens): pages of each sequence in random order; slots
    that hold no token, and pages that nobody owns, hold `fill` (default: random
    values). gap: unused elements between pages."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    n_pages = sum(need) + spare
    def pool():
        buf = torch.empty(n_pages, Hkv * page * D + gap, device=dev, dtype=dtype)
        buf.normal_(generator=gen)
        return buf[:, :Hkv * page * D].unflatten(1, (Hkv, page, D)) if gap else buf.view(n_pages, Hkv, page, D)
    k, v = pool(), pool()
    order = torch.randperm(n_pages, generator=gen, device=dev).int()
    table = torch.full((len(lens), max(need + [0]) + extra_columns), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    if fill is not None:
        owned = torch.zeros(n_pages, page, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            for t0 in range(0, max(n, 0), page):
                owned[int(table[b, t0 // page]), :min(page, n - t0)] = True
        for c in (k, v):
            c[(~owned)[:, None, :, None].expand(-1, Hkv, -1, D)] = fill
    return k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev)


def tokens_of(cache, table_row, n, page):
    """The first n tokens of a sequence, [Hkv, n, D] in float64, and which of them are mapped."""
    t = torch.arange(n, device=cache.device)
    pages = table_row[t // page].long()
    ok = (pages >= 0) & (pages < cache.shape[0])
    x = cache[torch.where(ok, pages, torch.zeros_like(pages)), :, t % page].double()   # [n, Hkv, D]
    return torch.where(ok[:, None, None], x, torch.zeros_like(x)).transpose(0, 1), ok


def attend(q, k, v, ok, pos_q, scale, softcap=0.0, slopes=None, window=0, up=0.0):
    """q [L, H, D] at positions pos_q [L] over k, v [Hkv, n, D] (float64), keys `ok` [n].
    Returns (out, bound) in float64."""
    L, H, D = q.shape
    Hkv, n = k.shape[0], k.shape[1]
    u = U[q.dtype]
    out = torch.zeros(L, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if n == 0:
        return out, bound
    dist = pos_q[:, None] - torch.arange(n, device=q.device)
    seen = (dist >= 0) & ok
    if window:
        seen = seen & (dist < window)
    for h in range(H):
        kh, vh, qh = k[h // (H // Hkv)], v[h // (H // Hkv)], q[:, h].double()
        s = qh @ kh.t().contiguous() * scale
        e = (D + 8) * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().t().contiguous()) + 2.0 ** -22
        if softcap:
            s = torch.tanh(s / softcap) * softcap
            e = e + softcap * 2.0 ** -20
        if slopes is not None:
            bias = slopes[h].double() * dist
            s = s - bias
            e = e + 2.0 ** -23 * bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m)), torch.zeros_like(s))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        # values that a row does not see count as zero (they may be anything)
        out[:, h] = p @ torch.where(ok[:, None], vh, torch.zeros_like(vh))
        worst = torch.where(seen, e, torch.zeros_like(e)).amax(-1, keepdim=True)
        keys = seen.sum(-1, keepdim=True)
        spread = p @ vh.abs()
        bound[:, h] = (u * out[:, h].abs() + (up + 4 * worst + 2.0 ** -24 * (16 + keys / 8.0)) * spread
                       + 2.0 ** -32 * keys * vh.abs().amax())
    return out, bound


def rows_of(lens, new):
    """[(sequence, its new rows' first row, rows, first position)]"""
    out, at = [], 0
    for b, n in enumerate(new):
        out.append((b, at, n, lens[b] - n))
        at += n
    return out


def offsets(new, dev):
    return torch.tensor([0] + list(new), device=dev).cumsum(0).int()


def attention(q, k, v, table, lens, new, scale, page, pair, prefix_pages=None, prefix_len=0, **opts):
    """The result and the bound for q's rows: new[b] rows of sequence b, its last tokens."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    up = (PAIR if pair else U)[q.dtype]
    for b, r0, n, pos in rows_of(lens, new):
        if n <= 0:
            continue
        live = min(max(lens[b], 0), table.shape[1] * page if not prefix_len else 10 ** 9)
        kb, ok = tokens_of(k, table[b], live, page)
        vb, _ = tokens_of(v, table[b], live, page)
        if prefix_len:
            m = min(prefix_len, live)
            kp, okp = tokens_of(k, prefix_pages, m, page)
            vp, _ = tokens_of(v, prefix_pages, m, page)
            kb, vb, ok = kb.clone(), vb.clone(), ok.clone()
            kb[:, :m], vb[:, :m], ok[:m] = kp, vp, okp
        p = torch.arange(pos, pos + n, device=q.device)
        out[r0:r0 + n], bound[r0:r0 + n] = attend(q[r0:r0 + n], kb, vb, ok, p, scale, up=up, **opts)
    return out, bound


def rotate(x, cos, sin):
    """x [n, heads, D], cos and sin [n, D], float64."""
    h = x.shape[-1] // 2
    lo, hi = x[..., :h], x[..., h:]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([lo * c[..., :h] - hi * s[..., :h], hi * c[..., h:] + lo * s[..., h:]], dim=-1)


def check(got, ref, bound):
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all())
    worst = (err / bound.clamp(min=1e-30)).max().item() if err.numel() else 0.0
    assert bool((err <= bound).all()), f"error {err.max().item():.3e}, {worst:.2f} times the bound"


def ragged(seed, B, lo, hi):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(B)]
