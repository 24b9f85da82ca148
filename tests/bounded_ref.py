"""Plain float64 restatements of drafted trees and of caches bounded by attention
weight, and their error bounds (tests/paged_ref.py has the paged cache's, whose terms
these use).

A weight is a sum of probabilities p. A kernel's p = 2^(t - m) / l is off by

* the score: e as in paged_ref.attend, with 16 steps more for t - m and the scaling in
  the log2 domain (values of the scores' size), and 2^-22 for exp2: a factor within
  1 +- 2 e for p and as much for the sum it is divided by: 4 e p;
* the sum l in any order: 2^-24 (16 + keys / 8) p, and the division 2^-22 p;

and adding N of them up, to what was there, by at most (N + 1) 2^-24 of the result's
size, in any order.
"""
from __future__ import annotations

import math

import torch

from tests import paged_ref as ref


def probabilities(q, k, seen, dist, scale, softcap=0.0, slopes=None, window=0):
    """q [L, H, D] over k [Hkv, n, D] (float64) where `seen` [L, n], at distances dist
    [L, n]: (p, relative bound) [H, L, n] in float64; zeros for rows that see nothing."""
    L, H, D = q.shape
    Hkv, n = k.shape[:2]
    if window:
        seen = seen & (dist < window)
    p, bound = [], []
    for h in range(H):
        qh, kh = q[:, h].double(), k[h // (H // Hkv)]
        s = qh @ kh.t().contiguous() * scale
        e = (D + 24) * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().t().contiguous()) + 2.0 ** -22
        if softcap:
            s = torch.tanh(s / softcap) * softcap
            e = e + softcap * 2.0 ** -20
        if slopes is not None:
            bias = slopes[h].double() * dist
            s = s - bias
            e = e + 2.0 ** -22 * bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
        x = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
        worst = torch.where(seen, e, torch.zeros_like(e)).amax(-1, keepdim=True)
        keys = seen.sum(-1, keepdim=True)
        p.append(x / x.sum(-1, keepdim=True).clamp(min=1e-300))
        bound.append((4 * worst + 2.0 ** -22 + 2.0 ** -24 * (16 + keys / 8.0)).expand(-1, n))
    return torch.stack(p), torch.stack(bound), seen


def attend(q, k, v, ok, seen, dist, scale, up, **opts):
    """(out, bound) [L, H, D] as paged_ref.attend, for any mask. ok [n]: mapped keys."""
    G = q.shape[1] // k.shape[0]
    p, rel, seen = probabilities(q, k, seen & ok, dist, scale, **opts)
    vh = v.repeat_interleave(G, 0)
    out = (p @ vh).transpose(0, 1)
    spread = ((p * (up + rel)) @ vh.abs()).transpose(0, 1)
    keys = seen.sum(-1)[:, None, None]
    return out, ref.U[q.dtype] * out.abs() + spread + 2.0 ** -32 * keys * v.abs().amax() if v.numel() else spread


def tree(q, k, v, table, lens, new, mask, positions, scale, page, **opts):
    """Attention of drafted trees. mask: for every row a Python integer; positions: a list or None."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, r0, n, ctx in ref.rows_of([max(x, 0) for x in lens], new):
        live = min(max(lens[b], 0), table.shape[1] * page)
        if n <= 0 or live == 0:
            continue
        kb, ok = ref.tokens_of(k, table[b], live, page)
        vb, _ = ref.tokens_of(v, table[b], live, page)
        kb = torch.where(ok[None, :, None], kb, torch.zeros_like(kb))
        at = [min(max(positions[r0 + i] if positions is not None else ctx + i, max(ctx, 0)), 1 << 30) for i in range(n)]
        seen = [[ctx + i >= 0 and (t < ctx or bool(mask[r0 + i] >> (t - ctx) & 1)) for t in range(live)]
                for i in range(n)]
        pos_k = [t if t < ctx else at[t - ctx] for t in range(live)]
        dist = torch.tensor(at, device=q.device)[:, None] - torch.tensor(pos_k, device=q.device)
        out[r0:r0 + n], bound[r0:r0 + n] = attend(q[r0:r0 + n], kb, vb, ok,
                                                  torch.tensor(seen, device=q.device).view(n, live), dist, scale,
                                                  ref.U[q.dtype], **opts)
    return out, bound


def words_of(mask, words, dev):
    """Rows of Python integers as int64 [rows, words]."""
    signed = lambda w: w - (1 << 64) if w >> 63 else w   # noqa: E731
    rows = [[signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in mask]
    return torch.tensor(rows, dtype=torch.int64, device=dev).view(len(mask), words)


def trees(rng, new, ctx):
    """Random trees: (mask, depth as position) of every row."""
    mask, pos = [], []
    for n, c in zip(new, ctx):
        seen, deep = [], []
        for i in range(n):
            parent = rng.randrange(-1, i)
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            deep.append(deep[parent] + 1 if parent >= 0 else c)
        mask += seen
        pos += deep
    return mask, pos


def weights(w, rows, q, k, table, lens, new, scale, page, observe=0, **opts):
    """w [R, Hkv, W] with the probabilities of every sequence's last rows added, and a bound."""
    G = q.shape[1] // k.shape[1]
    out = w.double().clone()
    bound = 2.0 ** -24 * out.abs()
    for b, r0, n, ctx in ref.rows_of(lens, new):
        live = min(max(lens[b], 0), table.shape[1] * page)
        row = b if rows is None else rows[b]
        if n <= 0 or live == 0 or not 0 <= row < w.shape[0]:
            continue
        skip = max(0, n - observe) if observe else 0
        kb, ok = ref.tokens_of(k, table[b], live, page)
        kb = torch.where(ok[None, :, None], kb, torch.zeros_like(kb))
        dist = torch.arange(ctx + skip, ctx + n, device=q.device)[:, None] - torch.arange(live, device=q.device)
        p, rel, _ = probabilities(q[r0 + skip:r0 + n], kb, (dist >= 0) & ok, dist, scale, **opts)
        add = p.sum(1).view(-1, G, live).sum(1)
        off = (p * rel).sum(1).view(-1, G, live).sum(1)
        m = min(live, w.shape[2])
        out[row, :, :m] += add[:, :m]
        bound[row, :, :m] += (off + add * (G * (n - skip) + 2) * 2.0 ** -24)[:, :m]
    return out, bound + 2.0 ** -24 * out.abs() + 1e-37


def select(w, lens, keep, first, recent, rows=None):
    """The kept slots [B, Hkv, keep] as lists, and the lengths."""
    kept, out = [], []
    for b, n in enumerate(lens):
        n = min(max(n, 0), w.shape[2])
        row = b if rows is None else rows[b]
        heads = []
        for h in range(w.shape[1]):
            x = w[row, h].tolist() if 0 <= row < w.shape[0] else [0.0] * w.shape[2]
            if n <= keep:
                pick = list(range(n))
            else:
                rest = sorted(range(first, n - recent),
                              key=lambda t: (not math.isnan(x[t]), 0.0 if math.isnan(x[t]) else -x[t], t))
                pick = sorted([*range(first), *range(n - recent, n), *rest[:keep - first - recent]])
            heads.append(pick + [-1] * (keep - len(pick)))
        kept.append(heads)
        out.append(min(n, keep))
    return kept, out


def compact(k, v, table, lens, kept, starts=None, w=None, rows=None):
    """The cache (and weights) with the tokens moved: new tensors."""
    k2, v2, page = k.clone(), v.clone(), k.shape[2]
    w2 = None if w is None else w.clone()
    capacity = table.shape[1] * page
    tab = table.tolist()

    def place(b, t):
        p = tab[b][t // page]
        return (p, t % page) if 0 <= p < k.shape[0] else None

    for b, n in enumerate(lens):
        n, start = min(max(n, 0), capacity), 0 if starts is None else starts[b]
        if not 0 <= start < n:
            continue
        for h in range(k.shape[1]):
            row = kept[b] if not isinstance(kept[b][0] if kept[b] else 0, list) else kept[b][h]
            for i, t in enumerate(row):
                if start + i < t < n and place(b, t) and place(b, start + i):
                    (p, s), (p2, s2) = place(b, t), place(b, start + i)
                    k2[p2, h, s2], v2[p2, h, s2] = k[p, h, s], v[p, h, s]
            r = b if rows is None else rows[b]
            if w is not None and 0 <= r < w.shape[0]:
                count = next((i for i, t in enumerate(row) if t < 0), len(row))
                for i in range(min(n, w.shape[2]) - start):
                    if i >= count:
                        w2[r, h, start + i] = 0.0
                    elif start + i < row[i] < n:
                        w2[r, h, start + i] = w[r, h, row[i]] if row[i] < w.shape[2] else 0.0
    return k2, v2, w2
