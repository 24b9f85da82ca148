"""Measured calls of the paged KV cache: appends with the rotary embedding, decode attention over ragged
batches, prompt attention, and decode behind a shared prefix.

With `own` false every operator runs in its plain form (elementary torch operations in fp32, rounded once);
with `own` true the calls go to llmik_cuda. Both read the same state: a cache of pages
[n_pages, n_kv_heads, page_size, head_dim] for K and V, a table [batch, max_pages] of each sequence's pages,
the live lengths, and for ragged batches the row offsets `cu_tokens` of each sequence's new tokens.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# (query heads, KV heads): the benchmark's 8B layout, its sibling with 8 heads per KV head, multi-head
# attention, and ratios that are no powers of two.
HEADS = [(32, 8), (32, 8), (64, 8), (32, 32), (16, 8), (28, 4), (40, 8), (24, 8)]
PAGES = [8, 16, 16, 24, 32, 64, 64, 128, 256]

# B sequences of lo .. hi tokens (drawn from `mix`; their new tokens where the call brings prompts), the last
# `pad` of them empty rows of a padded batch; `ctx`: at most so many tokens cached before a prompt's chunk;
# `prefix`: tokens that all sequences share in front of their own.
_BASE = {"dtype": "fp16", "D": 128, "H": 32, "Hkv": 8, "page": 64, "B": 1, "lo": 1, "hi": 1, "mix": 0, "pad": 0,
         "ctx": 0, "prefix": 0, "softcap": 0.0, "slopes": False, "window": 0}


def _case(**more):
    return {**_BASE, **more}


def listed():
    return [
        # One user's decode step: one token's q|k|v rotated and written. Launch latency.
        _case(name="append_step_b1", kind="append_step", lo=700, hi=700, page=16),
        # Five prompts of different lengths written at once, the largest append of a prefill step.
        _case(name="append_prompts_bf16", kind="append_prompt", dtype="bf16", B=5, lo=900, hi=2600, mix=2, page=32),
        # One user at a short context: the smallest attention call.
        _case(name="decode_b1_s700", kind="decode", lo=700, hi=700, page=16),
        # One user at a long context, heads of 64.
        _case(name="decode_b1_s50001_d64", kind="decode", D=64, lo=50001, hi=50001, page=128),
        # A serving batch whose sequences came at different times, in bf16, with padded rows.
        _case(name="decode_b32_ragged_bf16", kind="decode", dtype="bf16", B=32, lo=30, hi=8000, mix=3, pad=2),
        # A full batch at one length, scores capped: the largest cache.
        _case(name="decode_b64_s8192_cap", kind="decode", H=64, B=64, lo=8192, hi=8192, page=256, softcap=30.0),
        # Distance bias and a sliding window over small pages, 7 heads per KV head.
        _case(name="decode_b24_slopes_window", kind="decode", dtype="bf16", H=28, Hkv=4, B=24, lo=100, hi=12000,
              mix=4, page=24, slopes=True, window=4096),
        # Short prompts of three users in one call.
        _case(name="prefill_3_short", kind="prefill", B=3, lo=17, hi=150, mix=5, page=16),
        # One long prompt.
        _case(name="prefill_8192_bf16", kind="prefill", dtype="bf16", lo=8192, hi=8192),
        # Chunks of four prompts over what is cached of them already, scores capped.
        _case(name="prefill_chunks_cap", kind="prefill", B=4, lo=300, hi=1100, mix=6, ctx=6000, page=32, softcap=50.0),
        # A batch behind one system prompt, each sequence with up to a few hundred tokens of its own.
        _case(name="prefix_b64_p8192", kind="prefix", B=64, lo=10, hi=600, mix=7, prefix=8192),
        # A few users behind a shorter prefix that ends inside a page.
        _case(name="prefix_b6_p1500_bf16", kind="prefix", dtype="bf16", H=40, B=6, lo=3, hi=200, mix=8, page=16,
              prefix=1500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append_step", "append_prompt", "decode", "decode", "decode", "prefill", "prefill", "prefill",
                       "prefix", "prefix"])
    H, Hkv = rng.choice(HEADS)
    c = _case(kind=kind, dtype=rng.choice(["fp16", "bf16"]), D=rng.choice([128, 128, 64]), H=H, Hkv=Hkv,
              page=rng.choice(PAGES), mix=rng.randint(10, 10 ** 6))
    if kind == "append_step":
        c.update(B=_log(rng, 1, 256), lo=1, hi=_log(rng, 50, 600))
    elif kind == "append_prompt":
        c["B"] = rng.randint(1, 8)
        c["hi"] = _log(rng, 20, 8192 // c["B"])
        c["lo"] = rng.randint(1, c["hi"])
    elif kind == "decode":
        c["B"] = _log(rng, 1, 64)
        # no more cache than the largest listed one (64 x 8 x 8192 token rows)
        c["hi"] = _log(rng, 60, min(60000, 64 * 8 * 8192 // (c["B"] * Hkv) // 2))
        c["lo"] = rng.choice([c["hi"], rng.randint(1, c["hi"])])
    elif kind == "prefill":
        c["B"] = rng.choice([1, 1, 2, 3, 4, 6])
        c["hi"] = _log(rng, 4, 6000 // c["B"])
        c["lo"] = rng.randint(1, c["hi"])
        c["ctx"] = rng.choice([0, 0, _log(rng, 10, 5000)])
    else:
        c["B"] = _log(rng, 2, 96)
        c["prefix"] = _log(rng, 200, 8192)
        c["lo"], c["hi"] = 1, _log(rng, 4, 500)
    if kind in ("append_step", "decode") and c["B"] >= 8:
        c["pad"] = rng.choice([0, 1, c["B"] // 8])
    if kind in ("decode", "prefill", "prefix"):
        more = rng.choice(["", "", "softcap", "slopes", "window", "all"])
        if more in ("softcap", "all"):
            c["softcap"] = rng.choice([20.0, 30.0, 50.0])
        if more in ("slopes", "all"):
            c["slopes"] = True
        if more in ("window", "all"):
            c["window"] = _log(rng, 16, 4096)
    return c


def _shape(case):
    """(new tokens, cached tokens before them) of every sequence; one new token each where the call decodes."""
    rng = random.Random(case["mix"])
    n = [case["hi"] if case["lo"] == case["hi"] else _log(rng, case["lo"], case["hi"]) for _ in range(case["B"])]
    if case["kind"] in ("append_prompt", "prefill"):
        before = [rng.randint(1, case["ctx"]) if case["ctx"] else 0 for _ in n]
        return n, before
    live = case["B"] - case["pad"]
    return [1] * live, [case["prefix"] + t - 1 for t in n[:live]]


# ------------------------------------------------------------------ inputs

def _slopes(H):
    """The slopes of a distance bias: 2^-8/H, 2^-16/H, ... 2^-8."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hkv, D, ps, prefix = (case[n] for n in ("B", "H", "Hkv", "D", "page", "prefix"))
    dt = DTYPES[case["dtype"]]
    new, before = _shape(case)
    lens = [a + b for a, b in zip(new, before)]
    prompt = case["kind"] in ("append_prompt", "prefill")

    # Pages: those that lie wholly in the prefix are shared, the rest are each sequence's own, in any order.
    shared = prefix // ps
    need = [-(-n // ps) for n in lens]
    n_pages = shared + (1 if prefix % ps else 0) + sum(n - shared for n in need) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").int()
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    table[:len(need), :shared] = order[:shared]
    at = shared
    prefix_pages = None
    if prefix:
        prefix_pages = order[:-(-prefix // ps)].contiguous()
        at = prefix_pages.numel()
    for b, n in enumerate(need):
        table[b, shared:n] = order[at:at + n - shared]
        at += n - shared

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    st = {"case": case, "page_table": table, "prefix_pages": prefix_pages, "scale": 1.0 / math.sqrt(D),
          "slopes": _slopes(H) if case["slopes"] else None, "cu": None, "longest": max(lens), "chunk": max(new),
          "rows": sum(new), "n_pages": n_pages}
    st["seq_lens"] = torch.tensor(lens + [0] * (B - len(lens)), dtype=torch.int32, device="cuda")
    if prompt:
        st["cu"] = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    rows = sum(new) if prompt else B
    st["k"] = torch.empty(n_pages, Hkv, ps, D, device="cuda", dtype=dt).normal_(generator=gen)
    st["v"] = torch.empty(n_pages, Hkv, ps, D, device="cuda", dtype=dt).normal_(generator=gen)
    if case["kind"].startswith("append"):
        st["qkv"] = normal(rows, (H + 2 * Hkv) * D)
        # the tables of the positions that the model serves, rounded to its type where that is fp16
        ang = torch.arange(max(lens) + 64, device="cuda", dtype=torch.float64)[:, None] / (
            500000.0 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))[None]
        ang = torch.cat([ang, ang], dim=1)
        kept = torch.float16 if case["dtype"] == "fp16" else torch.float32
        st["cos"], st["sin"] = ang.cos().to(kept), ang.sin().to(kept)
    else:
        st["q"] = 2.0 * normal(rows, H, D)   # scores of a spread that a cap and a softmax meet
    return st


# ------------------------------------------------------------------ the operators

def _append_plain(st):
    c, qkv, cu, lens, n = st["case"], st["qkv"], st["cu"], st["seq_lens"].long(), st["rows"]
    H, Hkv, D, ps = c["H"], c["Hkv"], c["D"], c["page"]
    row = torch.arange(n, device="cuda")
    if cu is None:
        seq, pos = row, lens[:n] - 1
    else:
        seq = torch.searchsorted(cu[1:].long(), row, right=True)
        pos = lens[seq] - cu[1:].long()[seq] + row
    x = qkv[:n].float().view(n, H + 2 * Hkv, D)
    rot, v = x[:, :H + Hkv], x[:, H + Hkv:]
    cos, sin = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]
    rot = (rot * cos + torch.cat([-rot[..., D // 2:], rot[..., :D // 2]], dim=-1) * sin).to(qkv.dtype)
    page = st["page_table"][seq, pos // ps].long()
    st["k"][page, :, pos % ps] = rot[:, H:]
    st["v"][page, :, pos % ps] = v.to(qkv.dtype)
    q = torch.zeros(qkv.shape[0], H, D, dtype=qkv.dtype, device="cuda")
    q[:n] = rot[:, :H]
    return q, st["k"], st["v"]


def _gather(cache, pages):
    """[..., n] page numbers -> [..., Hkv, n * page, D] in fp32 (unmapped pages: any, they are masked)."""
    x = cache[pages.long().clamp(min=0)].transpose(-4, -3)
    return x.reshape(*x.shape[:-3], -1, x.shape[-1]).float()


def _scores(st, s, pos_q, pos_k, seen):
    """Scaled scores with the cap, the distance bias and the mask. s [B, Hkv, G, L, S]; pos_q [B, L], pos_k [S];
    seen: the mask so far, [B, 1, 1, L, S]."""
    c = st["case"]
    s = s * st["scale"]
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    dist = (pos_q[:, None, None, :, None] - pos_k).float()
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, c["Hkv"], -1, 1, 1) * dist
    seen = seen & (dist >= 0)
    if c["window"]:
        seen = seen & (dist < c["window"])
    return s.masked_fill(~seen, -math.inf)


def _softmax(s):
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _attention_plain(st, q, pos_q, klen):
    """q [B, L, H, D] at positions pos_q [B, L] over each sequence's first klen [B] tokens."""
    c = st["case"]
    B, L, H, D = q.shape
    Hkv, G = c["Hkv"], c["H"] // c["Hkv"]
    qh = q.float().view(B, L, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * L, D)
    own_from = st["prefix_pages"].numel() - (c["prefix"] % c["page"] > 0) if c["prefix"] else 0
    pages = st["page_table"][:, own_from:-(-st["longest"] // c["page"])]
    k, v = _gather(st["k"], pages), _gather(st["v"], pages)
    pos_k = torch.arange(k.shape[2], device="cuda") + own_from * c["page"]
    live = (pos_k < klen[:, None, None, None, None]) & (pos_k >= c["prefix"])
    s = torch.matmul(qh, k.transpose(2, 3).contiguous()).view(B, Hkv, G, L, -1)
    s = _scores(st, s, pos_q, pos_k, live)
    if c["prefix"]:
        kp, vp = _gather(st["k"], st["prefix_pages"]), _gather(st["v"], st["prefix_pages"])   # [Hkv, P, D]
        pos_p = torch.arange(kp.shape[1], device="cuda")
        sp = torch.matmul(qh.transpose(0, 1).reshape(Hkv, -1, D), kp.transpose(1, 2).contiguous())
        sp = sp.view(Hkv, B, G, L, -1).transpose(0, 1)
        sp = _scores(st, sp, pos_q, pos_p, (pos_p < klen[:, None, None, None, None]) & (pos_p < c["prefix"]))
        p = _softmax(torch.cat([sp, s], dim=-1))
        pp, p = p[..., :kp.shape[1]], p[..., kp.shape[1]:]
        o = torch.matmul(pp.transpose(0, 1).reshape(Hkv, B * G * L, -1), vp).view(Hkv, B, G * L, D).transpose(0, 1)
        o = o + torch.matmul(p.reshape(B, Hkv, G * L, -1), v)
    else:
        o = torch.matmul(_softmax(s).view(B, Hkv, G * L, -1), v)
    return o.view(B, Hkv, G, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H, D).to(q.dtype)


def _prefill_plain(st):
    q, cu, lens = st["q"], st["cu"].long(), st["seq_lens"].long()
    n = cu[1:] - cu[:-1]
    at = torch.arange(st["chunk"], device="cuda")
    rows = (cu[:-1, None] + at).clamp(max=q.shape[0] - 1)
    out = _attention_plain(st, q[rows], (lens - n)[:, None] + at, lens)
    row = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    return out[seq, row - cu[seq]]


def run(st):
    c = st["case"]
    kind = c["kind"]
    if not own:
        if kind.startswith("append"):
            return _append_plain(st)
        if kind == "prefill":
            return _prefill_plain(st)
        lens = st["seq_lens"].long()
        return _attention_plain(st, st["q"][:, None], lens[:, None] - 1, lens)[:, 0]
    llmik = _own()
    if kind.startswith("append"):
        q = llmik.rope_paged_append(st["qkv"], st["cos"], st["sin"], st["k"], st["v"], st["page_table"],
                                    st["seq_lens"], st["cu"])
        return q, st["k"], st["v"]
    mods = dict(softcap=c["softcap"], slopes=st["slopes"], window=c["window"])
    if kind == "decode":
        return llmik.paged_decode_attention(st["q"], st["k"], st["v"], st["page_table"], st["seq_lens"],
                                            st["scale"], **mods)
    if kind == "prefill":
        return llmik.paged_prefill_attention(st["q"], st["k"], st["v"], st["page_table"], st["seq_lens"], st["cu"],
                                             st["scale"], **mods)
    return llmik.paged_shared_prefix_attention(st["q"], st["k"], st["v"], st["page_table"], st["seq_lens"],
                                               st["prefix_pages"], c["prefix"], st["scale"], **mods)


def _own():
    pkg = os.path.join(os.getcwd(), "llm-inference-kernels_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import llmik_cuda
    return llmik_cuda


# ------------------------------------------------------------------ the work

def work(case):
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    new, before = _shape(case)
    rows = sum(new)
    if case["kind"].startswith("append"):
        table = 2 if case["dtype"] == "fp16" else 4
        positions = len({b + i for n, b in zip(new, before) for i in range(n)})
        return {"bytes": 2 * 2 * rows * (H + 2 * Hkv) * D + 2 * table * positions * D,
                "flops": 3 * rows * (H + Hkv) * D}
    w = case["window"] or 1 << 60
    pairs = sum(min(b + i + 1, w) for n, b in zip(new, before) for i in range(n))     # (row, key) pairs
    # tokens of the cache that some row of each sequence sees: from the first row's oldest key on
    spans = [(max(0, b + 1 - w), b + n) for n, b in zip(new, before)]
    P = case["prefix"]
    tokens = sum(e - max(s, P) for s, e in spans if e > max(s, P))
    if P:
        tokens += max(0, P - min(s for s, _ in spans))
    return {"bytes": 2 * 2 * tokens * Hkv * D + 2 * 2 * rows * H * D, "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------ in 64 bits

def _exact_append(st):
    c, dt = st["case"], st["qkv"].dtype
    H, Hkv, D, ps = c["H"], c["Hkv"], c["D"], c["page"]
    new, before = _shape(c)
    k, v = st["k"].double(), st["v"].double()
    q = torch.zeros(st["qkv"].shape[0], H, D, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, have) in enumerate(zip(new, before)):
        x = st["qkv"][at:at + n].double().view(n, H + 2 * Hkv, D)
        pos = torch.arange(have, have + n, device="cuda")
        cos, sin = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
        lo, hi = x[:, :H + Hkv, :D // 2], x[:, :H + Hkv, D // 2:]
        h = D // 2
        turned = torch.cat([lo * cos[..., :h] - hi * sin[..., :h], hi * cos[..., h:] + lo * sin[..., h:]], dim=-1)
        q[at:at + n] = turned[:, :H]
        slot = st["page_table"][b][pos // ps].long() * ps + pos % ps
        for cache, rows in ((k, turned[:, H:]), (v, x[:, H + Hkv:])):
            flat = cache.transpose(1, 2).reshape(-1, Hkv, D)
            flat[slot] = rows
            cache.copy_(flat.view(-1, ps, Hkv, D).transpose(1, 2))
        at += n
    return q, k, v


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"].startswith("append"):
        return _exact_append(st)
    H, Hkv, D, ps = case["H"], case["Hkv"], case["D"], case["page"]
    G = H // Hkv
    new, before = _shape(case)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, have) in enumerate(zip(new, before)):
        total = have + n
        pages = st["page_table"][b, :-(-total // ps)].long()
        k = st["k"][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :total]
        v = st["v"][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :total]
        if case["prefix"]:
            shared = st["prefix_pages"].long()
            k, v = k.clone(), v.clone()
            k[:, :case["prefix"]] = st["k"][shared].transpose(0, 1).reshape(Hkv, -1, D)[:, :case["prefix"]]
            v[:, :case["prefix"]] = st["v"][shared].transpose(0, 1).reshape(Hkv, -1, D)[:, :case["prefix"]]
        dist = torch.arange(have, total, device="cuda")[:, None] - torch.arange(total, device="cuda")
        hidden = dist < 0
        if case["window"]:
            hidden = hidden | (dist >= case["window"])
        for h in range(H):
            s = st["q"][at:at + n, h].double() @ k[h // G].double().t().contiguous() * st["scale"]
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            if case["slopes"]:
                s = s - st["slopes"][h].double() * dist
            s = s.masked_fill(hidden, -math.inf)
            out[at:at + n, h] = torch.softmax(s, dim=-1) @ v[h // G].double()
        at += n
    return out
