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
            lambda: lib.llmik_paged_decode_attention_weights(_at(c), 16, 16, 4, _at(o), _at(w), ws, n, None),
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
        assert lib.llmik_paged_decode_weights_workspace_size(_at(c), 4, _at(bad)) == 0


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

    need = lib.llmik_paged_decode_weights_workspace_size(_at(c), 4, _at(w))
    assert need > lib.llmik_paged_workspace_size(_at(c), 4, 0)
    decode = lambda q=16, out=16, ws=16, n=need: lib.llmik_paged_decode_attention_weights(   # noqa: E731
        _at(c), q, out, 4, _at(o), _at(w), ws, n, None)
    assert decode(n=need - 1) == WORKSPACE and decode(ws=None) == WORKSPACE
    assert decode(q=None) == INVALID and decode(out=24) == ALIGNMENT
    assert lib.llmik_paged_decode_attention_weights(_at(c), 16, 16, 4, _at(o), None, 16, need, None) == INVALID

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
