"""CPU: the paged cache's refusals, in the C layer and the Python ops, and
PagedKVCache's bookkeeping. No compute entry point is called with valid
arguments here."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from tests import helpers  # noqa: F401

H16, BF = torch.float16, torch.bfloat16
I32 = torch.int32


@pytest.fixture(scope="module")
def mod():
    import llmik_cuda
    return llmik_cuda


@pytest.fixture(scope="module")
def lib(mod):
    from llmik_cuda._lib import lib
    return lib


@pytest.fixture
def as_device(mod, monkeypatch):
    monkeypatch.setattr(mod, "_is_device", lambda t: True)
    return mod


def _cache(**more):
    from llmik_cuda._lib import PagedCache
    c = dict(k=16, v=16, page_table=16, seq_lens=16, page_stride=0, n_pages=4, page_size=16, max_pages=2, batch=2,
             n_kv_heads=2, head_dim=128, dtype=0)
    c.update(more)
    return PagedCache(**c)


def _options(**more):
    from llmik_cuda._lib import ScoreOptions
    c = dict(softmax_scale=0.1, softcap=0.0, slopes=None, window=0)
    c.update(more)
    return ScoreOptions(**c)


def _at(struct):
    return ctypes.addressof(struct)


INVALID, UNSUPPORTED, WORKSPACE, ALIGNMENT = -1, -2, -3, -4

CACHES = [
    (dict(head_dim=96), INVALID, "head_dim=64 and 128"),
    (dict(dtype=2), INVALID, "dtype must be"),
    (dict(n_kv_heads=0), INVALID, "head counts must be positive"),
    (dict(n_kv_heads=3), INVALID, "multiple of n_kv_heads"),
    (dict(page_size=0), INVALID, "positive multiple of 8"),
    (dict(page_size=12), INVALID, "positive multiple of 8"),
    (dict(page_size=1 << 21), UNSUPPORTED, "page_size above"),
    (dict(n_pages=0), INVALID, "no pages"),
    (dict(batch=-1), INVALID, "batch must be"),
    (dict(max_pages=0), INVALID, "at least one column"),
    (dict(page_stride=2 * 16 * 128 - 8), INVALID, "page_stride"),
    (dict(page_stride=2 * 16 * 128 + 4), INVALID, "page_stride"),
    (dict(batch=1 << 20, max_pages=1 << 20), UNSUPPORTED, "capacity too large"),
    (dict(k=None), INVALID, "null cache pointer"),
    (dict(page_table=None), INVALID, "null cache pointer"),
    (dict(v=24), ALIGNMENT, "k and v must be 16-byte"),
    (dict(seq_lens=18), ALIGNMENT, "4-byte"),
]


@pytest.mark.parametrize("case", CACHES, ids=lambda c: str(c[0]))
def test_c_layer_refuses_caches(lib, case):
    more, code, msg = case
    c, o = _cache(**more), _options()
    calls = [lambda: lib.llmik_rope_paged_append(_at(c), 16, 16, 16, 8, 0, 16, 16, 2, 4, None),
             lambda: lib.llmik_paged_decode_attention(_at(c), 16, 16, 4, _at(o), 16, 0, None),
             lambda: lib.llmik_paged_prefill_attention(_at(c), 16, 16, 16, 2, 4, _at(o), None, 0, None),
             lambda: lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 1, 5, _at(o), 16, 0, None)]
    for call in calls:
        assert call() == code and msg in lib.llmik_last_error().decode()


def test_c_layer_refuses_arguments(lib):
    c, o = _cache(), _options()
    err = lambda: lib.llmik_last_error().decode()   # noqa: E731
    append = lambda **a: lib.llmik_rope_paged_append(*{**dict(   # noqa: E731
        c=_at(c), qkv=16, cos=16, sin=16, n=8, f32=0, cu=16, q=16, rows=2, heads=4, stream=None), **a}.values())
    for a, code, msg in [(dict(c=None), INVALID, "null cache"), (dict(rows=-1), INVALID, "rows must be"),
                         (dict(cu=None, rows=3), INVALID, "one row per sequence"),
                         (dict(sin=None), INVALID, "come together"), (dict(n=-1), INVALID, "table_rows"),
                         (dict(qkv=None), INVALID, "null qkv"), (dict(q=8), ALIGNMENT, "16-byte"),
                         (dict(cos=20), ALIGNMENT, "16-byte"), (dict(cu=18), ALIGNMENT, "4-byte"),
                         (dict(rows=1 << 30), UNSUPPORTED, "too many rows")]:
        assert append(**a) == code and msg in err(), a
    for more, msg in [(dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"),
                      (dict(softcap=float("inf")), "softcap"), (dict(softcap=4097.0), "softcap"),
                      (dict(softcap=1e-38, softmax_scale=100.0), "softcap too small"), (dict(softmax_scale=float("nan")), "softmax_scale"),
                      (dict(softmax_scale=float("inf")), "softmax_scale"), (dict(window=-1), "window")]:
        bad = _options(**more)
        assert lib.llmik_paged_decode_attention(_at(c), 16, 16, 4, _at(bad), 16, 0, None) == INVALID and msg in err()
        assert lib.llmik_paged_prefill_attention(_at(c), 16, 16, 16, 2, 4, _at(bad), None, 0, None) == INVALID
        assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 1, 5, _at(bad), 16, 0, None) == INVALID
    assert lib.llmik_paged_decode_attention(_at(c), 16, 16, 4, None, 16, 0, None) == INVALID
    assert lib.llmik_paged_decode_attention(_at(c), None, 16, 4, _at(o), 16, 0, None) == INVALID
    assert lib.llmik_paged_decode_attention(_at(c), 24, 16, 4, _at(o), 16, 0, None) == ALIGNMENT
    assert lib.llmik_paged_decode_attention(_at(c), 16, 16, 5, _at(o), 16, 0, None) == INVALID
    # workspaces that are missing or too small
    need = lib.llmik_paged_workspace_size(_at(c), 4, 0)
    assert need > 16384
    assert lib.llmik_paged_decode_attention(_at(c), 16, 16, 4, _at(o), None, need, None) == WORKSPACE
    assert lib.llmik_paged_decode_attention(_at(c), 16, 16, 4, _at(o), 16, need - 1, None) == WORKSPACE
    more = lib.llmik_paged_workspace_size(_at(c), 4, 16)
    assert more > need
    assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 1, 16, _at(o), 16, need, None) == WORKSPACE
    long = _cache(max_pages=1000)
    parts = lib.llmik_paged_prefill_workspace_size(_at(long), 4, 2)
    assert parts > 16384
    assert lib.llmik_paged_prefill_attention(_at(long), 16, 16, 16, 2, 4, _at(o), 16, parts - 1, None) == WORKSPACE
    assert lib.llmik_paged_prefill_workspace_size(_at(c), 4, 2) == 0        # too few tokens to cut
    assert lib.llmik_paged_prefill_workspace_size(_at(long), 4, 1 << 20) == 0   # rows for every workgroup
    # prompts and prefixes
    assert lib.llmik_paged_prefill_attention(_at(c), 16, None, 16, 2, 4, _at(o), None, 0, None) == INVALID
    assert lib.llmik_paged_prefill_attention(_at(c), 16, 16, 16, -2, 4, _at(o), None, 0, None) == INVALID
    assert lib.llmik_paged_prefill_attention(_at(c), 16, 16, 16, 1 << 30, 4, _at(o), None, 0, None) == UNSUPPORTED
    assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 1, 17, _at(o), 16, more, None) == INVALID
    assert "fewer than prefix_len" in err()
    assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, None, 1, 9, _at(o), 16, more, None) == INVALID
    assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 1, -1, _at(o), 16, more, None) == INVALID


def test_workspace_sizes_do_not_depend_on_lengths_and_fit_the_counters(lib):
    """One counter per workgroup lies in the workspace's zeroed region; the parts
    are two slots per workgroup, whatever the table's capacity."""
    small, large = _cache(batch=8, max_pages=1000), _cache(batch=8, max_pages=100000)
    assert lib.llmik_paged_workspace_size(_at(small), 16, 0) == lib.llmik_paged_workspace_size(_at(large), 16, 0)
    one = _cache(batch=1, max_pages=1)
    slots = 2 * 2 * 2 * 8      # two KV heads, at most two pieces each, two slots, 8 heads
    assert lib.llmik_paged_workspace_size(_at(one), 16, 0) <= 16384 + 256 + slots * 2 * 4 * 2 + slots * 128 * 4 * 2


# ---------------------------------------------------------------- the Python ops

def _t(*shape, dtype=H16):
    return torch.zeros(*shape, dtype=dtype)


def _args(**more):
    a = dict(q=_t(2, 4, 128), k=_t(3, 2, 16, 128), v=_t(3, 2, 16, 128), table=_t(2, 2, dtype=I32),
             lens=_t(2, dtype=I32), cu=_t(3, dtype=I32), prefix=_t(1, dtype=I32), plen=8, scale=0.1, softcap=0.0,
             slopes=None, window=0)
    a.update(more)
    return a


def _calls(m, a):
    opts = (a["scale"], a["softcap"], a["slopes"], a["window"])
    base = (a["q"], a["k"], a["v"], a["table"], a["lens"])
    return [lambda: m.paged_decode_attention(*base, *opts),
            lambda: m.paged_prefill_attention(*base, a["cu"], *opts),
            lambda: m.paged_shared_prefix_attention(*base, a["prefix"], a["plen"], *opts)]


@pytest.mark.parametrize("more,msg", [
    (dict(q=_t(2, 4, 128, dtype=torch.float32)), "q must be fp16 or bf16"),
    (dict(q=_t(2, 4, 128, dtype=BF)), "must have q's dtype"),
    (dict(v=_t(3, 2, 16, 128, dtype=BF)), "must have q's dtype"),
    (dict(table=_t(2, 2, dtype=torch.int64)), "must be int32"),
    (dict(lens=_t(2)), "must be int32"),
    (dict(k=_t(3, 2, 16, 64)), "of one shape"),
    (dict(k=_t(2, 16, 128), v=_t(2, 16, 128)), "of one shape"),
    (dict(lens=_t(3, dtype=I32)), "seq_lens"),
    (dict(table=_t(4, 2, dtype=I32)[::2]), "must be contiguous"),
    (dict(k=_t(0, 2, 16, 128), v=_t(0, 2, 16, 128)), "no pages"),
    (dict(k=_t(3, 2, 12, 128), v=_t(3, 2, 12, 128)), "multiple of 8"),
    (dict(k=_t(3, 2, 16, 32), v=_t(3, 2, 16, 32)), "head_dim=64 and 128"),
    (dict(k=_t(3, 16, 2, 128).transpose(1, 2), v=_t(3, 16, 2, 128).transpose(1, 2)), "pages must be contiguous"),
    (dict(k=_t(6, 2, 16, 128)[::2]), "one stride in k_cache"),
    (dict(table=_t(2, 0, dtype=I32)), "at least one column"),
    (dict(), "CUDA tensors of one device"),
])
def test_python_refuses_caches(as_device, more, msg):
    for call in _calls(as_device, _args(**more)):
        with pytest.raises(RuntimeError, match=msg):
            call()


def test_python_checks_devices_first(mod):
    for call in _calls(mod, _args()):
        with pytest.raises(RuntimeError, match="all inputs must be CUDA tensors"):
            call()
    with pytest.raises(RuntimeError, match="all inputs must be CUDA tensors"):
        mod.rope_paged_append(_t(2, 8 * 128), None, None, _t(3, 2, 16, 128), _t(3, 2, 16, 128), _t(2, 2, dtype=I32),
                              _t(2, dtype=I32))


# ------------------------------------------------------------ PagedKVCache, on the host

@pytest.fixture
def cache():
    from llmik_cuda.kv_cache import PagedKVCache
    return PagedKVCache(10, 2, page_size=8, head_dim=64, device="cpu")


def test_batches_reserve_pages_and_describe_them(cache):
    a, b = cache.add(), cache.add()
    step = cache.batch([a, b], [17, 3])
    assert step.seq_lens.tolist() == [17, 3] and step.cu_tokens.tolist() == [0, 17, 20] and step.rows == 20
    assert step.page_table.shape == (2, 3) and step.page_table[1, 1:].tolist() == [-1, -1]
    used = step.page_table[step.page_table >= 0].tolist()
    assert len(set(used)) == 4 and cache.free_pages() == 6
    step = cache.batch([b, a])
    assert step.seq_lens.tolist() == [4, 18] and step.cu_tokens is None and step.rows == 2
    assert cache.free_pages() == 6 and step.prefix_pages is None
    step = cache.batch([a, b], [0, 5])
    assert step.cu_tokens.tolist() == [0, 0, 5] and cache.length(a) == 18 and cache.length(b) == 9
    assert cache.free_pages() == 5


def test_a_batch_that_does_not_fit_changes_nothing(cache):
    a, b = cache.add(), cache.add()
    cache.batch([a, b], [40, 30])
    with pytest.raises(RuntimeError, match="no free page"):
        cache.batch([a, b], [8, 9])
    assert cache.length(a) == 40 and cache.length(b) == 30 and cache.free_pages() == 1
    for bad, msg in [(([a, a],), "twice"), (([a, 77],), "no such"), (([a], [-1]), "counts"), (([a], [1, 2]), "one count")]:
        with pytest.raises(RuntimeError, match=msg):
            cache.batch(*bad)
    assert cache.length(a) == 40


def test_sharing_and_removal(cache):
    a = cache.add()
    first = cache.batch([a], [20]).page_table[0].tolist()
    cache.k[0, first[2], :, :4] = 3.0
    b = cache.add(share=a, tokens=18)
    assert cache.length(b) == 18 and cache.free_pages() == 6
    step = cache.batch([a, b])
    rows = step.page_table.tolist()
    assert rows[0][:2] == rows[1][:2] and rows[0][2] != rows[1][2]
    assert bool((cache.k[0, rows[1][2], :, :2] == 3.0).all()) and bool((cache.k[0, rows[1][2], :, 2:] == 0.0).all())
    cache.remove(a)
    assert cache.free_pages() == 7        # the two shared pages are still b's
    cache.remove(b)
    assert cache.free_pages() == 10
    with pytest.raises(RuntimeError, match="no such"):
        cache.remove(b)
    with pytest.raises(RuntimeError, match="no such"):
        cache.add(share=a)
    c = cache.add()
    with pytest.raises(RuntimeError, match="fewer tokens"):
        cache.add(share=c, tokens=1)


def test_a_fork_copies_the_last_page_in_every_layer():
    from llmik_cuda.kv_cache import PagedKVCache
    cache = PagedKVCache(6, 2, page_size=8, head_dim=64, device="cpu", n_layers=3)
    a = cache.add()
    src = cache.batch([a], [12]).page_table[0, 1]
    cache.k.normal_()
    cache.v.normal_()
    b = cache.add(share=a, tokens=11)
    dst = cache.batch([b]).page_table[0, 1]
    assert dst != src
    assert torch.equal(cache.k[:, dst, :, :3], cache.k[:, src, :, :3])
    assert torch.equal(cache.v[:, dst, :, :3], cache.v[:, src, :, :3])


def test_a_batch_knows_its_shared_prefix(cache):
    cache.SHARED_TOKENS, cache.SHARED_ROWS = 24, 2 * 24 * 2
    a = cache.add()
    cache.batch([a], [24])
    seqs = [a] + [cache.add(share=a, tokens=24) for _ in range(2)]
    step = cache.batch(seqs)
    assert step.prefix_len == 24 and step.prefix_pages.tolist() == step.page_table[0, :3].tolist()
    assert cache.batch([a]).prefix_pages is None                       # one sequence
    assert cache.batch(seqs, [2, 1, 1]).prefix_pages is None           # prompts
    other = cache.add()
    cache.batch([other], [5])
    assert cache.batch(seqs + [other]).prefix_len == 0                 # nothing in common
    cache.SHARED_ROWS += 1
    assert cache.batch(seqs).prefix_pages is None                      # too few rows to pay
    cache.SHARED_TOKENS, cache.SHARED_ROWS = 25, 2 * 24 * 2 // 16
    assert cache.batch(seqs).prefix_len == 24                          # few tokens, many rows
    cache.SHARED_ROWS += 1
    assert cache.batch(seqs).prefix_pages is None


def test_pages_are_never_lost_or_given_twice():
    """Random adds, forks, batches and removals: every page is free or held by as
    many sequences as count it, and only whole shared pages are held twice."""
    from llmik_cuda.kv_cache import PagedKVCache
    rng = random.Random(5)
    cache = PagedKVCache(40, 1, page_size=8, head_dim=64, device="cpu")
    live = []
    for _ in range(600):
        what = rng.random()
        try:
            if what < 0.2:
                live.append(cache.add())
            elif what < 0.35 and live:
                s = rng.choice(live)
                live.append(cache.add(share=s, tokens=rng.randint(0, cache.length(s))))
            elif what < 0.5 and live:
                cache.remove(live.pop(rng.randrange(len(live))))
            elif live:
                some = rng.sample(live, rng.randint(1, len(live)))
                cache.batch(some, [rng.randint(0, 20) for _ in some])
        except RuntimeError as e:
            assert "no free page" in str(e)
        held = [p for s in live for p in cache._pages[s]]
        assert len(set(held)) + cache.free_pages() == 40 and not set(held) & set(cache._free)
        assert all(held.count(p) == cache._users[p] for p in set(held))
        assert all(len(cache._pages[s]) == -(-cache.length(s) // 8) for s in live)


def test_a_window_decides_whether_the_prefix_is_read_once(monkeypatch):
    """What counts is what the window leaves of the shared prefix."""
    import llmik_cuda.kv_cache as kv
    taken = []
    monkeypatch.setattr(kv, "paged_decode_attention", lambda *a: taken.append(("decode", a[3], a[-1])))
    monkeypatch.setattr(kv, "paged_shared_prefix_attention", lambda *a: taken.append(("shared", a[3], a[-1])))
    cache = kv.PagedKVCache(600, 8, page_size=64, head_dim=64, device="cpu")
    a = cache.add()
    cache.batch([a], [8192])
    seqs = [a] + [cache.add(share=a, tokens=8192) for _ in range(63)]
    step = cache.batch(seqs)
    assert step.prefix_len == 8192 and step.shortest == 8193 and step.mean == 8193

    def path(step, window):
        cache.attention(step, None, 0.1, window=window)
        kind, table, w = taken.pop()
        assert w == window and table is step.page_table and bool((table[:, :128] >= 0).all())
        return kind

    assert path(step, 0) == "shared"
    for window, want in [(1, "decode"), (64, "decode"), (256, "decode"), (512, "decode"), (1024, "shared"),
                         (8192, "shared"), (10 ** 6, "shared")]:
        assert path(step, window) == want, window
    # sequences that have left the prefix behind see none of it; one short one among them changes little
    long = cache.batch(seqs[1:40], [300] * 39)
    assert long.prefix_pages is None                                    # prompts
    mixed = cache.batch(seqs[:40])
    assert mixed.shortest == 8194 and mixed.mean == 8194 + 39 * 300 // 40
    assert path(mixed, 280) == "decode" and path(mixed, 1024) == "shared"
    # a batch without the lengths (made by hand) counts the whole prefix
    assert path(step._replace(shortest=0, mean=0), 2048) == "shared"


def test_decode_for_all_batches():
    """shared_prefix=False: no batch is read through the shared prefix, whose
    probabilities have fewer bits."""
    from llmik_cuda.kv_cache import PagedKVCache
    for share in (True, False):
        cache = PagedKVCache(300, 8, page_size=64, head_dim=64, device="cpu", shared_prefix=share)
        a = cache.add()
        cache.batch([a], [8192])
        step = cache.batch([a] + [cache.add(share=a, tokens=8192) for _ in range(9)])
        assert (step.prefix_pages is not None) == share and step.prefix_len == (8192 if share else 0)


@pytest.mark.parametrize("more,msg", [
    (dict(softcap=1e-50), "softcap too small"), (dict(softcap=5e-46), "softcap too small"),
    (dict(softcap=-1e-50), "softcap must be"), (dict(softcap=float("nan")), "softcap must be"),
    (dict(softcap=4096.5), "softcap must be"), (dict(scale=1e39), "softmax_scale"),
    (dict(scale=float("nan")), "softmax_scale"), (dict(window=-1), "window"), (dict(window=1 << 31), "window"),
], ids=str)
def test_python_refuses_numbers(as_device, more, msg):
    """Before anything of the tensors is looked at; a cap that fp32 cannot hold is refused,
    not taken for none."""
    for call in _calls(as_device, _args(**more)):
        with pytest.raises(RuntimeError, match=msg):
            call()


def test_workspace_sizes_are_0_for_what_the_calls_refuse(lib):
    c, o = _cache(), _options()
    for prefix, code in [(-1, INVALID), (-2 ** 31, INVALID), ((1 << 30) + 1, UNSUPPORTED), (2 ** 31 - 64, UNSUPPORTED),
                         (2 ** 31 - 1, UNSUPPORTED)]:
        assert lib.llmik_paged_workspace_size(_at(c), 4, prefix) == 0, prefix
        assert lib.llmik_paged_shared_prefix_attention(_at(c), 16, 16, 4, 16, 2 ** 31 - 1, prefix, _at(o), 16, 1 << 60,
                                                       None) == code, prefix
    # rows that no launch holds: with a prefix only
    many = _cache(batch=1 << 20, max_pages=1, n_kv_heads=1)
    assert lib.llmik_paged_workspace_size(_at(many), 512, 16) == 0
    assert lib.llmik_paged_shared_prefix_attention(_at(many), 16, 16, 512, 16, 1, 16, _at(o), 16, 1 << 60,
                                                   None) == UNSUPPORTED
    assert lib.llmik_paged_workspace_size(_at(many), 512, 0) > 0
    # what is accepted: sizes that hold a part of every row, and for the longest prefix
    sizes = [lib.llmik_paged_workspace_size(_at(c), 4, n) for n in (0, 1, 64, 8192, 1 << 30)]
    assert 0 < sizes[0] < sizes[1] <= sizes[2] <= sizes[3] <= sizes[4] < 1 << 24
    for bad in (dict(head_dim=96), dict(page_size=12), dict(batch=-1)):
        assert lib.llmik_paged_workspace_size(_at(_cache(**bad)), 4, 16) == 0
        assert lib.llmik_paged_prefill_workspace_size(_at(_cache(**bad)), 4, 16) == 0
    assert lib.llmik_paged_prefill_workspace_size(_at(c), 4, -1) == 0
    assert lib.llmik_paged_prefill_workspace_size(_at(c), 4, 2 ** 31 - 1) == 0


@pytest.mark.parametrize("page,tiles", [(8, 1), (32, 1), (40, 2), (64, 2)])
def test_the_work_of_all_sequences_fits_32_bits(lib, page, tiles):
    """A slab counts its 32-token tiles, the last one begun too, and six more."""
    most = (2 ** 31 - 2) // (tiles + 6)
    fits = _cache(batch=most, max_pages=1, page_size=page, n_kv_heads=1)
    over = _cache(batch=most + 1, max_pages=1, page_size=page, n_kv_heads=1)
    o = _options()
    assert lib.llmik_paged_workspace_size(_at(fits), 1, 0) > 0
    assert lib.llmik_paged_workspace_size(_at(over), 1, 0) == 0
    assert lib.llmik_paged_decode_attention(_at(over), 16, 16, 1, _at(o), 16, 1 << 60, None) == UNSUPPORTED
