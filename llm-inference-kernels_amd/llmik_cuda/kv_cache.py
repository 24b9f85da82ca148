"""Cat-free quantised KV caches: preallocated buffers appended in place.

The reference keeps its INT4 KIVI cache as a list of packed chunks that it
torch.cat's onto the whole cache whenever a group of tokens is drained and
again, with the freshly quantised fp16 residual, before every decode-step
attention call (Int4KIVICache.append_only / get_quantized_for_attention,
integration/kv_int4_cache.py:104-144,168-206). Here the cache is one
preallocated buffer per tensor of capacity `max_len`; appends quantise
straight into it at the live offset (the *_into writers) and attention reads
it in place over the live length (`seqlen`). The stored codes and scales are
bit-identical to the reference cache's view after the same appends:

* Int4KIVICache: K per channel grouped along the sequence (full groups
  quantised once, from the same fp16 tokens the reference drains), the
  trailing partial group -- the reference's fp16 residual -- re-quantised on
  every append from the fp16 tokens kept here, exactly as the reference
  re-quantises its residual before each attention call; V per token.
* Int8KVCache: K and V per token (the INT8 path of the reference has no
  cache class; this is its prealloc_cache.PreallocCache layout,
  integration/prealloc_cache.py:42-79, in INT8).

PagedKVCache keeps fp16 or bf16 tokens of many sequences, each of its own
length, in one pool of pages; it drafts and accepts token trees, and, where it
records the tokens' attention weights, cuts sequences down to those that have
had the most (the reference has no counterpart).
"""
from __future__ import annotations

import warnings
from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import (_C, paged_compact, paged_decode_attention, paged_decode_attention_weights, paged_prefill_attention,
               paged_prefill_weights, paged_select_tokens, paged_shared_prefix_attention, paged_tree_attention,
               quantize_k_per_channel_groupwise_int4_into, quantize_per_token_into, quantize_v_per_token_int4_into,
               rope_paged_append)
# One-token steps at small batch are bound by the host: these three come from the
# extension, which checks types, shapes, strides and devices itself, rather
# than through the module's Python wrappers (a KIVI step of one token and
# attention, B=1 over 515 tokens, eager: 11.0 -> 9.4 us; 8.6 of it on the GPU).
from ._C import decode_attention_int4, decode_attention_int8, kivi_append_token_int4


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _check_append(k: torch.Tensor, v: torch.Tensor, batch: int, n_kv_heads: int, head_dim: int,
                  length: int, max_len: int) -> int:
    shape = k.shape
    if shape != v.shape or len(shape) != 4:
        raise RuntimeError("k and v must be [batch, n_kv_heads, n, head_dim]")
    if k.dtype != torch.float16 or v.dtype != torch.float16:
        raise RuntimeError("k and v must be fp16")
    b, h, n, d = shape
    if b != batch or h != n_kv_heads or d != head_dim:
        raise RuntimeError("k/v shape does not match the cache")
    if length + n > max_len:
        raise RuntimeError("append exceeds the cache capacity")
    return n


class Int8KVCache:
    """INT8 per-token K and V in preallocated [batch, n_kv_heads, max_len, ...]
    buffers; `append` quantises new tokens in place, `attention` runs the
    INT8 decode attention over the live length."""

    def __init__(self, batch: int, n_kv_heads: int, max_len: int, head_dim: int = 128,
                 device: Optional[torch.device] = None) -> None:
        dev = torch.device("cuda") if device is None else torch.device(device)
        self.batch, self.n_kv_heads, self.max_len, self.head_dim = batch, n_kv_heads, max_len, head_dim
        shape = (batch, n_kv_heads, max_len, head_dim)
        self.k_q = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.v_q = torch.zeros(shape, dtype=torch.int8, device=dev)
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float16, device=dev)
        self.v_scale = torch.zeros(shape[:3], dtype=torch.float16, device=dev)
        self.length = 0

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v [batch, n_kv_heads, n, head_dim] fp16."""
        n = _check_append(k, v, self.batch, self.n_kv_heads, self.head_dim, self.length,
                          self.max_len)
        if n == 0:
            return
        quantize_per_token_into(k, self.k_q, self.k_scale, self.length)
        quantize_per_token_into(v, self.v_q, self.v_scale, self.length)
        self.length += n

    def get_quantized_for_attention(self) -> Tuple[torch.Tensor, ...]:
        """(k_q, k_scale, v_q, v_scale, length): the whole buffers and the
        live length to pass as `seqlen`."""
        return self.k_q, self.k_scale, self.v_q, self.v_scale, self.length

    def attention(self, q: torch.Tensor, softmax_scale: float) -> torch.Tensor:
        """q [batch, n_heads, head_dim] fp16 over the live tokens."""
        _require(self.length > 0, "the cache is empty")
        return decode_attention_int8(q, self.k_q, self.k_scale, self.v_q, self.v_scale,
                                     float(softmax_scale), int(self.length))

    def reset(self) -> None:
        self.length = 0


class Int4KIVICache:
    """KIVI INT4 cache (K per channel in groups of `group_size` tokens along
    the sequence, V per token, packed two codes per byte) in preallocated
    buffers, with the fp16 tokens of the open (partial) K group kept for
    re-quantisation. Same stored codes and scales as the reference's
    Int4KIVICache after the same appends (see the module docstring)."""

    def __init__(self, batch: int, n_kv_heads: int, max_len: int, group_size: int = 32,
                 head_dim: int = 128, device: Optional[torch.device] = None) -> None:
        _require(group_size > 0, "group_size must be positive")
        dev = torch.device("cuda") if device is None else torch.device(device)
        self.batch, self.n_kv_heads, self.max_len = batch, n_kv_heads, max_len
        self.group_size, self.head_dim = group_size, head_dim
        n_groups = (max_len + group_size - 1) // group_size
        self.k_q = torch.zeros((batch, n_kv_heads, max_len, head_dim // 2), dtype=torch.int8,
                               device=dev)
        self.v_q = torch.zeros_like(self.k_q)
        self.k_scale = torch.zeros((batch, n_kv_heads, n_groups, head_dim), dtype=torch.float16,
                                   device=dev)
        self.v_scale = torch.zeros((batch, n_kv_heads, max_len), dtype=torch.float16, device=dev)
        # fp16 tokens of the open K group (positions group_start .. length-1)
        self.k_open = torch.zeros((batch, n_kv_heads, group_size, head_dim), dtype=torch.float16,
                                  device=dev)
        self.length = 0

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v [batch, n_kv_heads, n, head_dim] fp16."""
        n = _check_append(k, v, self.batch, self.n_kv_heads, self.head_dim, self.length,
                          self.max_len)
        if n == 0:
            return
        g = self.group_size
        if n == 1 and g <= 128 and self.head_dim == 128:
            # A decode step: one launch for the V token, the open group's new
            # fp16 token and its re-quantisation.
            kivi_append_token_int4(k, v, self.k_open, self.k_q, self.k_scale, self.v_q, self.v_scale,
                                   int(self.length), int(g))
            self.length += 1
            return
        if _C.kivi_append_int4(k, v, self.k_open, None, self.k_q, self.k_scale, self.v_q, self.v_scale,
                               self.length, g) is not None:
            self.length += n
            return
        quantize_v_per_token_int4_into(v, self.v_q, self.v_scale, self.length)
        pos = 0
        r = self.length % g
        if r:
            # Fill the open group and re-quantise it (still partial, or now full).
            take = min(g - r, n)
            self.k_open[:, :, r:r + take].copy_(k[:, :, :take])
            quantize_k_per_channel_groupwise_int4_into(
                self.k_open[:, :, :r + take], self.k_q, self.k_scale, self.length - r, g)
            pos = take
        full = (n - pos) // g * g
        if full:
            # Whole groups straight from the input.
            quantize_k_per_channel_groupwise_int4_into(
                k[:, :, pos:pos + full], self.k_q, self.k_scale, self.length + pos, g)
            pos += full
        rest = n - pos
        if rest:
            # A new open group.
            self.k_open[:, :, :rest].copy_(k[:, :, pos:])
            quantize_k_per_channel_groupwise_int4_into(
                self.k_open[:, :, :rest], self.k_q, self.k_scale, self.length + pos, g)
        self.length += n

    def append_with_view(self, k: torch.Tensor, v: torch.Tensor, v_open: torch.Tensor
                         ) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """append(k, v), and the cache's fp16 view from the same launch: K and
        V [batch, n_kv_heads, length, head_dim], fp16 code * scale of the full
        groups and the fp16 tokens of the open one. v_open [batch,
        n_kv_heads, group_size, head_dim] holds the open group's fp16 V tokens,
        as k_open does K's, and is kept up to date. None, with nothing done,
        where the launch does not take the call."""
        n = _check_append(k, v, self.batch, self.n_kv_heads, self.head_dim, self.length, self.max_len)
        views = _C.kivi_append_int4(k, v, self.k_open, v_open, self.k_q, self.k_scale, self.v_q, self.v_scale,
                                    self.length, self.group_size)
        if views is not None:
            self.length += n
        return views

    def view(self, v_open: torch.Tensor) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """The fp16 view alone (see append_with_view)."""
        return _C.kivi_append_int4(None, None, self.k_open, v_open, self.k_q, self.k_scale, self.v_q, self.v_scale,
                                   self.length, self.group_size)

    def get_quantized_for_attention(self) -> Tuple[torch.Tensor, ...]:
        """(k_q, k_scale, v_q, v_scale, length): the whole buffers and the
        live length to pass as `seqlen` (the reference returns freshly
        concatenated tensors of exactly the live length instead)."""
        return self.k_q, self.k_scale, self.v_q, self.v_scale, self.length

    def attention(self, q: torch.Tensor, softmax_scale: float) -> torch.Tensor:
        """q [batch, n_heads, head_dim] fp16 over the live tokens."""
        _require(self.length > 0, "the cache is empty")
        return decode_attention_int4(q, self.k_q, self.k_scale, self.v_q, self.v_scale,
                                     int(self.group_size), float(softmax_scale), int(self.length))

    def get_seq_length(self) -> int:
        return self.length

    def reset(self) -> None:
        self.length = 0


class PagedBatch(NamedTuple):
    """The sequences of one call and their new tokens, as the paged ops take
    them (PagedKVCache.batch)."""
    page_table: torch.Tensor            # [batch, max_pages] int32
    seq_lens: torch.Tensor              # [batch] int32, with the new tokens
    cu_tokens: Optional[torch.Tensor]   # [batch + 1] int32; None: one new token each
    rows: int                           # new tokens of all sequences
    prefix_pages: Optional[torch.Tensor]   # pages that all sequences share from the start on
    prefix_len: int
    shortest: int = 0                   # the shortest length, the mean length: how much of the
    mean: int = 0                       # prefix a window leaves
    positions: Optional[torch.Tensor] = None     # [rows] int32; None: the tokens' slots
    tree_mask: Optional[torch.Tensor] = None     # [rows, words] int64: a drafted tree (PagedKVCache.draft)
    weight_rows: Optional[torch.Tensor] = None   # [batch] int32: the sequences' rows of the weights
    shortened: bool = False                      # some sequence has lost tokens: slots are no positions
    queries: Optional[dict] = None               # layer -> a draft's q and score options, kept until it is accepted


class _Draft(NamedTuple):
    length: int            # of the sequence without the draft
    tokens: int            # drafted ones
    parents: List[int]
    row: int               # of its first token in the step's q
    queries: Optional[dict]   # of the step


class PagedKVCache:
    """Sequences of different lengths over a pool of `n_pages` pages of `page_size`
    tokens per layer: k, v [n_layers, n_pages, n_kv_heads, page_size, head_dim]. A
    page number means the same tokens in every layer.

    The host keeps each sequence's length and pages; `batch` reserves pages for
    a call's new tokens and hands the tables to the device, `append` rotates
    and writes the tokens, `attention` reads them:

        a = cache.add(); b = cache.add()
        step = cache.batch([a, b], [len(prompt_a), len(prompt_b)])
        q = cache.append(step, qkv, cos, sin)         # rows: a's tokens, then b's
        out = cache.attention(step, q, scale)
        step = cache.batch([a, b])                    # one more token each
        ...
        c = cache.add(share=a, tokens=1000)           # behind the first 1000 tokens of a
        cache.remove(b)

    One `batch` serves all layers: `append` and `attention` take the layer's
    number. All calls belong on one stream; not safe for several threads.

    A batch of single tokens behind whole shared pages may be read through
    paged_shared_prefix_attention, which rounds the prefix's probabilities to 16
    bits once where decode attention keeps a second part: a sequence's results
    then change (within the output type's rounding, fp16 2^-11, bf16 2^-8 of the
    values' weighted spread) with the sequences beside it. shared_prefix=False
    keeps decode attention for all batches.

    Drafted trees: `draft` reserves a tree of tokens behind each sequence,
    `append` and `attention` take its step like any other, and `accept` keeps one
    path of it:

        step = cache.draft([a, b], [parents_a, parents_b])
        ...                                           # every layer: append, attention
        cache.accept([a, b], [path_a, path_b])        # the tokens that the model agrees with

    A bounded cache: with track_rows > 0 up to so many sequences have a row of
    `weights` [n_layers, track_rows, n_kv_heads, track_tokens], to which
    `attention` adds what each token is given (of a prompt's chunk by its last
    `observe` rows, 0: by all), and `evict` cuts sequences down to the tokens of the
    largest weight, for every layer and KV head its own:

        cache.evict([a, b], keep=4096, first=4, recent=256)

    A drafted tree's attention adds nothing, as most of its tokens are dropped.
    With track_drafts=True the cache keeps a copy of the tree's q of every layer,
    and `accept` adds what the accepted tokens give, as decode steps of the same
    tokens would have (paged_prefill_weights of their rows). Without it the
    weights know nothing of drafted steps: accepted tokens count as ones that
    nothing has attended to, and an `evict` that meets them gives a warning.

    The tokens that stay keep their rotation, and new ones go on at the text's
    positions. A window or slopes are refused for a sequence that has lost
    tokens: distances would go by slots."""

    # A batch's shared prefix is read once for all sequences where that saves so many
    # token rows (of one KV head) and has so many tokens; a shorter one where it saves
    # sixteen times as many (_shared_prefix).
    SHARED_ROWS = 16384
    SHARED_TOKENS = 512

    def __init__(self, n_pages: int, n_kv_heads: int, page_size: int = 64, head_dim: int = 128,
                 dtype: torch.dtype = torch.float16, device: Optional[torch.device] = None,
                 n_layers: int = 1, shared_prefix: bool = True, track_rows: int = 0, track_tokens: int = 0,
                 observe: int = 0, track_drafts: bool = False) -> None:
        _require(n_pages > 0 and n_kv_heads > 0 and n_layers > 0, "n_pages, n_kv_heads and n_layers must be positive")
        _require(page_size > 0 and page_size % 8 == 0, "page_size must be a positive multiple of 8")
        _require(head_dim in (64, 128), "only head_dim=64 and 128 supported")
        _require(dtype in (torch.float16, torch.bfloat16), "dtype must be fp16 or bf16")
        _require(track_rows >= 0 and observe >= 0, "track_rows and observe must be >= 0")
        _require(track_rows == 0 or track_tokens > 0, "track_tokens must be positive where weights are recorded")
        _require(track_rows > 0 or not track_drafts, "track_drafts needs track_rows")
        self.device = torch.device("cuda") if device is None else torch.device(device)
        self.shared_prefix = bool(shared_prefix)
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = n_pages, n_kv_heads, page_size, head_dim
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=self.device)
        self.v = torch.zeros(shape, dtype=dtype, device=self.device)
        self.device = self.k.device   # with its index: batch() is not the current device's
        self._free = list(range(n_pages - 1, -1, -1))
        self._users = [0] * n_pages             # sequences that hold the page
        self._pages: dict[int, List[int]] = {}  # sequence -> its pages
        self._length: dict[int, int] = {}
        self._next = 0
        self._lost: dict[int, int] = {}               # sequence -> tokens that it has lost (its text is longer)
        self._drafts: dict[int, _Draft] = {}          # sequence -> its draft that is not accepted
        self.observe, self.track_drafts = int(observe), bool(track_drafts)
        self._unrecorded: set[int] = set()            # sequences with accepted tokens that no weights were recorded of
        self.weights: Optional[torch.Tensor] = None
        self._rows: dict[int, int] = {}               # sequence -> its row of the weights
        self._free_rows = list(range(track_rows - 1, -1, -1))
        if track_rows > 0:
            self.weights = torch.zeros(n_layers, track_rows, n_kv_heads, track_tokens, device=self.device)

    # ---- sequences ----

    def add(self, share: Optional[int] = None, tokens: int = 0) -> int:
        """A new sequence, empty or behind the first `tokens` tokens of the
        sequence `share`: whole pages are shared, the rest of the last one is
        copied. Returns its number. Recorded weights are copied; a sequence that
        has lost tokens is shared whole (of its first tokens it has not all)."""
        pages: List[int] = []
        _require(self.weights is None or len(self._free_rows) > 0, "the cache has no free row of weights")
        if share is not None:
            _require(share in self._pages, "no such sequence")
            _require(share not in self._drafts, "the shared sequence has a draft that is not accepted")
            _require(0 <= tokens <= self._length[share], "the shared sequence has fewer tokens")
            _require(self._lost[share] == 0 or tokens in (0, self._length[share]),
                     "a sequence that has lost tokens is shared whole")
            whole, rest = divmod(tokens, self.page_size)
            pages = self._pages[share][:whole]
            if rest:
                _require(len(self._free) > 0, "the cache has no free page")
                page, src = self._free.pop(), self._pages[share][whole]
                self._users[page] = 1
                self.k[:, page, :, :rest] = self.k[:, src, :, :rest]
                self.v[:, page, :, :rest] = self.v[:, src, :, :rest]
            for p in pages:
                self._users[p] += 1
            if rest:
                pages = pages + [page]
        else:
            _require(tokens == 0, "tokens are shared with a sequence")
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = list(pages), tokens
        self._lost[seq] = self._lost[share] if share is not None and tokens else 0
        if self.weights is not None:
            self._rows[seq] = row = self._free_rows.pop()
            self.weights[:, row].zero_()
            if share is not None:
                if share in self._unrecorded and tokens:
                    self._unrecorded.add(seq)
                n = min(tokens, self.weights.shape[3])
                self.weights[:, row, :, :n] = self.weights[:, self._rows[share], :, :n]
        return seq

    def remove(self, seq: int) -> None:
        """Ends a sequence; pages that no other one shares become free."""
        _require(seq in self._pages, "no such sequence")
        self._release(self._pages.pop(seq))
        del self._length[seq], self._lost[seq]
        self._drafts.pop(seq, None)
        self._unrecorded.discard(seq)
        if self.weights is not None:
            self._free_rows.append(self._rows.pop(seq))

    def _release(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)

    def _shorten(self, seq: int, tokens: int) -> None:
        """The sequence's first `tokens` slots stay; pages behind them are released."""
        keep = -(-tokens // self.page_size)
        self._release(self._pages[seq][keep:])
        del self._pages[seq][keep:]
        self._length[seq] = tokens

    def length(self, seq: int) -> int:
        return self._length[seq]

    def position(self, seq: int) -> int:
        """The text position of the sequence's next token: its length and what it has lost."""
        return self._length[seq] + self._lost[seq]

    def free_pages(self) -> int:
        return len(self._free)

    # ---- calls ----

    def batch(self, seqs: Sequence[int], new: Optional[Sequence[int]] = None) -> PagedBatch:
        """Reserves pages for new[i] (default 1) more tokens of seqs[i] and returns
        the call's tables. The tokens count as live from here on: `append` them
        before anything reads them. Nothing is reserved if the pages do not
        suffice."""
        return self._reserve(seqs, [1] * len(seqs) if new is None else [int(n) for n in new], None)

    def draft(self, seqs: Sequence[int], parents: Sequence[Sequence[int]]) -> PagedBatch:
        """`batch` for a drafted tree behind each sequence: parents[i][j] is the
        drafted token of seqs[i] that token j follows, an earlier one, or -1: the
        sequence's last token. The step's attention shows every drafted token the
        sequence and its own path, at the path's positions; `accept` ends the
        draft, and until then the sequence is in no other batch."""
        trees = [[int(p) for p in tree] for tree in parents]
        _require(len(trees) == len(seqs), "one tree per sequence")
        _require(all(-1 <= p < j for tree in trees for j, p in enumerate(tree)),
                 "a drafted token follows an earlier one or -1")
        return self._reserve(seqs, [len(tree) for tree in trees], trees)

    def accept(self, seqs: Sequence[int], paths: Sequence[Sequence[int]]) -> None:
        """Ends the drafts of `seqs`: of seqs[i] the drafted tokens paths[i] (numbers in
        the draft, ascending; none: all are dropped) become its next tokens, in
        every layer. The draft's step must have been appended to all layers that
        are read again. With track_drafts the weights that the accepted tokens give are
        recorded, in the layers that the step's `attention` was called for. A path begins at a token that follows the sequence and goes
        on from each token to one that follows it; other lists give a warning, as
        their tokens were rotated, and shown others, as what they then are not."""
        paths = [[int(j) for j in path] for path in paths]
        _require(len(paths) == len(seqs), "one path per sequence")
        _require(len(set(seqs)) == len(seqs), "a sequence occurs twice")
        _require(all(s in self._drafts for s in seqs), "a sequence has no draft")
        for s, path in zip(seqs, paths):
            _require(all(a < b for a, b in zip(path, path[1:])) and
                     all(0 <= j < self._drafts[s].tokens for j in path), "a path's tokens are ascending numbers of the draft")
        strays = [s for s, path in zip(seqs, paths) if [self._drafts[s].parents[j] for j in path] != [-1, *path][:len(path)]]
        if strays:
            warnings.warn(f"PagedKVCache.accept: what is accepted of the sequences {strays} is no path of their drafts: "
                          "its keys and values belong to other positions and other tokens before them", stacklevel=2)
        moved = [(s, path) for s, path in zip(seqs, paths) if path != list(range(len(path)))]
        if moved:
            ctx = [self._drafts[s].length for s, _ in moved]
            longest = max(len(path) for _, path in moved)
            kept = [[c + j for j in path] + [-1] * (longest - len(path)) for c, (_, path) in zip(ctx, moved)]
            self._compact([s for s, _ in moved], kept, ctx)
        drafts = [self._drafts.pop(s) for s in seqs]
        for s, path, draft in zip(seqs, paths, drafts):
            self._shorten(s, draft.length + len(path))
            if self.weights is not None and path and len(draft.queries or ()) < self.k.shape[0]:
                self._unrecorded.add(s)
        if self.track_drafts:
            self._record_accepted(seqs, paths, drafts)

    def _record_accepted(self, seqs: Sequence[int], paths: List[List[int]], drafts: List[_Draft]) -> None:
        """The weights that accepted tokens give: they are the sequences' last ones now, in order, as
        a prompt's are."""
        steps: dict[int, list] = {}
        for s, path, draft in zip(seqs, paths, drafts):
            if path and draft.queries:
                steps.setdefault(id(draft.queries), []).append((s, path, draft))
        for items in steps.values():
            b, width = len(items), max(len(self._pages[s]) for s, _, _ in items)
            cu = [0]
            for _, path, _ in items:
                cu.append(cu[-1] + len(path))
            flat = [self._length[s] for s, _, _ in items] + [self._rows[s] for s, _, _ in items] + cu
            flat += [p for s, _, _ in items for p in self._pages[s] + [-1] * (width - len(self._pages[s]))]
            flat += [draft.row + j for _, path, draft in items for j in path]
            dev = self._to_device(flat)
            table, rows = dev[3 * b + 1:3 * b + 1 + b * width].view(b, width), dev[len(flat) - cu[-1]:]
            for layer, (q, *options) in items[0][2].queries.items():
                paged_prefill_weights(q.index_select(0, rows), self.k[layer], table, dev[:b], dev[2 * b:3 * b + 1],
                                      self.weights[layer], *options, 0, dev[b:2 * b])

    def evict(self, seqs: Sequence[int], keep: int, first: int = 0, recent: int = 0) -> None:
        """Cuts the sequences down to `keep` tokens for every layer and KV head: the
        first `first`, the last `recent` and, of the others, those of the largest
        recorded weight (paged_select_tokens). Shorter ones stay as they are. Pages
        that other sequences share are copied first: nothing is changed if the free
        pages do not suffice. A sequence that accepted drafted tokens without their
        weights (track_drafts) gives a warning."""
        _require(self.weights is not None, "the cache records no weights (track_rows)")
        _require(len(set(seqs)) == len(seqs), "a sequence occurs twice")
        _require(all(s in self._pages for s in seqs), "no such sequence")
        _require(keep > 0 and first >= 0 and recent >= 0 and first + recent <= keep,
                 "first and recent must be >= 0, together at most keep")
        _require(all(s not in self._drafts for s in seqs), "a sequence has a draft that is not accepted")
        long = [s for s in seqs if self._length[s] > keep]
        _require(all(self._length[s] <= self.weights.shape[3] for s in long),
                 "a sequence has more tokens than weights (track_tokens)")
        if not long:
            return
        whole = -(-keep // self.page_size)
        shared = [(s, i) for s in long for i, p in enumerate(self._pages[s][:whole]) if self._users[p] > 1]
        # (a page that only these sequences share: the last of them keeps it)
        left = dict((p, self._users[p]) for s in long for p in self._pages[s])
        copies = []
        for s, i in shared:
            p = self._pages[s][i]
            if left[p] > 1:
                left[p] -= 1
                copies.append((s, i))
        _require(len(copies) <= len(self._free), "the cache has no free page")
        blind = [s for s in long if s in self._unrecorded]
        if blind:
            warnings.warn(f"PagedKVCache.evict: the weights of the sequences {blind} hold nothing of drafted tokens that "
                          "were accepted, which go first (track_drafts=True records them)", stacklevel=2)
            self._unrecorded.difference_update(blind)
        if copies:
            src = [self._pages[s][i] for s, i in copies]
            dst = [self._free.pop() for _ in copies]
            self.k[:, dst] = self.k[:, src]
            self.v[:, dst] = self.v[:, src]
            for (s, i), old, page in zip(copies, src, dst):
                self._users[page], self._pages[s][i] = 1, page
                self._release([old])
        self._compact(long, None, None, keep, first, recent)
        for s in long:
            self._lost[s] += self._length[s] - keep
            self._shorten(s, keep)

    def _compact(self, seqs: Sequence[int], kept: Optional[List[List[int]]], starts: Optional[List[int]],
                 keep: int = 0, first: int = 0, recent: int = 0) -> None:
        """Selection (where no lists are given) and moves of all layers in one launch each:
        the layers' pools are one, whose pages and weight rows are numbered on."""
        layers, b = self.k.shape[0], len(seqs)
        width = max(len(self._pages[s]) for s in seqs)
        flat = [self._length[s] for s in seqs] + (starts or [0] * b)
        flat += [self._rows.get(s, 0) for s in seqs] + [n for row in kept or [] for n in row]
        flat += [p for s in seqs for p in self._pages[s] + [-1] * (width - len(self._pages[s]))]
        dev = self._to_device(flat)
        lens, first_slots, rows = (dev[i * b:(i + 1) * b].repeat(layers) for i in range(3))
        pages = dev[len(flat) - b * width:].view(b, width)
        layer = torch.arange(layers, dtype=torch.int32, device=self.device)[:, None, None]
        table = torch.where(pages >= 0, pages + layer * self.n_pages, -1).view(-1, width)
        k, v = self.k.flatten(0, 1), self.v.flatten(0, 1)
        if kept is not None:
            lists = dev[3 * b:3 * b + b * len(kept[0])].view(b, -1).repeat(layers, 1)
            paged_compact(k, v, table, lens, lists, first_slots)
            return
        weights = self.weights.flatten(0, 1)
        rows = rows + (layer.view(-1, 1) * self.weights.shape[1]).expand(-1, b).reshape(-1)
        lists, _ = paged_select_tokens(weights, lens, keep, first, recent, rows)
        paged_compact(k, v, table, lens, lists, None, weights, rows)

    def _to_device(self, flat: List[int]) -> torch.Tensor:
        host = torch.tensor(flat, dtype=torch.int32)
        return host.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else host

    def _reserve(self, seqs: Sequence[int], counts: List[int], trees: Optional[List[List[int]]]) -> PagedBatch:
        _require(len(counts) == len(seqs), "one count per sequence")
        _require(len(set(seqs)) == len(seqs), "a sequence occurs twice in the batch")
        _require(all(s in self._pages for s in seqs), "no such sequence")
        _require(all(n >= 0 for n in counts), "counts must be >= 0")
        _require(all(s not in self._drafts for s in seqs), "a sequence has a draft that is not accepted")
        before = [self._length[s] for s in seqs]
        need = [-(-(self._length[s] + n) // self.page_size) - len(self._pages[s]) for s, n in zip(seqs, counts)]
        _require(sum(need) <= len(self._free), "the cache has no free page")
        for s, n, m in zip(seqs, counts, need):
            for _ in range(m):
                page = self._free.pop()
                self._users[page] = 1
                self._pages[s].append(page)
            self._length[s] += n
        pages = [self._pages[s] for s in seqs]
        lens = [self._length[s] for s in seqs]
        ragged = trees is not None or any(n != 1 for n in counts)
        lost = any(self._lost[s] for s in seqs)
        positions: List[int] = []
        words, masks = 0, []
        queries: Optional[dict] = {} if trees is not None and self.track_drafts else None
        if trees is not None:
            words = max(1, -(-max([len(t) for t in trees] + [0]) // 64))
            for s, n, tree in zip(seqs, before, trees):
                self._drafts[s] = _Draft(n, len(tree), tree, len(positions), queries)
                seen: List[int] = []
                deep: List[int] = []
                for j, parent in enumerate(tree):
                    seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
                    deep.append(deep[parent] + 1 if parent >= 0 else n + self._lost[s])
                masks += [(m >> 32 * w) & 0xFFFFFFFF for m in seen for w in range(2 * words)]
                positions += deep
        elif lost:
            positions = [n + self._lost[s] + j for s, n, c in zip(seqs, before, counts) for j in range(c)]
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        shared = 0 if ragged or not self.shared_prefix or self.weights is not None else self._shared_prefix(pages, lens)
        width = max([len(p) for p in pages] + [1])
        # One copy to the device: lengths, row offsets, then the table, and what else there is.
        flat = lens + cu + [p for row in pages for p in row + [-1] * (width - len(row))]
        ends = [len(flat)]
        for more in (positions, [self._rows[s] for s in seqs] if self.weights is not None else []):
            flat += more
            ends.append(len(flat))
        flat += [0] * (len(flat) % 2) + [m - (1 << 32) if m >> 31 else m for m in masks]   # (64-bit words)
        dev = self._to_device(flat)
        b = len(seqs)
        table = dev[2 * b + 1:ends[0]].view(b, width) if b else torch.zeros((0, width), dtype=torch.int32, device=self.device)
        tree_mask = None
        if trees is not None:
            tree_mask = dev[len(flat) - len(masks):].view(torch.int64).view(cu[-1], words)
        return PagedBatch(table, dev[:b], dev[b:2 * b + 1] if ragged else None, cu[-1],
                          table[0, :shared] if shared else None, shared * self.page_size,
                          min(lens, default=0), sum(lens) // max(b, 1),
                          dev[ends[0]:ends[1]] if lost or trees is not None else None, tree_mask,
                          dev[ends[1]:ends[2]] if self.weights is not None else None, lost, queries)

    def _shared_prefix(self, pages: List[List[int]], lens: List[int]) -> int:
        """Whole pages that all sequences share from the start on, or 0 where reading
        them once for all does not pay (_pays)."""
        if len(pages) < 2:
            return 0
        n = min(min(len(p) for p in pages), (min(lens) - 1) // self.page_size)
        first = pages[0]
        same = 0
        while same < n and all(p[same] == first[same] for p in pages):
            same += 1
        tokens = same * self.page_size
        return same if self._pays(tokens, tokens * (len(pages) - 1)) else 0

    def _pays(self, tokens: int, again: int) -> bool:
        """Whether to read `tokens` shared tokens once for all, where the sequences but
        one would read `again` of them again: partial results and a second launch
        against those rows. us, decode against shared, sequences x shared tokens, heads
        of 128: 8 KV heads 2 x 1024 10.5, 11.1; 2 x 2048 12.3, 11.5; 4 x 512 10.4, 11.2;
        4 x 1024 12.8, 11.5; 8 x 512 12.4, 11.5; 64 x 256 16.0, 16.8; 64 x 512 27.5, 18.4;
        32 KV heads 2 x 256 9.4, 10.7; 2 x 512 12.9, 11.2; 16 x 256 13.4, 13.2; 64 x 256
        53.6, 38.6."""
        least = self.SHARED_ROWS * (1 if tokens >= self.SHARED_TOKENS else 16)
        return tokens > 0 and again * self.n_kv_heads >= least

    def _window_pays(self, step: PagedBatch, window: int) -> bool:
        """_pays for what a window leaves of the shared prefix: the shortest sequence
        sees the most of it, the mean length stands for all. us, decode against shared,
        64 sequences behind 8192 tokens, windows of 64, 256, 512, 1024, 4096: 8.6, 21.4;
        13.7, 23.5; 19.1, 29.3; 33.6, 29.5; 91, 29.7; 16 behind 2048, 64, 512, 1024: 7.4,
        12.8; 11.7, 14.7; 17.4, 14.7. (8 behind 8192 with 1024 go the wrong way: 15.8, 16.6.)"""
        sees = lambda length: min(max(step.prefix_len - max(length - window, 0), 0), step.prefix_len)  # noqa: E731
        return self._pays(sees(step.shortest), sees(step.mean) * (step.page_table.shape[0] - 1))

    def append(self, step: PagedBatch, qkv: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor],
               layer: int = 0) -> torch.Tensor:
        """rope_paged_append of the batch's new tokens to a layer; returns the
        rotated q [rows, n_heads, head_dim]."""
        return rope_paged_append(qkv, cos, sin, self.k[layer], self.v[layer], step.page_table, step.seq_lens,
                                 step.cu_tokens, step.positions)

    def attention(self, step: PagedBatch, q: torch.Tensor, softmax_scale: float, softcap: float = 0.0,
                  slopes: Optional[torch.Tensor] = None, window: int = 0, layer: int = 0) -> torch.Tensor:
        """Attention of the batch's new tokens in a layer: decode, decode behind a
        shared prefix, prompts, or a drafted tree, by the batch (and what a window leaves
        of the prefix). Where the cache records weights, those of decode steps and prompts
        are added: once for every call (a tree's by `accept`, of the layer's last call)."""
        k, v = self.k[layer], self.v[layer]
        _require(not step.shortened or (slopes is None and window <= 0),
                 "window and slopes need sequences that have lost no tokens")
        if step.tree_mask is not None:
            out = paged_tree_attention(q, k, v, step.page_table, step.seq_lens, step.cu_tokens, step.tree_mask,
                                       softmax_scale, softcap, slopes, window, step.positions)
            if step.queries is not None:
                step.queries[layer] = (q.clone(), softmax_scale, softcap, slopes, window)
            return out
        if step.cu_tokens is not None:
            if self.weights is not None:
                paged_prefill_weights(q, k, step.page_table, step.seq_lens, step.cu_tokens, self.weights[layer],
                                      softmax_scale, softcap, slopes, window, self.observe, step.weight_rows)
            return paged_prefill_attention(q, k, v, step.page_table, step.seq_lens, step.cu_tokens, softmax_scale,
                                           softcap, slopes, window)
        if self.weights is not None:
            return paged_decode_attention_weights(q, k, v, step.page_table, step.seq_lens, self.weights[layer],
                                                  softmax_scale, softcap, slopes, window, step.weight_rows)
        if step.prefix_pages is not None and (window <= 0 or self._window_pays(step, window)):
            return paged_shared_prefix_attention(q, k, v, step.page_table, step.seq_lens, step.prefix_pages,
                                                 step.prefix_len, softmax_scale, softcap, slopes, window)
        return paged_decode_attention(q, k, v, step.page_table, step.seq_lens, softmax_scale, softcap, slopes, window)
