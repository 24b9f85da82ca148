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
length, in one pool of pages (the reference has no counterpart).
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import (_C, paged_decode_attention, paged_prefill_attention, paged_shared_prefix_attention,
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
    keeps decode attention for all batches."""

    # A batch's shared prefix is read once for all sequences where that saves so many
    # token rows (of one KV head) and has so many tokens; a shorter one where it saves
    # sixteen times as many (_shared_prefix).
    SHARED_ROWS = 16384
    SHARED_TOKENS = 512

    def __init__(self, n_pages: int, n_kv_heads: int, page_size: int = 64, head_dim: int = 128,
                 dtype: torch.dtype = torch.float16, device: Optional[torch.device] = None,
                 n_layers: int = 1, shared_prefix: bool = True) -> None:
        _require(n_pages > 0 and n_kv_heads > 0 and n_layers > 0, "n_pages, n_kv_heads and n_layers must be positive")
        _require(page_size > 0 and page_size % 8 == 0, "page_size must be a positive multiple of 8")
        _require(head_dim in (64, 128), "only head_dim=64 and 128 supported")
        _require(dtype in (torch.float16, torch.bfloat16), "dtype must be fp16 or bf16")
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

    # ---- sequences ----

    def add(self, share: Optional[int] = None, tokens: int = 0) -> int:
        """A new sequence, empty or behind the first `tokens` tokens of the
        sequence `share`: whole pages are shared, the rest of the last one is
        copied. Returns its number."""
        pages: List[int] = []
        if share is not None:
            _require(share in self._pages, "no such sequence")
            _require(0 <= tokens <= self._length[share], "the shared sequence has fewer tokens")
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
        return seq

    def remove(self, seq: int) -> None:
        """Ends a sequence; pages that no other one shares become free."""
        _require(seq in self._pages, "no such sequence")
        for p in self._pages.pop(seq):
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)
        del self._length[seq]

    def length(self, seq: int) -> int:
        return self._length[seq]

    def free_pages(self) -> int:
        return len(self._free)

    # ---- calls ----

    def batch(self, seqs: Sequence[int], new: Optional[Sequence[int]] = None) -> PagedBatch:
        """Reserves pages for new[i] (default 1) more tokens of seqs[i] and returns
        the call's tables. The tokens count as live from here on: `append` them
        before anything reads them. Nothing is reserved if the pages do not
        suffice."""
        counts = [1] * len(seqs) if new is None else [int(n) for n in new]
        _require(len(counts) == len(seqs), "one count per sequence")
        _require(len(set(seqs)) == len(seqs), "a sequence occurs twice in the batch")
        _require(all(s in self._pages for s in seqs), "no such sequence")
        _require(all(n >= 0 for n in counts), "counts must be >= 0")
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
        ragged = any(n != 1 for n in counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        shared = 0 if ragged or not self.shared_prefix else self._shared_prefix(pages, lens)
        width = max([len(p) for p in pages] + [1])
        # One copy to the device: lengths, row offsets, then the table.
        flat = lens + cu + [p for row in pages for p in row + [-1] * (width - len(row))]
        host = torch.tensor(flat, dtype=torch.int32)
        if self.device.type == "cuda":
            dev = host.pin_memory().to(self.device, non_blocking=True)
        else:
            dev = host
        b = len(seqs)
        table = dev[2 * b + 1:].view(b, width) if b else torch.zeros((0, width), dtype=torch.int32, device=self.device)
        return PagedBatch(table, dev[:b], dev[b:2 * b + 1] if ragged else None, cu[-1],
                          table[0, :shared] if shared else None, shared * self.page_size,
                          min(lens, default=0), sum(lens) // max(b, 1))

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
                                 step.cu_tokens)

    def attention(self, step: PagedBatch, q: torch.Tensor, softmax_scale: float, softcap: float = 0.0,
                  slopes: Optional[torch.Tensor] = None, window: int = 0, layer: int = 0) -> torch.Tensor:
        """Attention of the batch's new tokens in a layer: decode, decode behind a
        shared prefix, or prompts, by the batch (and what a window leaves of the prefix)."""
        k, v = self.k[layer], self.v[layer]
        if step.cu_tokens is not None:
            return paged_prefill_attention(q, k, v, step.page_table, step.seq_lens, step.cu_tokens, softmax_scale,
                                           softcap, slopes, window)
        if step.prefix_pages is not None and (window <= 0 or self._window_pays(step, window)):
            return paged_shared_prefix_attention(q, k, v, step.page_table, step.seq_lens, step.prefix_pages,
                                                 step.prefix_len, softmax_scale, softcap, slopes, window)
        return paged_decode_attention(q, k, v, step.page_table, step.seq_lens, softmax_scale, softcap, slopes, window)
