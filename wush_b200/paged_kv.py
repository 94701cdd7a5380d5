"""Paged key-value cache of a decoder layer, and the attention of new tokens over it.

Decoding one token at a time needs, next to the quantized linear layers, a cache of the keys and values of every
sequence.  It is kept in pages of a common pool, so that sequences grow without moving: token p of sequence b lies in
page ``block_table[b, p // page_size]`` at row ``p % page_size``.  The operators:

  paged_kv_append         rotate new queries and keys by their positions, write keys and values into their pages
  paged_kv_bounds         smallest and largest value of every key channel of the pages the newest tokens lie in
  paged_select_pages      the pages on which a new query can have its largest logits
  paged_decode_attention  attention of one new token per sequence over all its tokens, the last `window` of them, or the
                          selected pages

The reference has no counterpart: its quantized layers (inference_lib/src/fp_quant/module/linear.py:51-386) run inside
another library's models, whose cache and attention they use.  ``wush_b200.block.ShardedDecoderBlock`` calls these
operators (``prefill`` and ``decode``); they can equally be called by themselves.

Every operator runs on the current stream of its tensors' device, without a host synchronization, and can be captured
into a CUDA graph.  Inference only: results carry no gradient.  Lengths, positions, tables and selected pages are int32
tensors on the device.  An entry that lies outside what it indexes (a page outside the pool, a length beyond the table,
...) is skipped by the kernels and reported by ``_lib.check_status(device)``.
"""
from __future__ import annotations

import functools
from struct import Struct
from typing import Optional, Tuple

import torch

from . import _lib

# The structs of include/wush_b200.h: wush_kv_pages comes packed from the cache, the rest of a call's arguments follow it.
# (Packing one struct costs a tenth of converting as many arguments, and a small call is bound by its host time.)
_PAGES = Struct("@2P6q3Pq5i4x")
_APPEND = Struct("@P3q" + 5 * "P2q" + "5P2q4i")
_BOUNDS = Struct("@P3q3Pq")
_SELECT = Struct("@P3qP2q4PQ2P5i4x")
_ATTENTION = Struct("@P3q" + 2 * "P2q" + "5PQ2Pq3if")
_NO_HEADS = (0, 0, 0)

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}
MAX_DIM = 256
MAX_TOKENS = 2 ** 31 - 1 - 2 ** 16      # of a sequence


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 [max_positions, rotary_dim]: the cosines of the rotary_dim / 2 angles of every position, then the sines.
    Pair i of position p turns by p * base^(-2 i / rotary_dim); angles are computed in float64.  Any table of this
    layout can be passed to ``paged_kv_append``, so scaled or multi-axis positions are a matter of its rows."""
    if rotary_dim <= 0 or rotary_dim % 2 or max_positions <= 0:
        raise ValueError("rotary_dim must be even and positive, max_positions positive")
    freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).to(torch.float32)


class PagedKVCache:
    """The pool of pages of one layer: ``k`` and ``v`` [num_pages, page_size, n_kv_heads, head_dim], bfloat16, float16 or
    float8_e4m3fn, with unit channel stride and any order of the other axes (``allocate(layout="hnd")`` keeps a head's
    rows of a page together).  head_dim is a multiple of 8 (16 for 8-bit pages) and at most 256.

    8-bit pages hold key / k_scale and value / v_scale (float32 [n_kv_heads], positive, given by the caller).  ``bounds``
    [num_pages, n_kv_heads, 2, head_dim] (bfloat16 or float16; the type of 16-bit pages) is what ``paged_kv_bounds``
    fills and ``paged_select_pages`` reads.  The object keeps references to its tensors; replacing them needs a new one.
    Copies (``copy``, ``pickle``) are made anew around their tensors, so a deep copy has pages of its own."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None, bounds: Optional[torch.Tensor] = None):
        for t in (k, v, k_scale, v_scale, bounds):
            if t is not None and not t.is_cuda:
                raise _lib.WushB200Error("wush_b200 ops need CUDA tensors; there is no CPU fallback")
        _check_pool(k, v, k_scale, v_scale, bounds)
        self.k, self.v, self.k_scale, self.v_scale, self.bounds = k, v, k_scale, v_scale, bounds
        self.num_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        ptr = lambda t: t.data_ptr() if t is not None else 0
        self._packed = _PAGES.pack(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1),
                                   v.stride(2), ptr(k_scale), ptr(v_scale), ptr(bounds), *k.shape, TYPES[k.dtype],
                                   TYPES[bounds.dtype] if bounds is not None else 0)
        self._index = k.get_device()
        self._status = _lib.status_word(self.device).data_ptr()
        self._query_types = (torch.bfloat16, torch.float16) if k.dtype == torch.float8_e4m3fn else (k.dtype,)
        self._attention_scratch = {}                          # bytes by number of query heads

    def __getstate__(self):
        eight = self.dtype == torch.float8_e4m3fn             # (pickle does not know 8-bit floats)
        k, v = (t.view(torch.uint8) if eight else t for t in (self.k, self.v))
        return {**self.__dict__, "k": k, "v": v}

    def __setstate__(self, state):                            # the packed addresses become those of the copy's tensors
        k, v = (t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t for t in (state["k"], state["v"]))
        self.__init__(k, v, state["k_scale"], state["v_scale"], state["bounds"])
        for name, value in state.items():                     # (what a caller has hung on the object)
            self.__dict__.setdefault(name, value)

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype=torch.bfloat16, device=None,
                 layout: str = "nhd", k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                 bounds: bool = False) -> "PagedKVCache":
        """A pool of its own; layout "nhd": [pages, rows, heads, channels] in memory, "hnd": [pages, heads, rows, channels]."""
        if layout not in ("nhd", "hnd"):
            raise ValueError(f"layout must be 'nhd' or 'hnd', not {layout!r}")
        if dtype not in TYPES:
            raise ValueError(f"unsupported cache dtype: {dtype}")

        def pool():
            if layout == "nhd":
                return torch.zeros(num_pages, page_size, n_kv_heads, head_dim, dtype=dtype, device=device)
            return torch.zeros(num_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device).transpose(1, 2)
        bt = torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype
        b = torch.zeros(num_pages, n_kv_heads, 2, head_dim, dtype=bt, device=device) if bounds else None
        return cls(pool(), pool(), k_scale=k_scale, v_scale=v_scale, bounds=b)


class DecodeStep:
    """What the layers of a model share in one decoding step (or the prompt pass before it): lengths, tables, rotation and
    the form of the attention.  ``wush_b200.block.ShardedDecoderBlock.decode`` takes it.

    block_table  int32 [sequences, pages]
    seq_lens     int32 [sequences]: tokens of every sequence, the new one included; 0 for a padded row.  It may be written
                 in place between steps (another sequence in a row), between replays of a captured step as well
    rope         fp32 table for ``paged_kv_append`` (None: no rotation), interleaved its pairing
    scale, window  of ``paged_decode_attention``
    top_pages    attend to this many selected pages per key head (0: all); needs caches with bounds
    """

    def __init__(self, block_table: torch.Tensor, seq_lens: torch.Tensor, rope: Optional[torch.Tensor] = None,
                 interleaved: bool = False, scale: Optional[float] = None, window: int = 0, top_pages: int = 0):
        if top_pages < 0 or (top_pages and window):
            raise ValueError("top_pages must not be negative; a window and selected pages exclude each other")
        if seq_lens.dim() != 1 or seq_lens.dtype != torch.int32:
            raise ValueError("seq_lens must be an int32 [sequences] tensor")
        self.block_table, self.seq_lens, self.rope, self.interleaved = block_table, seq_lens, rope, interleaved
        self.scale, self.window, self.top_pages = scale, window, top_pages
        self.seq_ids = torch.arange(seq_lens.shape[0], dtype=torch.int32, device=seq_lens.device)
        self.positions = seq_lens - 1                         # of the new tokens, -1 in a padded row; attend() writes it

    def advance(self) -> None:
        """The next token of every sequence (padded rows stay padding); in place, so that captured steps see it."""
        self.seq_lens += self.seq_lens > 0
        torch.sub(self.seq_lens, 1, out=self.positions)

    def attend(self, cache: PagedKVCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Append the new tokens' keys and values ([sequences, heads, head_dim]) to a layer's cache and attend.  ``q`` is
        overwritten, first by the rotated queries, then by the result, and returned."""
        torch.sub(self.seq_lens, 1, out=self.positions)       # (here, in every layer: nothing tells when seq_lens was written)
        paged_kv_append(cache, k, v, self.block_table, self.seq_ids, self.positions, q=q, rope=self.rope,
                        interleaved=self.interleaved, q_out=q)
        if cache.bounds is not None:
            paged_kv_bounds(cache, self.block_table, self.seq_lens)
        pages = counts = None
        if self.top_pages:
            pages, counts = paged_select_pages(q, cache, self.block_table, self.seq_lens, self.top_pages,
                                               sink=min(1, self.top_pages - 1))
        return paged_decode_attention(q, cache, self.block_table, self.seq_lens, scale=self.scale, window=self.window,
                                      pages=pages, counts=counts, out=q)


def _check_pool(k, v, k_scale, v_scale, bounds) -> None:
    if k.dim() != 4 or k.shape != v.shape or min(k.shape) < 1:
        raise ValueError("k and v must be [num_pages, page_size, n_kv_heads, head_dim] tensors of one shape")
    if k.dtype not in TYPES or v.dtype != k.dtype:
        raise ValueError("k and v must be of one type: bfloat16, float16 or float8_e4m3fn")
    d, e = k.shape[3], k.element_size()
    if d > MAX_DIM or (d * e) % 16:
        raise ValueError(f"head_dim must be a multiple of {16 // e} and at most {MAX_DIM}")
    for t in (k, v):
        if t.stride(3) != 1:
            raise ValueError("the channels of a head must be contiguous")
        if t.data_ptr() % 16 or any((s * e) % 16 for s in t.stride()[:3]):
            raise ValueError("pages, rows and heads must start on 16-byte boundaries")
    eight = k.dtype == torch.float8_e4m3fn
    for t in (k_scale, v_scale):
        if (t is not None) != eight:
            raise ValueError("k_scale and v_scale go with 8-bit pages, and only with them")
        if eight and (t.dtype != torch.float32 or tuple(t.shape) != (k.shape[2],) or not t.is_contiguous()):
            raise ValueError("k_scale and v_scale must be contiguous float32 [n_kv_heads] tensors")
    if bounds is not None:
        if tuple(bounds.shape) != (k.shape[0], k.shape[2], 2, d) or not bounds.is_contiguous() or bounds.data_ptr() % 16:
            raise ValueError("bounds must be a contiguous [num_pages, n_kv_heads, 2, head_dim] tensor")
        if bounds.dtype not in ((torch.bfloat16, torch.float16) if eight else (k.dtype,)):
            raise ValueError("bounds must be of the pages' type (bfloat16 or float16 for 8-bit pages)")
    if any(t is not None and t.device != k.device for t in (v, k_scale, v_scale, bounds)):
        raise ValueError("the tensors of a cache must be on one device")


def _int32(t: torch.Tensor, shape, what: str, index: int) -> int:
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape} on cuda:{index}")
    return t.data_ptr()


def _table(cache: PagedKVCache, block_table: torch.Tensor):
    """(pointer, row stride, sequences, pages a sequence)"""
    shape = block_table.shape
    if block_table.dtype is not torch.int32 or len(shape) != 2 or block_table.get_device() != cache._index or shape[1] < 1:
        raise ValueError(f"block_table must be an int32 [sequences, pages] tensor on {cache.device}")
    seqs, width = shape
    row, col = block_table.stride()
    if (col != 1 and width > 1) or row < 0:
        raise ValueError("block_table must have a unit column stride")
    if width * cache.page_size > MAX_TOKENS:
        raise ValueError(f"a block table can hold at most {MAX_TOKENS} tokens per sequence")
    return block_table.data_ptr(), row, seqs, width


def _heads(cache: PagedKVCache, t: torch.Tensor, rows: int, heads: int, dtype, what: str):
    """(pointer, row stride, head stride) of a [rows, heads, head_dim] tensor"""
    if t.shape != (rows, heads, cache.head_dim):
        raise ValueError(f"{what} must be a [{rows}, {heads}, {cache.head_dim}] tensor")
    if t.get_device() != cache._index:
        if not t.is_cuda:
            raise _lib.WushB200Error("wush_b200 ops need CUDA tensors; there is no CPU fallback")
        raise ValueError(f"{what} is on {t.device}, the cache on {cache.device}")
    if t.dtype is not dtype:
        raise ValueError(f"{what} must be {dtype}")
    row, head, channel = t.stride()
    p = t.data_ptr()
    if channel != 1 or p & 15 or row & 7 or head & 7:
        raise ValueError(f"{what}: channels must be contiguous, and rows and heads start on 16-byte boundaries")
    return p, row, head


def _output(cache: PagedKVCache, t: torch.Tensor, rows: int, heads: int, dtype, what: str):
    """_heads of a tensor that is written: its rows and heads must not be one and the same (an expanded tensor)."""
    p, row, head = _heads(cache, t, rows, heads, dtype, what)
    if (row == 0 and rows > 1) or (head == 0 and heads > 1):
        raise ValueError(f"{what}: rows and heads must not overlap")
    return p, row, head


def _query_type(cache: PagedKVCache, t: torch.Tensor, what: str):
    """Element type of a call's queries, keys and values: that of 16-bit pages, either 16-bit type for 8-bit pages."""
    if t.dtype not in cache._query_types:
        raise ValueError(f"{what} must be " + " or ".join(str(x) for x in cache._query_types))
    return t.dtype


def _q_heads(cache: PagedKVCache, q: torch.Tensor) -> int:
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % cache.n_kv_heads:
        raise ValueError(f"q must be [rows, heads, {cache.head_dim}] with a multiple of {cache.n_kv_heads} heads")
    return q.shape[1]


def _on_its_device(at: int):
    """Run an operator (its cache is positional argument `at`) with the cache's device as the current one.  Switching costs
    more than a small call, so only when it is another."""
    def decorate(op):
        @functools.wraps(op)
        def run(*args, **kwargs):
            cache = args[at] if len(args) > at else kwargs.get("cache")
            if not isinstance(cache, PagedKVCache):
                raise TypeError(f"{op.__name__} needs a PagedKVCache")
            if torch.cuda.current_device() == cache._index:
                return op(*args, **kwargs)
            with torch.cuda.device(cache._index):
                return op(*args, **kwargs)
        return run
    return decorate


def _stream(cache: PagedKVCache) -> int:
    # torch.cuda.current_stream(...).cuda_stream without the two objects in between
    return torch._C._cuda_getCurrentRawStream(cache._index)


def _finish(cache: PagedKVCache, rc: int, what: str) -> None:
    if rc:
        _lib.check(rc, what)
    if _lib.CHECK_EVERY_OP:
        _lib.check_status(cache.device, what)


@_on_its_device(0)
def paged_kv_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, seq_ids: torch.Tensor,
                    positions: torch.Tensor, q: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None,
                    interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                    k_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the keys and values of new tokens into their pages, rotated by their positions; returns the rotated
    queries (None without ``q``).

    k, v       [rows, n_kv_heads, head_dim], q [rows, heads, head_dim]: slices of one fused projection will do
    seq_ids    int32 [rows]: row of ``block_table`` (int32 [sequences, pages]) the token belongs to
    positions  int32 [rows]: its position in that sequence.  A row with a negative id or position is padding: nothing is
               written for it.  No two rows may name the same token.
    rope       fp32 [positions, rotary_dim] (see ``rope_table``), rotary_dim a multiple of 16; None: no rotation.
               Channels behind rotary_dim are copied.  ``interleaved`` False: channel i turns with i + rotary_dim/2,
               True: channel 2i with 2i + 1.
    q_out      receives the rotated queries instead of a new (zeroed) tensor and may be ``q``; ``k_out`` likewise receives
               the rotated keys and may be ``k``.  Otherwise outputs must not overlap inputs.
    """
    typ = _query_type(cache, k, "k")
    rows, kv_heads = k.shape[0], cache.n_kv_heads
    hk = _heads(cache, k, rows, kv_heads, typ, "k")
    hv = _heads(cache, v, rows, kv_heads, typ, "v")
    table = _table(cache, block_table)
    ids = _int32(seq_ids, (rows,), "seq_ids", cache._index)
    pos = _int32(positions, (rows,), "positions", cache._index)
    hq = hqo = hko = _NO_HEADS
    n_heads = 0
    if q is not None:
        n_heads = _q_heads(cache, q)
        hq = _heads(cache, q, rows, n_heads, typ, "q")
        if q_out is None:
            q_out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        hqo = _output(cache, q_out, rows, n_heads, typ, "q_out")
    elif q_out is not None:
        raise ValueError("q_out goes with q")
    if k_out is not None:
        hko = _output(cache, k_out, rows, kv_heads, typ, "k_out")
    rope_ptr, rope_rows, rotary = 0, 0, 0
    if rope is not None:
        if rope.dim() != 2 or rope.dtype is not torch.float32 or not rope.is_contiguous() or rope.get_device() != cache._index \
                or rope.data_ptr() % 16:
            raise ValueError(f"rope must be a contiguous float32 [positions, rotary_dim] tensor on {cache.device}")
        rope_rows, rotary = rope.shape
        if rope_rows < 1 or rotary < 16 or rotary % 16 or rotary > cache.head_dim:
            raise ValueError("rotary_dim must be a multiple of 16 and at most head_dim")
        rope_ptr = rope.data_ptr()
    if rows == 0:
        return q_out
    rc = _lib.load().wush_kv_append(cache._packed + _APPEND.pack(
        *table, *hq, *hqo, *hk, *hv, *hko, rope_ptr, ids, pos, cache._status, _stream(cache), rows, rope_rows, TYPES[typ], n_heads,
        rotary, interleaved))
    _finish(cache, rc, "wush_kv_append")
    return q_out


@_on_its_device(0)
def paged_kv_bounds(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, new_tokens: int = 1) -> None:
    """Recompute ``cache.bounds`` for the pages that hold the last ``new_tokens`` of the ``seq_lens`` tokens of every
    sequence: the smallest and the largest stored key of every channel over the page's filled rows (NaN if one is).
    Call it after ``paged_kv_append``, with the largest number of tokens a sequence received."""
    if cache.bounds is None:
        raise ValueError("the cache has no bounds")
    if new_tokens < 0:
        raise ValueError("new_tokens must not be negative")
    table = _table(cache, block_table)
    lens = _int32(seq_lens, (table[2],), "seq_lens", cache._index)
    rc = _lib.load().wush_kv_bounds(cache._packed + _BOUNDS.pack(*table, lens, cache._status, _stream(cache), new_tokens))
    _finish(cache, rc, "wush_kv_bounds")


@_on_its_device(1)
def paged_select_pages(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, top: int,
                       sink: int = 1, recent: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages worth attending to: (pages int32 [sequences, n_kv_heads, top], counts int32 [sequences, n_kv_heads]).

    For every sequence and key head: its first ``sink`` and last ``recent`` pages, then the pages with the largest
    scores up to ``top`` in all (equal scores: the lowest page first).  A page's score is the largest, over the queries
    that share the key head, of sum_d max(q_d lower_d, q_d upper_d): no logit on the page exceeds it.  Scores near the border
    are summed in 64 bits: exactly, whatever the order, where the terms of a page and their partial sums fit 53 bits, and to
    64-bit rounding (dim * 2^-53 of the terms' magnitude) otherwise.  A page one of whose bounds is not finite, and a score
    that is not finite, count as +infinity.  Pages come in ascending order, followed by -1; a sequence of at most ``top``
    pages gets all of them.  (Right but slow where more than 256 pages share the score at the border, as with bounds that
    nobody filled, or a query is not finite: 0.7 ms for 2047 pages.)  q: [sequences, heads, head_dim], as
    ``paged_decode_attention`` takes it; ``cache.bounds`` must be up to date (``paged_kv_bounds``)."""
    if cache.bounds is None:
        raise ValueError("the cache has no bounds")
    if top < 1 or sink < 0 or recent < 0 or sink + recent > top:
        raise ValueError("top must be at least 1 and at least sink + recent, which must not be negative")
    typ = _query_type(cache, q, "q")
    table = _table(cache, block_table)
    _, _, seqs, width = table
    n_heads = _q_heads(cache, q)
    hq = _heads(cache, q, seqs, n_heads, typ, "q")
    lens = _int32(seq_lens, (seqs,), "seq_lens", cache._index)
    pages = seq_lens.new_empty((seqs, cache.n_kv_heads, top))
    counts = seq_lens.new_empty((seqs, cache.n_kv_heads))
    if seqs == 0:
        return pages, counts
    lib, stream = _lib.load(), _stream(cache)
    with _lib.workspace_lock:
        work = _lib.stream_workspace(cache._index, stream, lib.wush_kv_select_workspace_bytes(seqs, cache.n_kv_heads, width))
        rc = lib.wush_kv_select_pages(cache._packed + _SELECT.pack(
            *table, *hq, lens, pages.data_ptr(), counts.data_ptr(), work.data_ptr(), work.numel(), cache._status, stream,
            TYPES[typ], n_heads, top, sink, recent))
    _finish(cache, rc, "wush_kv_select_pages")
    return pages, counts


@_on_its_device(1)
def paged_decode_attention(q: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                           scale: Optional[float] = None, window: int = 0, pages: Optional[torch.Tensor] = None,
                           counts: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                           return_lse: bool = False):
    """softmax(scale * q K^T) V for one new token per sequence: [sequences, heads, head_dim] in q's type (and, with
    ``return_lse``, float32 [sequences, heads]: the log of the sum of exponentials).

    q          [sequences, heads, head_dim]; query head h reads key head h // (heads / n_kv_heads)
    seq_lens   int32 [sequences]: tokens in the cache, the new one included.  No token (<= 0): zeros, and -inf.  A key or
               value that is not finite in a token that counts makes what it meets NaN or infinite (a logit of -inf weighs
               nothing); in one that does not count it has no effect.
    scale      softmax scale, 1 / sqrt(head_dim) by default
    window     only the last ``window`` tokens; 0: all
    pages, counts  attend to the tokens of these pages only: for every sequence and key head the first counts[b, h]
               entries of pages[b, h], logical page numbers as ``paged_select_pages`` returns them (any order; a page
               listed twice counts twice; no page at a count <= 0).  Not together with a window.
    out        receives the result instead of a new tensor; it may be ``q``, and must not overlap it otherwise
    """
    typ = _query_type(cache, q, "q")
    table = _table(cache, block_table)
    seqs = table[2]
    n_heads = _q_heads(cache, q)
    hq = _heads(cache, q, seqs, n_heads, typ, "q")
    lens = _int32(seq_lens, (seqs,), "seq_lens", cache._index)
    if window < 0:
        raise ValueError("window must not be negative")
    top, pages_ptr, counts_ptr = 0, 0, 0
    if (pages is None) != (counts is None):
        raise ValueError("pages and counts go together")
    if pages is not None:
        if window:
            raise ValueError("a window and selected pages exclude each other")
        if pages.dim() != 3 or pages.shape[2] < 1 or pages.shape[2] * cache.page_size > MAX_TOKENS:
            raise ValueError(f"pages must be [sequences, n_kv_heads, top] and hold at most {MAX_TOKENS} tokens")
        top = pages.shape[2]
        pages_ptr = _int32(pages, (seqs, cache.n_kv_heads, top), "pages", cache._index)
        counts_ptr = _int32(counts, (seqs, cache.n_kv_heads), "counts", cache._index)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ho = _output(cache, out, seqs, n_heads, typ, "out")
    lse = torch.empty((seqs, n_heads), dtype=torch.float32, device=cache.device) if return_lse else None
    if seqs > 0:
        lib, stream = _lib.load(), _stream(cache)
        nbytes = cache._attention_scratch.get(n_heads)
        if nbytes is None:
            nbytes = cache._attention_scratch[n_heads] = lib.wush_kv_attention_workspace_bytes(cache._packed, n_heads)
        with _lib.workspace_lock:
            work = _lib.stream_workspace(cache._index, stream, nbytes)
            rc = lib.wush_kv_attention(cache._packed + _ATTENTION.pack(
                *table, *hq, *ho, lse.data_ptr() if return_lse else 0, lens, pages_ptr, counts_ptr, work.data_ptr(), work.numel(),
                cache._status, stream, window, TYPES[typ], n_heads, top, cache.head_dim ** -0.5 if scale is None else scale))
        _finish(cache, rc, "wush_kv_attention")
    return (out, lse) if return_lse else out
