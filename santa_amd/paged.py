"""Paged KV caches that sequences share, and the exact attention that reads them.

The reference's caches are contiguous, one per sequence
(tutorial_code/runtime_common.py:340-397).  Here a cache is a pool of pages per
layer, [num_pages, page_size, KVH, D] for K and for V (the pools that
``decode_systematic_paged`` of the extension modules reads), and a block table:
token n of a sequence is row ``n % page_size`` of page
``block_table[seq, n // page_size]``.  Sequences forked from one another hold
the same pages until they write:

    cache = PagedKVCache(layers, num_pages=8192, page_size=16, kv_heads=8, head_dim=128, max_seqs=64, max_len=65536)
    prompt, = cache.add([0])
    logits = model.extend(prompt_tokens, cache, [prompt])   # santa_amd.runtime.RandomLlama
    seqs = [prompt, *cache.fork(prompt, 63)]
    logits = model.extend(next_tokens, cache, seqs)         # the prompt's K and V are read once for all 64

* ``PagedKVCache`` adds, lengthens, forks, frees and compacts sequences;
* ``PagedPlan`` cuts up the attention's work for one set of lengths (built on
  the host once per step, used by every layer);
* ``rope_append`` rotates new tokens' q and k and writes k and v to their pages;
* ``paged_attention`` is exact attention over pages, for one or several new
  tokens per sequence;
* ``copy_pages`` copies pages within pools.

On a GPU all of them run the library's kernels (santa_paged.hip); torch
expressions are the CPU path and that of calls that the attention kernel does
not take (float32, head_dim other than 64 and 128, autograd).
"""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from .runtime import _FusedOps, _plain

__all__ = ["PagedKVCache", "PagedPlan", "paged_attention", "rope_append", "copy_pages"]

_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
_IP = ctypes.POINTER(ctypes.c_int)


class _PlanInfo(ctypes.Structure):
    _fields_ = ([(n, _I) for n in ("tokens", "groups", "items", "merge_tokens", "max_len", "max_row", "heads",
                                   "kv_heads")]
                + [(n, _L) for n in ("records", "ints", "pos_at", "merge_at", "parts_at", "list_at")]
                + [("rounded", _I)])


_lib_ready = None


def _lib():
    global _lib_ready
    if _lib_ready is None:
        L = _FusedOps.lib()
        info = ctypes.POINTER(_PlanInfo)
        L.santa_pages_create.argtypes = [_I] * 4 + [ctypes.POINTER(_P)]
        L.santa_pages_destroy.argtypes = [_P]
        L.santa_pages_destroy.restype = None
        L.santa_pages_add.argtypes = [_P, _IP, _I, _IP]
        L.santa_pages_extend.argtypes = [_P, _IP, _IP, _I]
        L.santa_pages_shrink.argtypes = [_P, _IP, _IP, _I]
        L.santa_pages_fork.argtypes = [_P, _I, _I, _IP]
        L.santa_pages_free.argtypes = [_P, _IP, _I]
        L.santa_pages_compact.argtypes = [_P]
        L.santa_pages_changes.argtypes = [_P, ctypes.POINTER(_IP), _IP, ctypes.POINTER(_IP), _IP, _IP]
        L.santa_pages_length.argtypes = [_P, _I]
        L.santa_pages_used.argtypes = [_P]
        L.santa_pages_row.argtypes = [_P, _I, ctypes.POINTER(_IP)]
        L.santa_pages_shared.argtypes = [_P, _IP, _IP, _I, _IP, _IP, _IP]
        L.santa_pages_apply.argtypes = [_P, ctypes.POINTER(_P), _I, _L, _L, _P, _L, _I, _P]
        L.santa_paged_copy.argtypes = [ctypes.POINTER(_P), _I, _L, _L, _I, _IP, _I, _P]
        L.santa_paged_plan.argtypes = [_IP, _IP, _IP, _I, _IP, _IP, _I, _I, _I, _I, info, _P, _L]
        L.santa_paged_workspace_size.argtypes = [info, _I]
        L.santa_paged_workspace_size.restype = ctypes.c_size_t
        L.santa_paged_attention.argtypes = [_P] * 4 + [_I] * 4 + [ctypes.POINTER(_L), _P, _L, _I, info, _P,
                                                                  ctypes.c_float, _P, ctypes.c_size_t, _P]
        L.santa_paged_rope_append.argtypes = [_P] * 6 + [_I] * 4 + [ctypes.POINTER(_L), _P, _L, _I, info, _P, _P]
        _lib_ready = L
    return _lib_ready


_check = _FusedOps._check


def _launch(device: torch.device, call, *args):
    """call(*args, stream) on device and its current stream (the raw handle: an
    object of it costs as much as a launch)."""
    if torch._C._cuda_getDevice() == device.index:
        _check(call(*args, torch._C._cuda_getCurrentRawStream(device.index)))
        return
    with torch.cuda.device(device):
        _check(call(*args, torch._C._cuda_getCurrentRawStream(device.index)))


def _device(device) -> torch.device:
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        return torch.device("cuda", torch.cuda.current_device())
    return device


def _int_list(values, what: str) -> List[int]:
    """Host integers: a list, a range, an array or a CPU tensor."""
    if isinstance(values, torch.Tensor):
        if values.is_cuda:
            raise ValueError(f"{what} must be host integers; reading a GPU tensor would wait for the GPU")
        values = values.tolist()
    if isinstance(values, int):
        raise ValueError(f"{what} must be a list")
    values = list(values)
    ints = [int(v) for v in values]
    if ints != values:
        raise ValueError(f"{what} must be whole numbers")
    return ints


def _ints(values: Sequence[int]):
    for v in values:
        if not -(1 << 31) <= v < 1 << 31:
            raise ValueError(f"{v} does not fit 32 bits")
    return (ctypes.c_int * len(values))(*values)


# ------------------------------------------------------------------- pages
class PagedKVCache:
    """K and V page pools of `layers` layers, and the sequences that hold pages
    of them.  Which pages a sequence holds is kept on the host: a call that does
    not fit raises and changes nothing, and none waits for the GPU.  What a call
    changes on the GPU (block_table, copies of pages) runs on the current
    stream.  A cache is used by one host thread at a time, and its streams are
    ordered by the caller.

    `k`, `v`: the pools, one [num_pages, page_size, kv_heads, head_dim] per
    layer (their contents start at 0); `block_table`: int32 [max_seqs,
    ceil(max_len / page_size)], row s that of sequence s."""

    def __init__(self, layers: int, num_pages: int, page_size: int, *, kv_heads: int, head_dim: int, max_seqs: int,
                 max_len: int, dtype=torch.bfloat16, device="cuda"):
        self._pages = None
        device = _device(device)
        if layers < 0 or kv_heads <= 0 or head_dim <= 0 or max_len <= 0 or page_size <= 0:
            raise ValueError("a cache needs layers, heads and room for tokens")
        row_pages = -(-int(max_len) // int(page_size))
        handle = _P()
        _check(_lib().santa_pages_create(*_ints([num_pages, page_size, max_seqs, row_pages]), ctypes.byref(handle)))
        self._pages = handle
        self.device, self.dtype = device, dtype
        self.layers, self.num_pages, self.page_size = layers, num_pages, page_size
        self.kv_heads, self.head_dim, self.max_seqs = kv_heads, head_dim, max_seqs
        shape = (num_pages, page_size, kv_heads, head_dim)
        with torch.inference_mode(False):  # they are written to in any mode
            self.k = tuple(torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers))
            self.v = tuple(torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers))
            self.block_table = torch.zeros(max_seqs, row_pages, dtype=torch.int32, device=device)
        self._page_bytes = page_size * kv_heads * head_dim * self.block_table.new_empty(0, dtype=dtype).element_size()
        if device.type == "cuda" and self._page_bytes % 16:
            raise ValueError("pages must be whole 16-byte pieces")
        pools = [t.data_ptr() for t in (*self.k, *self.v)]
        self._pools = (_P * len(pools))(*pools)

    def __del__(self):
        if getattr(self, "_pages", None) is not None and _lib_ready is not None:
            _lib_ready.santa_pages_destroy(self._pages)

    # ------------------------------------------------------------ sequences
    @property
    def used_pages(self) -> int:
        return _lib().santa_pages_used(self._pages)

    @property
    def free_pages(self) -> int:
        return self.num_pages - self.used_pages

    def lengths(self, seqs: Sequence[int]) -> List[int]:
        seqs = _int_list(seqs, "seqs")
        out = [_lib().santa_pages_length(self._pages, s) for s in _ints(seqs)]
        if min(out, default=0) < 0:
            raise RuntimeError(f"no sequence {seqs[out.index(-1)]} in the cache")
        return out

    def pages(self, seq: int) -> List[int]:
        """The pages that a sequence holds, first tokens first."""
        row = _IP()
        n = _lib().santa_pages_row(self._pages, *_ints([seq]), ctypes.byref(row))
        if n < 0:
            raise RuntimeError(f"no sequence {seq} in the cache")
        return row[:n]

    def add(self, lengths: Sequence[int]) -> List[int]:
        """New sequences with pages for that many tokens each (whose K and V the
        caller writes): the lowest free rows of the block table, pages of the
        lowest numbers."""
        lengths = _int_list(lengths, "lengths")
        self._may_change()
        out = (ctypes.c_int * len(lengths))()
        _check(_lib().santa_pages_add(self._pages, _ints(lengths), len(lengths), out))
        self._apply()
        return list(out)

    def extend(self, seqs: Sequence[int], tokens: Union[int, Sequence[int]] = 1) -> None:
        """Pages for that many more tokens of each sequence.  A last page that
        is partly filled and that other sequences hold too is copied first, in
        every layer."""
        seqs = _int_list(seqs, "seqs")
        tokens = [tokens] * len(seqs) if isinstance(tokens, int) else _int_list(tokens, "tokens")
        if len(tokens) != len(seqs):
            raise ValueError(f"tokens must be an int or have one entry per sequence ({len(seqs)})")
        self._may_change()
        _check(_lib().santa_pages_extend(self._pages, _ints(seqs), _ints(tokens), len(seqs)))
        self._apply()

    def _take_back(self, seqs: Sequence[int], tokens: Sequence[int]) -> None:
        """Those many last tokens, whose K and V were never written, leave the
        sequences again (a last page that extend() copied stays theirs)."""
        _check(_lib().santa_pages_shrink(self._pages, _ints(seqs), _ints(tokens), len(seqs)))

    def fork(self, seq: int, n: int = 1) -> List[int]:
        """n new sequences with the same tokens, which hold the same pages."""
        self._may_change()
        if not 0 <= n <= self.max_seqs:
            raise ValueError(f"n must be in [0, {self.max_seqs}]; got {n}")
        out = (ctypes.c_int * n)()
        _check(_lib().santa_pages_fork(self._pages, *_ints([seq, n]), out))
        self._apply()
        return list(out)

    def free(self, seqs: Sequence[int]) -> None:
        """The sequences end; pages that no other sequence holds are free."""
        seqs = _int_list(seqs, "seqs")
        self._may_change()
        _check(_lib().santa_pages_free(self._pages, _ints(seqs), len(seqs)))

    def compact(self) -> int:
        """Moves pages so that those in use are the first ones of the pools;
        returns their number."""
        self._may_change()
        _check(_lib().santa_pages_compact(self._pages))
        self._apply()
        return self.used_pages

    def tables(self, seqs: Sequence[int]) -> torch.Tensor:
        """The rows of the block table of these sequences, in their order (for
        calls that take row b for sequence b)."""
        seqs = _int_list(seqs, "seqs")
        self.lengths(seqs)
        if seqs == list(range(seqs[0], seqs[0] + len(seqs))) if seqs else True:
            return self.block_table[seqs[0]:seqs[0] + len(seqs)] if seqs else self.block_table[:0]
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the rows of these sequences do not follow one another: they cannot be gathered while a "
                               "graph is captured")
        at = torch.tensor(seqs, dtype=torch.int64, pin_memory=self.device.type == "cuda")
        return self.block_table.index_select(0, at.to(self.device, non_blocking=True))

    def plan(self, seqs: Sequence[int], heads: int, new_tokens: Union[int, Sequence[int]] = 1, *,
             fixed: bool = False) -> "PagedPlan":
        """The plan of these sequences' attention, the last new_tokens of each
        being its queries; tokens that sequences hold in the same pages are read
        once."""
        seqs = _int_list(seqs, "seqs")
        lens = self.lengths(seqs)
        own = [new_tokens] * len(seqs) if isinstance(new_tokens, int) else _int_list(new_tokens, "new_tokens")
        if len(own) != len(seqs):
            raise ValueError(f"new_tokens must be an int or have one entry per sequence ({len(seqs)})")
        n = len(seqs)
        group, shared, groups = (ctypes.c_int * n)(), (ctypes.c_int * max(1, n))(), ctypes.c_int()
        _check(_lib().santa_pages_shared(self._pages, _ints(seqs), _ints(own), n, group, shared, ctypes.byref(groups)))
        members: List[List[int]] = [[] for _ in range(groups.value)]
        for i, g in enumerate(group):
            if g >= 0:
                members[g].append(i)
        return PagedPlan(lens, heads=heads, kv_heads=self.kv_heads, new_tokens=own, rows=seqs, fixed=fixed,
                         prefixes=[(m, shared[g]) for g, m in enumerate(members)], device=self.device)

    # -------------------------------------------------------------- changes
    def _may_change(self) -> None:
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a cache's sequences cannot change while a graph is captured: a replay would not "
                               "change them again")

    def _apply(self) -> None:
        """What the last call asks of the pools and the block table."""
        table = self.block_table
        if self.device.type == "cuda":
            _launch(self.device, _lib().santa_pages_apply, self._pages, self._pools, len(self._pools), self._page_bytes,
                    self._page_bytes, table.data_ptr(), table.shape[1], self.max_seqs)
            return
        copies, edits = _IP(), _IP()
        n_copies, n_edits, remap = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _check(_lib().santa_pages_changes(self._pages, *map(ctypes.byref, (copies, n_copies, edits, n_edits, remap))))
        pairs = copies[:2 * n_copies.value] if n_copies.value else []
        src, dst = pairs[::2], pairs[1::2]
        for t in (*self.k, *self.v) if src else ():
            t[dst] = t[src]
        for i in range(n_edits.value):
            row, col, count, value = edits[4 * i:4 * i + 4]
            table[row, col:col + count] = (table[-1 - value, col:col + count] if value < 0
                                           else torch.arange(value, value + count, dtype=torch.int32))
        if remap.value:
            to = torch.arange(self.num_pages, dtype=torch.int32)
            to[src] = torch.tensor(dst, dtype=torch.int32)
            table.copy_(to[table.long()])


def copy_pages(pools: Union[torch.Tensor, Iterable[torch.Tensor]], src: Sequence[int], dst: Sequence[int]) -> None:
    """pool[dst[i]] = pool[src[i]] for every i in each pool [num_pages, ...]
    (pages contiguous; all pools with the same number of pages).  No page is
    written twice, or both read and written.  On a GPU pages are whole 16-byte
    pieces, and the copies run on the current stream, a captured call's replays
    included."""
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    src, dst = _int_list(src, "src"), _int_list(dst, "dst")
    if len(src) != len(dst):
        raise ValueError("src and dst must be of one length")
    if not pools:
        return
    num_pages, device = pools[0].shape[0] if pools[0].dim() else 0, pools[0].device
    groups = {}
    for t in pools:
        if t.dim() < 2 or t.shape[0] != num_pages or t.device != device:
            raise ValueError("pools must be [num_pages, ...] tensors of one number of pages on one device")
        page = t[0] if num_pages else t
        if not page.is_contiguous() or (num_pages > 1 and t.stride(0) < page.numel()):
            raise ValueError("the pages of a pool must be contiguous")
        size = page.numel() * t.element_size() if num_pages else 0
        stride = t.stride(0) * t.element_size() if num_pages > 1 else size
        groups.setdefault((size, stride), []).append(t)
    if device.type == "cuda":
        pairs = _ints([p for pair in zip(src, dst) for p in pair])
        if any(size % 16 or stride % 16 for size, stride in groups) or any(t.data_ptr() % 16 for t in pools):
            raise RuntimeError("pages must be whole 16-byte pieces, 16-byte aligned")
        for (size, stride), ts in groups.items():
            if size == 0 and all(0 <= p < num_pages for p in pairs):
                continue
            pointers = (_P * len(ts))(*[t.data_ptr() for t in ts])
            _launch(device, _lib().santa_paged_copy, pointers, len(ts), size, stride, num_pages, pairs, len(src))
        return
    for p in (*src, *dst):
        if not 0 <= p < num_pages:
            raise RuntimeError(f"no page {p} in a pool of {num_pages}")
    if len(set(dst)) != len(dst):
        raise RuntimeError("a page is written twice")
    if set(src) & set(dst):
        raise RuntimeError("a page is both read and written")
    if src:
        for t in pools:
            t[dst] = t[src]


# --------------------------------------------------------------------- plan
class PagedPlan:
    """How ``paged_attention`` and ``rope_append`` treat a batch: sequence b
    holds seq_lens[b] tokens in row rows[b] (default b) of the block table, and
    the last new_tokens[b] of them (an int for all, or one per sequence; 0 is
    allowed) are the batch's tokens, sequence after sequence.  A sequence may
    be shorter than its new tokens (a slot not in use): tokens of a negative
    position are not written and attend to nothing, which gives zeros.

    prefixes: [(members, tokens)]: the sequences in `members` (indices into
    seq_lens; a sequence is in one prefix at most) have their first `tokens`
    tokens in common, which lie before the new tokens of each; they are read
    once for all, through the row of one of them.

    The plan is built on the host and copied to the device on the current
    stream.  `update(seq_lens)` makes it that of other lengths of the same
    sequences.  With fixed=True an update keeps the launches and workspaces of
    the kernels' calls the same, so that a captured graph can be replayed after
    it (at the cost of workgroups without work), up to the lengths that the
    captured calls' block tables have room for.  A plan that a graph holds in
    another way is not updated, and one that a graph holds is kept as long as
    the graph."""

    def __init__(self, seq_lens: Sequence[int], *, heads: int, kv_heads: int, new_tokens: Union[int, Sequence[int]] = 1,
                 prefixes: Sequence[Tuple[Sequence[int], int]] = (), rows: Optional[Sequence[int]] = None,
                 device="cuda", fixed: bool = False):
        lens = _int_list(seq_lens, "seq_lens")
        B = len(lens)
        self.heads, self.kv_heads = _ints([int(heads), int(kv_heads)])
        self.fixed = bool(fixed)
        self.device = _device(device)
        self.new_tokens = [new_tokens] * B if isinstance(new_tokens, int) else _int_list(new_tokens, "new_tokens")
        self.rows = list(range(B)) if rows is None else _int_list(rows, "rows")
        if len(self.new_tokens) != B or len(self.rows) != B:
            raise ValueError(f"new_tokens and rows must have one entry per sequence ({B})")
        self.prefixes = [(_int_list(m, "members"), int(n)) for m, n in prefixes]
        group = [-1] * B
        for g, (members, _) in enumerate(self.prefixes):
            for b in members:
                if not 0 <= b < B:
                    raise ValueError(f"no sequence {b} in a batch of {B}")
                if group[b] >= 0:
                    raise ValueError(f"sequence {b} is named in two prefixes")
                group[b] = g
        self._args = (_ints(self.new_tokens), _ints(self.rows), B, _ints(group),
                      _ints([n for _, n in self.prefixes]), len(self.prefixes))
        self._info = _PlanInfo()
        # room for a plan: its items, in whole pieces of 256 rows and a cut for every workgroup, and what it says of
        # each token; one that is larger is built again
        tokens, rows = sum(max(0, t) for t in self.new_tokens), max(1, 256 * self.kv_heads // max(1, self.heads))
        self._size = min(1 << 22, 16 * (B + 2 * (tokens // rows) + len(self.prefixes) + 256 // max(1, self.kv_heads) + 1)
                         + 12 * tokens + 2)
        self._data = self._stream = None
        self._room = None  # what captured calls have room for
        self.update(lens)

    def update(self, seq_lens: Sequence[int]) -> None:
        """The plan of other lengths.  Calls that use the plan on other streams,
        and replays of graphs that hold them, are ordered by the caller."""
        lens = _int_list(seq_lens, "seq_lens")
        new, rows, B, group, shared, groups = self._args
        if len(lens) != B:
            raise ValueError(f"seq_lens must have one entry per sequence ({B})")
        cuda = self.device.type == "cuda"
        if cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a plan cannot be made while a graph is captured: a replay would not make it again")
        if self._room is not None and max(lens, default=0) > self._room:
            if self._room < 0:
                raise RuntimeError("a captured call holds this plan's lengths: only the kernels' calls of a plan with "
                                   "fixed=True follow an update")
            raise RuntimeError(f"seq_lens exceeds the block table's capacity in a captured call: {max(lens)} > "
                               f"{self._room}")
        info = _PlanInfo()

        def build(buffer, n):
            if cuda:  # the plan is cut to that device's compute units
                with torch.cuda.device(self.device):
                    return _lib().santa_paged_plan(_ints(lens), new, rows, B, group, shared, groups, self.heads,
                                                   self.kv_heads, int(self.fixed), ctypes.byref(info), buffer, n)
            return _lib().santa_paged_plan(_ints(lens), new, rows, B, group, shared, groups, self.heads, self.kv_heads,
                                           int(self.fixed), ctypes.byref(info), buffer, n)

        with torch.inference_mode(False):  # updated in any mode
            host = torch.empty(self._size, dtype=torch.int32, pin_memory=cuda)
            rc = build(host.data_ptr(), self._size)
            if rc != 0 and info.ints > self._size:
                host = torch.empty(info.ints, dtype=torch.int32, pin_memory=cuda)
                rc = build(host.data_ptr(), info.ints)
            _check(rc)
            host = host[:max(1, info.ints)]
            if self._data is not None and self._data.shape == host.shape:
                self._used()
                self._data.copy_(host, non_blocking=True)
            else:
                self._data = host.to(self.device, non_blocking=True)
                if cuda:
                    self._stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        self._info, self.seq_lens = info, lens

    def _captured(self, room: int, follows: bool) -> None:
        """Where a graph is captured, notes that it holds a call with a block
        table for `room` tokens, whose replays follow an update (a kernel's,
        which reads the plan) or do not."""
        if self._stream is not None and torch._C._cuda_isCurrentStreamCapturing():
            self._hold(room if follows and self.fixed else -1)

    def _hold(self, room: int) -> None:
        self._room = room if self._room is None else min(room, self._room)

    def _used(self) -> None:
        """Before a call on the current stream: the plan's memory, where it comes
        from another stream, is not given out again before the call has ended."""
        if self._stream is not None and torch._C._cuda_getCurrentRawStream(self.device.index) != self._stream:
            self._data.record_stream(torch.cuda.current_stream(self.device))

    @property
    def tokens(self) -> int:
        """Tokens of the batch: the sum of new_tokens."""
        return self._info.tokens

    @property
    def positions(self) -> torch.Tensor:
        """The position of every token of the batch, int32 [tokens] on the device."""
        at = self._info.pos_at
        return self._data[at:at + 2 * self.tokens:2]


def _check_pools(k_pages, v_pages, block_table, plan: PagedPlan, like: torch.Tensor) -> None:
    shape, device = k_pages.shape, like.device
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be [num_pages, page_size, KVH, D] tensors of one shape")
    if k_pages.dtype != like.dtype or v_pages.dtype != like.dtype:
        raise ValueError("k_pages and v_pages must have the dtype of the new tokens")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or (block_table.shape[1] > 1
                                                                      and block_table.stride(1) != 1):
        raise ValueError("block_table must be an int32 [sequences, pages] tensor with contiguous rows")
    if k_pages.device != device or v_pages.device != device or block_table.device != device:
        raise ValueError("device mismatch")
    if plan.device != device:
        raise ValueError(f"the plan is for {plan.device}, the tensors are on {device}")
    num_pages, page_size, kv_heads, _ = shape
    if page_size < 8 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two in [8, 1048576]. Got page_size={page_size}")
    if num_pages == 0:
        raise ValueError("num_pages must be > 0")
    if kv_heads != plan.kv_heads:
        raise ValueError(f"the plan is for {plan.kv_heads} KV heads, the pages hold {kv_heads}")
    info, (rows, width) = plan._info, block_table.shape
    if info.max_row >= rows:
        raise ValueError(f"the plan names block table row {info.max_row} of {rows}")
    if info.max_len > width * page_size:
        raise ValueError(f"seq_lens exceeds the block table's capacity: {info.max_len} > {width * page_size}")


def _strides(t: torch.Tensor, what: str) -> Sequence[int]:
    """The leading strides of [.., D]; those of dimensions of size 1, which are
    never used and can be any number, as if packed."""
    strides = t.stride()
    if 1 in t.shape:
        strides, packed = list(strides), 1
        for i in range(t.dim() - 1, -1, -1):
            if t.shape[i] == 1:
                strides[i] = packed
            packed *= t.shape[i]
    bad = strides[-1] != 1 or t.data_ptr() % 16
    for s in strides[:-1]:
        bad = bad or s % 8 or s < 0
    if bad:
        raise ValueError(f"{what} must be 16-byte aligned, its last dimension contiguous and its other strides "
                         "multiples of 8 elements")
    return strides[:-1]


def _overlaps(t: torch.Tensor) -> bool:
    """Whether elements of t share memory, or dimensions interleave."""
    span = 1
    if not t.is_contiguous():
        for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
            if stride < span:
                return True
            span += stride * (size - 1)
    return False


def _packed(t: torch.Tensor) -> torch.Tensor:
    """t, contiguous and 16-byte aligned."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _table_rows(table: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The table as the kernels address it, and its row stride: rows that do
    not overlap."""
    if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        table = table.contiguous()
    return table, table.stride(0) if table.shape[0] > 1 else table.shape[1]


def _token_slots(block_table, plan: PagedPlan, page_size: int):
    """(token of the batch, pool row) of the tokens that have a position."""
    token, seq, pos, t0 = [], [], [], 0
    for row, n, t in zip(plan.rows, plan.seq_lens, plan.new_tokens):
        for i in range(max(0, t - n), t):
            token.append(t0 + i)
            seq.append(row)
            pos.append(n - t + i)
        t0 += t
    token, seq, pos = (torch.tensor(x, dtype=torch.int64, device=block_table.device) for x in (token, seq, pos))
    return token, block_table[seq, pos // page_size].long() * page_size + pos % page_size


def rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                block_table: torch.Tensor, plan: PagedPlan) -> torch.Tensor:
    """RoPE of the batch's tokens with their write into pages: qkv [tokens, H +
    2 KVH, D], cos and sin [tokens, D] (rotate-half convention).  The k heads
    are rotated and written to k_pages, the v heads to v_pages, at the tokens'
    positions; returns the rotated q heads [tokens, H, D].  float32 arithmetic,
    rounded once.  Two tokens of one position and page (sequences that share a
    page they write to) leave one of the two there: ``PagedKVCache.extend``
    gives every sequence its own."""
    if qkv.dim() != 3 or qkv.shape[:2] != (plan.tokens, plan.heads + 2 * plan.kv_heads):
        raise ValueError(f"qkv must be [{plan.tokens}, {plan.heads + 2 * plan.kv_heads}, D]; got {tuple(qkv.shape)}")
    D, H, KVH = qkv.shape[2], plan.heads, plan.kv_heads
    _check_pools(k_pages, v_pages, block_table, plan, qkv)
    if k_pages.shape[3] != D:
        raise ValueError(f"D mismatch: qkv {D}, pages {k_pages.shape[3]}")
    if D % 2 or cos.shape != (plan.tokens, D) or sin.shape != cos.shape:
        raise ValueError(f"cos and sin must be [{plan.tokens}, D], D even")
    device, dtype = qkv.device, qkv.dtype
    if cos.device != device or sin.device != device or cos.dtype != dtype or sin.dtype != dtype:
        raise ValueError("cos and sin must have the device and dtype of qkv")
    if (device.type == "cuda" and dtype in (torch.bfloat16, torch.float16) and D % 16 == 0
            and _plain(qkv, cos, sin, k_pages, v_pages)):
        strides = (*_strides(k_pages, "k_pages"), *_strides(v_pages, "v_pages"))
        if _overlaps(k_pages) or _overlaps(v_pages):
            raise ValueError("rows of pages that are written must not overlap")
        qkv, cos, sin = _packed(qkv), _packed(cos), _packed(sin)
        q = qkv.new_empty((plan.tokens, H, D))
        table, row = _table_rows(block_table)
        if plan.tokens:
            plan._used()
            _launch(device, _lib().santa_paged_rope_append, qkv.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                    q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), int(dtype == torch.float16), D,
                    k_pages.shape[0], k_pages.shape[1], (_L * 6)(*strides), table.data_ptr(), row, table.shape[0],
                    ctypes.byref(plan._info), plan._data.data_ptr())
            plan._captured(block_table.shape[1] * k_pages.shape[1], True)
        return q
    wide = torch.float64 if qkv.dtype == torch.float64 else torch.float32
    x, c, s = qkv[:, :H + KVH].to(wide), cos.to(wide)[:, None], sin.to(wide)[:, None]
    turned = (x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], dim=-1) * s).to(qkv.dtype)
    token, slot = _token_slots(block_table, plan, k_pages.shape[1])
    page, row = slot // k_pages.shape[1], slot % k_pages.shape[1]
    k_pages[page, row] = turned[token, H:]
    v_pages[page, row] = qkv[token, H + KVH:]
    plan._captured(0, False)
    return turned[:, :H]


# ---------------------------------------------------------------- attention
def _weighted(p, v, seen):
    """p @ v [KVH, rows, D] over the tokens that a row attends to (seen [rows,
    n]): an infinity or a NaN among a later token's values stays out, where its
    product with a probability of 0 would be NaN."""
    bad = ~torch.isfinite(v)
    o = torch.bmm(p, v.masked_fill(bad, 0.0))
    weighs, none = ((seen & (p.detach() > 0)).to(v.dtype), (seen & ~(p.detach() > 0)).to(v.dtype))
    plus, minus = (torch.bmm(weighs, (v.detach() == x).to(v.dtype)) > 0 for x in (math.inf, -math.inf))
    lost = torch.bmm(weighs, v.detach().isnan().to(v.dtype)) + torch.bmm(none, bad.to(v.dtype)) > 0
    for where, value in ((plus, math.inf), (minus, -math.inf), (lost, math.nan)):
        o = o + torch.where(where, value, 0.0).to(o.dtype)
    return o


def _attention_expressions(q, k_pages, v_pages, block_table, plan: PagedPlan, scale: float) -> torch.Tensor:
    """paged_attention sequence by sequence, float32 (float64 for float64)."""
    N, H, D = q.shape
    page_size, KVH = k_pages.shape[1:3]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    out, t0 = [], 0
    for row, n, t in zip(plan.rows, plan.seq_lens, plan.new_tokens):
        blind = min(t, max(0, t - n))  # tokens of a negative position
        if blind:
            out.append(torch.zeros_like(q[t0:t0 + blind]))
        if t > blind:
            at = torch.arange(n, device=q.device)
            page, r = block_table[row, at // page_size].long(), at % page_size
            k = k_pages[page, r].to(wide).permute(1, 2, 0).contiguous()                      # [KVH, D, n]
            v = v_pages[page, r].to(wide).permute(1, 0, 2).contiguous()                      # [KVH, n, D]
            x = q[t0 + blind:t0 + t].to(wide).reshape(t - blind, KVH, H // KVH, D).permute(1, 0, 2, 3)
            s = torch.bmm(x.reshape(KVH, -1, D).contiguous(), k) * scale                     # [KVH, tokens * GH, n]
            pos = torch.arange(n - t + blind, n, device=q.device).repeat_interleave(H // KVH)
            s = s.masked_fill(at[None, :] > pos[:, None], float("-inf"))
            o = _weighted(torch.softmax(s, dim=-1), v, at[None, :] <= pos[:, None]) if t > 1 else \
                torch.bmm(torch.softmax(s, dim=-1), v)
            o = o.view(KVH, t - blind, H // KVH, D).permute(1, 0, 2, 3)
            out.append(o.reshape(t - blind, H, D).to(q.dtype))
        t0 += t
    return torch.cat(out) if out else torch.empty_like(q)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    plan: Union[PagedPlan, Sequence[int]], *, scale: Optional[float] = None,
                    rounded: Optional[bool] = None) -> torch.Tensor:
    """Exact attention of a batch's tokens over paged caches: q [tokens, H, D]
    (the tokens of the plan, sequence after sequence), k_pages and v_pages
    [num_pages, page_size, KVH, D] which hold the tokens themselves already,
    block_table int32 [sequences, pages] -> [tokens, H, D].  A token attends to
    the tokens of its sequence up to itself; one at a negative position gives
    zeros.  plan: a PagedPlan, or the lengths of the sequences, each with one
    new token.  scale: of the scores, positive, 1 / sqrt(D) by default.

    bf16 and f16 of head_dim 64 and 128 on a GPU run as one kernel over all
    sequences (and one that joins parts, where the tokens of a sequence are
    split).  Prefixes of the plan are read once for all their members.  Scores,
    softmax and sums are float32.  rounded: whether the probabilities are
    rounded to the 16-bit type for the second product (as in a prefill), or
    enter it as the sum of two such values, which gives the values of float32
    probabilities and takes up to a third longer where many rows read the same
    tokens.  By default they are rounded where a sequence has several new
    tokens, and more than 32 rows of them (tokens x query heads per KV head);
    up to 16 rows that pass over a KV head's tokens together are not rounded
    either way.  The expressions for other calls never round them."""
    if q.dim() != 3:
        raise ValueError(f"q must be [tokens, H, D]; got {tuple(q.shape)}")
    N, H, D = q.shape
    if not isinstance(plan, PagedPlan):
        plan = PagedPlan(plan, heads=H, kv_heads=k_pages.shape[2], device=q.device)
    if (N, H) != (plan.tokens, plan.heads):
        raise ValueError(f"the plan is for {plan.tokens} tokens of {plan.heads} heads; q has {N} of {H}")
    _check_pools(k_pages, v_pages, block_table, plan, q)
    if k_pages.shape[3] != D:
        raise ValueError(f"D mismatch: q {D}, pages {k_pages.shape[3]}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-37 < scale < 1e37:  # normal in float32, times log2(e) too
        raise ValueError(f"scale must be positive and finite; got {scale}")
    device = q.device
    if not (device.type == "cuda" and q.dtype in (torch.bfloat16, torch.float16) and D in (64, 128)
            and _plain(q, k_pages, v_pages)):
        out = _attention_expressions(q, k_pages, v_pages, block_table, plan, scale)
        plan._captured(0, False)
        return out
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if N == 0:
        return out
    try:
        sq = _strides(q, "q")
    except ValueError:
        q = _packed(q)
        sq = _strides(q, "q")
    strides = (_L * 8)(*sq, *_strides(k_pages, "k_pages"), *_strides(v_pages, "v_pages"))
    table, row = _table_rows(block_table)
    info = plan._info
    if rounded is not None and bool(info.rounded) != rounded:
        info = _PlanInfo.from_buffer_copy(info)
        info.rounded = int(rounded)
    info = ctypes.byref(info)
    lib = _lib()
    workspace = torch.empty(lib.santa_paged_workspace_size(info, D), dtype=torch.uint8, device=device)
    plan._used()
    _launch(device, lib.santa_paged_attention, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(),
            int(q.dtype == torch.float16), D, k_pages.shape[0], k_pages.shape[1], strides, table.data_ptr(), row,
            table.shape[0], info, plan._data.data_ptr(), scale, workspace.data_ptr(), workspace.numel())
    plan._captured(block_table.shape[1] * k_pages.shape[1], True)
    return out
