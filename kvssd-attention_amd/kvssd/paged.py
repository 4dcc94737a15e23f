"""A packed cache that grows token by token: pages, append, attention, eviction.

The reference's cache is written once (src/kvssd/store.py:46-63) and then only
read, one sequence at a time.  Here a pool of pages in the same packed layout
holds many sequences:

* :func:`append_tokens` -- new tokens' keys (rotated on the way) and values,
  quantised by the framework's codec into their sequences' pages;
* ``HipAttentionBackend.run_paged`` / ``prepare_paged`` -- one new token's
  attention per sequence, optionally summing each slot's attention weight;
* ``run_paged_tokens`` / ``prepare_paged_tokens`` -- attention of many new tokens
  a sequence: prompts, chunks of prompts, trees of drafted tokens;
* :func:`keep_tokens` -- the accepted ones of a sequence's drafted tokens moved
  together, the others dropped;
* :func:`evict_tokens` -- every sequence cut to a budget of slots by that sum;
* :class:`PagedKVCache` -- the pool, its free pages, the sequences' lengths and
  positions, and these operators over them.

Attention takes a sliding window and a few first tokens that stay visible.

The functions launch on the current stream and never wait for the GPU.
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence

import torch

from . import _native
from .backends import AttentionBackend, PackedBatch, PagedBatch, resolve_attention_backend
from .backends.hip import current_stream_handle, on_device
from .backends.paged import native_cache
from .rotary import _DTYPES, Rotary, check_heads, empty_heads, heads_of, refuse_grad


def _gpu_index(batch: PagedBatch) -> int:
    device = batch.packed_k.device
    if device.type != "cuda":
        raise ValueError(f"a paged cache requires ROCm GPU tensors, got {device.type}")
    return device.index if device.index is not None else torch.cuda.current_device()


def _int32(t: torch.Tensor, name: str, count: int, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != (count,) or t.device != device:
        raise ValueError(f"{name} must be int32 [{count}] on {device}")
    return t if t.is_contiguous() else t.contiguous()


def append_tokens(
    batch: PagedBatch,
    keys: torch.Tensor,
    values: torch.Tensor,
    *,
    offsets: torch.Tensor | None = None,
    rotary: Rotary | None = None,
    query: torch.Tensor | None = None,
    first_positions: torch.Tensor | None = None,
    lengths_out: torch.Tensor | None = None,
    parents: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor]:
    """Write new tokens behind their sequences' slots: (rotated query or None, new lengths).

    ``keys`` and ``values`` are [tokens, kv_heads, head_dim] (float16, bfloat16 or float32, any token and head
    strides).  With ``offsets`` (int32 [sequences + 1]) tokens offsets[b] .. offsets[b+1]-1 belong to sequence b;
    without, there is one token a sequence.  A sequence's i-th new token goes to slot lengths[b] + i (dropped past
    the page table's end or where the table names no page) and has position first_positions[b] + i (int32
    [sequences]; default: its slot).  The pages of those slots must be no other sequence's.  With ``rotary`` the keys
    are turned by their positions and rounded to their type before they are quantised, and so is ``query`` [tokens,
    query_heads, head_dim], if given.  Where the batch has them, the slots' positions are stored and their weights set
    to 0.  Tokens of no sequence (before offsets[0], from offsets[sequences] on) are dropped, their queries turned as
    at position 0.

    With ``parents`` (int32 [tokens]) a sequence's new tokens are a tree, as ``run_paged_tokens`` takes it: the i-th
    goes to its slot all the same, and its position is the first's plus its depth (0 of a token whose parent is none of
    the sequence's earlier new tokens).

    ``batch.lengths`` stays as it is unless it is passed as ``lengths_out`` (one token a sequence only); by default
    the new lengths are a new tensor."""
    batch.validate()
    index = _gpu_index(batch)
    device = batch.packed_k.device
    dtype, tokens = keys.dtype, keys.shape[0] if keys.ndim else 0
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype}")
    kv_heads, sequences = batch.packed_k.shape[2], batch.lengths.shape[0]
    for name, t in (("keys", keys), ("values", values)):
        check_heads(t, name, tokens, batch.head_dim, dtype, device)
        if t.shape[1] != kv_heads:
            raise ValueError("keys and values must be [tokens, kv_heads, head_dim]")
    if query is not None:
        if rotary is None:
            raise ValueError("a query is only taken to be rotated")
        check_heads(query, "query", tokens, batch.head_dim, dtype, device)
    if rotary is not None:
        if rotary.head_dim != batch.head_dim:
            raise ValueError("rotary head_dim differs from the cache's")
        if rotary.frequencies.device != device:
            raise ValueError("rotary frequencies and paged cache must share a device")
    refuse_grad(keys, values, query)
    if offsets is not None:
        offsets = _int32(offsets, "offsets", sequences + 1, device)
    elif tokens != sequences:
        raise ValueError("without offsets there is one token a sequence")
    if first_positions is not None:
        first_positions = _int32(first_positions, "first_positions", sequences, device)
    if parents is not None:
        parents = _int32(parents, "parents", tokens, device)
    if lengths_out is None:
        lengths_out = torch.empty_like(batch.lengths)
    elif _int32(lengths_out, "lengths_out", sequences, device) is not lengths_out:
        raise ValueError("lengths_out must be contiguous")
    keys, values = (t if t.stride(2) == 1 else t.contiguous() for t in (keys, values))
    turned, turns = None, ()
    if query is not None:
        query = query if query.stride(2) == 1 else query.contiguous()
        turned = empty_heads(query)
        if query.shape[1]:
            turns = heads_of(query, turned)
    args = _native.PagedAppendArgs(
        heads_of(keys), heads_of(values), turns, tokens, None if offsets is None else offsets.data_ptr(),
        None if first_positions is None else first_positions.data_ptr(),
        None if parents is None else parents.data_ptr(),
        None if rotary is None else ctypes.pointer(rotary.spec()), lengths_out.data_ptr(), _DTYPES[dtype], 0,
    )
    cache = native_cache(batch)
    with on_device(index):
        rc = _native.load().kvssd_hip_paged_append(
            ctypes.addressof(cache), ctypes.addressof(args), current_stream_handle(index)
        )
    if rc:
        _native.check(rc, "kvssd_hip_paged_append")
    return turned, lengths_out


def evict_tokens(
    batch: PagedBatch, budget: int, *, sink: int = 0, recent: int = 0
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence to at most ``budget`` slots: new (lengths, weights, positions).

    Kept are the slots whose position is below ``sink`` or among the last ``recent`` (above the sequence's largest
    position - recent), then those of the largest weights (NaN counts as -inf); of equals the lower slot, and
    ``budget`` in all.  The n-th kept slot at or past the budget moves into the n-th freed slot before it: only
    those rows are copied, within the sequence's pages (which no other sequence, and no second place of the table,
    may name).  Every slot of a sequence that is cut has to lie in a page of the pool: a row without one cannot move,
    and the slot that it was to fill would keep an evicted token's under its own weight and position (attention and
    append skip such slots; :class:`PagedKVCache` makes none).  The batch's own lengths, weights and positions stay as
    they are; the returned ones describe the cache after the cut (weight 0 and position -1 past the new length)."""
    batch.validate()
    index = _gpu_index(batch)
    if batch.weights is None or batch.positions is None:
        raise ValueError("eviction needs a cache with weights and positions")
    if budget < 1:
        raise ValueError("budget must be positive")
    if sink < 0 or recent < 0:
        raise ValueError("sink and recent counts must be non-negative")
    if sink + recent > budget:
        raise ValueError("sink and recent must fit the budget")
    budget = min(budget, 2**31 - 1)
    lengths, weights, positions = (torch.empty_like(t) for t in (batch.lengths, batch.weights, batch.positions))
    lib = _native.load()
    cache = native_cache(batch)
    args = _native.PagedEvictArgs(
        budget, min(sink, budget), min(recent, budget), 0, lengths.data_ptr(), weights.data_ptr(), positions.data_ptr()
    )
    need = ctypes.c_size_t(0)
    where = ctypes.addressof(cache), ctypes.addressof(args)
    _native.check(lib.kvssd_hip_paged_evict_workspace_bytes(*where, ctypes.byref(need)), "kvssd_hip_paged_evict")
    work = torch.empty((need.value,), dtype=torch.uint8, device=batch.packed_k.device)
    args.workspace, args.workspace_bytes = work.data_ptr(), need.value
    with on_device(index):
        rc = lib.kvssd_hip_paged_evict(*where, current_stream_handle(index))
    if rc:
        _native.check(rc, "kvssd_hip_paged_evict")
    return lengths, weights, positions


def keep_tokens(
    batch: PagedBatch, drafted: torch.Tensor, kept: torch.Tensor, *, lengths_out: torch.Tensor | None = None
) -> torch.Tensor:
    """Keep some of each sequence's last ``drafted`` (int32 [sequences]) slots and drop the others: the new lengths.

    ``kept`` (int32 [sequences, width]) lists the kept ones' places among them, ascending; a sequence's list ends at the
    first entry that is not above the one before it or not a drafted token's (-1, say).  With base = length - drafted,
    slot base + j takes the row of slot base + kept[b, j], and its weight and position where the cache has them; the new
    length is base plus the list's.  Rows move in place, within the sequence's pages (which no other sequence may name),
    and each of those slots has to lie in a page of the pool: a row without one does not move.

    ``batch.lengths`` stays as it is unless it is passed as ``lengths_out``; by default the new lengths are a new
    tensor."""
    batch.validate()
    index = _gpu_index(batch)
    device, sequences = batch.packed_k.device, batch.lengths.shape[0]
    drafted = _int32(drafted, "drafted", sequences, device)
    if kept.dtype != torch.int32 or kept.ndim != 2 or kept.shape[0] != sequences or kept.device != device:
        raise ValueError(f"kept must be int32 [{sequences}, width] on {device}")
    kept = kept if kept.is_contiguous() else kept.contiguous()
    if lengths_out is None:
        lengths_out = torch.empty_like(batch.lengths)
    elif _int32(lengths_out, "lengths_out", sequences, device) is not lengths_out:
        raise ValueError("lengths_out must be contiguous")
    args = _native.PagedKeepArgs(drafted.data_ptr(), kept.data_ptr(), lengths_out.data_ptr(), kept.shape[1], 0)
    cache = native_cache(batch)
    with on_device(index):
        rc = _native.load().kvssd_hip_paged_keep(
            ctypes.addressof(cache), ctypes.addressof(args), current_stream_handle(index)
        )
    if rc:
        _native.check(rc, "kvssd_hip_paged_keep")
    return lengths_out


class PagedKVCache:
    """The packed cache of one layer for up to ``sequences`` sequences at a time, in pages that they take from a
    common pool as they grow and give back as they are cut or end.

    Lengths and free pages are kept on the host (they follow from the calls, so that no call waits for the GPU),
    with a copy of the lengths on the device for the kernels.  ``track_weights`` keeps each slot's position and
    summed attention weight, which :meth:`evict` needs: 8 bytes for each of the ``max_pages`` * ``page_tokens`` slots
    that each sequence may grow to (``max_pages`` defaults to the whole pool), and a cut writes as many again.  From the
    first cut on, positions differ from slots and are copied from the host at every append.  One stream at a time:
    calls on different streams have to be ordered by the caller.  :meth:`append`, :meth:`keep` and :meth:`evict` change
    host state and so cannot be captured in a graph; the operators under them can.

    A step with drafted tokens is :meth:`append` with their ``parents``, :meth:`attend_tokens` with the same, and
    :meth:`keep` with each sequence's accepted path; until then the cache holds all of them, and only those calls and
    :meth:`clear` are taken."""

    def __init__(
        self,
        pages: int,
        page_tokens: int,
        kv_heads: int,
        head_dim: int,
        *,
        bits: int = 4,
        group_size: int = 32,
        sequences: int = 1,
        max_pages: int | None = None,
        track_weights: bool = False,
        device: str | torch.device = "cuda",
        attention_backend: str | AttentionBackend | None = None,
    ):
        if min(pages, page_tokens, kv_heads, head_dim, sequences) < 1:
            raise ValueError("pages, page_tokens, kv_heads, head_dim and sequences must be positive")
        if bits not in (2, 4):
            raise ValueError("bits must be 2 or 4")
        if head_dim % 32 or head_dim > 256:
            raise ValueError("head_dim must be a multiple of 32 up to 256")
        if group_size < 32 or group_size & (group_size - 1) or head_dim % group_size:
            raise ValueError("group_size must be a power of two, 32 or more, that divides head_dim")
        max_pages = pages if max_pages is None else max_pages
        if max_pages < 1:
            raise ValueError("max_pages must be positive")
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:  # this GPU, whichever is the current one later on
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.page_tokens, self.max_pages, self.sequences = page_tokens, max_pages, sequences
        self.backend = resolve_attention_backend(attention_backend, device)
        shape = (pages, page_tokens, kv_heads)
        codes = [torch.zeros((*shape, head_dim * bits // 8), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros((*shape, head_dim // group_size), dtype=torch.float16, device=device) for _ in range(2)]
        slots = (sequences, max_pages * page_tokens)
        self.batch = PagedBatch(
            *codes, *scales,
            torch.full((sequences, max_pages), -1, dtype=torch.int32, device=device),
            torch.zeros((sequences,), dtype=torch.int32, device=device), bits, group_size,
            torch.zeros(slots, dtype=torch.float32, device=device) if track_weights else None,
            torch.full(slots, -1, dtype=torch.int32, device=device) if track_weights else None,
        )
        self.batch.validate()
        self._free = list(range(pages - 1, -1, -1))  # taken from the end: lowest id first
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self.lengths = [0] * sequences  # slots in use, per sequence
        self.next_positions = [0] * sequences  # position of the next token, per sequence
        self._plan: tuple | None = None  # of `attend`: what it was planned for, and the prepared decode
        self._tokens_plan: tuple | None = None  # of `attend_tokens`, the same
        # the last append's tokens of each sequence, while they can be kept in part, and whether they are a tree
        self._latest: list[int] | None = None
        self._drafting = False
        # of a tree: its parents, on the host or on their way there until the event, and the sequences' places among them
        self._tree: tuple[list[int] | torch.Tensor, torch.cuda.Event | None, list[int]] | None = None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _host_to_device(self, values: list[int] | list[list[int]]) -> torch.Tensor:
        host = torch.tensor(values, dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        return host.to(self.device, non_blocking=True)

    def _resize(self, lengths: Sequence[int]) -> None:
        """Take or give back pages so that sequence b holds lengths[b] slots; nothing changes where the pool or a
        row of the page table is too small."""
        room = self.page_tokens
        if not any(n > len(have) * room or n <= (len(have) - 1) * room for n, have in zip(lengths, self._pages)):
            return
        want = [-(-n // room) for n in lengths]
        if max(want) > self.max_pages:
            raise ValueError(f"a sequence may hold at most {self.max_pages * self.page_tokens} tokens")
        back = sum(max(0, len(have) - n) for have, n in zip(self._pages, want))
        more = sum(max(0, n - len(have)) for have, n in zip(self._pages, want))
        if more > len(self._free) + back:
            raise RuntimeError(f"the pool has {len(self._free) + back} free pages, {more} are needed")
        rows = []
        for b, n in enumerate(want):
            if len(self._pages[b]) != n:
                rows.append(b)
            while len(self._pages[b]) > n:
                self._free.append(self._pages[b].pop())
        for b, n in enumerate(want):
            while len(self._pages[b]) < n:
                self._pages[b].append(self._free.pop())
        if rows:
            table = [self._pages[b] + [-1] * (self.max_pages - want[b]) for b in rows]
            if len(rows) == self.sequences:
                self.batch.page_table.copy_(self._host_to_device(table))
            else:
                self.batch.page_table[self._host_to_device(rows).long()] = self._host_to_device(table)

    def _no_drafts(self) -> None:
        if self._drafting:
            raise RuntimeError("the cache holds drafted tokens; keep those that are accepted first")

    def append(
        self,
        keys: torch.Tensor,
        values: torch.Tensor,
        counts: Sequence[int] | None = None,
        *,
        rotary: Rotary | None = None,
        query: torch.Tensor | None = None,
        parents: torch.Tensor | Sequence[int] | None = None,
    ) -> torch.Tensor | None:
        """Append counts[b] tokens to sequence b (default: one to each), as they lie in ``keys`` and ``values``
        [tokens, kv_heads, head_dim], sequence after sequence; returns the rotated query, if one was given.

        ``parents`` [tokens] (int32 on the cache's device, or numbers) makes each sequence's tokens a tree of drafted
        ones (see :func:`append_tokens`), of which :meth:`keep` has to take those that are accepted next."""
        self._no_drafts()
        one = counts is None
        counts = [1] * self.sequences if one else [int(n) for n in counts]
        if len(counts) != self.sequences or min(counts) < 0:
            raise ValueError("counts must hold one non-negative number per sequence")
        if keys.ndim != 3 or sum(counts) != keys.shape[0]:
            raise ValueError("counts must add up to the number of tokens")
        after = [n + more for n, more in zip(self.lengths, counts)]
        offsets = None
        if not one and any(n != 1 for n in counts):
            ends = [0]
            for n in counts:
                ends.append(ends[-1] + n)
            offsets = self._host_to_device(ends)
        first = None
        if self.next_positions != self.lengths:
            first = self._host_to_device(self.next_positions)
        drafting, given = parents is not None and any(counts), None
        if parents is not None:
            given = parents if isinstance(parents, torch.Tensor) else [int(x) for x in parents]
            parents = self._parents(given, keys.shape[0])
        held = list(self.lengths)
        self._resize(after)
        try:
            turned, lengths = append_tokens(
                self.batch, keys, values, offsets=offsets, rotary=rotary, query=query, first_positions=first,
                lengths_out=self.batch.lengths if offsets is None else None, parents=parents,
            )
        except Exception:
            self._resize(held)
            raise
        if offsets is not None:
            self.batch.lengths.copy_(lengths)
        self.lengths = after
        self.next_positions = [n + more for n, more in zip(self.next_positions, counts)]
        self._latest, self._drafting = counts, drafting
        self._tree = self._tree_of(given, counts) if drafting else None
        return turned

    def _parents(self, parents: torch.Tensor | Sequence[int], tokens: int) -> torch.Tensor:
        if not isinstance(parents, torch.Tensor):
            parents = [int(x) for x in parents]
            if len(parents) != tokens:
                raise ValueError("parents must hold one number per token")
            parents = self._host_to_device([x if -1 <= x < tokens else -1 for x in parents])
        return parents

    def _tree_of(self, parents: torch.Tensor | list[int], counts: Sequence[int]) -> tuple:
        """What :meth:`keep` checks paths by.  A tensor on the GPU is on its way to the host when this returns."""
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        if not isinstance(parents, torch.Tensor):
            return parents, None, starts
        if parents.device.type != "cuda":
            return parents.tolist(), None, starts
        with on_device(self.device.index):
            host = torch.empty(parents.shape, dtype=parents.dtype, pin_memory=True)
            host.copy_(parents, non_blocking=True)
            copied = torch.cuda.Event()
            copied.record()
        return host, copied, starts

    def _check_paths(self, paths: Sequence[Sequence[int]]) -> None:
        """Kept tokens have the positions that follow the slots before them: they are a row's first ones, or each the
        child of the one before it."""
        if not self._drafting:
            if any(path != list(range(len(path))) for path in paths):
                raise ValueError("of tokens in a row the first ones are kept")
            return
        parents, copied, starts = self._tree
        if copied is not None:
            copied.synchronize()
            parents = parents.tolist()
            self._tree = parents, None, starts
        for path, start in zip(paths, starts):
            for above, x in zip([-1, *path], path):
                up = parents[start + x]
                if (up if 0 <= up < x else -1) != above:
                    raise ValueError("a tree's path must lead from a token without a parent from child to child")

    def keep(self, paths: Sequence[Sequence[int] | None]) -> None:
        """Of the last append's tokens, keep paths[b] of sequence b -- their places among its tokens, ascending: of tokens
        in a row the first ones, of a tree a path from one without a parent from child to child -- and drop the others
        (:func:`keep_tokens`); pages behind are given back.  None keeps all, of a sequence whose tokens are no tree.  Where
        the append's parents were a tensor, this waits until that append has read them."""
        counts = self._latest
        if counts is None:
            raise RuntimeError("there are no tokens to choose from: keep follows an append")
        if len(paths) != self.sequences:
            raise ValueError("paths must hold one list (or None) per sequence")
        chosen = []
        for path, n in zip(paths, counts):
            if path is None and self._drafting and n > 1:
                raise ValueError("a tree's tokens are kept by their path")
            path = list(range(n)) if path is None else [int(x) for x in path]
            if any(not 0 <= x < n for x in path) or any(a >= b for a, b in zip(path, path[1:])):
                raise ValueError("a path must hold ascending places among the sequence's new tokens")
            chosen.append(path)
        self._check_paths(chosen)
        width = max(len(path) for path in chosen)
        drafted = self._host_to_device(counts)
        kept = self._host_to_device([path + [-1] * (width - len(path)) for path in chosen])
        keep_tokens(self.batch, drafted, kept.view(self.sequences, width), lengths_out=self.batch.lengths)
        dropped = [n - len(path) for n, path in zip(counts, chosen)]
        self.lengths = [n - less for n, less in zip(self.lengths, dropped)]
        self.next_positions = [n - less for n, less in zip(self.next_positions, dropped)]
        self._latest, self._drafting, self._tree = None, False, None
        self._resize(self.lengths)

    def attend(
        self,
        query: torch.Tensor,
        sm_scale: float | None = None,
        *,
        out_dtype: torch.dtype | None = None,
        accumulate: bool = False,
        window: int = 0,
        sink: int = 0,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """(out, lse) of one query per sequence, [sequences, query_heads, head_dim]; see
        ``HipAttentionBackend.run_paged``.  The scale defaults to 1/sqrt(head_dim).  A ``window`` counts slots, and so is
        taken as long as none was evicted only."""
        self._no_drafts()
        self._no_cuts(window)
        scale = self.batch.head_dim ** -0.5 if sm_scale is None else sm_scale
        visible = dict(window=window, sink=sink) if window or sink else {}
        if getattr(self.backend, "name", None) != "hip":
            return self.backend.run_paged(query, self.batch, scale, out_dtype=out_dtype, accumulate=accumulate, **visible)
        shape = (query.shape, query.dtype, query.device, scale, out_dtype, accumulate, window, sink)
        self._plan = self._planned(
            self._plan, shape,
            lambda **hints: self.backend.prepare_paged(
                query, self.batch, scale, out_dtype=out_dtype, accumulate=accumulate, **hints, **visible
            ),
        )
        return self._plan[5](query)

    def _planned(self, plan: tuple | None, shape: tuple, prepare) -> tuple:
        """Checked and planned anew where the shape changes or the lengths have grown or shrunk by an eighth: between,
        the plan's hints are an eighth high at most, and the kernel goes by the lengths that there are."""
        longest, total = max(self.lengths), sum(self.lengths)
        if plan is None or plan[0] != shape or not (plan[1] <= longest <= plan[2] and plan[3] <= total <= plan[4]):
            hints = [n + n // 8 + 1 for n in (longest, total)]
            run = prepare(max_length=hints[0], total_tokens=hints[1])
            plan = (shape, longest - longest // 8, hints[0], total - total // 8, hints[1], run)
        return plan

    def _no_cuts(self, window: int) -> None:
        if window and self.next_positions != self.lengths:
            raise ValueError("a window needs slots in the order of their positions, which eviction gives up")

    def attend_tokens(
        self,
        query: torch.Tensor,
        counts: Sequence[int] | None = None,
        sm_scale: float | None = None,
        *,
        parents: torch.Tensor | Sequence[int] | None = None,
        out_dtype: torch.dtype | None = None,
        window: int = 0,
        sink: int = 0,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """(out, lse) of each sequence's last counts[b] tokens (default: one of each), [tokens, query_heads, head_dim],
        which are in the cache already: what a prompt's or a chunk's tokens see, or, with ``parents``, a tree's; see
        ``HipAttentionBackend.run_paged_tokens``.  Weights are not summed.  Scale and window as in :meth:`attend`.
        The lists are copied from the host, so that a call cannot be captured in a graph (that operator can)."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("attend_tokens copies lists from the host; capture run_paged_tokens")
        self._no_cuts(window)
        counts = [1] * self.sequences if counts is None else [int(n) for n in counts]
        if len(counts) != self.sequences or min(counts) < 0:
            raise ValueError("counts must hold one non-negative number per sequence")
        if self._drafting and (parents is None or counts != self._latest):
            raise RuntimeError("the cache holds drafted tokens; attend them with their parents, or keep the accepted ones")
        if query.ndim != 3 or sum(counts) != query.shape[0]:
            raise ValueError("counts must add up to the number of tokens")
        if any(n > length for n, length in zip(counts, self.lengths)):
            raise ValueError("a sequence holds fewer tokens than that")
        ends = [0]
        for n in counts:
            ends.append(ends[-1] + n)
        offsets = self._host_to_device(ends)
        if parents is not None:
            parents = self._parents(parents, query.shape[0])
        scale = self.batch.head_dim ** -0.5 if sm_scale is None else sm_scale
        visible = dict(window=window, sink=sink, out_dtype=out_dtype)
        if getattr(self.backend, "name", None) != "hip":
            return self.backend.run_paged_tokens(query, self.batch, scale, offsets, parents, **visible)
        shape = (query.shape, query.dtype, query.device, scale, out_dtype, window, sink)
        self._tokens_plan = self._planned(
            self._tokens_plan, shape,
            lambda **hints: self.backend.prepare_paged_tokens(query, self.batch, scale, **hints, **visible),
        )
        return self._tokens_plan[5](query, offsets, parents)

    def evict(self, budget: int, *, sink: int = 0, recent: int = 0) -> None:
        """Cut every sequence to at most ``budget`` tokens (:func:`evict_tokens`) and give back the pages behind.

        ``batch`` keeps its arrays, so that decodes prepared before, and graphs of them, go on with the cut cache."""
        self._no_drafts()
        longest = max(self.lengths)
        lengths, weights, positions = evict_tokens(self.batch, budget, sink=sink, recent=recent)
        self.batch.lengths.copy_(lengths)
        self.batch.weights[:, :longest].copy_(weights[:, :longest])  # (none of the sequences has slots behind)
        self.batch.positions[:, :longest].copy_(positions[:, :longest])
        self.lengths = [min(n, budget) for n in self.lengths]
        self._latest = None
        self._resize(self.lengths)

    def clear(self, sequence: int) -> None:
        """End a sequence: its pages go back to the pool, and its row starts empty."""
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"sequence must lie in [0, {self.sequences})")
        self.lengths[sequence] = self.next_positions[sequence] = 0
        if self._latest is not None:
            self._latest[sequence] = 0
            self._drafting = self._drafting and any(self._latest)
        self.batch.lengths[sequence].zero_()
        self._resize(self.lengths)

    def load(self, sequence: int, blocks: PackedBatch) -> None:
        """Fill an empty sequence with a packed layer's blocks (as ``gather_records`` or ``stack_blocks`` give them,
        page_tokens tokens each, all full but the last), positions counted from 0."""
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"sequence must lie in [0, {self.sequences})")
        self._no_drafts()
        if self.lengths[sequence]:
            raise ValueError("sequence is not empty")
        if (blocks.bits, blocks.group_size) != (self.batch.bits, self.batch.group_size):
            raise ValueError("blocks and cache differ in bits or group_size")
        if blocks.packed_k.shape[1:] != self.batch.packed_k.shape[1:] or blocks.scales_k.shape[1:] != self.batch.scales_k.shape[1:]:
            raise ValueError("blocks and pages differ in shape")
        valid = blocks.valid_tokens.tolist()
        if not valid:
            return
        if any(n != self.page_tokens for n in valid[:-1]) or not 0 < valid[-1] <= self.page_tokens:
            raise ValueError("every block but the last must be full")
        length = sum(valid)
        lengths = list(self.lengths)
        lengths[sequence] = length
        self._resize(lengths)
        rows = self._host_to_device(self._pages[sequence]).long()
        for name in ("packed_k", "packed_v", "scales_k", "scales_v"):
            getattr(self.batch, name)[rows] = getattr(blocks, name).to(self.device)
        if self.batch.positions is not None:
            self.batch.positions[sequence, :length] = torch.arange(length, dtype=torch.int32, device=self.device)
            self.batch.weights[sequence, :length] = 0.0
        self.batch.lengths[sequence] = length
        if self._latest is not None:
            self._latest[sequence] = 0
        self.lengths[sequence] = self.next_positions[sequence] = length
