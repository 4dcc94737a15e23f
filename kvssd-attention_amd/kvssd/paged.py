"""A packed cache that grows token by token: pages, append, attention, eviction.

The reference's cache is written once (src/kvssd/store.py:46-63) and then only
read, one sequence at a time.  Here a pool of pages in the same packed layout
holds many sequences:

* :func:`append_tokens` -- new tokens' keys (rotated on the way) and values,
  quantised by the framework's codec into their sequences' pages;
* ``HipAttentionBackend.run_paged`` / ``prepare_paged`` -- one new token's
  attention per sequence, optionally summing each slot's attention weight;
* :func:`evict_tokens` -- every sequence cut to a budget of slots by that sum;
* :class:`PagedKVCache` -- the pool, its free pages, the sequences' lengths and
  positions, and the three operators over them.

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


class PagedKVCache:
    """The packed cache of one layer for up to ``sequences`` sequences at a time, in pages that they take from a
    common pool as they grow and give back as they are cut or end.

    Lengths and free pages are kept on the host (they follow from the calls, so that no call waits for the GPU),
    with a copy of the lengths on the device for the kernels.  ``track_weights`` keeps each slot's position and
    summed attention weight, which :meth:`evict` needs: 8 bytes for each of the ``max_pages`` * ``page_tokens`` slots
    that each sequence may grow to (``max_pages`` defaults to the whole pool), and a cut writes as many again.  From the
    first cut on, positions differ from slots and are copied from the host at every append.  One stream at a time:
    calls on different streams have to be ordered by the caller.  :meth:`append` and :meth:`evict` change host state and
    so cannot be captured in a graph; the operators under them can."""

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

    def append(
        self,
        keys: torch.Tensor,
        values: torch.Tensor,
        counts: Sequence[int] | None = None,
        *,
        rotary: Rotary | None = None,
        query: torch.Tensor | None = None,
    ) -> torch.Tensor | None:
        """Append counts[b] tokens to sequence b (default: one to each), as they lie in ``keys`` and ``values``
        [tokens, kv_heads, head_dim], sequence after sequence; returns the rotated query, if one was given."""
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
        held = list(self.lengths)
        self._resize(after)
        try:
            turned, lengths = append_tokens(
                self.batch, keys, values, offsets=offsets, rotary=rotary, query=query, first_positions=first,
                lengths_out=self.batch.lengths if offsets is None else None,
            )
        except Exception:
            self._resize(held)
            raise
        if offsets is not None:
            self.batch.lengths.copy_(lengths)
        self.lengths = after
        self.next_positions = [n + more for n, more in zip(self.next_positions, counts)]
        return turned

    def attend(
        self,
        query: torch.Tensor,
        sm_scale: float | None = None,
        *,
        out_dtype: torch.dtype | None = None,
        accumulate: bool = False,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """(out, lse) of one query per sequence, [sequences, query_heads, head_dim]; see
        ``HipAttentionBackend.run_paged``.  The scale defaults to 1/sqrt(head_dim)."""
        scale = self.batch.head_dim ** -0.5 if sm_scale is None else sm_scale
        if getattr(self.backend, "name", None) != "hip":
            return self.backend.run_paged(query, self.batch, scale, out_dtype=out_dtype, accumulate=accumulate)
        # Checked and planned anew where the shape changes or the lengths have grown or shrunk by an eighth: between,
        # the plan's hints are an eighth high at most, and the kernel goes by the lengths that there are.
        shape = (query.shape, query.dtype, query.device, scale, out_dtype, accumulate)
        longest, total = max(self.lengths), sum(self.lengths)
        plan = self._plan
        if plan is None or plan[0] != shape or not (plan[1] <= longest <= plan[2] and plan[3] <= total <= plan[4]):
            hints = [n + n // 8 + 1 for n in (longest, total)]
            run = self.backend.prepare_paged(
                query, self.batch, scale, out_dtype=out_dtype, accumulate=accumulate, max_length=hints[0],
                total_tokens=hints[1],
            )
            plan = self._plan = (shape, longest - longest // 8, hints[0], total - total // 8, hints[1], run)
        return plan[5](query)

    def evict(self, budget: int, *, sink: int = 0, recent: int = 0) -> None:
        """Cut every sequence to at most ``budget`` tokens (:func:`evict_tokens`) and give back the pages behind.

        ``batch`` keeps its arrays, so that decodes prepared before, and graphs of them, go on with the cut cache."""
        longest = max(self.lengths)
        lengths, weights, positions = evict_tokens(self.batch, budget, sink=sink, recent=recent)
        self.batch.lengths.copy_(lengths)
        self.batch.weights[:, :longest].copy_(weights[:, :longest])  # (none of the sequences has slots behind)
        self.batch.positions[:, :longest].copy_(positions[:, :longest])
        self.lengths = [min(n, budget) for n in self.lengths]
        self._resize(self.lengths)

    def clear(self, sequence: int) -> None:
        """End a sequence: its pages go back to the pool, and its row starts empty."""
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"sequence must lie in [0, {self.sequences})")
        self.lengths[sequence] = self.next_positions[sequence] = 0
        self.batch.lengths[sequence].zero_()
        self._resize(self.lengths)

    def load(self, sequence: int, blocks: PackedBatch) -> None:
        """Fill an empty sequence with a packed layer's blocks (as ``gather_records`` or ``stack_blocks`` give them,
        page_tokens tokens each, all full but the last), positions counted from 0."""
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"sequence must lie in [0, {self.sequences})")
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
        self.lengths[sequence] = self.next_positions[sequence] = length
