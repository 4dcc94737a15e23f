"""One decode shape over a paged cache, its checks done once.

Used by ``HipAttentionBackend.prepare_paged`` / ``run_paged`` (one token a
sequence) and ``prepare_paged_tokens`` / ``run_paged_tokens`` (many); as the
prepared decode of a packed batch (``hip.py``), for batches of sequences in
pages.
"""

from __future__ import annotations

import ctypes
import threading

import torch

from .. import _native
from .base import PagedBatch, refuse_grad

_BLOCK_BYTES = 16 << 20  # outputs allocated at a time, at most


def native_cache(batch: PagedBatch) -> _native.PagedCache:
    """kvssd_paged_cache of a validated batch."""
    pages, page_tokens, kv_heads, _ = batch.packed_k.shape
    sequences, max_pages = batch.page_table.shape
    return _native.PagedCache(
        batch.bits, kv_heads, batch.head_dim, batch.group_size, pages, page_tokens, sequences, max_pages,
        batch.packed_k.data_ptr(), batch.packed_v.data_ptr(), batch.scales_k.data_ptr(), batch.scales_v.data_ptr(),
        batch.page_table.data_ptr(), batch.lengths.data_ptr(),
        None if batch.weights is None else batch.weights.data_ptr(),
        None if batch.positions is None else batch.positions.data_ptr(),
    )


class PreparedPagedDecode:
    """Calling it with a query of the prepared shape, dtype and device attends over the batch as its arrays are then
    (``lengths``, ``page_table`` and pages may change in place between calls) and returns a fresh (out, lse).

    Partials go to a workspace per stream and host thread.  Outputs are rows of blocks allocated a few at a time; two
    calls never share a row.  Under graph capture every call allocates its own workspace and outputs, so that captured
    graphs share nothing with each other or with eager calls."""

    _MAX_SLOTS = 8

    def __init__(
        self, query, batch: PagedBatch, sm_scale, out_dtype, accumulate, max_length, total_tokens, window=0, sink=0, rows=64
    ):
        batch.validate()
        batch.validate_query(query)
        batch.validate_visible(window, sink, accumulate)
        self._check(query, out_dtype, max_length, total_tokens)
        self._keep(query, batch, out_dtype)
        self._args = _native.PagedDecodeArgs(
            None, None, None, None, 0, float(sm_scale), int(total_tokens), int(min(max_length, 2**31 - 1)),
            query.shape[1], _native.QUERY_DTYPES[query.dtype], int(self._out_dtype != torch.float32), int(accumulate),
            min(window, 2**31 - 1), min(sink, 2**31 - 1), 0,
        )
        self._plan("kvssd_hip_paged_decode", query, rows)

    @staticmethod
    def _check(query, out_dtype, max_length, total_tokens) -> None:
        if query.device.type != "cuda":
            raise ValueError(f"HIP backend requires ROCm GPU tensors, got {query.device.type}")
        if query.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise ValueError(f"unsupported query dtype {query.dtype}")
        if out_dtype is not None and out_dtype not in (torch.float32, query.dtype):
            raise ValueError(f"out_dtype must be torch.float32 or the query's dtype {query.dtype}, got {out_dtype}")
        if max_length < 0 or total_tokens < 0:
            raise ValueError("max_length and total_tokens must be >= 0")

    def _keep(self, query, batch: PagedBatch, out_dtype) -> None:
        self._batch = batch  # keeps the arrays alive
        self._device = query.device
        self._index = query.device.index if query.device.index is not None else torch.cuda.current_device()
        self._qsize, self._qdtype = query.shape, query.dtype
        self._out_dtype = torch.float32 if out_dtype is None else out_dtype
        self._cache = native_cache(batch)
        self._cache_addr = ctypes.addressof(self._cache)

    def _plan(self, entry: str, query, rows: int) -> None:
        lib = _native.load()
        need = ctypes.c_size_t(0)
        plan = getattr(lib, entry + "_workspace_bytes")
        _native.check(
            plan(self._cache_addr, ctypes.addressof(self._args), ctypes.byref(need)), entry + "_workspace_bytes"
        )
        self._need = int(need.value)
        self._entry, self._fn = entry, getattr(lib, entry)
        out_bytes = query.numel() * self._out_dtype.itemsize + 4 * query.shape[0] * query.shape[1]
        self._rows = max(1, min(rows, _BLOCK_BYTES // max(out_bytes, 1)))
        # (stream, thread): [args, its address, next row, outs, lses, workspace]
        self._slots: dict[tuple[int, int], list] = {}

    def _slot(self, old: list | None, rows: int) -> list:
        if old is None:
            args = type(self._args).from_buffer_copy(self._args)
            work = torch.empty((max(self._need, 1),), dtype=torch.uint8, device=self._device)
            args.workspace, args.workspace_bytes = work.data_ptr(), work.numel()
        else:
            args, work = old[0], old[5]
        outs = torch.empty((rows, *self._qsize), dtype=self._out_dtype, device=self._device).unbind(0)
        lses = torch.empty((rows, *self._qsize[:2]), dtype=torch.float32, device=self._device).unbind(0)
        return [args, ctypes.addressof(args), 0, outs, lses, work]

    def _match(self, query: torch.Tensor) -> None:
        if query.dtype is not self._qdtype or query.shape != self._qsize or query.get_device() != self._index:
            raise ValueError(
                f"query {tuple(query.shape)} {query.dtype} on {query.device} does not match the prepared decode "
                f"({tuple(self._qsize)} {self._qdtype} on {self._device})"
            )
        refuse_grad(query)

    def __call__(self, query: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        self._match(query)
        if not query.is_contiguous() or query.data_ptr() % 16:  # the kernel reads 16 bytes at a time
            query = query.clone(memory_format=torch.contiguous_format)
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self._launch(query.data_ptr())
        return self._launch(query.data_ptr())

    def _launch(self, query, *lists: int | None) -> tuple[torch.Tensor, torch.Tensor]:
        from .hip import current_stream_handle

        handle = current_stream_handle(self._index)
        if torch.cuda.is_current_stream_capturing():
            slot = self._slot(None, 1)
        else:
            key = (handle, threading.get_ident())
            slot = self._slots.get(key)
            if slot is None or slot[2] == self._rows:
                if slot is None and len(self._slots) >= self._MAX_SLOTS:
                    self._slots.pop(next(iter(self._slots)), None)
                slot = self._slots[key] = self._slot(slot, self._rows)
        row = slot[2]
        slot[2] = row + 1
        args, out, lse = slot[0], slot[3][row], slot[4][row]
        args.query, args.out, args.lse = query, out.data_ptr(), lse.data_ptr()
        if lists:
            args.offsets, args.parents = lists
        rc = self._fn(self._cache_addr, slot[1], handle)
        if rc:
            _native.check(rc, self._entry)
        return out, lse


class PreparedPagedTokens(PreparedPagedDecode):
    """As PreparedPagedDecode for many new tokens a sequence: calling it with a query [tokens, query_heads, head_dim] of
    the prepared shape (any token and head strides), the sequences' ``offsets`` in it and, for trees, the tokens'
    ``parents`` returns a fresh (out, lse).  Workspaces and outputs as there."""

    def __init__(self, query, batch: PagedBatch, sm_scale, out_dtype, window, sink, max_length, total_tokens, rows=64):
        batch.validate()
        batch.validate_tokens(query)
        batch.validate_visible(window, sink)
        self._check(query, out_dtype, max_length, total_tokens)
        self._keep(query, batch, out_dtype)
        heads = _native.Heads(None, None, 0, 0, 0, 0, query.shape[1], 0)
        self._args = _native.PagedTokensArgs(
            heads, None, None, None, None, None, 0, float(sm_scale), query.shape[0], int(total_tokens),
            int(min(max_length, 2**31 - 1)), min(window, 2**31 - 1), min(sink, 2**31 - 1),
            _native.QUERY_DTYPES[query.dtype], int(self._out_dtype != torch.float32), 0,
        )
        self._plan("kvssd_hip_paged_tokens", query, rows)

    def __call__(
        self, query: torch.Tensor, offsets: torch.Tensor, parents: torch.Tensor | None = None
    ) -> tuple[torch.Tensor, torch.Tensor]:
        self._match(query)
        self._batch.validate_lists(query.shape[0], offsets, parents)
        token, head, one = query.stride()
        if one != 1 or query.data_ptr() % 16 or token * query.itemsize % 16 or head * query.itemsize % 16:
            query = query.clone(memory_format=torch.contiguous_format)  # the kernel reads 16 bytes at a time
        offsets = offsets if offsets.is_contiguous() else offsets.contiguous()
        if parents is not None and not parents.is_contiguous():
            parents = parents.contiguous()
        heads = _native.Heads(query.data_ptr(), None, query.stride(0), query.stride(1), 0, 0, query.shape[1], 0)
        lists = offsets.data_ptr(), None if parents is None else parents.data_ptr()
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                return self._launch(heads, *lists)
        return self._launch(heads, *lists)
