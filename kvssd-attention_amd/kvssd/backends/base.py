"""Attention backend contract (reference: src/kvssd/backends/base.py:9-69).

A backend consumes a ``PackedBatch`` (query ``[QH, D]``, packed K/V
``[NB, BT, KVH, D*bits/8]`` uint8, fp16 scales ``[NB, BT, KVH, D/g]``, valid
token counts ``[NB]`` int32) and returns the softmax-normalised output
``[QH, D]`` fp32 with its log-sum-exp ``[QH]`` fp32.  Returning the
log-normaliser is what lets independently computed chunks merge exactly.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Protocol, runtime_checkable

import torch
from torch.autograd import forward_ad


def refuse_grad(*tensors: torch.Tensor | None) -> None:
    """The generation operators have no derivative, backward or forward: say so, rather than cut the graph or drop a
    tangent."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("this operator has no backward pass; call it under torch.no_grad() or on detached tensors")
    if getattr(forward_ad, "_current_level", 0) >= 0:  # (within forward_ad.dual_level only)
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise ValueError("this operator has no forward derivative; call it on the tensors' primal values")


@dataclass(frozen=True)
class BackendAvailability:
    name: str
    available: bool
    accelerated: bool
    direct: bool
    reason: str
    device_type: str


@dataclass(frozen=True)
class PackedBatch:
    packed_k: torch.Tensor
    packed_v: torch.Tensor
    scales_k: torch.Tensor
    scales_v: torch.Tensor
    valid_tokens: torch.Tensor
    bits: int
    group_size: int

    def validate(self, query: torch.Tensor) -> None:
        """Raise ValueError on a malformed batch (messages as src/kvssd/backends/base.py:29-55)."""
        if query.ndim != 2:
            raise ValueError("query must be [query_heads, head_dim]")
        if self.packed_k.ndim != 4 or self.packed_k.shape != self.packed_v.shape:
            raise ValueError("packed KV must match [blocks,tokens,kv_heads,packed_dim]")
        if self.scales_k.ndim != 4 or self.scales_k.shape != self.scales_v.shape:
            raise ValueError("KV scales must match [blocks,tokens,kv_heads,groups]")
        if self.valid_tokens.shape != (self.packed_k.shape[0],):
            raise ValueError("valid_tokens must contain one count per block")
        if self.bits not in (2, 4):
            raise ValueError("bits must be 2 or 4")
        head_dim = query.shape[-1]
        if self.group_size <= 0 or head_dim % self.group_size:
            raise ValueError("group_size must divide head_dim")
        if self.packed_k.shape[-1] != head_dim * self.bits // 8:
            raise ValueError("packed dimension does not match query head dimension")
        if query.shape[0] % self.packed_k.shape[2]:
            raise ValueError("query heads must be divisible by KV heads")
        tensors = (self.packed_k, self.packed_v, self.scales_k, self.scales_v, self.valid_tokens)
        if any(t.device != query.device for t in tensors):
            raise ValueError("query and packed batch must share a device")


@dataclass(frozen=True)
class PagedBatch:
    """A paged packed cache: a pool of pages in the PackedBatch layout and, per
    sequence, the pages that hold it.

    * ``packed_k``, ``packed_v``: uint8 ``[pages, page_tokens, KVH, D*bits/8]``;
      ``scales_k``, ``scales_v``: fp16 ``[pages, page_tokens, KVH, D/g]``;
    * ``page_table``: int32 ``[sequences, max_pages]``; slot s of sequence b lies
      in page ``page_table[b, s // page_tokens]``, row ``s % page_tokens``;
    * ``lengths``: int32 ``[sequences]``, slots in use;
    * ``weights`` (fp32) and ``positions`` (int32), or None: ``[sequences,
      max_pages * page_tokens]``, each slot's summed attention weight and its
      token's position.

    Several sequences may name the same page, to be attended; appending and
    eviction write, and the pages they write have to be the sequence's own.

    No counterpart in the reference, whose batches are one sequence's blocks."""

    packed_k: torch.Tensor
    packed_v: torch.Tensor
    scales_k: torch.Tensor
    scales_v: torch.Tensor
    page_table: torch.Tensor
    lengths: torch.Tensor
    bits: int
    group_size: int
    weights: torch.Tensor | None = None
    positions: torch.Tensor | None = None

    @property
    def head_dim(self) -> int:
        return self.scales_k.shape[-1] * self.group_size

    @property
    def capacity(self) -> int:
        """Slots a sequence's row of the page table can name."""
        return self.page_table.shape[1] * self.packed_k.shape[1]

    def validate(self) -> None:
        """Raise ValueError on a malformed cache."""
        if self.bits not in (2, 4):
            raise ValueError("bits must be 2 or 4")
        if self.packed_k.ndim != 4 or self.packed_k.shape != self.packed_v.shape:
            raise ValueError("packed pages must match [pages,tokens,kv_heads,packed_dim]")
        if self.scales_k.ndim != 4 or self.scales_k.shape != self.scales_v.shape:
            raise ValueError("page scales must match [pages,tokens,kv_heads,groups]")
        if self.scales_k.shape[:3] != self.packed_k.shape[:3]:
            raise ValueError("scale dimension mismatch")
        if self.group_size < 32 or self.group_size & (self.group_size - 1):
            raise ValueError("group_size must be a power of two, 32 or more, that divides head_dim")
        if self.packed_k.shape[-1] * 8 != self.head_dim * self.bits:
            raise ValueError("packed dimension does not match scales and group_size")
        if self.page_table.ndim != 2 or self.lengths.shape != (self.page_table.shape[0],):
            raise ValueError("page_table must be [sequences,max_pages] and lengths [sequences]")
        slots = (self.page_table.shape[0], self.capacity)
        device = self.packed_k.device
        for name, t, dtype in (
            ("packed KV", self.packed_k, torch.uint8), ("packed KV", self.packed_v, torch.uint8),
            ("scales", self.scales_k, torch.float16), ("scales", self.scales_v, torch.float16),
            ("page_table", self.page_table, torch.int32), ("lengths", self.lengths, torch.int32),
            ("weights", self.weights, torch.float32), ("positions", self.positions, torch.int32),
        ):
            if t is None:
                continue
            if t.dtype is not dtype:
                raise ValueError(f"{name} must be {str(dtype).removeprefix('torch.')}")
            if t.device != device:
                raise ValueError("a paged cache must lie on one device")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if name in ("weights", "positions") and t.shape != slots:
                raise ValueError(f"{name} must be [sequences, max_pages * page_tokens]")

    def validate_query(self, query: torch.Tensor) -> None:
        if query.ndim != 3 or query.shape[0] != self.lengths.shape[0]:
            raise ValueError("query must be [sequences, query_heads, head_dim]")
        if query.shape[2] != self.head_dim:
            raise ValueError("packed dimension does not match query head dimension")
        if query.shape[1] == 0 or query.shape[1] % self.packed_k.shape[2]:
            raise ValueError("query heads must be divisible by KV heads")
        if query.device != self.packed_k.device:
            raise ValueError("query and paged cache must share a device")

    def validate_tokens(self, query: torch.Tensor) -> None:
        """Of a query with many tokens a sequence."""
        if query.ndim != 3:
            raise ValueError("query must be [tokens, query_heads, head_dim]")
        if query.shape[2] != self.head_dim:
            raise ValueError("packed dimension does not match query head dimension")
        if query.shape[1] == 0 or query.shape[1] % self.packed_k.shape[2]:
            raise ValueError("query heads must be divisible by KV heads")
        if query.device != self.packed_k.device:
            raise ValueError("query and paged cache must share a device")

    def validate_lists(self, tokens: int, offsets: torch.Tensor, parents: torch.Tensor | None) -> None:
        """Of the sequences' places among ``tokens`` tokens and the tokens' parents."""
        for name, t, count in (("offsets", offsets, self.lengths.shape[0] + 1), ("parents", parents, tokens)):
            if t is None:
                continue
            if t.dtype != torch.int32 or t.shape != (count,) or t.device != self.lengths.device:
                raise ValueError(f"{name} must be int32 [{count}] on {self.lengths.device}")

    def validate_visible(self, window: int, sink: int, accumulate: bool = False) -> None:
        if window < 0 or sink < 0:
            raise ValueError("window and sink must be >= 0")
        if window and accumulate:
            raise ValueError("weights are summed over whole sequences, not over a window")
        if accumulate and self.weights is None:
            raise ValueError("accumulate needs a cache with weights")


@runtime_checkable
class AttentionBackend(Protocol):
    name: str

    def probe(self, device: torch.device) -> BackendAvailability: ...

    def run(
        self,
        query: torch.Tensor,
        batch: PackedBatch,
        sm_scale: float,
    ) -> tuple[torch.Tensor, torch.Tensor]: ...
