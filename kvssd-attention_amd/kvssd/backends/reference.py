"""Portable PyTorch dequantize-then-attend backend.

Same contract and arithmetic as the reference's ReferenceAttentionBackend
(src/kvssd/backends/reference.py:9-50): fp32 dequantisation, concatenation of
each block's first ``valid`` rows, GQA map ``qh // (QH/KVH)``, fp32 scores,
log-sum-exp and softmax.  It is the reference API's portable backend (the only
one on CPU) and never reports itself as accelerated, so the pipeline does not
route its streamed GPU path through it.
"""

from __future__ import annotations

import torch

from ..quant import unpack_codes
from .base import BackendAvailability, PackedBatch, PagedBatch


class ReferenceAttentionBackend:
    name = "reference"

    def probe(self, device: torch.device) -> BackendAvailability:
        return BackendAvailability(
            self.name, True, False, False, "portable PyTorch dequantize-then-attend reference", device.type
        )

    def run(self, query: torch.Tensor, batch: PackedBatch, sm_scale: float) -> tuple[torch.Tensor, torch.Tensor]:
        batch.validate(query)
        head_dim = query.shape[-1]
        mid = 1 << (batch.bits - 1)

        def dequant(packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
            codes = unpack_codes(packed, batch.bits, head_dim).float() - mid
            return codes * scales.float().repeat_interleave(batch.group_size, dim=-1)

        keys = dequant(batch.packed_k, batch.scales_k)
        values = dequant(batch.packed_v, batch.scales_v)
        # block i contributes the rows [i, :valid[i]] (Python slice rules: a
        # negative count drops that many rows from the end of the block)
        counts = [int(v) for v in batch.valid_tokens.tolist()]
        keys = torch.cat([keys[i, :n] for i, n in enumerate(counts)], dim=0)
        values = torch.cat([values[i, :n] for i, n in enumerate(counts)], dim=0)
        q_heads, kv_heads = query.shape[0], keys.shape[1]
        head_map = torch.arange(q_heads, device=query.device) // (q_heads // kv_heads)
        scores = torch.einsum("hd,thd->ht", query.float(), keys[:, head_map]) * sm_scale
        lse = torch.logsumexp(scores, dim=-1)
        out = torch.einsum("ht,thd->hd", torch.softmax(scores, dim=-1), values[:, head_map])
        return out, lse

    def run_paged(
        self,
        query: torch.Tensor,
        batch: PagedBatch,
        sm_scale: float,
        out_dtype: torch.dtype | None = None,
        accumulate: bool = False,
        max_length: int = 0,
        total_tokens: int = 0,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """Attention of one query per sequence over its pages, sequence by sequence (what
        HipAttentionBackend.run_paged computes); see there for the arguments.  The hints have nothing to size here, and
        weights are summed outside of any graph."""
        batch.validate()
        batch.validate_query(query)
        if accumulate and batch.weights is None:
            raise ValueError("accumulate needs a cache with weights")
        page_tokens = batch.packed_k.shape[1]
        outs, lses = [], []
        for b, length in enumerate(batch.lengths.tolist()):
            slots = torch.arange(max(0, min(length, batch.capacity)), device=query.device)
            pages = batch.page_table[b].long()[slots // page_tokens]
            slots = slots[(pages >= 0) & (pages < batch.packed_k.shape[0])]
            rows = batch.page_table[b].long()[slots // page_tokens] * page_tokens + slots % page_tokens
            one = PackedBatch(
                *(t.flatten(0, 1)[rows].unsqueeze(0)
                  for t in (batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v)),
                torch.tensor([len(slots)], dtype=torch.int32, device=query.device), batch.bits, batch.group_size,
            )
            if len(slots) == 0:
                outs.append(torch.zeros_like(query[b], dtype=torch.float32))
                lses.append(torch.full((query.shape[1],), -torch.inf, device=query.device))
                continue
            out, lse = self.run(query[b], one, sm_scale)
            outs.append(out)
            lses.append(lse)
            if accumulate:
                mid = 1 << (batch.bits - 1)
                keys = unpack_codes(one.packed_k[0], batch.bits, query.shape[2]).float() - mid
                keys = keys * one.scales_k[0].float().repeat_interleave(batch.group_size, dim=-1)
                grouped = query[b].float().reshape(keys.shape[1], -1, keys.shape[2])
                scores = torch.matmul(grouped, keys.permute(1, 2, 0).contiguous()) * sm_scale
                weights = torch.exp(scores - lse.reshape(*scores.shape[:2], 1)).sum((0, 1)).detach()
                batch.weights[b, slots] += weights
        out = torch.stack(outs)
        return out.to(out_dtype or torch.float32), torch.stack(lses)
