"""Selection, SSD prefetch, record-native staging and fused decode on one GPU.

Reference: src/kvssd/pipeline.py:19-196.  The same public surface
(``KVSSDPipeline(store, device, io_depth, stage_blocks, require_cuda_kernel,
attention_backend)``, ``decode(query, layer, selector)``, context manager),
re-planned for MI355X:

* The streamed path moves records, not parsed blocks: the loader's I/O
  threads read a chunk's raw records straight into a page-locked staging slot,
  one ``hipMemcpyAsync`` per chunk carries them to the device on the transfer
  stream, and on the compute stream the GPU gather checks every header and
  payload CRC-32 and lays out the PackedBatch arrays for the fused decode
  (``kvssd.staging``).  The host never parses, checksums, clones or stacks a
  block (the reference does all four, loader.py:73-91, pipeline.py:98-109).
* Each chunk's (O, LSE) folds into a running accumulator with one HIP merge
  kernel (the reference issues about six torch launches, pipeline.py:147-153).
* Two resident tiers sit above the SSD: ``load_host_resident`` keeps a layer's
  raw records in page-locked host memory, so a decode of it only streams
  PCIe (read by the gather kernel itself, or copied where ``stage_blocks``
  makes chunks of 8 MiB or more); ``load_resident`` keeps the gathered PackedBatch of a layer in HBM
  (288 GB per MI355X), and a decode of it is a single fused call over a device
  block table with no SSD or PCIe traffic.
"""

from __future__ import annotations

import math
from collections.abc import Sequence
from dataclasses import dataclass, field

import torch

from .attention import packed_attention, resolve_required
from .backends import AttentionBackend, PackedBatch
from .loader import AsyncBlockLoader
from .paged import PagedKVCache
from .records_hip import gather_records, raise_for_status
from .selectors import AllBlocks, BlockSelector
from .staging import HostRecords, RecordStager
from .store import KVCacheStore


@dataclass
class _Resident:
    batch: PackedBatch
    row_of: dict[int, int]
    ids: list[int]  # block id of each row, in row order
    # device block tables of recent selections (selection -> int32 rows)
    tables: dict[tuple[int, ...], torch.Tensor] = field(default_factory=dict)
    # prepared HIP decodes: (table address or None, query shape, dtype, scale) -> PreparedDecode
    prepared: dict[tuple, object] = field(default_factory=dict)
    # the prepared decode of the whole layer in row order last used (AllBlocks)
    whole: object | None = None


_TABLE_CACHE = 8  # selections whose device block tables a resident layer keeps


class KVSSDPipeline:
    """End-to-end selection, SSD prefetch, pinned staging, and packed attention pipeline."""

    def __init__(
        self,
        store: KVCacheStore,
        device: str | torch.device = "cuda",
        io_depth: int = 2,
        stage_blocks: int = 4,
        require_cuda_kernel: bool = False,
        attention_backend: str | AttentionBackend | None = None,
        defer_record_checks: bool = False,
    ):
        self.store = store
        self.device = torch.device(device)
        if self.device.type == "cuda" and not torch.cuda.is_available():
            raise RuntimeError("CUDA device requested but CUDA is unavailable")
        if stage_blocks < 1:
            raise ValueError("stage_blocks must be positive")
        self.loader = AsyncBlockLoader(store, depth=io_depth, pinned=self.device.type == "cuda", device=self.device)
        self.stage_blocks = stage_blocks
        self.require_cuda_kernel = require_cuda_kernel
        self.attention_backend = resolve_required(require_cuda_kernel, attention_backend, self.device)
        # resident decodes through the HIP backend's prepared decodes
        self._hip = getattr(self.attention_backend, "name", None) == "hip"
        gpu = self.device.type == "cuda"
        self.transfer_stream = torch.cuda.Stream(device=self.device) if gpu else None
        # a second copy stream: successive chunks alternate between the two
        self._transfer_alt = torch.cuda.Stream(device=self.device) if gpu else None
        self.compute_stream = torch.cuda.Stream(device=self.device) if gpu else None
        # streamed decodes check their records' CRC and headers before
        # returning (the reference's behaviour); deferred, a decode returns
        # without waiting for the GPU and a bad record raises at the next
        # streamed decode, synchronize() or close()
        self.defer_record_checks = defer_record_checks
        self._stager: RecordStager | None = None
        self._resident: dict[int, _Resident] = {}
        self._host: dict[int, HostRecords] = {}

    # ------------------------------------------------------------ helpers ---
    def _require_gpu(self, what: str) -> None:
        if self.device.type != "cuda":
            raise RuntimeError(f"{what} need a GPU device")

    def _staging(self) -> RecordStager:
        if self._stager is None:
            assert self.transfer_stream is not None and self.compute_stream is not None
            self._stager = RecordStager(
                self.store.spec,
                self.device,
                self.stage_blocks,
                self.attention_backend,
                [self.transfer_stream, self._transfer_alt],
                self.compute_stream,
            )
            self._stager.defer_checks = self.defer_record_checks
        return self._stager

    def _read_layer(self, layer: int) -> HostRecords:
        ids = self.store.blocks_for_layer(layer)
        if not ids:
            raise ValueError(f"layer {layer} has no blocks")
        records = torch.empty((len(ids), self.store.spec.record_bytes), dtype=torch.uint8, pin_memory=True)
        self.loader.read_records(layer, ids, records)
        return HostRecords(records, ids)

    # ---------------------------------------------------------- streamed ---
    def _decode_streamed(self, query: torch.Tensor, layer: int, selected: list[int]) -> torch.Tensor:
        stager = self._staging()
        host = self._host.get(layer)
        if host is not None:
            fill = stager.host_fill(host)
        else:
            fill = stager.read_fill(lambda ids, rows: self.loader.read_records_async(layer, ids, rows))
        out, _ = stager.run(query, 1.0 / math.sqrt(query.shape[-1]), layer, selected, fill)
        return out.to(query.dtype)

    # ---------------------------------------------------------- resident ---
    def load_host_resident(self, layers: Sequence[int] | None = None) -> None:
        """Keep whole layers' raw records in page-locked host memory; later
        decodes of them stream PCIe only (records are still CRC-checked on the GPU)."""
        self._require_gpu("host-resident layers")
        for layer in layers if layers is not None else range(self.store.spec.layers):
            self._host[layer] = self._read_layer(layer)

    def release_host_resident(self, layers: Sequence[int] | None = None) -> None:
        for layer in list(self._host) if layers is None else layers:
            self._host.pop(layer, None)

    def load_resident(self, layers: Sequence[int] | None = None) -> None:
        """Copy whole layers into device memory; later decodes of them read HBM only.
        The records cross PCIe once and are checked and gathered on the GPU."""
        self._require_gpu("resident layers")
        spec = self.store.spec
        for layer in layers if layers is not None else range(spec.layers):
            host = self._host.get(layer) or self._read_layer(layer)
            raw = host.records.view(-1).to(self.device)
            kp, vp, ks, vs, valid, status = gather_records(raw, spec, len(host.block_ids))
            raise_for_status(status, layer, host.block_ids)
            del raw
            batch = PackedBatch(kp, vp, ks, vs, valid, spec.bits, spec.group_size)
            self._resident[layer] = _Resident(batch, dict(host.row_of), list(host.block_ids))

    def release_resident(self, layers: Sequence[int] | None = None) -> None:
        for layer in list(self._resident) if layers is None else layers:
            self._resident.pop(layer, None)

    def paged_cache(self, layer: int, *, spare_pages: int = 0, track_weights: bool = False) -> PagedKVCache:
        """A resident layer as a paged cache of one sequence that can grow: its blocks copied into pages of
        block_tokens tokens, with ``spare_pages`` free ones behind them."""
        res = self._resident.get(layer)
        if res is None:
            raise ValueError(f"layer {layer} is not resident")
        spec = self.store.spec
        cache = PagedKVCache(
            len(res.ids) + spare_pages, spec.block_tokens, spec.kv_heads, spec.head_dim, bits=spec.bits,
            group_size=spec.group_size, track_weights=track_weights, device=self.device,
            attention_backend=self.attention_backend,
        )
        cache.load(0, res.batch)
        return cache

    def _table(self, res: _Resident, selected: list[int]) -> torch.Tensor | None:
        """Device block table for ``selected``; None when it is every row in order."""
        if selected is res.ids or selected == res.ids:
            return None
        key = tuple(selected)
        table = res.tables.get(key)
        if table is None:
            rows = [res.row_of[b] for b in selected]
            table = torch.tensor(rows, dtype=torch.int32).to(self.device)
            if len(res.tables) >= _TABLE_CACHE:
                res.tables.pop(next(iter(res.tables)))
            res.tables[key] = table
        return table

    def _decode_resident(self, query: torch.Tensor, layer: int, selected: list[int]) -> torch.Tensor:
        res = self._resident[layer]
        if self._hip:
            # checks, descriptor and pointers once per (selection, query shape
            # and dtype; the scale follows from the shape); the merge writes
            # the query's dtype itself (no separate cast)
            table = self._table(res, selected)
            key = (None if table is None else table.data_ptr(), query.shape, query.dtype)
            prepared = res.prepared.get(key)
            if prepared is None:
                scale = 1.0 / math.sqrt(query.shape[-1])
                prepared = self.attention_backend.prepare(query, res.batch, scale, block_table=table, out_dtype=query.dtype)
                if len(res.prepared) >= 2 * _TABLE_CACHE:
                    res.prepared.pop(next(iter(res.prepared)))
                res.prepared[key] = prepared
            out, _ = prepared(query)
            if table is None:
                res.whole = prepared
            return out
        else:
            scale = 1.0 / math.sqrt(query.shape[-1])
            run = self.attention_backend.run
            rows = [res.row_of[b] for b in selected]
            idx = torch.tensor(rows, dtype=torch.long, device=self.device)
            b = res.batch
            sub = PackedBatch(
                b.packed_k[idx], b.packed_v[idx], b.scales_k[idx], b.scales_v[idx], b.valid_tokens[idx], b.bits, b.group_size
            )
            out, _ = run(query, sub, scale)
        return out.to(query.dtype)

    # ------------------------------------------------------------ public ---
    def decode(
        self,
        query: torch.Tensor,
        layer: int,
        selector: BlockSelector | None = None,
    ) -> torch.Tensor:
        res = self._resident.get(layer)
        if res is not None and (selector is None or type(selector) is AllBlocks):
            # every block of an HBM-resident layer, in the store's order: its
            # batch's row order (a store's block lists never change), with no
            # copy or compare of the id list on the per-call path; a query of
            # the shape, dtype and device of the last such call goes straight
            # to that call's prepared decode
            if res.whole is not None:
                r = res.whole.try_call(query)
                if r is not None:
                    return r[0]
            if res.ids:
                return self._decode_resident(query.to(self.device), layer, res.ids)
            raise ValueError("selector returned no blocks")
        selector = selector or AllBlocks()
        selected = selector.select(self.store.blocks_for_layer(layer))
        if not selected:
            raise ValueError("selector returned no blocks")
        query = query.to(self.device)
        if res is not None:
            return self._decode_resident(query, layer, selected)
        if self.device.type == "cuda" and (layer in self._host or self.attention_backend.probe(self.device).accelerated):
            return self._decode_streamed(query, layer, selected)
        blocks = list(self.loader.iter_blocks(layer, selected))
        return packed_attention(
            query,
            blocks,
            sm_scale=1.0 / math.sqrt(query.shape[-1]),
            require_cuda_kernel=self.require_cuda_kernel,
            attention_backend=self.attention_backend,
        )

    def synchronize(self) -> None:
        """Wait for the pipeline's GPU work; raise for any deferred record error."""
        if self._stager is not None:
            self._stager.check_pending()
        if self.device.type == "cuda":
            torch.cuda.synchronize(self.device)

    def close(self) -> None:
        try:
            if self._stager is not None:
                self._stager.check_pending()
        finally:
            self.loader.close()
            self._resident.clear()
            self._host.clear()

    def __enter__(self) -> "KVSSDPipeline":
        return self

    def __exit__(self, *_: object) -> None:
        self.close()
