"""The paged cache without a GPU: the portable backend, the host's bookkeeping, and every refusal."""

from __future__ import annotations

import ctypes
import dataclasses

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, Rotary, _native, append_tokens, evict_tokens
from kvssd.backends import PackedBatch, PagedBatch
from kvssd.backends.hip import HipAttentionBackend
from kvssd.backends.reference import ReferenceAttentionBackend
from paged_oracle import as_double, attend, evict, make_pool, make_table


def small(lengths=(20, 0, 33), bits=4, bt=16, kvh=2, d=64, g=32, tracked=True):
    rng = np.random.default_rng(1)
    pages = sum(-(-n // bt) for n in lengths) + 1
    pool = make_pool(rng, pages, bt, kvh, d, g, bits)
    table = make_table(rng, lengths, bt, 4, pages)
    slots = (len(lengths), 4 * bt)
    t = torch.from_numpy
    batch = PagedBatch(*map(t, pool), t(table), torch.tensor(lengths, dtype=torch.int32), bits, g,
                       torch.zeros(slots) if tracked else None,
                       torch.zeros(slots, dtype=torch.int32) if tracked else None)
    return batch, pool, table


def test_portable_backend_matches_the_oracle():
    for bits in (2, 4):
        batch, pool, table = small(bits=bits)
        table[2, 1] = -1
        batch.page_table.copy_(torch.from_numpy(table))
        q = torch.from_numpy(np.random.default_rng(2).standard_normal((3, 4, 64))).float()
        want = attend(as_double(q), pool, table, [20, 0, 33], bits, 0.125, np.zeros((3, 64)))
        out, lse = ReferenceAttentionBackend().run_paged(q, batch, 0.125, accumulate=True)
        # 32-bit sums of 64 products: the packed backend's tolerance
        np.testing.assert_allclose(out.numpy(), want["out"], atol=2e-5, rtol=2e-5)
        np.testing.assert_allclose(lse.numpy(), want["lse"], atol=2e-5, rtol=2e-5)
        np.testing.assert_allclose(batch.weights.numpy(), want["weights"], atol=2e-5, rtol=2e-5)
        half, _ = ReferenceAttentionBackend().run_paged(q.half(), batch, 0.125, out_dtype=torch.float16)
        assert half.dtype == torch.float16


def test_the_oracle_of_eviction_keeps_what_it_should():
    # by hand: positions 0 and 4 are held (sink 1, recent 1), then weights 9 and 5 (the lower of the two fives)
    assert evict(np.array([1.0, 5, 9, 5, 0, 2]), np.array([0, 1, 2, 3, 5, 4]), 6, 4, 1, 1) == [0, 1, 2, 4]
    assert evict(np.array([1.0, 5, 9]), np.array([0, 1, 2]), 3, 1, 0, 0) == [2]
    assert evict(np.array([1.0, 5]), np.array([0, 1]), 2, 7, 0, 0) == [0, 1]


@pytest.mark.parametrize(("change", "match"), [
    (dict(bits=3), "bits must be 2 or 4"),
    (dict(bits=2), "packed dimension"),
    (dict(group_size=16), "group_size"),
    (dict(group_size=96), "group_size"),
    (dict(group_size=64), "packed dimension"),
    (dict(packed_k=torch.zeros(5, 16, 2, 32)), "uint8"),
    (dict(packed_k=torch.zeros(5, 16, 2, dtype=torch.uint8)), "must match"),
    (dict(scales_k=torch.zeros(5, 16, 2, 2)), "float16"),
    (dict(page_table=torch.zeros(3, 4, dtype=torch.int64)), "page_table must be int32"),
    (dict(page_table=torch.zeros(3, dtype=torch.int32)), "max_pages"),
    (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(6, dtype=torch.int32)[::2]), "contiguous"),
    (dict(weights=torch.zeros(3, 63)), "weights must be"),
    (dict(weights=torch.zeros(3, 64, dtype=torch.float64)), "weights must be float32"),
    (dict(positions=torch.zeros(2, 64, dtype=torch.int32)), "positions must be"),
])
def test_malformed_caches_are_refused(change, match):
    batch, _, _ = small()
    pages = batch.packed_k.shape[0]
    change = {k: (v[:1].expand(pages, *v.shape[1:]) if isinstance(v, torch.Tensor) and k.startswith(("packed", "scales"))
                  else v) for k, v in change.items()}
    for name in ("packed", "scales"):
        if f"{name}_k" in change:
            change[f"{name}_v"] = change[f"{name}_k"]
    with pytest.raises(ValueError, match=match):
        dataclasses.replace(batch, **change).validate()


@pytest.mark.parametrize(("shape", "match"), [
    ((2, 4, 64), "sequences"), ((3, 4), "sequences"), ((3, 3, 64), "divisible"), ((3, 0, 64), "divisible"),
    ((3, 4, 32), "head dimension"),
])
def test_queries_that_do_not_fit_are_refused(shape, match):
    batch, _, _ = small()
    for backend in (ReferenceAttentionBackend(), HipAttentionBackend()):
        with pytest.raises(ValueError, match=match):
            backend.run_paged(torch.zeros(shape), batch, 1.0)


def test_accumulation_needs_weights():
    batch, _, _ = small(tracked=False)
    for backend in (ReferenceAttentionBackend(),):
        with pytest.raises(ValueError, match="with weights"):
            backend.run_paged(torch.zeros(3, 4, 64), batch, 1.0, accumulate=True)


def test_cpu_tensors_are_refused_by_the_kernels():
    batch, _, _ = small()
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        HipAttentionBackend().run_paged(torch.zeros(3, 4, 64), batch, 1.0)
    with pytest.raises(ValueError, match="GPU"):
        append_tokens(batch, x, x)
    with pytest.raises(ValueError, match="GPU"):
        evict_tokens(batch, 4)


# ------------------------------------------------------------------------------------------- the library's own checks


def native(**change):
    """A well-formed kvssd_paged_cache over addresses that nothing reads: every call below fails a check first."""
    values = dict(bits=4, kv_heads=2, head_dim=64, group_size=32, num_pages=5, page_tokens=16, sequences=3, max_pages=4,
                  packed_k=4096, packed_v=4096, scales_k=4096, scales_v=4096, page_table=4096, lengths=4096,
                  weights=4096, positions=4096)
    return _native.PagedCache(**{**values, **change})


BAD_CACHES = [
    (dict(bits=3), "bits must be 2 or 4"), (dict(kv_heads=0), "packed pages"), (dict(num_pages=0), "packed pages"),
    (dict(page_tokens=0), "packed pages"), (dict(head_dim=288), "head_dim"), (dict(head_dim=48), "head_dim"),
    (dict(group_size=16), "group_size"), (dict(group_size=48), "group_size"), (dict(group_size=128), "group_size"),
    (dict(sequences=0), "page_table"), (dict(sequences=(1 << 20) + 1), "page_table"), (dict(max_pages=0), "page_table"),
    (dict(max_pages=1 << 28), r"2\^30"), (dict(num_pages=1 << 28), r"2\^30"), (dict(packed_v=None), "NULL"),
    (dict(lengths=None), "NULL"), (dict(scales_k=4098), "aligned"), (dict(packed_k=4104), "aligned"),
]


@pytest.mark.parametrize(("change", "match"), BAD_CACHES, ids=lambda x: str(x))
def test_bad_caches_fail_every_entry_point(change, match):
    lib = _native.load()
    cache = native(**change)
    n = ctypes.c_size_t(0)
    decode, append, evict_args = _native.PagedDecodeArgs(), _native.PagedAppendArgs(), _native.PagedEvictArgs()
    for rc in (
        lambda: lib.kvssd_hip_paged_decode(ctypes.byref(cache), ctypes.byref(decode), None),
        lambda: lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), ctypes.byref(decode), ctypes.byref(n)),
        lambda: lib.kvssd_hip_paged_append(ctypes.byref(cache), ctypes.byref(append), None),
        lambda: lib.kvssd_hip_paged_evict(ctypes.byref(cache), ctypes.byref(evict_args), None),
        lambda: lib.kvssd_hip_paged_evict_workspace_bytes(ctypes.byref(cache), ctypes.byref(evict_args), ctypes.byref(n)),
    ):
        with pytest.raises(ValueError, match=match):
            _native.check(rc(), "entry point")


def test_null_structures_are_errors():
    lib = _native.load()
    cache, n = native(), ctypes.c_size_t(0)
    for rc in (
        lambda: lib.kvssd_hip_paged_decode(None, None, None),
        lambda: lib.kvssd_hip_paged_decode(ctypes.byref(cache), None, None),
        lambda: lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), None, ctypes.byref(n)),
        lambda: lib.kvssd_hip_paged_append(ctypes.byref(cache), None, None),
        lambda: lib.kvssd_hip_paged_evict(ctypes.byref(cache), None, None),
        lambda: lib.kvssd_hip_rotary(None, None, 0, 1, 0, None, 1, None),
    ):
        with pytest.raises(ValueError, match="NULL"):
            _native.check(rc(), "entry point")


def test_bad_decodes_are_errors():
    lib = _native.load()
    cache, n = native(), ctypes.c_size_t(0)
    good = dict(query=4096, out=4096, lse=4096, workspace=4096, workspace_bytes=1 << 30, sm_scale=1.0, query_heads=4)

    def call(cache=cache, **change):
        args = _native.PagedDecodeArgs(**{**good, **change})
        _native.check(lib.kvssd_hip_paged_decode(ctypes.byref(cache), ctypes.byref(args), None), "decode")

    for change, match in (
        (dict(query_heads=3), "divisible"), (dict(query_heads=0), "divisible"), (dict(query_dtype=3), "dtype"),
        (dict(query_dtype=-1), "dtype"), (dict(out_query_dtype=2), "out_query_dtype"), (dict(max_length=-1), ">= 0"),
        (dict(total_tokens=-1), ">= 0"), (dict(query=None), "NULL"), (dict(out=None), "NULL"), (dict(lse=None), "NULL"),
        (dict(workspace_bytes=8, accumulate=1), "workspace too small: need"), (dict(workspace=4097), "256-byte"),
    ):
        with pytest.raises(ValueError, match=match):
            call(**change)
    with pytest.raises(ValueError, match="with weights"):
        call(native(weights=None), accumulate=1)
    # the workspace of a decode grows with its runs, and with its scores where weights are summed
    args = _native.PagedDecodeArgs(**good)
    assert lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), ctypes.byref(n)) == 0
    plain = n.value
    args.accumulate = 1
    assert lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), ctypes.byref(n)) == 0
    assert n.value == plain + 3 * 4 * 64 * 4


def test_bad_appends_are_errors():
    lib = _native.load()
    heads = lambda n=2, data=4096, out=4096: _native.Heads(data, out, 128, 64, 128, 64, n, 0)  # noqa: E731
    spec = _native.RotarySpec(4096, 1.0, 64, 64, 0, 0)

    def call(cache=None, **change):
        args = _native.PagedAppendArgs(**{**dict(keys=heads(), values=heads(), tokens=3, dtype=0), **change})
        _native.check(lib.kvssd_hip_paged_append(ctypes.byref(cache or native()), ctypes.byref(args), None), "append")

    for change, match in (
        (dict(dtype=3), "dtype"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 24), "tokens"),
        (dict(tokens=4), "one token a sequence"), (dict(keys=heads(3)), "kv_heads"), (dict(values=heads(1)), "kv_heads"),
        (dict(keys=heads(data=None)), "NULL"), (dict(query=heads(4)), "rotated"),
        (dict(offsets=4096, lengths_out=4096), "lengths_out"),
        (dict(rotary=ctypes.pointer(_native.RotarySpec(4096, 1.0, 32, 32, 0, 0))), "differs"),
        (dict(rotary=ctypes.pointer(_native.RotarySpec(4096, 1.0, 64, 31, 0, 0))), "even"),
        (dict(rotary=ctypes.pointer(_native.RotarySpec(None, 1.0, 64, 64, 0, 0))), "NULL"),
        (dict(rotary=ctypes.pointer(spec), query=heads(4, out=None)), "NULL"),
        (dict(rotary=ctypes.pointer(spec), query=heads(0)), "heads"),
    ):
        with pytest.raises(ValueError, match=match):
            call(**change)


def test_bad_evictions_are_errors():
    lib = _native.load()
    good = dict(budget=20, sink=2, recent=5, lengths_out=8192, weights_out=8192, positions_out=8192, workspace=8192,
                workspace_bytes=1 << 20)

    def call(cache=None, **change):
        args = _native.PagedEvictArgs(**{**good, **change})
        _native.check(lib.kvssd_hip_paged_evict(ctypes.byref(cache or native()), ctypes.byref(args), None), "evict")

    for change, match in (
        (dict(budget=0), "budget"), (dict(sink=-1), "non-negative"), (dict(recent=-1), "non-negative"),
        (dict(recent=19), "fit the budget"), (dict(sink=2**31 - 1, recent=2**31 - 1), "fit the budget"),
        (dict(lengths_out=None), "NULL"), (dict(weights_out=4096), "their own"), (dict(lengths_out=4096), "their own"),
        (dict(positions_out=4096), "their own"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=100), "workspace too small"),
    ):
        with pytest.raises(ValueError, match=match):
            call(**change)
    with pytest.raises(ValueError, match="weights and positions"):
        call(native(weights=None))
    with pytest.raises(ValueError, match="weights and positions"):
        call(native(positions=None))


def test_bad_rotations_are_errors():
    lib = _native.load()
    heads = (_native.Heads * 2)(_native.Heads(4096, 4096, 64, 64, 64, 64, 1, 0), _native.Heads(4096, None, 64, 64, 64, 64, 1, 0))

    def call(spec=(4096, 1.0, 64, 64, 0, 0), positions=4096, tokens=1, dtype=0, count=1, tensors=heads):
        spec = _native.RotarySpec(*spec)
        _native.check(lib.kvssd_hip_rotary(ctypes.byref(spec), positions, 0, tokens, dtype, tensors, count, None), "rotary")

    for change, match in (
        (dict(spec=(None, 1.0, 64, 64, 0, 0)), "NULL"), (dict(spec=(4096, 1.0, 64, 0, 0, 0)), "even"),
        (dict(spec=(4096, 1.0, 64, 66, 0, 0)), "even"), (dict(spec=(4096, 1.0, 2048, 64, 0, 0)), "1024"),
        (dict(dtype=3), "dtype"), (dict(count=0), "one or two"), (dict(count=3), "one or two"),
        (dict(tensors=None), "one or two"), (dict(count=2), "NULL"), (dict(positions=None), "NULL"),
        (dict(tokens=-1), "tokens"), (dict(tokens=1 << 24), "tokens"),
    ):
        with pytest.raises(ValueError, match=match):
            call(**change)


# -------------------------------------------------------------------------------------------- the host's bookkeeping


def host_cache(**change):
    return PagedKVCache(**{**dict(pages=6, page_tokens=4, kv_heads=1, head_dim=32, sequences=3, max_pages=3,
                                  track_weights=True, device="cpu"), **change})


def test_pages_are_taken_and_given_back():
    cache = host_cache()
    cache._resize([5, 0, 4])
    assert cache.free_pages == 3
    table = cache.batch.page_table.tolist()
    assert table == [[0, 1, -1], [-1, -1, -1], [2, -1, -1]]
    cache._resize([1, 9, 4])  # one given back and taken again in the same call
    assert cache.free_pages == 1
    used = [p for row in cache.batch.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 5 and cache.batch.page_table.tolist()[0][0] == 0
    with pytest.raises(RuntimeError, match="1 free pages, 2 are needed"):
        cache._resize([9, 9, 4])
    with pytest.raises(ValueError, match="at most 12 tokens"):
        cache._resize([13, 0, 0])
    assert cache.free_pages == 1 and cache.batch.page_table.tolist()[2][0] == 2  # nothing changed
    cache._resize([0, 0, 0])
    assert cache.free_pages == 6 and (cache.batch.page_table == -1).all()


def test_a_refused_append_leaves_the_cache_as_it_was():
    cache = host_cache()
    x = torch.zeros(3, 1, 32)
    with pytest.raises(ValueError, match="GPU"):
        cache.append(x, x)
    assert cache.free_pages == 6 and cache.lengths == [0, 0, 0] and (cache.batch.page_table == -1).all()
    for counts, match in (([1, 1], "one non-negative number"), ([4, -1, 0], "one non-negative number"), ([1, 1, 2], "add up")):
        with pytest.raises(ValueError, match=match):
            cache.append(x, x, counts)


def test_blocks_are_loaded_into_pages():
    rng = np.random.default_rng(3)
    cache = host_cache()
    pool = [torch.from_numpy(a) for a in make_pool(rng, 2, 4, 1, 32, 32, 4)]
    cache._resize([0, 0, 1])
    cache.lengths[2] = 1
    cache.load(0, PackedBatch(*pool, torch.tensor([4, 3], dtype=torch.int32), 4, 32))
    assert cache.lengths == [7, 0, 1] and cache.next_positions == [7, 0, 0] and cache.batch.lengths.tolist()[0] == 7
    ids = cache.batch.page_table[0, :2].long()
    assert torch.equal(cache.batch.packed_k[ids], pool[0]) and torch.equal(cache.batch.scales_v[ids], pool[3])
    assert cache.batch.positions[0, :7].tolist() == list(range(7))
    q = torch.from_numpy(rng.standard_normal((3, 2, 32))).float()
    out, _ = cache.attend(q)
    want, _ = ReferenceAttentionBackend().run(q[0], PackedBatch(*pool, torch.tensor([4, 3], dtype=torch.int32), 4, 32), 32 ** -0.5)
    torch.testing.assert_close(out[0], want)
    with pytest.raises(ValueError, match="not empty"):
        cache.load(0, PackedBatch(*pool, torch.tensor([4, 3], dtype=torch.int32), 4, 32))
    with pytest.raises(ValueError, match="must be full"):
        cache.load(1, PackedBatch(*pool, torch.tensor([3, 4], dtype=torch.int32), 4, 32))
    with pytest.raises(ValueError, match="differ in bits"):
        cache.load(1, PackedBatch(*pool, torch.tensor([4, 4], dtype=torch.int32), 2, 32))
    with pytest.raises(ValueError, match="sequence must lie"):
        cache.load(3, PackedBatch(*pool, torch.tensor([4, 4], dtype=torch.int32), 4, 32))
    cache.clear(0)
    assert cache.lengths == [0, 0, 1] and cache.free_pages == 5
    with pytest.raises(ValueError, match="sequence must lie"):
        cache.clear(-1)


@pytest.mark.parametrize(("change", "match"), [
    (dict(pages=0), "positive"), (dict(sequences=0), "positive"), (dict(bits=8), "bits"), (dict(head_dim=48), "head_dim"),
    (dict(head_dim=512), "head_dim"), (dict(group_size=64), "group_size"), (dict(group_size=8), "group_size"),
    (dict(max_pages=0), "max_pages"),
])
def test_refused_caches(change, match):
    with pytest.raises(ValueError, match=match):
        host_cache(**change)


def test_rotary_and_cache_have_to_fit():
    assert Rotary(32, device="cpu").spec(True).inverse == 1 and Rotary(32, device="cpu").spec().inverse == 0


def test_a_pool_of_one_row_is_taken_whatever_its_scales():
    lib = _native.load()
    for groups in (1, 2, 3):
        cache = native(num_pages=1, page_tokens=1, kv_heads=1, max_pages=1, head_dim=32 * groups)
        args, n = _native.PagedDecodeArgs(query_heads=1), ctypes.c_size_t(0)
        _native.check(
            lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), ctypes.byref(n)), "decode"
        )


def test_a_cut_writes_into_the_arrays_that_there_are(monkeypatch):
    cache = host_cache()
    cache._resize([9, 2, 0])
    cache.lengths = [9, 2, 0]
    cache.batch.lengths.copy_(torch.tensor([9, 2, 0]))
    before = cache.batch
    arrays = {f.name: getattr(before, f.name) for f in dataclasses.fields(before)}
    slots = before.weights.shape
    cut = (torch.tensor([4, 2, 0], dtype=torch.int32), torch.arange(36.0).view(slots),
           torch.arange(36, dtype=torch.int32).view(slots))
    monkeypatch.setattr("kvssd.paged.evict_tokens", lambda *a, **k: cut)
    cache.evict(4)
    assert cache.batch is before and all(getattr(before, n) is a for n, a in arrays.items())
    for got, want in zip((before.lengths, before.weights, before.positions), cut):
        assert torch.equal(got[..., :9], want[..., :9])
    assert cache.lengths == [4, 2, 0] and cache.free_pages == 4


def test_the_scores_workspace_goes_by_the_hints():
    """16 sequences that may each grow into a whole pool of 262,144 slots (a table's row), 32 query heads."""
    lib = _native.load()
    cache = native(kv_heads=8, head_dim=128, num_pages=4096, page_tokens=64, sequences=16, max_pages=4096)
    sizes = []
    for accumulate in (0, 1):
        for hints in ({}, dict(max_length=4700, total_tokens=70000), dict(total_tokens=70000), dict(max_length=4700)):
            args, n = _native.PagedDecodeArgs(query_heads=32, accumulate=accumulate, **hints), ctypes.c_size_t(0)
            _native.check(
                lib.kvssd_hip_paged_decode_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), ctypes.byref(n)), "decode"
            )
            sizes.append(n.value)
    scores = [b - a for a, b in zip(sizes[:4], sizes[4:])]
    stage = 32 * 64 * 4  # bytes of 64 slots' scores
    assert scores[0] == 16 * 4096 * stage  # no hint: every slot of the table
    assert scores[1] == scores[2] == (70000 // 64 + 16) * stage and scores[3] == 16 * 74 * stage


def test_a_cache_stays_on_the_gpu_that_was_current(monkeypatch):
    made = []

    class Stop(Exception):
        pass

    def resolve(name, device):
        made.append(device)
        raise Stop

    monkeypatch.setattr("kvssd.paged.resolve_attention_backend", resolve)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for device, want in (("cuda", "cuda:3"), ("cuda:1", "cuda:1"), ("cpu", "cpu")):
        with pytest.raises(Stop):
            host_cache(device=device)
        assert made.pop() == torch.device(want)


def test_the_portable_backend_takes_hints_and_keeps_weights_out_of_graphs():
    batch, pool, table = small()
    q = torch.from_numpy(np.random.default_rng(4).standard_normal((3, 4, 64))).float().requires_grad_()
    out, _ = ReferenceAttentionBackend().run_paged(q, batch, 0.125, accumulate=True, max_length=33, total_tokens=53)
    assert not batch.weights.requires_grad and batch.weights.sum().item() == pytest.approx(8.0, rel=1e-5)
    out.sum().backward()  # (this backend has a backward pass)
    assert torch.isfinite(q.grad).all() and (q.grad[1] == 0).all()
