"""Windows, many tokens a sequence, trees and kept drafts over a paged cache without a GPU: the portable backend, the
host's bookkeeping, and every refusal."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, _native, append_tokens, keep_tokens
from kvssd.backends import PagedBatch
from kvssd.backends.hip import HipAttentionBackend
from kvssd.backends.reference import ReferenceAttentionBackend
from paged_oracle import as_double, make_pool, make_table
from test_paged import BAD_CACHES, native, small
from tokens_oracle import attend_tokens, keep, visible


def test_the_oracle_of_what_is_seen():
    # by hand: 3 slots before, a tree of 4 (1 and 2 under 0, 3 under 2)
    assert visible(7, 4, [-1, 0, 0, 2], 0, 0).astype(int).tolist() == [
        [1, 1, 1, 1, 0, 0, 0], [1, 1, 1, 1, 1, 0, 0], [1, 1, 1, 1, 0, 1, 0], [1, 1, 1, 1, 0, 1, 1]]
    # token 3 is at position 5: a window of 3 holds positions 3, 4 and 5, a sink of 1 position 0
    assert visible(7, 4, [-1, 0, 0, 2], 3, 1)[3].astype(int).tolist() == [1, 0, 0, 1, 0, 1, 1]
    assert visible(4, 2, None, 2, 0).astype(int).tolist() == [[0, 1, 1, 0], [0, 0, 1, 1]]
    assert visible(1, 3, None, 0, 0).astype(int).tolist() == [[0], [0], [1]]


def test_the_oracle_of_keeping():
    pool = [np.arange(8.0).reshape(2, 4, 1, 1) for _ in range(4)]
    pools, lengths, weights, _ = keep(pool, np.array([[1, 0]]), [7], [5], [[1, 3, 3, 4]], np.arange(8.0)[None])
    # slots 2, 3 (base 2) take slots 3 and 5: rows 7 and 1 of the pool go to 6 and 7; the list ends at the second 3
    assert lengths.tolist() == [4] and pools[0].ravel().tolist() == [0, 1, 2, 3, 4, 5, 7, 1]
    assert weights[0].tolist() == [0, 1, 3, 5, 4, 5, 6, 7]


@pytest.mark.parametrize("bits", [2, 4])
@pytest.mark.parametrize(("tree", "window", "sink"), [(False, 0, 0), (False, 9, 2), (True, 0, 0), (True, 4, 30), (False, 1, 0)])
def test_the_portable_backend_matches_the_oracle(bits, tree, window, sink):
    batch, pool, table = small(bits=bits)
    table[2, 1] = -1
    batch.page_table.copy_(torch.from_numpy(table))
    # tokens 0 and 17 of no sequence; sequence 1 has one more than slots (none)
    offsets, lengths = [1, 8, 9, 17], [20, 0, 33]
    rng = np.random.default_rng(3)
    q = torch.from_numpy(rng.standard_normal((18, 4, 64))).float()
    parents = rng.integers(-1, 8, 18).astype(np.int32) if tree else None
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, 0.125, parents, window, sink)
    off = torch.tensor(offsets, dtype=torch.int32)
    up = None if parents is None else torch.from_numpy(parents)
    out, lse = ReferenceAttentionBackend().run_paged_tokens(q, batch, 0.125, off, up, window=window, sink=sink, max_length=33)
    # 32-bit sums of 64 products: the packed backend's tolerance
    np.testing.assert_allclose(out.numpy(), want["out"], atol=2e-5, rtol=2e-5)
    np.testing.assert_allclose(lse.numpy(), want["lse"], atol=2e-5, rtol=2e-5)
    assert (lse[[0, 8, 17]] == -torch.inf).all() and (out[[0, 8, 17]] == 0).all()
    if not tree:  # one token a sequence is the single-token decode
        one, one_lse = ReferenceAttentionBackend().run_paged(q[:3], batch, 0.125, window=window, sink=sink)
        many, many_lse = ReferenceAttentionBackend().run_paged_tokens(
            q[:3], batch, 0.125, torch.arange(4, dtype=torch.int32), window=window, sink=sink)
        torch.testing.assert_close(one, many)
        torch.testing.assert_close(one_lse, many_lse)
    half, _ = ReferenceAttentionBackend().run_paged_tokens(q.half(), batch, 0.125, off, out_dtype=torch.float16)
    assert half.dtype == torch.float16
    none, none_lse = ReferenceAttentionBackend().run_paged_tokens(q[:0], batch, 0.125, torch.zeros(4, dtype=torch.int32))
    assert none.shape == (0, 4, 64) and none_lse.shape == (0, 4)


# ------------------------------------------------------------------------------------------------------------ refusals


OFF, UP = torch.tensor([0, 1, 1, 3], dtype=torch.int32), torch.tensor([-1, -1, 0], dtype=torch.int32)


@pytest.mark.parametrize(("change", "match"), [
    (dict(query=torch.zeros(4, 64)), "tokens, query_heads, head_dim"),
    (dict(query=torch.zeros(3, 4, 32)), "packed dimension"),
    (dict(query=torch.zeros(3, 3, 64)), "divisible"),
    (dict(query=torch.zeros(3, 0, 64)), "divisible"),
    (dict(offsets=OFF.long()), "offsets must be int32"),
    (dict(offsets=OFF[:3]), r"offsets must be int32 \[4\]"),
    (dict(parents=UP[:2]), r"parents must be int32 \[3\]"),
    (dict(parents=UP.float()), "parents must be int32"),
    (dict(window=-1), "window and sink"),
    (dict(sink=-1), "window and sink"),
], ids=str)
def test_calls_that_do_not_fit_are_refused(change, match):
    batch, _, _ = small()
    args = {**dict(query=torch.zeros(3, 4, 64), batch=batch, sm_scale=1.0, offsets=OFF), **change}
    with pytest.raises(ValueError, match=match):
        ReferenceAttentionBackend().run_paged_tokens(**args)
    if not {"offsets", "parents"} & set(change):  # checked when the prepared call is made
        with pytest.raises(ValueError, match=match):
            HipAttentionBackend().run_paged_tokens(**args)


def test_windows_and_weights_exclude_each_other():
    batch, _, _ = small()
    for backend in (ReferenceAttentionBackend(), HipAttentionBackend()):
        with pytest.raises(ValueError, match="not over a window"):
            backend.run_paged(torch.zeros(3, 4, 64), batch, 1.0, accumulate=True, window=5)
        for visible_slots in (dict(window=-1), dict(sink=-1)):
            with pytest.raises(ValueError, match="window and sink"):
                backend.run_paged(torch.zeros(3, 4, 64), batch, 1.0, **visible_slots)


def test_cpu_tensors_are_refused_by_the_kernels():
    batch, _, _ = small()
    with pytest.raises(ValueError, match="GPU"):
        HipAttentionBackend().run_paged_tokens(torch.zeros(3, 4, 64), batch, 1.0, OFF)
    with pytest.raises(ValueError, match="GPU"):
        keep_tokens(batch, OFF[:3], torch.zeros(3, 2, dtype=torch.int32))
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        append_tokens(batch, x, x, parents=UP)


@pytest.mark.parametrize(("change", "match"), BAD_CACHES, ids=str)
def test_bad_caches_fail_every_entry_point(change, match):
    lib, n = _native.load(), ctypes.c_size_t(0)
    cache, tokens, kept = native(**change), _native.PagedTokensArgs(), _native.PagedKeepArgs()
    for rc in (
        lambda: lib.kvssd_hip_paged_tokens(ctypes.byref(cache), ctypes.byref(tokens), None),
        lambda: lib.kvssd_hip_paged_tokens_workspace_bytes(ctypes.byref(cache), ctypes.byref(tokens), ctypes.byref(n)),
        lambda: lib.kvssd_hip_paged_keep(ctypes.byref(cache), ctypes.byref(kept), None),
    ):
        with pytest.raises(ValueError, match=match):
            _native.check(rc(), "entry point")


def test_null_structures_are_errors():
    lib, cache, n = _native.load(), native(), ctypes.c_size_t(0)
    tokens = _native.PagedTokensArgs()
    for rc in (
        lambda: lib.kvssd_hip_paged_tokens(None, None, None),
        lambda: lib.kvssd_hip_paged_tokens(ctypes.byref(cache), None, None),
        lambda: lib.kvssd_hip_paged_tokens_workspace_bytes(ctypes.byref(cache), None, ctypes.byref(n)),
        lambda: lib.kvssd_hip_paged_tokens_workspace_bytes(ctypes.byref(cache), ctypes.byref(tokens), None),
        lambda: lib.kvssd_hip_paged_keep(None, None, None),
        lambda: lib.kvssd_hip_paged_keep(ctypes.byref(cache), None, None),
    ):
        with pytest.raises(ValueError, match="NULL"):
            _native.check(rc(), "entry point")


def tokens_args(**change):
    heads = lambda n=4, data=4096, stride=256: _native.Heads(data, None, stride, 64, 0, 0, n, 0)  # noqa: E731
    query = heads(**change.pop("query", {}))
    return _native.PagedTokensArgs(**{**dict(query=query, out=4096, lse=4096, offsets=4096, workspace=4096,
                                             workspace_bytes=1 << 30, sm_scale=1.0, tokens=3), **change})


@pytest.mark.parametrize(("change", "match"), [
    (dict(query=dict(n=3)), "divisible"), (dict(query=dict(n=0)), "divisible"), (dict(query_dtype=3), "dtype"),
    (dict(query_dtype=-1), "dtype"), (dict(out_query_dtype=2), "out_query_dtype"), (dict(max_length=-1), ">= 0"),
    (dict(total_tokens=-1), ">= 0"), (dict(window=-1), "window and sink"), (dict(sink=-1), "window and sink"),
    (dict(tokens=-1), r"2\^30"), (dict(tokens=1 << 40), r"2\^30"), (dict(tokens=1 << 28, query=dict(n=8)), r"2\^30"),
    (dict(tokens=1 << 28), "too many"), (dict(query=dict(data=None)), "NULL"), (dict(out=None), "NULL"),
    (dict(lse=None), "NULL"), (dict(offsets=None), "NULL"), (dict(query=dict(data=4104)), "16-byte"),
    (dict(query=dict(stride=260), query_dtype=1), "16-byte"), (dict(out=4100), "16-byte"), (dict(workspace=4097), "256-byte"),
], ids=str)
def test_bad_token_calls_are_errors(change, match):
    lib, cache, args = _native.load(), native(), tokens_args(**dict(change))
    with pytest.raises(ValueError, match=match):
        _native.check(lib.kvssd_hip_paged_tokens(ctypes.byref(cache), ctypes.byref(args), None), "tokens")


def workspace(cache=None, **change) -> int:
    n, args = ctypes.c_size_t(0), tokens_args(**change)
    _native.check(_native.load().kvssd_hip_paged_tokens_workspace_bytes(
        ctypes.byref(cache or native()), ctypes.byref(args), ctypes.byref(n)), "tokens")
    return n.value


def test_the_workspace_of_tokens():
    lib = _native.load()
    long = dict(kv_heads=8, head_dim=128, num_pages=4096, page_tokens=64, sequences=1, max_pages=4096)
    # no call is too small to plan, and none that is whole needs any
    assert workspace(tokens=0) == 0 and workspace() == 0
    assert workspace(native(**long), query=dict(n=32), tokens=1 << 14) == 0
    split = workspace(native(**long), query=dict(n=32), tokens=8)
    assert split > 0
    for short in (dict(max_length=64), dict(total_tokens=64), dict(window=10), dict(window=2**31 - 1, sink=2**31 - 1, max_length=64)):
        assert workspace(native(**long), query=dict(n=32), tokens=8, **short) < split
    assert workspace(native(**long), query=dict(n=32), tokens=8, window=2**31 - 1, sink=2**31 - 1) == split
    args = tokens_args(query=dict(n=32), tokens=8, workspace_bytes=split - 1)
    for bad in (dict(workspace_bytes=split - 1), dict(workspace=None)):
        args = tokens_args(query=dict(n=32), tokens=8, **bad)
        with pytest.raises(ValueError, match=f"workspace too small: need {split} bytes"):
            _native.check(lib.kvssd_hip_paged_tokens(ctypes.byref(native(**long)), ctypes.byref(args), None), "tokens")
    # many sequences' places: two numbers for each and for the tokens before and behind them
    places = workspace(native(sequences=1000), tokens=1000, max_length=64)
    assert places == (2 * 1003 + 1) * 4 // 256 * 256 + 256
    # whatever the hints and the numbers of sequences and tokens, planning ends and the sum fits
    for sequences in (1, 62, 63, 4096, 1 << 20):
        for tokens in (0, 1, 100, 1 << 20):
            for hints in ({}, dict(max_length=1), dict(total_tokens=1), dict(window=1)):
                assert workspace(native(sequences=sequences), tokens=tokens, **hints) < 1 << 40


def test_a_call_without_tokens_does_nothing():
    args = _native.PagedTokensArgs()
    assert _native.load().kvssd_hip_paged_tokens(ctypes.byref(native()), ctypes.byref(args), None) == 0


def test_bad_windows_of_single_tokens_are_errors():
    good = dict(query=4096, out=4096, lse=4096, workspace=4096, workspace_bytes=1 << 30, sm_scale=1.0, query_heads=4)
    for change, match in ((dict(window=-1), "window and sink"), (dict(sink=-1), "window and sink"),
                          (dict(window=5, accumulate=1), "not over a window")):
        args = _native.PagedDecodeArgs(**{**good, **change})
        with pytest.raises(ValueError, match=match):
            _native.check(_native.load().kvssd_hip_paged_decode(ctypes.byref(native()), ctypes.byref(args), None), "decode")
    cache, n = native(num_pages=4096, max_pages=4096), ctypes.c_size_t(0)
    for window in (1, 2**31 - 1):
        args = _native.PagedDecodeArgs(**good, window=window, sink=2**31 - 1)
        _native.check(_native.load().kvssd_hip_paged_decode_workspace_bytes(
            ctypes.byref(cache), ctypes.byref(args), ctypes.byref(n)), "decode")


def test_bad_keeps_are_errors():
    good = dict(drafted=4096, kept=4096, lengths_out=4096, width=3)
    for change, match in ((dict(width=-1), "width"), (dict(drafted=None), "NULL"), (dict(kept=None), "NULL"),
                          (dict(lengths_out=None), "NULL"), (dict(width=0, lengths_out=None), "NULL")):
        args = _native.PagedKeepArgs(**{**good, **change})
        with pytest.raises(ValueError, match=match):
            _native.check(_native.load().kvssd_hip_paged_keep(ctypes.byref(native()), ctypes.byref(args), None), "keep")


def test_structures_are_the_headers():
    # bytes, as a C compiler lays them out
    sizes = [ctypes.sizeof(t) for t in (_native.PagedTokensArgs, _native.PagedKeepArgs, _native.PagedDecodeArgs, _native.PagedAppendArgs)]
    assert sizes == [152, 32, 88, 224]
    assert _native.PagedTokensArgs.tokens.offset == 112 and _native.PagedAppendArgs.rotary.offset == 200


# --------------------------------------------------------------------------------------------------- the host's part


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose appends and keeps change lengths alone."""
    calls = []

    def append(batch, keys, values, *, offsets=None, lengths_out=None, query=None, parents=None, **_):
        counts = torch.ones_like(batch.lengths) if offsets is None else offsets[1:] - offsets[:-1]
        calls.append(("append", counts.tolist(), None if parents is None else parents.tolist()))
        lengths = batch.lengths + counts
        return query, lengths if lengths_out is None else lengths_out.copy_(lengths)

    def kept(batch, drafted, paths, *, lengths_out):
        calls.append(("keep", drafted.tolist(), paths.tolist()))
        return lengths_out.copy_(batch.lengths - drafted + (paths >= 0).sum(1).int())

    monkeypatch.setattr("kvssd.paged.append_tokens", append)
    monkeypatch.setattr("kvssd.paged.keep_tokens", kept)
    made = PagedKVCache(pages=9, page_tokens=4, kv_heads=1, head_dim=32, sequences=3, max_pages=5, track_weights=True, device="cpu")
    made.calls = calls
    return made


def rows(n):
    return torch.zeros(n, 1, 32)


def test_a_drafted_step(cache):
    cache.append(rows(7), rows(7), [5, 2, 0])
    assert cache.lengths == [5, 2, 0] and cache.free_pages == 6
    cache.append(rows(9), rows(9), [6, 3, 0], parents=[-1, 0, 0, 1, 1, 99, -7, 0, 1])
    assert cache.calls[-1] == ("append", [6, 3, 0], [-1, 0, 0, 1, 1, -1, -1, 0, 1])  # (what is no token's place is -1)
    assert cache.lengths == cache.next_positions == [11, 5, 0] and cache.free_pages == 4
    q = torch.zeros(9, 2, 32)
    for call in (lambda: cache.attend(q[:3]), lambda: cache.append(rows(3), rows(3)), lambda: cache.evict(4),
                 lambda: cache.attend_tokens(q, [6, 3, 0]), lambda: cache.attend_tokens(q[:3], parents=[-1] * 3),
                 lambda: cache.load(2, None)):
        with pytest.raises(RuntimeError, match="drafted"):
            call()
    for paths, match in (([[0], [0]], "one list"), ([[0, 6], [], []], "ascending places"), ([[1, 0], [], []], "ascending"),
                         ([[0, 0], [], []], "ascending"), ([[-1], [], []], "ascending"), ([[0], [0], [0]], "ascending"),
                         ([None, [], []], "by their path")):
        with pytest.raises(ValueError, match=match):
            cache.keep(paths)
    assert cache.lengths == [11, 5, 0]  # nothing has changed
    cache.keep([[0, 2], [], None])
    assert cache.calls[-1] == ("keep", [6, 3, 0], [[0, 2], [-1, -1], [-1, -1]])
    assert cache.lengths == cache.next_positions == [7, 2, 0] and cache.batch.lengths.tolist() == [7, 2, 0]
    assert cache.free_pages == 6 and (cache.batch.page_table >= 0).sum(1).tolist() == [2, 1, 0]
    with pytest.raises(RuntimeError, match="follows an append"):
        cache.keep([[], [], []])


def test_drafts_of_one_path_and_drafts_given_up(cache):
    cache.append(rows(6), rows(6), [1, 4, 1])
    cache.keep([None, [0, 1], []])  # tokens in a row: the first ones
    assert cache.lengths == [1, 2, 0]
    cache.append(rows(3), rows(3), parents=[-1, -1, -1])
    cache.keep([None, None, []])  # one token a sequence is no tree
    assert cache.lengths == [2, 3, 0]
    cache.append(rows(2), rows(2), [0, 2, 0], parents=torch.tensor([-1, 0], dtype=torch.int32))
    cache.clear(1)  # with all that was drafted
    assert cache.lengths == [2, 0, 0]
    cache.append(rows(3), rows(3))
    cache.append(rows(0), rows(0), [0, 0, 0], parents=[])  # nothing is drafted
    cache.append(rows(3), rows(3))
    assert cache.lengths == [4, 2, 2]
    with pytest.raises(ValueError, match="one number per token"):
        cache.append(rows(3), rows(3), parents=[0])
    assert cache.lengths == [4, 2, 2]
    cache._latest = [1, 1, 1]
    cache.append(rows(4), rows(4), [2, 2, 0], parents=[-1, 0, -1, 0])
    cache.clear(0)
    with pytest.raises(RuntimeError, match="drafted"):  # the other sequence's are left
        cache.append(rows(3), rows(3))
    cache.keep([[], [0], []])
    assert cache.lengths == [0, 3, 2]


def test_attention_of_the_last_tokens(cache):
    rng = np.random.default_rng(5)
    pool = make_pool(rng, 9, 4, 1, 32, 32, 4)
    cache.append(rows(12), rows(12), [8, 3, 1])
    for name, a in zip(("packed_k", "packed_v", "scales_k", "scales_v"), pool):
        assert getattr(cache.batch, name).shape == a.shape
    for t, a in zip((cache.batch.packed_k, cache.batch.scales_k, cache.batch.packed_v, cache.batch.scales_v),
                    (pool[0], pool[2], pool[1], pool[3])):
        t.copy_(torch.from_numpy(a))
    table = cache.batch.page_table.numpy()
    q = torch.from_numpy(rng.standard_normal((7, 2, 32))).float()
    for window, parents in ((0, None), (3, None), (0, [-1, 0, 0, 1, -1, -1, 0])):
        out, lse = cache.attend_tokens(q, [4, 3, 0], window=window, sink=1 if window else 0, parents=parents)
        want = attend_tokens(as_double(q), pool, table, cache.lengths, [0, 4, 7, 7], 4, 32 ** -0.5, parents, window, 1 if window else 0)
        np.testing.assert_allclose(out.numpy(), want["out"], atol=2e-5, rtol=2e-5)
        np.testing.assert_allclose(lse.numpy(), want["lse"], atol=2e-5, rtol=2e-5)
    one, _ = cache.attend_tokens(q[:3])
    many, _ = cache.attend(q[:3])
    torch.testing.assert_close(one, many)
    torch.testing.assert_close(cache.attend(q[:3], window=2, sink=1)[0], cache.attend_tokens(q[:3], window=2, sink=1)[0])
    for counts, match in (([4, 3], "one non-negative"), ([8, -1, 0], "one non-negative"), ([4, 4, 0], "add up"),
                          ([3, 4, 0], "fewer tokens")):
        with pytest.raises(ValueError, match=match):
            cache.attend_tokens(q, counts)
    with pytest.raises(ValueError, match="one number per token"):
        cache.attend_tokens(q, [4, 3, 0], parents=[0])
    cache.next_positions[0] += 1  # as after an eviction
    for call in (lambda: cache.attend(q[:3], window=2), lambda: cache.attend_tokens(q[:3], window=2)):
        with pytest.raises(ValueError, match="slots in the order of their positions"):
            call()


@pytest.mark.parametrize("path", [[1], [0, 2], [1, 2], [0, 1, 3], [2, 3]], ids=str)
def test_tokens_in_a_row_are_kept_from_the_first_on(cache, path):
    # a later one behind a gap would lie in a slot before its position, which the next token would get too
    cache.append(rows(5), rows(5), [4, 1, 0])
    with pytest.raises(ValueError, match="the first ones"):
        cache.keep([path, None, None])
    assert cache.lengths == cache.next_positions == [4, 1, 0] and cache.calls[-1][0] == "append"
    cache.keep([[0, 1, 2], [], []])
    assert cache.lengths == cache.next_positions == [3, 0, 0]


@pytest.mark.parametrize("given", ["numbers", "tensor"])
@pytest.mark.parametrize("path", [[1], [3], [0, 1, 2], [0, 3], [0, 1, 4], [5, 6], [0, 1, 3, 4], [4]], ids=str)
def test_a_tree_is_kept_by_a_path_of_children(cache, path, given):
    # 0 -> 1 -> 3, 0 -> 2, 4 -> 5, and 6 (a parent that is no earlier token is none); another sequence's 0 -> 1 -> 2
    parents = [-1, 0, 0, 1, 4, 4, 9] + [-1, 0, 1]
    cache.append(rows(4), rows(4), [2, 1, 1])
    up = parents if given == "numbers" else torch.tensor(parents, dtype=torch.int32)
    cache.append(rows(10), rows(10), [7, 0, 3], parents=up)
    if given == "tensor":
        up.fill_(-1)  # what the tokens' positions came from counts
    refused = path != [4]
    if refused:
        with pytest.raises(ValueError, match="from child to child"):
            cache.keep([path, [], [0, 1]])
        assert cache.lengths == [9, 1, 4] and cache.calls[-1][0] == "append"
    with pytest.raises(ValueError, match="from child to child"):
        cache.keep([[0], [], [1, 2]])
    if refused:
        cache.keep([[0, 1, 3], [], [0, 1, 2]])
        assert cache.lengths == cache.next_positions == [5, 1, 4]
    else:
        cache.clear(2)  # and with it its part of the tree
        cache.keep([[4, 5], None, []])
        assert cache.lengths == cache.next_positions == [4, 1, 0]
    with pytest.raises(RuntimeError, match="follows an append"):
        cache.keep([[], [], []])
