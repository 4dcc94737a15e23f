"""Attention over part of a paged cache on the GPU -- windows with sinks, many tokens a sequence, trees -- and keeping
drafted tokens, against 64-bit oracles.

Tolerances.  Let A = sum_t p_t |v_t| (per output value), u = 2^-24.
* A score is a 32-bit sum of head_dim products whose terms add up to at most ``reach`` (returned by the oracle), then a
  product per group and their sum: off by at most E = (head_dim + 16) u reach.  Softmax weights are then off by at most
  a factor e^(2E) ~ 1 + 2E + ..., lse by E, and 2^x and the logarithm add a few u.
* With 16-bit results a weight is rounded to fp16 (2^-11 of it) and so is a value, code times scale (2^-11); both are
  scaled beforehand so that what falls below fp16's normal range is 2^-33 or less of the largest: nothing beside it.
  One-token attention rounds their product once (less).  With 32-bit results both are sums of two fp16 parts (2^-22).
* Sums over n slots in 32 bits: at most n u A.
* The result's rounding: eps/2 of the value.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, Rotary, append_tokens, keep_tokens
from kvssd.backends import PagedBatch
from kvssd.backends.hip import HipAttentionBackend
from kvssd.backends.reference import ReferenceAttentionBackend
from paged_oracle import as_double, make_pool, make_table
from tokens_oracle import attend_tokens, chain, keep

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def paged(dev, pool, table, lengths, bits, g, weights=None, positions=None) -> PagedBatch:
    t = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return PagedBatch(*(t(a) for a in pool), t(table.astype(np.int32)), t(np.asarray(lengths, np.int32)), bits, g,
                      t(weights), t(positions))


def ints(dev, values) -> torch.Tensor:
    return torch.tensor([int(x) for x in values], dtype=torch.int32, device=dev)


def check(out, lse, want, d, longest, dtype, precise):
    e = (d + 16) * U * want["reach"] + 8 * U
    weight = 2 * e + (2.0 ** -21 if precise else 2.0 ** -10) + (longest + 8) * U
    tol = want["size"] * weight * (1 + weight) + np.abs(want["out"]) * torch.finfo(dtype).eps / 2
    tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    got, got_lse = as_double(out), as_double(lse)
    empty = np.isinf(want["lse"])
    assert (got_lse[empty] == -np.inf).all() and (got[empty] == 0).all()
    err = np.abs(got - want["out"])
    assert (err <= tol).all(), f"out: largest error over its bound {np.nanmax(err / np.maximum(tol, 1e-300))}"
    lerr = np.abs(got_lse[~empty] - want["lse"][~empty])
    ltol = e + (np.abs(want["lse"][~empty]) + 40) * 4 * U
    assert (lerr <= ltol).all(), f"lse: {(lerr / ltol).max()}"


def random_parents(rng, counts, chainy=0.5):
    out = []
    for n in counts:
        out += [-1 if i == 0 or rng.random() < 0.1 else (i - 1 if rng.random() < chainy else int(rng.integers(0, i)))
                for i in range(n)]
    return np.array(out, np.int32)


def problem(dev, bits, qh, kvh, d, g, bt, before, counts, dtype, seed, scale=(0.2, 0.5)):
    rng = np.random.default_rng(seed)
    lengths = [a + n for a, n in zip(before, counts)]
    width = max(1, max(-(-n // bt) for n in lengths)) + 1
    pages = sum(-(-n // bt) for n in lengths) + 2
    pool = make_pool(rng, pages, bt, kvh, d, g, bits, scale)
    table = make_table(rng, lengths, bt, width, pages)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    q = torch.from_numpy(rng.standard_normal((int(offsets[-1]), qh, d))).to(dtype).to(dev)
    return rng, pool, table, lengths, offsets, q


# bits, query heads, kv heads, head_dim, group, page_tokens, slots before, new tokens, dtype, window, sink
SHAPES = [
    (4, 1, 1, 32, 32, 16, [0], [1], torch.float16, 0, 0),
    (4, 32, 8, 128, 32, 64, [0, 5, 300, 64, 1000], [130, 33, 1, 0, 64], torch.bfloat16, 0, 0),
    (4, 32, 8, 128, 32, 128, [4096], [8], torch.float16, 0, 0),
    (4, 8, 2, 128, 32, 64, [0], [517], torch.bfloat16, 100, 4),
    (4, 8, 2, 128, 32, 64, [700, 3], [70, 200], torch.float16, 64, 65),
    (4, 8, 2, 128, 64, 64, [900], [40], torch.float16, 1, 0),            # a token sees itself alone
    (4, 8, 2, 128, 128, 24, [100, 0], [61, 31], torch.bfloat16, 31, 100),  # pages that end inside a tile
    (2, 32, 8, 128, 32, 32, [777, 10], [19, 260], torch.bfloat16, 0, 0),
    (2, 8, 2, 128, 64, 1, [40], [9], torch.float16, 17, 3),               # a page a token
    (4, 10, 2, 96, 32, 16, [333], [45], torch.bfloat16, 0, 0),            # three groups
    (2, 6, 3, 96, 32, 40, [121, 90], [5, 40], torch.float32, 50, 2),
    (4, 16, 1, 64, 32, 64, [700, 5], [50, 3], torch.float16, 0, 0),
    (4, 40, 1, 64, 64, 7, [129], [64], torch.bfloat16, 40, 1),
    (2, 4, 2, 64, 32, 128, [1000], [100], torch.float32, 0, 0),
    (4, 18, 9, 256, 32, 64, [100, 260], [20, 33], torch.bfloat16, 0, 0),
    (2, 32, 2, 256, 64, 48, [513], [40], torch.float16, 200, 7),
    (4, 4, 1, 256, 256, 64, [600, 1], [90, 1], torch.float32, 0, 0),
    (4, 10, 5, 160, 32, 32, [200, 31], [30, 64], torch.bfloat16, 90, 4),  # five groups
    (2, 2, 1, 224, 32, 56, [111], [70], torch.float16, 0, 0),
    (4, 2, 2, 192, 64, 64, [70], [200], torch.bfloat16, 0, 0),
    (4, 128, 1, 128, 32, 64, [300], [6], torch.bfloat16, 0, 0),           # a token's heads over several tiles
    (2, 16, 16, 32, 32, 20, [41, 60, 0], [7, 1, 19], torch.bfloat16, 25, 2),
    (4, 7, 1, 128, 32, 64, [50], [77], torch.float16, 0, 0),              # rows of tokens that end inside a tile
    (4, 64, 4, 128, 32, 64, [2000, 0], [16, 300], torch.float32, 0, 0),
]
NAMES = lambda s: "-".join(map(str, s[:6])) + f"-{len(s[6])}-w{s[9]}"  # noqa: E731


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("shape", SHAPES, ids=NAMES)
def test_tokens_match_the_oracle(cuda_device, shape, tree, out32):
    bits, qh, kvh, d, g, bt, before, counts, dtype, window, sink = shape
    rng, pool, table, lengths, offsets, q = problem(cuda_device, bits, qh, kvh, d, g, bt, before, counts, dtype, sum(shape[:6]))
    parents = random_parents(rng, counts) if tree else None
    batch = paged(cuda_device, pool, table, lengths, bits, g)
    scale = 1 / math.sqrt(d)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, scale, parents, window, sink)
    out_dtype = torch.float32 if out32 else dtype
    precise = out_dtype == torch.float32
    backend = HipAttentionBackend()
    up = ints(cuda_device, parents) if tree else None
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), dict(max_length=1, total_tokens=1)):
        out, lse = backend.run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), up, window=window, sink=sink,
                                            out_dtype=out_dtype, **hints)
        assert out.dtype == out_dtype
        check(out, lse, want, d, max(lengths), out_dtype, precise)


# lengths with every relation to window, sinks and the stages' borders
@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize(("window", "sink"), [(1, 0), (64, 0), (64, 64), (100, 4), (63, 65), (129, 1), (1000, 200), (5, 3000)])
@pytest.mark.parametrize(("bits", "qh", "kvh", "d", "g", "bt", "dtype"), [
    (4, 32, 8, 128, 32, 64, torch.bfloat16), (4, 8, 2, 64, 32, 20, torch.float16), (2, 10, 5, 96, 32, 32, torch.float32),
    (2, 16, 2, 256, 64, 128, torch.float16),
])
def test_a_window_for_single_tokens(cuda_device, bits, qh, kvh, d, g, bt, dtype, window, sink, out32):
    lengths = [0, 1, 63, 64, 65, 128, 200, 1001, 2500]
    rng, pool, table, _, offsets, q = problem(cuda_device, bits, qh, kvh, d, g, bt, [n - 1 for n in lengths], [1] * 9, dtype,
                                              window + sink + d)
    table[8, 300 // bt:700 // bt] = -1  # pages that nobody sees may be gone (sinks of 3000: skipped slots)
    batch = paged(cuda_device, pool, table, lengths, bits, g)
    scale = 1 / math.sqrt(d)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, scale, None, window, sink)
    out_dtype = torch.float32 if out32 else dtype
    backend = HipAttentionBackend()
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), dict(max_length=1, total_tokens=1)):
        out, lse = backend.run_paged(q, batch, scale, out_dtype=out_dtype, window=window, sink=sink, **hints)
        check(out, lse, want, d, max(lengths), out_dtype, out_dtype == torch.float32)
    # as many tokens a sequence: one
    out, lse = backend.run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), out_dtype=out_dtype, window=window, sink=sink)
    check(out, lse, want, d, max(lengths), out_dtype, out_dtype == torch.float32)


@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize(("context", "count"), [(0, 700), (5000, 3), (20000, 16), (3000, 300)])
def test_long_sequences_are_split_and_joined(cuda_device, context, count, tree):
    counts = [count, 1, min(count, 9)]
    before = [context, 0, context // 3]
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 4, 2, 64, 32, 64, before, counts, torch.float16, context + count)
    parents = random_parents(rng, counts, 0.2) if tree else None
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125, parents)
    up = ints(cuda_device, parents) if tree else None
    backend = HipAttentionBackend()
    for out_dtype in (torch.float16, torch.float32):
        out, lse = backend.run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets), up, out_dtype=out_dtype,
                                            max_length=max(lengths), total_tokens=sum(lengths))
        check(out, lse, want, 64, max(lengths), out_dtype, out_dtype == torch.float32)
        again, again_lse = backend.run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets), up, out_dtype=out_dtype,
                                                    max_length=max(lengths), total_tokens=sum(lengths))
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_deep_and_wide_trees(cuda_device):
    counts = [300, 257, 64]
    before = [10, 0, 129]
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 4, 2, 64, 32, 64, before, counts, torch.float16, 11)
    star = np.concatenate([[-1], np.zeros(256, np.int64)])  # all children of one
    deep = np.arange(300) - 1
    odd = rng.integers(-1000, 1000, 64)  # numbers that are no earlier token's make children of the context
    parents = np.concatenate([deep, star, odd]).astype(np.int32)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    for window, sink in ((0, 0), (40, 3)):
        want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125, parents, window, sink)
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets), ints(cuda_device, parents),
                                                          window=window, sink=sink, out_dtype=torch.float16)
        check(out, lse, want, 64, max(lengths), torch.float16, False)
    # a chain is a causal chunk
    causal, _ = HipAttentionBackend().run_paged_tokens(q[:300], paged(cuda_device, pool, table[:1], lengths[:1], 4, 32), 0.125,
                                                       ints(cuda_device, [0, 300]))
    tree, _ = HipAttentionBackend().run_paged_tokens(q[:300], paged(cuda_device, pool, table[:1], lengths[:1], 4, 32), 0.125,
                                                     ints(cuda_device, [0, 300]), ints(cuda_device, deep))
    torch.testing.assert_close(causal, tree, atol=2e-5, rtol=2e-5)  # 32-bit grade, another order of sums at most


def test_tokens_of_no_sequence_and_offsets_of_any_kind(cuda_device):
    rng, pool, table, lengths, _, q = problem(cuda_device, 4, 4, 2, 64, 32, 16, [20, 0, 40, 7], [10, 5, 0, 9], torch.float16, 3)
    q = torch.cat([q, q, q])[:40]
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    offsets = np.array([6, 16, 21, 21, 30])
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets))
    check(out, lse, want, 64, 60, torch.float32, True)
    assert (out[:6] == 0).all() and (out[30:] == 0).all() and (lse[30:] == -torch.inf).all()
    # more tokens than slots: the first ones have none
    batch = paged(cuda_device, pool, table, [4, 2, 0, 16], 4, 32)
    want = attend_tokens(as_double(q), pool, table, [4, 2, 0, 16], offsets, 4, 0.125)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets))
    check(out, lse, want, 64, 60, torch.float32, True)
    # lengths past the table's row, or negative
    batch = paged(cuda_device, pool, table, [10000, -5, 3, 16], 4, 32)
    want = attend_tokens(as_double(q), pool, table, [10000, -5, 3, 16], offsets, 4, 0.125)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets))
    check(out, lse, want, 64, 200, torch.float32, True)
    # offsets past the tokens name those that there are; falling ones name none
    for offsets in ([0, 50, 60, 60, 70], [-9, 12, 12, 12, 12], [0, 10, 5, 5, 5], [40, 40, 40, 40, 40], [50, 60, 70, 80, 90]):
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets))
        assert torch.isfinite(out).all() and not torch.isnan(lse).any()
    empty, empty_lse = HipAttentionBackend().run_paged_tokens(q[:0], batch, 0.125, ints(cuda_device, [0] * 5))
    assert empty.shape == (0, 4, 64) and empty_lse.shape == (0, 4)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_what_a_token_does_not_see_has_no_part_whatever_it_holds(cuda_device, dtype):
    """Infinities and NaN as scales of slots that are masked for some tokens and seen by others, of slots that nobody
    sees, of unused slots; NaN in one token's query."""
    counts, before = [40, 30], [100, 70]
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 4, 2, 64, 32, 32, before, counts, dtype, 8)
    parents = random_parents(rng, counts, 0.0)
    pk, pv, sk, sv = (x.copy() for x in pool)
    clean = (pk, pv, sk, sv)
    dirty = tuple(x.copy() for x in clean)
    base = np.array(before)
    bad = {0: [3, 50, 100 + 17, 100 + 39], 1: [0, 70 + 12]}  # slots: outside windows, and among the new tokens
    seen_bad = {}
    for b, slots in bad.items():
        for x, slot in enumerate(slots):
            row = table[b][slot // 32] * 32 + slot % 32
            for which, value in ((2, np.nan), (3, (np.inf, np.nan, -np.inf)[x % 3])):
                dirty[which].reshape(-1, 2, 2)[row, x % 2] = value
    used = {table[b][s // 32] * 32 + s % 32 for b in range(2) for s in range(lengths[b])}
    unused = np.array([r for r in range(pk.shape[0] * 32) if r not in used])
    for which in (2, 3):
        dirty[which].reshape(-1, 2, 2)[unused] = np.nan
    q = q.clone()
    q[offsets[1] + 3, 1] = float("nan")
    from tokens_oracle import visible

    for up, window, sink in ((None, 0, 0), (None, 25, 3), (parents, 0, 0), (parents, 20, 0)):
        want = attend_tokens(as_double(q), clean, table, lengths, offsets, 4, 0.125, up, window, sink)
        out, lse = HipAttentionBackend().run_paged_tokens(
            q, paged(cuda_device, dirty, table, lengths, 4, 32), 0.125, ints(cuda_device, offsets),
            None if up is None else ints(cuda_device, up), window=window, sink=sink, out_dtype=dtype)
        touched = np.zeros((70, 4), bool)
        touched[offsets[1] + 3, 1] = True
        for b, slots in bad.items():
            seen = visible(lengths[b], counts[b], None if up is None else up[offsets[b]:offsets[b + 1]], window, sink)
            for x, slot in enumerate(slots):
                heads = slice(2 * (x % 2), 2 * (x % 2) + 2)
                touched[offsets[b]:offsets[b + 1], heads] |= seen[:, slot][:, None]
        assert touched.any() and not touched.all()
        got, got_lse = as_double(out), as_double(lse)
        assert np.isnan(got_lse[touched]).all()  # (NaN keys) and what does not see them is as without them:
        ok = ~touched
        part = dict(out=want["out"][ok], lse=want["lse"][ok], size=want["size"][ok], reach=want["reach"])
        check(torch.from_numpy(got[ok]).to(dtype), torch.from_numpy(got_lse[ok]).float(), part, 64, 140, dtype, dtype == torch.float32)
    # infinite values alone: seen they are infinite or NaN, and nothing elsewhere
    for value in (np.inf, -np.inf, np.nan):
        only = tuple(x.copy() for x in clean)
        row = table[0][(100 + 17) // 32] * 32 + (100 + 17) % 32
        only[3].reshape(-1, 2, 2)[row, 0, 1] = value
        want = attend_tokens(as_double(q), clean, table, lengths, offsets, 4, 0.125)
        out, lse = HipAttentionBackend().run_paged_tokens(q, paged(cuda_device, only, table, lengths, 4, 32), 0.125,
                                                          ints(cuda_device, offsets), out_dtype=dtype)
        got = as_double(out)
        assert not np.isfinite(got[17:40, :2, 32:]).any()
        ok = np.isfinite(got)
        ok[17:40, :2, 32:] = True
        assert ok[:43].all() and ok[44:].all()
        err = np.abs(got - want["out"])[np.isfinite(got)]
        assert (err <= 2e-2).all()  # (sizes of 1: 2^-10 and the type's rounding are far below)


def test_pages_that_are_not_there(cuda_device):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 32, [200, 64], [70, 5], torch.bfloat16, 14)
    table[0, 1], table[0, 6], table[1, 0] = -1, 100000, -7
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    for window in (0, 50):
        want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.1, None, window)
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.1, ints(cuda_device, offsets), window=window,
                                                          out_dtype=torch.bfloat16)
        check(out, lse, want, 128, 270, torch.bfloat16, False)
    table[:] = -1
    out, lse = HipAttentionBackend().run_paged_tokens(q, paged(cuda_device, pool, table, lengths, 4, 32), 0.1,
                                                      ints(cuda_device, offsets))
    assert (out == 0).all() and (lse == -torch.inf).all()


@pytest.mark.parametrize("scales", [(6e-8, 3e-7), (1e-5, 1e-3), (5e3, 6e4)], ids=["subnormal", "small", "large"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_any_size(cuda_device, scales, dtype):
    """Value scales over fp16's whole range, keys' scales as usual; a sequence whose later slots are far larger."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 64, [300, 10], [40, 100], dtype, 15)
    pool = list(pool)
    pool[3] = np.exp(rng.uniform(*np.log(scales), pool[3].shape)).astype(np.float16)
    rows = [table[0][s // 64] * 64 + s % 64 for s in range(150, 170)]
    pool[3].reshape(-1, 2, 4)[rows] *= np.float16(1.0 if scales[1] > 1e3 else 200.0)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    scale = 1 / math.sqrt(128)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, scale)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), out_dtype=dtype)
    check(out, lse, want, 128, 340, dtype, dtype == torch.float32)


@pytest.mark.parametrize("factor", [1e-4, 30.0, 1000.0])
def test_queries_and_scales_of_any_size(cuda_device, factor):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 64, [300, 10], [40, 100], torch.float32, 16)
    q = (q * torch.exp(2 * torch.randn(q.shape[:2], generator=torch.Generator().manual_seed(1)).to(q))[..., None] * factor)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = q.to(dtype)
        for scale in (0.125 / factor, -0.125 / factor, 0.0):
            batch = paged(cuda_device, pool, table, lengths, 4, 32)
            want = attend_tokens(as_double(x), pool, table, lengths, offsets, 4, scale)
            out, lse = HipAttentionBackend().run_paged_tokens(x, batch, scale, ints(cuda_device, offsets), out_dtype=dtype)
            # (of rows that the type holds: an infinite query has no scores)
            ok = torch.isfinite(x).all(-1).cpu().numpy()
            assert ok.any()
            part = dict(out=want["out"][ok], lse=want["lse"][ok], size=want["size"][ok], reach=want["reach"])
            check(out.cpu()[torch.from_numpy(ok)], lse.cpu()[torch.from_numpy(ok)], part, 64, 340, dtype, dtype == torch.float32)


@pytest.mark.parametrize("layout", ["fused", "heads first", "every second dim", "one byte off"])
def test_queries_of_any_strides(cuda_device, layout):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 96, 32, 64, [30, 10], [40, 21], torch.bfloat16, 17)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    if layout == "fused":
        wide = torch.randn((61, 13, 96), device=cuda_device).bfloat16()
        wide[:, 2:10] = q
        x = wide[:, 2:10]
    elif layout == "heads first":
        x = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "every second dim":
        wide = torch.zeros((61, 8, 192), device=cuda_device).bfloat16()
        wide[..., ::2] = q
        x = wide[..., ::2]
    else:
        flat = torch.zeros(61 * 8 * 96 + 1, device=cuda_device).bfloat16()
        flat[1:] = q.flatten()
        x = flat[1:].view(61, 8, 96)
    assert torch.equal(x, q)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.1)
    out, lse = HipAttentionBackend().run_paged_tokens(x, batch, 0.1, ints(cuda_device, offsets), out_dtype=torch.bfloat16)
    assert out.is_contiguous()
    check(out, lse, want, 96, 70, torch.bfloat16, False)
    run = HipAttentionBackend().prepare_paged_tokens(q, batch, 0.1, out_dtype=torch.bfloat16)
    again, _ = run(x, ints(cuda_device, offsets))
    assert torch.equal(out, again)


def test_offsets_past_32_bits(cuda_device):
    """A pool of 4.4 GB of codes, a sequence in its last pages."""
    kvh, d, bt = 16, 256, 64
    pages = 33600  # rows of 2,048 bytes: 2^32 bytes end at page 32,768
    codes = [torch.zeros((pages, bt, kvh, d // 2), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    scales = [torch.zeros((pages, bt, kvh, d // 32), dtype=torch.float16, device=cuda_device) for _ in range(2)]
    rng = np.random.default_rng(18)
    small = make_pool(rng, 4, bt, kvh, d, 32, 4)
    for big, part in zip((codes[0], codes[1], scales[0], scales[1]), small):
        big[-4:] = torch.from_numpy(part).to(cuda_device)
    small_table = np.array([[2, 0, 3, 1]], np.int32)
    table = small_table + pages - 4
    q = torch.from_numpy(rng.standard_normal((30, 16, d))).half().to(cuda_device)
    want = attend_tokens(as_double(q), small, small_table, [230], [0, 30], 4, 0.06)
    batch = PagedBatch(*codes, *scales, ints(cuda_device, table[0]).view(1, 4), ints(cuda_device, [230]), 4, 32)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.06, ints(cuda_device, [0, 30]), out_dtype=torch.float16)
    check(out, lse, want, d, 230, torch.float16, False)
    one, one_lse = HipAttentionBackend().run_paged(q[29:], batch, 0.06, out_dtype=torch.float16, window=60, sink=2)
    want = attend_tokens(as_double(q[29:]), small, small_table, [230], [0, 1], 4, 0.06, None, 60, 2)
    check(one, one_lse, want, d, 230, torch.float16, False)
    lengths = keep_tokens(batch, ints(cuda_device, [30]), ints(cuda_device, [5, 7, 29]).view(1, 3))
    assert lengths.tolist() == [203]
    pools, _, _, _ = keep(small, small_table, [230], [30], [[5, 7, 29]])
    for big, part in zip((codes[0], codes[1], scales[0], scales[1]), pools):
        assert np.array_equal(big[-4:].cpu().numpy(), part)


def test_another_stream_and_a_captured_step(cuda_device):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 64, [3000, 10], [16, 16], torch.float16, 19)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    parents = random_parents(rng, [16, 16])
    off, up = ints(cuda_device, offsets), ints(cuda_device, parents)
    backend = HipAttentionBackend()
    run = backend.prepare_paged_tokens(q, batch, 0.08, out_dtype=torch.float16)
    one = backend.prepare_paged(q[:2], batch, 0.08, out_dtype=torch.float16, window=200, sink=4)
    want, want_lse = run(q, off, up)
    want_one, _ = one(q[:2])
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_lse = run(q, off, up)
        got_one, _ = one(q[:2])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse) and torch.equal(got_one, want_one)
    graphs, outs = [], []
    for _ in range(2):  # two graphs share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((*run(q, off, up), one(q[:2])[0]))
        graphs.append(graph)
    first = batch.lengths.clone()
    for more in (0, -7, 0, -300):  # (the first sequence alone)
        batch.lengths.copy_(first)
        batch.lengths[0] += more
        want, want_lse = run(q, off, up)
        want_one, _ = one(q[:2])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, lse, single in outs:
            assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(single, want_one)


def test_prepared_calls_keep_apart(cuda_device):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 64, [30, 10], [7, 2], torch.float16, 20)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    run = HipAttentionBackend().prepare_paged_tokens(q, batch, 0.125, out_dtype=torch.float16)
    off = ints(cuda_device, offsets)
    outs = [run(q * (1 + i), off)[0] for i in range(70)]
    fresh = [HipAttentionBackend().run_paged_tokens(q * (1 + i), batch, 0.125, off, out_dtype=torch.float16)[0] for i in range(70)]
    assert all(torch.equal(a, b) for a, b in zip(outs, fresh))
    for bad in (q[:8], q.float(), q[:, :4]):
        with pytest.raises(ValueError, match="does not match the prepared"):
            run(bad, off)
    with pytest.raises(ValueError, match="offsets must be int32"):
        run(q, off.long())
    with pytest.raises(ValueError, match="parents must be int32"):
        run(q, off, ints(cuda_device, [0] * 8))
    with pytest.raises(ValueError, match="no backward pass"):
        run(q.clone().requires_grad_(), off)


def test_the_portable_backend_computes_the_same(cuda_device):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 16, [30, 0], [17, 12], torch.float16, 21)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    parents = ints(cuda_device, random_parents(rng, [17, 12]))
    off = ints(cuda_device, offsets)
    for up, window, sink in ((None, 0, 0), (parents, 0, 0), (parents, 9, 2), (None, 9, 2)):
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, off, up, window=window, sink=sink)
        ref, ref_lse = ReferenceAttentionBackend().run_paged_tokens(q, batch, 0.125, off, up, window=window, sink=sink)
        # both 32-bit grade: 2e-5 is the tolerance of the packed decodes' 32-bit kernels
        torch.testing.assert_close(out, ref, atol=2e-5, rtol=2e-5)
        torch.testing.assert_close(lse, ref_lse, atol=2e-5, rtol=2e-5)
    out, lse = HipAttentionBackend().run_paged(q[:2], batch, 0.125, window=9, sink=2)
    ref, ref_lse = ReferenceAttentionBackend().run_paged(q[:2], batch, 0.125, window=9, sink=2)
    torch.testing.assert_close(out, ref, atol=2e-5, rtol=2e-5)
    torch.testing.assert_close(lse, ref_lse, atol=2e-5, rtol=2e-5)


# ------------------------------------------------------------------------------------------------------------ keeping


@pytest.mark.parametrize(("bits", "kvh", "d", "g", "bt"), [
    (4, 8, 128, 32, 64), (2, 1, 32, 32, 16), (4, 3, 96, 32, 20), (2, 5, 32, 32, 1), (4, 2, 256, 256, 128), (2, 3, 64, 64, 24),
])
@pytest.mark.parametrize("tracked", [False, True])
def test_kept_rows(cuda_device, bits, kvh, d, g, bt, tracked):
    rng = np.random.default_rng(bits + kvh + d)
    lengths = [0, 1, 30, 100, 65, 64, 700, 40, 10]
    drafted = [0, 1, 30, 40, 64, 70, 600, 8, -3]
    width = 600
    kept = np.full((9, width), -1, np.int32)
    lists = [[], [0], [29], sorted(rng.choice(40, 17, False)), list(range(64)), [1, 5, 5, 6], sorted(rng.choice(600, 590, False)),
             [2, 3, 8, 9], [0, 1]]
    for b, x in enumerate(lists):
        kept[b, :len(x)] = x
    pages = sum(-(-n // bt) for n in lengths) + 2
    pool = make_pool(rng, pages, bt, kvh, d, g, bits)
    table = make_table(rng, lengths, bt, -(-700 // bt) + 1, pages)
    shape = (9, table.shape[1] * bt)
    weights = rng.uniform(0, 3, shape).astype(np.float32) if tracked else None
    positions = rng.integers(0, 1 << 20, shape).astype(np.int32) if tracked else None
    batch = paged(cuda_device, pool, table, lengths, bits, g, weights, positions)
    want = keep(pool, table, lengths, drafted, kept, weights, positions)
    got = keep_tokens(batch, ints(cuda_device, drafted), torch.from_numpy(kept).to(cuda_device))
    assert got.tolist() == list(want[1]) and batch.lengths.tolist() == lengths
    for a, b in zip((batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v), want[0]):
        assert np.array_equal(a.cpu().numpy().view(np.uint8), b.view(np.uint8))
    if tracked:
        assert np.array_equal(batch.weights.cpu().numpy(), want[2]) and np.array_equal(batch.positions.cpu().numpy(), want[3])
    # nothing kept, without a list; then the lengths in place
    assert keep_tokens(batch, ints(cuda_device, drafted), torch.empty((9, 0), dtype=torch.int32, device=cuda_device)).tolist() == [
        n - max(0, min(x, n)) for n, x in zip(lengths, drafted)]
    got = keep_tokens(batch, ints(cuda_device, [0, 1, 1, 1, 0, 0, 0, 0, 1]), torch.from_numpy(kept[:, :1].copy()).to(cuda_device),
                      lengths_out=batch.lengths)
    assert got is batch.lengths and got.tolist() == [0, 1, 29, 99 + (kept[3, 0] == 0), 65, 64, 700, 40, 10]


def test_kept_rows_without_a_page_do_not_move(cuda_device):
    rng = np.random.default_rng(31)
    pool = make_pool(rng, 8, 16, 2, 64, 32, 4)
    table = np.array([[3, 1, -1, 5], [0, 100, 2, 4]], np.int32)
    kept = np.array([[4, 12, 20, 21], [1, 3, 25, 30]], np.int32)
    batch = paged(cuda_device, pool, table, [60, 60], 4, 32)
    got = keep_tokens(batch, ints(cuda_device, [40, 50]), torch.from_numpy(kept).to(cuda_device))
    want = keep(pool, table, [60, 60], [40, 50], kept)
    assert got.tolist() == list(want[1]) == [24, 14]
    for a, b in zip((batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v), want[0]):
        assert np.array_equal(a.cpu().numpy(), b)


# ------------------------------------------------------------------------------------------------------ a run of them


@pytest.mark.parametrize(("bits", "layout"), [(4, "half"), (2, "interleaved")])
def test_drafting_leaves_the_cache_that_plain_decoding_does(cuda_device, bits, layout):
    """Steps of drafted trees, of which a path is kept, against a cache that is given those tokens one by one: codes,
    scales, positions and lengths are the same bits, and attention over them agrees."""
    rng = np.random.default_rng(41)
    kvh, qh, d, sequences = 2, 8, 64, 3
    make = lambda: PagedKVCache(60, 16, kvh, d, bits=bits, sequences=sequences, max_pages=20, track_weights=True,  # noqa: E731
                                device=cuda_device)
    drafting, plain = make(), make()
    rotary = Rotary(d, layout=layout, device=cuda_device)

    def heads(n, h):
        return torch.from_numpy(rng.standard_normal((n, h, d))).bfloat16().to(cuda_device)

    counts = [40, 3, 0]
    keys, values, query = heads(43, kvh), heads(43, kvh), heads(43, qh)
    for cache in (drafting, plain):
        turned = cache.append(keys, values, counts, rotary=rotary, query=query)
    out, lse = drafting.attend_tokens(turned, counts, window=20, sink=2)
    lengths = list(drafting.lengths)
    pool = [t.cpu().numpy() for t in (drafting.batch.packed_k, drafting.batch.packed_v, drafting.batch.scales_k, drafting.batch.scales_v)]
    want = attend_tokens(as_double(turned), pool, drafting.batch.page_table.cpu().numpy(), lengths, [0, 40, 43, 43], bits, 0.125,
                         None, 20, 2)
    check(out, lse, want, d, 40, torch.float32, True)
    for step in range(6):
        counts = [int(n) for n in rng.integers(1, 14, sequences)]
        if step == 3:
            counts[1] = 0
        parents = random_parents(rng, counts)
        n = sum(counts)
        keys, values, query = heads(n, kvh), heads(n, kvh), heads(n, qh)
        up = ints(cuda_device, parents) if step % 2 else parents.tolist()
        turned = drafting.append(keys, values, counts, rotary=rotary, query=query, parents=up)
        with pytest.raises(RuntimeError, match="drafted"):
            drafting.attend(query[:3])
        with pytest.raises(RuntimeError, match="drafted"):
            drafting.append(keys, values, counts)
        out, lse = drafting.attend_tokens(turned, counts, parents=up)
        ends = np.concatenate([[0], np.cumsum(counts)])
        pool = [t.cpu().numpy() for t in (drafting.batch.packed_k, drafting.batch.packed_v, drafting.batch.scales_k, drafting.batch.scales_v)]
        want = attend_tokens(as_double(turned), pool, drafting.batch.page_table.cpu().numpy(), drafting.lengths, ends, bits, 0.125, parents)
        check(out, lse, want, d, max(drafting.lengths), torch.float32, True)
        paths = []
        for b in range(sequences):
            path = chain(parents[ends[b]:ends[b + 1]], int(rng.integers(0, counts[b])))[::-1] if counts[b] else []
            paths.append(path[:int(rng.integers(0, len(path) + 1))])
        drafting.keep(paths)
        # the same tokens, one after the other, in the other cache; their attention is what the tree's was
        longest = max(len(p) for p in paths)
        for j in range(longest):
            now = [int(j < len(p)) for p in paths]
            rows = [int(ends[b]) + p[j] for b, p in enumerate(paths) if j < len(p)]
            q = plain.append(keys[rows], values[rows], now, rotary=rotary, query=query[rows])
            assert torch.equal(q, turned[rows])
            one, one_lse = plain.attend_tokens(q, now)
            torch.testing.assert_close(one, out[rows], atol=2e-5, rtol=2e-5)
            torch.testing.assert_close(one_lse, lse[rows], atol=2e-5, rtol=2e-5)
        assert drafting.lengths == plain.lengths and drafting.next_positions == plain.next_positions
        assert drafting.free_pages == plain.free_pages
        assert torch.equal(drafting.batch.lengths, plain.batch.lengths)
        for b, length in enumerate(plain.lengths):
            slots = torch.arange(length, device=cuda_device)
            rows = [c.batch.page_table[b].long()[slots // 16] * 16 + slots % 16 for c in (drafting, plain)]
            for name in ("packed_k", "packed_v", "scales_k", "scales_v"):
                a, other = (getattr(c.batch, name).flatten(0, 1)[r] for c, r in zip((drafting, plain), rows))
                assert torch.equal(a, other)
            assert torch.equal(drafting.batch.positions[b, :length], plain.batch.positions[b, :length])
        query = heads(sequences, qh)
        for window in (0, 9):
            a, _ = drafting.attend(query, window=window, sink=1 if window else 0)
            other, _ = plain.attend(query, window=window, sink=1 if window else 0)
            torch.testing.assert_close(a, other, atol=2e-5, rtol=2e-5)
    # after an eviction positions differ from slots: trees go on, windows are refused
    drafting.attend(query, accumulate=True)
    drafting.evict(20, sink=2, recent=5)
    with pytest.raises(ValueError, match="window"):
        drafting.attend(query, window=9)
    with pytest.raises(ValueError, match="window"):
        drafting.attend_tokens(query, window=9)
    first = list(drafting.next_positions)
    base = list(drafting.lengths)
    keys, values, query = heads(9, kvh), heads(9, kvh), heads(9, qh)
    parents = [-1, 0, 0] * 3
    turned = drafting.append(keys, values, [3, 3, 3], rotary=rotary, query=query, parents=parents)
    assert [drafting.batch.positions[b, base[b]:base[b] + 3].tolist() for b in range(3)] == [[p, p + 1, p + 1] for p in first]
    out, _ = drafting.attend_tokens(turned, [3, 3, 3], parents=parents)
    assert torch.isfinite(out).all()
    drafting.keep([[0, 2], [], [0]])
    assert drafting.next_positions == [first[0] + 2, first[1], first[2] + 1]
    assert drafting.batch.positions[0, base[0]:base[0] + 2].tolist() == [first[0], first[0] + 1]


def test_positions_of_a_tree(cuda_device):
    """append_tokens turns a tree's keys and queries by first + depth."""
    rng = np.random.default_rng(51)
    counts = [30, 0, 64, 5]
    parents = random_parents(rng, counts)
    first = np.array([7, 100, 1000000, 0])
    d, kvh = 64, 2
    n = sum(counts)
    x = torch.from_numpy(rng.standard_normal((n, kvh, d))).half().to(cuda_device)
    q = torch.from_numpy(rng.standard_normal((n, 4, d))).half().to(cuda_device)
    rotary = Rotary(d, device=cuda_device)
    ends = np.concatenate([[0], np.cumsum(counts)])
    places = np.concatenate([
        [first[b] + len(chain(parents[ends[b]:ends[b + 1]], i)) - 1 for i in range(c)] for b, c in enumerate(counts)
    ]).astype(np.int64)

    def cache():
        rng = np.random.default_rng(1)
        pool = make_pool(rng, 16, 16, kvh, d, 32, 4)
        table = make_table(rng, [40, 1, 80, 10], 16, 6, 16)
        return paged(cuda_device, pool, table, [3, 1, 9, 0], 4, 32, np.zeros((4, 96), np.float32), np.full((4, 96), -1, np.int32))

    a, b = cache(), cache()
    turned, lengths = append_tokens(a, x, x, offsets=ints(cuda_device, ends), rotary=rotary, query=q,
                                    first_positions=ints(cuda_device, first), parents=ints(cuda_device, parents))
    want_q, want_k = rotary(torch.from_numpy(places).to(cuda_device), q, x)
    assert torch.equal(turned, want_q) and lengths.tolist() == [33, 1, 73, 5]
    append_tokens(b, want_k, x, offsets=ints(cuda_device, ends))
    for name in ("packed_k", "packed_v", "scales_k", "scales_v"):
        assert torch.equal(getattr(a, name), getattr(b, name))
    for s, (length, c) in enumerate(zip([3, 1, 9, 0], counts)):
        assert a.positions[s, length:length + c].tolist() == places[ends[s]:ends[s + 1]].tolist()
