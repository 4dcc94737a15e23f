"""Batches of many sequences with few new tokens each, deep trees, and calls at the edges of what is allowed, on the GPU
against the 64-bit oracles (tolerances: test_gpu_paged_tokens)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, keep_tokens
from kvssd.backends.hip import HipAttentionBackend
from paged_oracle import as_double, make_pool, make_table
from test_gpu_paged_tokens import check, ints, paged, problem, random_parents
from tokens_oracle import attend_tokens, chain, keep, visible

pytestmark = pytest.mark.gpu


# bits, query heads, kv heads, head_dim, group, page_tokens, slots before, new tokens, window, sink: at most 32 rows of a
# kv head and sequence on average
FEW = [
    (4, 32, 8, 128, 32, 64, [0, 5, 63, 64, 255, 256, 1000], [1, 8, 1, 4, 8, 2, 8], 0, 0),
    (4, 32, 8, 128, 128, 24, [700, 3], [8, 8], 100, 30),
    (2, 16, 4, 128, 64, 64, [513, 40, 0], [6, 0, 9], 0, 0),
    (4, 8, 2, 96, 32, 16, [300, 20], [7, 3], 0, 0),
    (2, 4, 2, 96, 32, 40, [130, 600], [5, 10], 64, 4),
    (4, 16, 1, 64, 32, 64, [1500], [2], 0, 0),
    (2, 2, 2, 32, 32, 7, [290, 0, 0, 31], [20, 1, 0, 9], 33, 2),
    (4, 5, 1, 64, 64, 128, [900, 260], [6, 6], 0, 0),
    (4, 8, 2, 256, 64, 64, [500, 3], [5, 5], 0, 0),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "-".join(map(str, s[:6])) + f"-{len(s[6])}-w{s[8]}")
def test_few_tokens_a_sequence(cuda_device, shape, tree, dtype):
    bits, qh, kvh, d, g, bt, before, counts, window, sink = shape
    rng, pool, table, lengths, offsets, q = problem(cuda_device, bits, qh, kvh, d, g, bt, before, counts, dtype, 60 + qh)
    parents = random_parents(rng, counts) if tree else None
    scale = 1 / d ** 0.5
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, scale, parents, window, sink)
    batch = paged(cuda_device, pool, table, lengths, bits, g)
    up = None if parents is None else ints(cuda_device, parents)
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), dict(max_length=1, total_tokens=1)):
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), up, window=window,
                                                          sink=sink, out_dtype=dtype, **hints)
        check(out, lse, want, d, max(lengths), dtype, False)


@pytest.mark.parametrize("sequences", [62, 63, 64, 200, 1100])
def test_many_sequences(cuda_device, sequences):
    rng = np.random.default_rng(sequences)
    before, counts = rng.integers(0, 40, sequences), rng.integers(0, 4, sequences)
    before[sequences // 2], counts[sequences // 2] = 700, 60  # one far longer
    before[7:12] = counts[7:12] = 0
    _, pool, table, lengths, offsets, q = problem(cuda_device, 4, 4, 2, 64, 32, 16, before.tolist(), counts.tolist(), torch.float16, 70)
    q = torch.cat([q[:3], q, q[:2]])  # tokens of no sequence at both ends
    offsets = offsets + 3
    parents = np.concatenate([[5, 0, -1], random_parents(rng, counts.tolist()), [0, 1]])
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    off = ints(cuda_device, offsets)
    for up, window in ((None, 0), (parents, 0), (None, 9)):
        want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125, up, window, 2)
        for hints in ({}, dict(max_length=760, total_tokens=int(sum(lengths)))):
            out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, off, None if up is None else ints(cuda_device, up),
                                                              window=window, sink=2, out_dtype=torch.float16, **hints)
            check(out, lse, want, 64, 760, torch.float16, False)
    # offsets of any kind, none of which may be left without an end
    for bad in (rng.integers(-5, len(q) + 9, sequences + 1), np.arange(sequences + 1)[::-1], np.tile([0, len(q)], sequences)[:sequences + 1]):
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, bad), out_dtype=torch.float16)
        assert out.shape == q.shape


def test_many_sequences_in_a_graph(cuda_device):
    rng = np.random.default_rng(71)
    sequences = 90
    before, counts = rng.integers(0, 300, sequences).tolist(), [3] * sequences
    _, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 16, before, counts, torch.bfloat16, 72)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    off, up = ints(cuda_device, offsets), ints(cuda_device, random_parents(rng, counts))
    run = HipAttentionBackend().prepare_paged_tokens(q, batch, 0.09, out_dtype=torch.bfloat16)
    run(q, off, up)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(q, off, up))
        graphs.append(graph)
    first = batch.lengths.clone()
    for shift in (0, 30, 1, 0):
        batch.lengths.copy_(first.roll(shift).clamp(max=int(first.max())))
        want, want_lse = run(q, off, up)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, lse in outs:
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("window", [0, 50])
def test_trees_of_thousands(cuda_device, window):
    """More tokens than parents are kept nearby; one of the trees is a path."""
    counts, before = [1500, 1100], [40, 7]
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 2, 1, 64, 32, 64, before, counts, torch.float16, 73)
    parents = np.concatenate([random_parents(rng, counts[:1], 0.2), np.arange(1100) - 1]).astype(np.int32)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125, parents, window, 3 if window else 0)
    out, lse = HipAttentionBackend().run_paged_tokens(
        q, paged(cuda_device, pool, table, lengths, 4, 32), 0.125, ints(cuda_device, offsets), ints(cuda_device, parents),
        window=window, sink=3 if window else 0, out_dtype=torch.float16)
    check(out, lse, want, 64, 1540, torch.float16, False)
    # the path sees what a prompt does
    plain, plain_lse = HipAttentionBackend().run_paged_tokens(
        q, paged(cuda_device, pool, table, lengths, 4, 32), 0.125, ints(cuda_device, offsets), window=window,
        sink=3 if window else 0, out_dtype=torch.float16)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 0.125, None, window, 3 if window else 0)
    check(plain, plain_lse, want, 64, 1540, torch.float16, False)


@pytest.mark.parametrize("window, sink", [(2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (1, 2**31 - 1), (2**40, 2**40), (1 << 30, 5)])
def test_windows_past_everything_hide_nothing(cuda_device, window, sink):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 64, [500, 10], [6, 2], torch.float16, 74)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    off, up = ints(cuda_device, offsets), ints(cuda_device, random_parents(rng, [6, 2]))
    for parents in (None, up):
        out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, off, parents, out_dtype=torch.float16)
        got, got_lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, off, parents, window=window, sink=sink, out_dtype=torch.float16)
        # (the same slots, in stages and runs that may differ: two results of one bound)
        torch.testing.assert_close(got, out, atol=2e-3, rtol=2e-3)
        torch.testing.assert_close(got_lse, lse, atol=1e-5, rtol=1e-5)
    one, one_lse = HipAttentionBackend().run_paged(q[:2], batch, 0.125)
    got, got_lse = HipAttentionBackend().run_paged(q[:2], batch, 0.125, window=window, sink=sink)
    torch.testing.assert_close(got, one, atol=1e-5, rtol=1e-5)
    torch.testing.assert_close(got_lse, one_lse, atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("counts", [[4], [40], [300]], ids=str)
def test_a_value_that_is_not_finite_is_seen_in_any_split(cuda_device, counts):
    """Its slot's weight may be nothing beside a later run's: NaN all the same, as 0 * NaN is, and alike in every split."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 64, [5000], counts, torch.float16, 75)
    pool = tuple(x.copy() for x in pool)
    pool[2].reshape(-1, 2, 4)[table[0][0] * 64:table[0][0] * 64 + 64] = 0  # keys of the first page: scores of 0
    row = table[0][0] * 64 + 10
    pool[3].reshape(-1, 2, 4)[row, 1, 2] = np.inf
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    for scale in (0.1, 20.0):
        for hints in ({}, dict(max_length=64, total_tokens=64)):
            out, lse = HipAttentionBackend().run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), out_dtype=torch.float16, **hints)
            bad = torch.isnan(out)
            assert bad[:, 4:, 64:96].all() and not bad[:, :4].any() and not bad[:, 4:, :64].any() and not bad[:, 4:, 96:].any()
            assert torch.isfinite(lse).all()


def test_a_query_broadcast_over_tokens_and_heads(cuda_device):
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 64, [100, 3], [5, 9], torch.float16, 76)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    off = ints(cuda_device, offsets)
    for x in (q[:1].expand(14, 8, 64), q[:, :1].expand(14, 8, 64), q[:1, :1].expand(14, 8, 64), q.flip(0)):
        got = HipAttentionBackend().run_paged_tokens(x, batch, 0.125, off)
        want = HipAttentionBackend().run_paged_tokens(x.contiguous(), batch, 0.125, off)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_of_a_caches_tokens_is_not_captured(cuda_device):
    cache = PagedKVCache(4, 16, 2, 64, sequences=2, device=cuda_device)
    x = torch.randn(2, 2, 64, device=cuda_device, dtype=torch.float16)
    cache.append(x, x)
    graph, before = torch.cuda.CUDAGraph(), torch.cuda.current_stream()
    with pytest.raises(RuntimeError, match="capture run_paged_tokens"):
        with torch.cuda.graph(graph):
            cache.attend_tokens(x)
    assert torch.cuda.current_stream() == before
    out, _ = cache.attend_tokens(x)
    assert torch.isfinite(out).all()


def test_a_step_of_trees_in_a_graph(cuda_device):
    """Attention over the drafted tokens and keeping a path of them, captured and replayed over changing trees."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 64, 32, 16, [90, 30, 0], [8, 8, 8], torch.float16, 77)
    table[:, 7:] = -1  # (lists no page past the sequences' own)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    off, up = ints(cuda_device, offsets), ints(cuda_device, np.tile(np.arange(8) - 1, 3))
    drafted, kept = ints(cuda_device, [8, 8, 8]), torch.zeros(3, 4, dtype=torch.int32, device=cuda_device)
    after = torch.empty_like(batch.lengths)
    run = HipAttentionBackend().prepare_paged_tokens(q, batch, 0.125, out_dtype=torch.float16)
    arrays = (batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v)
    start = [t.clone() for t in arrays]
    run(q, off, up)
    keep_tokens(batch, drafted, kept.fill_(-1), lengths_out=after)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = run(q, off, up)
        keep_tokens(batch, drafted, kept, lengths_out=after)
    for step in range(4):
        parents = random_parents(rng, [8, 8, 8])
        paths = [chain(parents[8 * b:8 * b + 8], int(rng.integers(0, 8)))[::-1][:4] for b in range(3)]
        up.copy_(ints("cpu", parents))
        kept.copy_(torch.tensor([p + [-1] * (4 - len(p)) for p in paths], dtype=torch.int32))
        for t, s in zip(arrays, start):
            t.copy_(s)
        want, want_lse = run(q, off, up)
        want_after = keep_tokens(batch, drafted, kept)
        moved = [t.clone() for t in arrays]
        for t, s in zip(arrays, start):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(after, want_after)
        assert after.tolist() == [n - 8 + len(p) for n, p in zip(lengths, paths)]
        assert all(torch.equal(t, m) for t, m in zip(arrays, moved))


def test_what_stands_behind_a_lists_end(cuda_device):
    """A list ends at its first entry that is not above the one before it or not a drafted token's; what follows may be
    anything, ascending numbers from far below 0 among it."""
    rng = np.random.default_rng(78)
    low, high = -2**31, 2**31 - 1
    lists = [
        [3, -2000000000, -1999999999, -1999999998],
        [low, low + 1, low + 2, -1, 0, 1],
        [-5, -4, -3, 0, 1, 2],
        [0, 1, high, -7, -6, -5, 2, 3],
        [2, 40, 41, -100000, -99999, 5, 6],
        [0, 5, 5, 6, 7, 8, 9],
        [1, 0, 4, 5, 6],
        list(range(512)) + [-1] + list(range(-3000000, -2999913)),          # (600 entries)
        list(range(0, 1024, 2)) + list(range(-88, 0)),
        list(range(3, 603)),
    ]
    width = 600
    kept = np.sort(rng.integers(low, high, (16, width)), axis=1).astype(np.int32)  # ascending numbers of any size
    for b, x in enumerate(lists):
        kept[b, :min(len(x), width)] = x[:width]
    kept[11] = rng.integers(low, high, width)
    kept[12] = rng.integers(-40, 40, width)
    kept[13, :9] = [4, 5, 9, 20, 21, 22, 23, 24, 39]
    drafted = [40] * 7 + [700, 1100, 650] + [40] * 4 + [0, high]
    lengths = [50] * 7 + [900, 1200, 700] + [50] * 6
    pages = sum(-(-n // 16) for n in lengths) + 2
    pool = make_pool(rng, pages, 16, 2, 64, 32, 4)
    table = make_table(rng, lengths, 16, 80, pages)
    weights = rng.uniform(0, 3, (16, 1280)).astype(np.float32)
    positions = rng.integers(0, 1 << 20, (16, 1280)).astype(np.int32)
    batch = paged(cuda_device, pool, table, lengths, 4, 32, weights, positions)
    want = keep(pool, table, lengths, drafted, kept, weights, positions)
    got = keep_tokens(batch, ints(cuda_device, drafted), torch.from_numpy(kept).to(cuda_device))
    assert got.tolist() == list(want[1])
    assert (got - ints(cuda_device, lengths) + ints(cuda_device, drafted)).tolist()[:10] == [1, 0, 0, 2, 1, 2, 1, 512, 512, 600]
    for a, b in zip((batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v), want[0]):
        assert np.array_equal(a.cpu().numpy().view(np.uint8), b.view(np.uint8))
    assert np.array_equal(batch.weights.cpu().numpy(), want[2]) and np.array_equal(batch.positions.cpu().numpy(), want[3])


@pytest.mark.parametrize(("d", "bits"), [(64, 4), (96, 2), (128, 4)])
def test_few_tokens_repeat_bit_for_bit(cuda_device, d, bits):
    """Waves that exchange keys, values and flags among their own lanes: the same bits in every pass, with slots that lie
    in no page and a value scale that is not finite among them."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, bits, 8, 2, d, 32, 32, [1500, 70, 0], [8, 6, 3], torch.float16, 79)
    pool = tuple(x.copy() for x in pool)
    table[0, [3, 17]] = -1
    pool[3].reshape(-1, 2, d // 32)[table[0][9] * 32 + 5, 1, 1] = np.inf
    batch = paged(cuda_device, pool, table, lengths, bits, 32)
    off, up = ints(cuda_device, offsets), ints(cuda_device, random_parents(rng, [8, 6, 3]))
    run = HipAttentionBackend().prepare_paged_tokens(q, batch, 0.1, out_dtype=torch.float16)
    first, first_lse = run(q, off, up)
    poisoned = torch.isnan(first)
    assert poisoned[:8, 4:, 32:64].all() and poisoned.sum() == 8 * 4 * 32
    for _ in range(50):
        out, lse = run(q, off, up)
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(first)) and torch.equal(torch.isnan(out), poisoned)
        assert torch.equal(lse, first_lse)


def test_paths_of_a_tree_given_as_a_tensor(cuda_device):
    """What is kept is checked by the parents that the append read, whatever has become of the tensor, on its stream too."""
    cache = PagedKVCache(20, 16, 2, 64, sequences=2, device=cuda_device)
    x = torch.randn(9, 2, 64, device=cuda_device, dtype=torch.float16)
    parents = [-1, 0, 0, 1, 4] + [-1, 0, 1, 1]
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(cuda_device)):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            wide = ints(cuda_device, np.repeat(parents, 2))
            cache.append(x, x, [5, 4], parents=wide[::2])  # (any stride)
            wide.fill_(-1)
            held = list(cache.lengths)
            for paths in ([[0, 3], []], [[4], [1]], [[0, 1, 2], []], [[0, 4], []], [[], [0, 1, 2, 3]]):
                with pytest.raises(ValueError, match="from child to child"):
                    cache.keep(paths)
            assert cache.lengths == held == cache.batch.lengths.tolist()
            cache.keep([[0, 1, 3], [0, 1, 3]])
            assert cache.lengths == cache.next_positions == [held[0] - 2, held[1] - 1] == cache.batch.lengths.tolist()
        torch.cuda.current_stream().wait_stream(stream)


@pytest.mark.parametrize("sequences", [4, 70])
def test_offsets_that_fall(cuda_device, sequences):
    """They name no tokens where they fall; tokens that are then named once, by a sequence or as none's, have their result."""
    rng = np.random.default_rng(sequences + 80)
    tokens = 60
    before = rng.integers(10, 60, sequences).tolist()
    _, pool, table, lengths, _, q = problem(cuda_device, 4, 4, 2, 64, 32, 16, before, [tokens] * sequences, torch.float16, 80)
    q = q[:tokens]
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    for trial in range(6):
        offsets = np.sort(rng.integers(-5, tokens + 10, sequences + 1))
        at = int(rng.integers(0, sequences))
        offsets[at], offsets[at + 1] = offsets[at + 1] + 3, offsets[at] - 2  # one pair the wrong way round
        ends = np.clip(offsets, 0, tokens)
        named, out, size = np.zeros(tokens, int), np.zeros(q.shape), np.zeros(q.shape)
        lse, reach = np.full(q.shape[:2], -np.inf), 0.0
        named[:ends[0]] += 1
        named[ends[-1]:] += 1
        for b in range(sequences):
            a, e = int(ends[b]), int(ends[b + 1])
            if e > a:
                one = attend_tokens(as_double(q), pool, table[b:b + 1], lengths[b:b + 1], [a, e], 4, 0.125)
                named[a:e] += 1
                out[a:e], lse[a:e], size[a:e] = one["out"][a:e], one["lse"][a:e], one["size"][a:e]
                reach = max(reach, one["reach"])
        assert (named > 0).all() and (named == 1).any()
        got, got_lse = HipAttentionBackend().run_paged_tokens(q, batch, 0.125, ints(cuda_device, offsets), out_dtype=torch.float16)
        ok = torch.from_numpy(named == 1)
        part = dict(out=out[named == 1], lse=lse[named == 1], size=size[named == 1], reach=reach)
        check(got.cpu()[ok], got_lse.cpu()[ok], part, 64, 120, torch.float16, False)
        assert not torch.isnan(got).any() and not torch.isnan(got_lse).any()
