"""The paged cache's operators at the edges of what a call may hold: thousands of sequences, shared pages, pools past
4 GiB, queries of any alignment and stride, two host threads, and codes bit for bit over millions of values."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, Rotary, append_tokens, evict_tokens
from kvssd.backends import PagedBatch
from kvssd.backends.hip import HipAttentionBackend
from paged_oracle import as_double, attend, evict, make_pool, make_table
from test_gpu_paged import check_attention, paged

pytestmark = pytest.mark.gpu


MANY = [
    # lengths, bits, query heads, kv heads, head_dim, page_tokens
    ([0] * 99 + [20000], 4, 4, 1, 32, 64),  # one long sequence behind a wave of empty ones
    ([20000] + [1] * 200, 2, 2, 2, 64, 32),
    ([(37 * i) % 301 for i in range(130)], 4, 8, 2, 64, 16),
    ([i % 3 for i in range(1500)], 4, 2, 1, 32, 8),
    ([5] * 64, 2, 16, 8, 128, 64),
    ([64 * i for i in range(65)], 4, 4, 4, 32, 64),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: f"{len(c[0])}-{max(c[0])}-int{c[1]}")
def test_attention_over_many_sequences(cuda_device, case):
    lengths, bits, qh, kvh, d, bt = case
    rng = np.random.default_rng(len(lengths))
    width = max(-(-n // bt) for n in lengths) + 1
    pages = sum(-(-n // bt) for n in lengths) + 1
    pool = make_pool(rng, pages, bt, kvh, d, 32, bits)
    table = make_table(rng, lengths, bt, width, pages)
    batch = paged(cuda_device, pool, table, lengths, bits, 32)
    q = torch.from_numpy(rng.standard_normal((len(lengths), qh, d))).half().to(cuda_device)
    want = attend(as_double(q), pool, table, lengths, bits, 0.125)
    backend = HipAttentionBackend()
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), dict(max_length=64, total_tokens=1)):
        for out_dtype in (torch.float16, torch.float32):
            out, lse = backend.run_paged(q, batch, 0.125, out_dtype=out_dtype, **hints)
            check_attention(out, lse, want, d, max(lengths), out_dtype, out_dtype == torch.float32)


def test_seventy_thousand_sequences(cuda_device):
    """More than a grid's second dimension holds, for the summed weights and for eviction's moves."""
    n, bt, width = 70_000, 16, 40
    rng = np.random.default_rng(54)
    pool = make_pool(rng, 43, bt, 1, 32, 32, 2)
    table = rng.integers(0, 3, (n, width)).astype(np.int32)  # (attention may share pages)
    table[-1] = 3 + np.arange(width)
    lengths = [i % 4 for i in range(n - 1)] + [width * bt]
    slots = (n, width * bt)
    pos = np.tile(np.arange(slots[1], dtype=np.int32), (n, 1))
    batch = paged(cuda_device, pool, table, lengths, 2, 32, np.zeros(slots, np.float32), pos)
    q = torch.from_numpy(rng.standard_normal((n, 1, 32))).half().to(cuda_device)
    out, lse = HipAttentionBackend().run_paged(q, batch, 0.125, accumulate=True)
    some = [0, 1, 2, 3, 65533, 65534, 65535, 65536, 65537, 65538, 65539, n - 2, n - 1]
    want = attend(as_double(q[some]), pool, table[some], [lengths[i] for i in some], 2, 0.125, np.zeros((len(some), slots[1])))
    check_attention(out[some], lse[some], want, 32, width * bt, torch.float32, True)
    got = as_double(batch.weights[some])
    assert np.abs(got - want["weights"]).max() < 2.0 ** -18  # (scores below 16: each off by less than 2^-19)
    sums = batch.weights.double().sum(1).cpu().numpy()
    assert np.abs(sums - (np.array(lengths) > 0)).max() < 2.0 ** -14
    # a budget whose moves take a launch of their own; all but the last sequence are shorter
    w = batch.weights.clone()
    new_lengths, new_w, new_p = evict_tokens(batch, 300, recent=10)
    assert torch.equal(new_lengths, batch.lengths.clamp(max=300))
    source = evict(w[-1].cpu().numpy(), pos[-1], width * bt, 300, 0, 10)
    assert new_p[-1, :300].tolist() == source and torch.equal(new_w[-1, :300], w[-1][source])
    assert torch.equal(new_w[:-1, :4], w[:-1, :4])
    old = torch.from_numpy(pool[0][3:].reshape(-1, 8))
    assert torch.equal(batch.packed_k[3:].cpu().view(-1, 8)[:300], old[source])
    assert torch.equal(batch.packed_k[:3].cpu(), torch.from_numpy(pool[0][:3]))


def test_queries_of_any_alignment_and_stride(cuda_device):
    rng = np.random.default_rng(50)
    lengths = [100, 33]
    pool = make_pool(rng, 12, 16, 2, 64, 32, 4)
    table = make_table(rng, lengths, 16, 7, 12)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    backend = HipAttentionBackend()
    flat = torch.from_numpy(rng.standard_normal(2 * 8 * 64 + 8)).half().to(cuda_device)
    for shift in (1, 3, 4):  # 2, 6 and 8 bytes past a 16-byte border
        q = flat[shift:shift + 2 * 8 * 64].view(2, 8, 64)
        run = backend.prepare_paged(q, batch, 0.1)
        for a, b in zip(run(q), backend.run_paged(q.clone(), batch, 0.1)):
            assert torch.equal(a, b)
    strided = flat[:2 * 8 * 64].view(8, 2, 64).transpose(0, 1)
    broadcast = flat[:64].view(1, 1, 64).expand(2, 8, 64)
    for q in (strided, broadcast):
        for a, b in zip(backend.run_paged(q, batch, 0.1), backend.run_paged(q.contiguous(), batch, 0.1)):
            assert torch.equal(a, b)


def test_sequences_may_share_pages(cuda_device):
    rng = np.random.default_rng(51)
    pool = make_pool(rng, 12, 32, 2, 64, 32, 4)
    table = np.array([[3, 5, 7, -1], [3, 5, 8, 9], [3, 3, 3, 3]])
    lengths = [70, 128, 100]
    batch = paged(cuda_device, pool, table, lengths, 4, 32, np.zeros((3, 128), np.float32))
    q = torch.from_numpy(rng.standard_normal((3, 4, 64))).half().to(cuda_device)
    want = attend(as_double(q), pool, table, lengths, 4, 0.125)
    out, lse = HipAttentionBackend().run_paged(q, batch, 0.125, accumulate=True)
    check_attention(out, lse, want, 64, 128, torch.float32, True)
    # a slot's weights are the sequence's own, shared page or not
    sums = batch.weights.double().sum(1).cpu().numpy()
    assert np.abs(sums - 4).max() < 4 * 2.0 ** -12 and (batch.weights[0, 70:] == 0).all()


def test_two_threads_on_one_prepared_decode(cuda_device):
    rng = np.random.default_rng(52)
    lengths = [3000, 100]
    pool = make_pool(rng, 50, 64, 2, 128, 32, 4)
    table = make_table(rng, lengths, 64, 48, 50)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    queries = torch.from_numpy(rng.standard_normal((2, 2, 8, 128))).half().to(cuda_device)
    run = HipAttentionBackend().prepare_paged(queries[0], batch, 0.1)
    want = [run(q) for q in queries]
    got: list[list] = [[], []]

    def work(i):
        torch.cuda.set_device(cuda_device)
        stream = torch.cuda.Stream(cuda_device)
        stream.wait_stream(torch.cuda.default_stream(cuda_device))
        with torch.cuda.stream(stream):
            for _ in range(100):
                got[i].append(run(queries[i]))
        stream.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for i in range(2):
        assert len(got[i]) == 100
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


@pytest.mark.parametrize(("dtype", "bits", "layout", "kvh", "d", "counts"), [
    (torch.bfloat16, 4, "half", 8, 128, [5000, 1, 3999]),      # eight tokens a workgroup
    (torch.float16, 4, "interleaved", 8, 128, [9000]),
    (torch.bfloat16, 2, "half", 3, 96, [4100, 0, 4101]),
    (torch.float16, 2, "half", 16, 128, [2100, 200]),           # two, more words than threads
    (torch.float32, 4, "half", 1, 32, [8192 + 5]),
    (torch.float32, 2, "interleaved", 4, 64, [3000, 3000]),
    (torch.bfloat16, 4, "half", 5, 256, [6000]),
])
def test_appended_codes_are_the_rotated_keys_over_millions_of_values(cuda_device, dtype, bits, layout, kvh, d, counts):
    """A value rounded once to 16 bits, rather than to 32 and then to 16, differs in 2^-17 of the cases: too few for a
    small test."""
    total, bt = sum(counts), 128
    width = max(-(-n // bt) for n in counts)
    gen = torch.Generator(cuda_device).manual_seed(7)
    shape = (len(counts) * width, bt, kvh)
    rotary = Rotary(d, layout=layout, device=cuda_device)
    k, v = (torch.randn((total, kvh, d), generator=gen, device=cuda_device).to(dtype) for _ in range(2))
    q = torch.randn((total, 2, d), generator=gen, device=cuda_device).to(dtype)
    offsets = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device=cuda_device)
    first = torch.arange(len(counts), dtype=torch.int32, device=cuda_device) * 1000
    batches = []
    for _ in range(2):
        codes = [torch.zeros((*shape, d * bits // 8), dtype=torch.uint8, device=cuda_device) for _ in "kv"]
        scales = [torch.zeros((*shape, d // 32), dtype=torch.float16, device=cuda_device) for _ in "kv"]
        table = torch.arange(len(counts) * width, dtype=torch.int32, device=cuda_device).view(len(counts), width)
        batches.append(PagedBatch(*codes, *scales, table, torch.zeros_like(first), bits, 32))
    turned, lengths = append_tokens(batches[0], k, v, offsets=offsets, rotary=rotary, query=q, first_positions=first)
    position = torch.cat([torch.arange(n, device=cuda_device) + 1000 * i for i, n in enumerate(counts)])
    tq, tk = rotary(position, q, k)
    append_tokens(batches[1], tk, v, offsets=offsets)
    assert lengths.tolist() == counts and torch.equal(turned, tq)
    for name in ("packed_k", "packed_v", "scales_k", "scales_v"):
        a, b = (getattr(x, name).view(torch.uint8) for x in batches)
        assert torch.equal(a, b), (name, int((a != b).sum()))
    # the rotation itself: 64 bits, rounded to 32 and then to the type (torch's conversions)
    angle = position.double()[:, None, None] * rotary.frequencies
    c, s, x = torch.cos(angle), torch.sin(angle), k.double()
    a, b = (x[..., : d // 2], x[..., d // 2:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    lo, hi = a * c - b * s, b * c + a * s
    want = torch.cat((lo, hi), -1) if layout == "half" else torch.stack((lo, hi), -1).flatten(-2)
    # sines off by a few 2^-53 and a product fused or not: the 32-bit rounding hides all but a border's two sides
    far = (tk.double() - want).abs() - want.abs() * torch.finfo(dtype).eps / 2 - (a.abs() + b.abs()).amax() * 2.0 ** -24
    assert far.max() <= torch.finfo(dtype).smallest_normal


def test_a_pool_past_4_gib(cuda_device):
    """Pages at both ends of a pool whose code arrays pass 2^32 bytes; the same pages of a small pool beside them."""
    pages, bt, kvh, d = 66000, 128, 8, 128
    if torch.cuda.mem_get_info(cuda_device)[0] < 24 << 30:
        pytest.skip("needs 24 GiB of GPU memory")
    ends = [pages - 1, 0, pages - 2, 65537, pages - 3, 1]
    assert (pages - 3) * bt * kvh * d // 2 > 1 << 32
    big = PagedBatch(
        *(torch.empty((pages, bt, kvh, d // 2), dtype=torch.uint8, device=cuda_device) for _ in "kv"),
        *(torch.empty((pages, bt, kvh, d // 32), dtype=torch.float16, device=cuda_device) for _ in "kv"),
        torch.tensor([ends[:3], ends[3:]], dtype=torch.int32, device=cuda_device),
        torch.zeros(2, dtype=torch.int32, device=cuda_device), 4, 32,
        torch.zeros((2, 3 * bt), device=cuda_device), torch.full((2, 3 * bt), -1, dtype=torch.int32, device=cuda_device),
    )
    small = PagedBatch(
        *(torch.empty((6, *t.shape[1:]), dtype=t.dtype, device=cuda_device)
          for t in (big.packed_k, big.packed_v, big.scales_k, big.scales_v)),
        torch.arange(6, dtype=torch.int32, device=cuda_device).view(2, 3), big.lengths.clone(), 4, 32,
        big.weights.clone(), big.positions.clone(),
    )
    gen = torch.Generator(cuda_device).manual_seed(3)
    counts = [380, 300]
    k, v = (torch.randn((680, kvh, d), generator=gen, device=cuda_device).bfloat16() for _ in range(2))
    q = torch.randn((2, 32, d), generator=gen, device=cuda_device).bfloat16()
    offsets = torch.tensor([0, 380, 680], dtype=torch.int32, device=cuda_device)
    rotary, backend = Rotary(d, device=cuda_device), HipAttentionBackend()
    results = []
    for batch in (big, small):
        _, lengths = append_tokens(batch, k, v, offsets=offsets, rotary=rotary)
        batch.lengths.copy_(lengths)
        first = backend.run_paged(q, batch, 0.1, accumulate=True)
        lengths, weights, positions = evict_tokens(batch, 200, sink=2, recent=50)
        batch.lengths.copy_(lengths)
        second = backend.run_paged(q, batch, 0.1)
        ids = batch.page_table.flatten().long()
        results.append([*first, *second, lengths, weights, positions,
                        *(t[ids] for t in (batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v))])
    assert results[0][4].tolist() == [min(n, 200) for n in counts]
    for i, (a, b) in enumerate(zip(*results)):
        if i < 7:
            assert torch.equal(a, b), i
        else:  # slots past the appended ones hold whatever the memory held
            n = [torch.arange(3 * bt) < c for c in counts]
            used = torch.stack(n).view(6, bt).to(cuda_device)
            assert torch.equal(a[used].view(torch.uint8), b[used].view(torch.uint8)), i


def test_operators_run_on_another_stream(cuda_device):
    rng = np.random.default_rng(53)
    pool = make_pool(rng, 10, 32, 2, 64, 32, 4)
    table = make_table(rng, [160, 160], 32, 5, 10)
    slots = (2, 160)
    pos = np.tile(np.arange(160, dtype=np.int32), (2, 1))
    w = rng.uniform(0, 1, slots).astype(np.float32)
    a, b = (paged(cuda_device, pool, table, [150, 60], 4, 32, w, pos) for _ in "ab")
    k, v, q = (torch.from_numpy(rng.standard_normal((2, h, 64))).half().to(cuda_device) for h in (2, 2, 4))
    rotary = Rotary(64, device=cuda_device)
    results = []
    side = torch.cuda.Stream(cuda_device)
    torch.cuda.synchronize()
    for batch, stream in ((a, torch.cuda.current_stream(cuda_device)), (b, side)):
        with torch.cuda.stream(stream):
            turned, lengths = append_tokens(batch, k, v, rotary=rotary, query=q)
            batch.lengths.copy_(lengths)
            out, lse = HipAttentionBackend().run_paged(turned, batch, 0.125, accumulate=True)
            cut = evict_tokens(batch, 50, recent=8)
            results.append([turned, lengths, out, lse, *cut, batch.packed_k, batch.scales_v, batch.weights])
    torch.cuda.synchronize()
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_a_cache_plans_anew_as_its_lengths_change(cuda_device):
    rng = np.random.default_rng(55)
    make = lambda h, n=2: torch.from_numpy(rng.standard_normal((n, h, 64))).half().to(cuda_device)  # noqa: E731
    cache = PagedKVCache(60, 16, 2, 64, sequences=2, max_pages=30, track_weights=True, device=cuda_device)
    backend = HipAttentionBackend()
    plans = set()

    def attend_and_check(query, **options):
        out, lse = cache.attend(query, **options)
        plans.add(id(cache._plan[5]))
        keep.append(cache._plan)
        want, want_lse = backend.run_paged(query, cache.batch, 64 ** -0.5, out_dtype=options.get("out_dtype"))
        # a plan of other runs sums in another order: 32-bit grade, as elsewhere; 16-bit results by their rounding too
        tol = dict(atol=2e-5, rtol=2e-5) if out.dtype == torch.float32 else dict(atol=2e-3, rtol=2.0 ** -10)
        torch.testing.assert_close(out, want, **tol)
        torch.testing.assert_close(lse, want_lse, atol=2e-5, rtol=2e-5)

    keep: list = []
    query = make(8)
    attend_and_check(query)  # empty
    cache.append(make(2, 40), make(2, 40), [37, 3])
    for _ in range(150):
        cache.append(make(2), make(2))
        attend_and_check(query, accumulate=True)
    assert 3 < len(plans) < 40
    cache.evict(100, sink=2, recent=8)
    assert cache.lengths == [100, 100] and cache.batch.lengths.tolist() == [100, 100]
    attend_and_check(query, accumulate=True)
    sums = cache.batch.weights.double().sum(1)
    attend_and_check(query, accumulate=True)  # into the weights of the cut cache
    assert ((cache.batch.weights.double().sum(1) - sums - 8).abs() < 1e-3).all()
    cache.clear(0)
    attend_and_check(query[:, :2].contiguous())
    attend_and_check(query, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="query must be"):
        cache.attend(query[:1])


def test_inplace_rotation_of_one_tensor_twice_is_refused(cuda_device):
    x = torch.randn((3, 4, 32), device=cuda_device)
    positions = torch.arange(3, device=cuda_device)
    rotary = Rotary(32, device=cuda_device)
    before = x.clone()
    with pytest.raises(ValueError, match="share no element"):
        rotary(positions, x, x, inplace=True)
    with pytest.raises(ValueError, match="share no element"):
        rotary(positions, x, x[:, :1], inplace=True)
    assert torch.equal(x, before)
    both = rotary(positions, x, x)  # (into tensors of their own)
    rotary(positions, x[:, :3], x[:, 3:], inplace=True)  # the slices of one tensor
    assert torch.equal(x, both[0]) and torch.equal(both[0], both[1])


@pytest.mark.parametrize(("bits", "qh", "kvh", "d", "bt", "length"), [
    (4, 9, 9, 64, 64, 60000),    # workgroups of five kv heads, the second with one too few
    (2, 14, 7, 128, 32, 50000),  # seven waves, one workgroup over the heads
    (4, 5, 5, 160, 24, 40000),   # three waves and two, slots' rows found lane by lane
    (4, 24, 3, 128, 128, 90000),  # two head tiles a kv head
])
def test_long_runs_of_heads_that_fill_no_workgroup(cuda_device, bits, qh, kvh, d, bt, length):
    rng = np.random.default_rng(56)
    lengths = [length, 700]
    width = -(-length // bt)
    pages = width + -(-700 // bt)
    pool = make_pool(rng, pages, bt, kvh, d, 32, bits)
    table = make_table(rng, lengths, bt, width, pages)
    batch = paged(cuda_device, pool, table, lengths, bits, 32)
    q = torch.from_numpy(rng.standard_normal((2, qh, d))).bfloat16().to(cuda_device)
    want = attend(as_double(q), pool, table, lengths, bits, d ** -0.5)
    backend = HipAttentionBackend()
    for out_dtype in (torch.bfloat16, torch.float32):
        out, lse = backend.run_paged(q, batch, d ** -0.5, out_dtype=out_dtype)
        check_attention(out, lse, want, d, length, out_dtype, out_dtype == torch.float32)
        for a, b in zip((out, lse), backend.run_paged(q, batch, d ** -0.5, out_dtype=out_dtype)):
            assert torch.equal(a, b)


@pytest.mark.parametrize(("bits", "kvh", "d", "g", "bt", "pages"), [
    (4, 1, 32, 32, 1, 1),    # one row, one scale
    (4, 1, 64, 64, 7, 9),
    (2, 3, 32, 32, 5, 11),
    (4, 1, 96, 32, 1, 1),    # three groups
    (4, 3, 96, 32, 7, 9),
    (2, 1, 96, 32, 3, 25),
    (4, 3, 160, 32, 5, 13),  # five
    (2, 5, 224, 32, 9, 9),   # seven
])
def test_scales_that_end_an_odd_pool(cuda_device, bits, kvh, d, g, bt, pages):
    """A pool with an odd number of scales, its last row in use: the last scale fills half a word, and what lies behind
    the array (NaN here) has no part."""
    rng = np.random.default_rng(57)
    pool = list(make_pool(rng, pages, bt, kvh, d, g, bits))
    for table, length in ((np.arange(pages)[None], pages * bt), (np.full((1, 1), pages - 1), bt)):  # all; the last page
        lengths = [length]
        batch = paged(cuda_device, pool, table, lengths, bits, g)
        tails = []
        for a in pool[2:]:
            flat = torch.full((a.size + 8,), float("nan"), dtype=torch.float16, device=cuda_device)
            flat[:a.size] = torch.from_numpy(a).flatten().to(cuda_device)
            tails.append(flat[:a.size].view(a.shape))
        batch = PagedBatch(batch.packed_k, batch.packed_v, *tails, batch.page_table, batch.lengths, bits, g)
        q = torch.from_numpy(rng.standard_normal((1, 2 * kvh, d))).half().to(cuda_device)
        want = attend(as_double(q), pool, table, lengths, bits, d ** -0.5)
        for out_dtype in (torch.float16, torch.float32):
            out, lse = HipAttentionBackend().run_paged(q, batch, d ** -0.5, out_dtype=out_dtype)
            check_attention(out, lse, want, d, length, out_dtype, out_dtype == torch.float32)


def test_decodes_prepared_before_a_cut_follow_the_cache(cuda_device):
    """A prepared decode and a captured one go on after an eviction as a call made anew does, and add to the weights
    that the next cut reads."""
    rng = np.random.default_rng(58)
    make = lambda n, h: torch.from_numpy(rng.standard_normal((n, h, 64))).half().to(cuda_device)  # noqa: E731
    cache = PagedKVCache(24, 16, 2, 64, sequences=2, max_pages=12, track_weights=True, device=cuda_device)
    backend, query = HipAttentionBackend(), make(2, 8)
    run = backend.prepare_paged(query, cache.batch, 0.125, accumulate=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(query)
    cache.append(make(250, 2), make(250, 2), [150, 100])
    for r in range(3):
        cache.attend(query, 0.125, accumulate=True)
        cache.evict(80 - 20 * r, sink=2, recent=8)
        assert cache.batch.lengths.tolist() == cache.lengths == [80 - 20 * r] * 2
        want = backend.run_paged(query, cache.batch, 0.125)
        sums = cache.batch.weights.double().sum(1)
        for n in (1, 2):
            if n == 1:
                got = run(query)
            else:
                graph.replay()
                got = captured
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            # 8 heads' weights a call: each a sum of at most 80 numbers within 2^-17 of themselves
            assert ((cache.batch.weights.double().sum(1) - sums - 8 * n).abs() < 16 * 2.0 ** -15).all()
        cache.append(make(2, 2), make(2, 2))
    del graph


def test_tangents_are_refused_by_every_operator(cuda_device):
    from torch.autograd import forward_ad

    rng = np.random.default_rng(59)
    pool = make_pool(rng, 4, 16, 2, 64, 32, 4)
    batch = paged(cuda_device, pool, np.arange(4).reshape(2, 2), [20, 3], 4, 32)
    k, q = (torch.from_numpy(rng.standard_normal((2, h, 64))).half().to(cuda_device) for h in (2, 4))
    rotary, backend = Rotary(64, device=cuda_device), HipAttentionBackend()
    run = backend.prepare_paged(q, batch, 0.125)
    positions = torch.arange(2, device=cuda_device)
    before = batch.packed_k.clone()
    with forward_ad.dual_level():
        dk, dq = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (k, q))
        for call in (
            lambda: rotary(positions, dq), lambda: rotary(positions, q, dk), lambda: append_tokens(batch, dk, k),
            lambda: append_tokens(batch, k, dk), lambda: append_tokens(batch, k, k, rotary=rotary, query=dq),
            lambda: run(dq), lambda: backend.run_paged(dq, batch, 0.125),
        ):
            with pytest.raises(ValueError, match="no forward derivative"):
                call()
        run(q)
    assert torch.equal(batch.packed_k, before)


@pytest.mark.parametrize(("lengths", "bits", "qh", "kvh", "d", "g", "bt", "dtype"), [
    ([3000, 0, 64, 777], 4, 32, 8, 128, 32, 64, torch.bfloat16),
    ([500, 1, 130], 2, 12, 2, 96, 32, 24, torch.float16),          # three groups, slots' rows found lane by lane
    ([200, 65], 4, 6, 3, 256, 256, 40, torch.float32),
    ([300, 40], 2, 2, 2, 64, 64, 32, torch.float32),
    ([(37 * i) % 301 for i in range(130)], 4, 8, 2, 64, 32, 16, torch.float16),
    ([5] * 70 + [20000], 4, 4, 1, 32, 32, 64, torch.bfloat16),
])
def test_weights_of_lengths_past_the_hints(cuda_device, lengths, bits, qh, kvh, d, g, bt, dtype):
    """Scores have as many places as the hints make out; a slot past them gets the same weight, from its key."""
    rng = np.random.default_rng(60)
    width = max(-(-n // bt) for n in lengths) + 1
    pages = sum(-(-n // bt) for n in lengths) + 1
    pool = make_pool(rng, pages, bt, kvh, d, g, bits)
    table = make_table(rng, lengths, bt, width, pages)
    table[0, 1] = -1  # slots without a page
    start = rng.uniform(0, 3, (len(lengths), width * bt)).astype(np.float32)
    q = torch.from_numpy(rng.standard_normal((len(lengths), qh, d))).to(dtype).to(cuda_device)
    scale = d ** -0.5
    want = attend(as_double(q), pool, table, lengths, bits, scale, start)
    u = 2.0 ** -24
    e = 2 * (d + 16) * u * want["reach"] + (np.abs(want["lse"][np.isfinite(want["lse"])]).max() + 60) * 8 * u
    added = want["weights"] - start
    tol = added * (e + qh * u) * 2 + np.abs(want["weights"]) * u * 2
    backend = HipAttentionBackend()
    half = dict(max_length=max(lengths), total_tokens=sum(lengths) // 2)
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), half, dict(max_length=1, total_tokens=1),
                  dict(max_length=70), dict(total_tokens=1)):
        batch = paged(cuda_device, pool, table, lengths, bits, g, start)
        run = backend.prepare_paged(q, batch, scale, accumulate=True, **hints)
        out, lse = run(q)
        check_attention(out, lse, want, d, max(lengths), torch.float32, True)
        got = as_double(batch.weights)
        assert (np.abs(got - want["weights"]) <= tol).all(), hints
        untouched = added == 0
        assert (got[untouched] == start.astype(np.float64)[untouched]).all(), hints


def test_a_cache_of_an_unnumbered_device(cuda_device):
    cache = PagedKVCache(4, 16, 1, 32, sequences=2, device="cuda")
    assert cache.device == cache.batch.packed_k.device == cuda_device
    x = torch.ones((5, 1, 32), device=cuda_device)
    cache.append(x, x, [3, 2])
    out, _ = cache.attend(torch.ones((2, 2, 32), device=cuda_device))
    # a one is held as code 7 times the scale 1/7, which its rounding to fp16 puts off by at most 2^-11 of itself; the
    # mean of equal values is that value to 32-bit grade
    assert ((out - 1).abs() <= 2.0 ** -11 + 2.0 ** -16).all() and cache.batch.lengths.tolist() == [3, 2]


def test_tokens_of_no_sequence_are_dropped(cuda_device):
    """A padded batch: offsets that begin behind the first token and end before the last."""
    from kvssd import RotaryScaling

    rng = np.random.default_rng(61)
    pool = make_pool(rng, 8, 16, 2, 64, 32, 4)
    table = np.arange(8).reshape(2, 4)
    slots = np.zeros((2, 64))
    a, b = (paged(cuda_device, pool, table, [3, 14], 4, 32, slots.astype(np.float32) + 7, slots.astype(np.int32) - 1)
            for _ in "ab")
    k, v, q = (torch.from_numpy(rng.standard_normal((40, h, 64))).half().to(cuda_device) for h in (2, 2, 4))
    rotary = Rotary(64, scaling=RotaryScaling("yarn", 4.0), device=cuda_device)
    offsets = torch.tensor([5, 20, 31], dtype=torch.int32, device=cuda_device)
    turned, lengths = append_tokens(a, k, v, offsets=offsets, rotary=rotary, query=q)
    want, want_lengths = append_tokens(b, k[5:31], v[5:31], offsets=offsets - 5, rotary=rotary, query=q[5:31])
    assert lengths.tolist() == want_lengths.tolist() == [18, 25] and torch.equal(turned[5:31], want)
    for name in ("packed_k", "packed_v", "scales_k", "scales_v", "weights", "positions"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    at_0 = rotary(torch.zeros(40, dtype=torch.int64, device=cuda_device), q)
    assert torch.equal(turned[:5], at_0[:5]) and torch.equal(turned[31:], at_0[31:])


@pytest.mark.parametrize(("lengths", "budget", "bt", "width"), [
    ([300, 150, 20], 100, 24, 20), ([5000, 120], 4000, 64, 80), ([9000, 4100], 3000, 64, 200),
], ids=["one", "rows moved apart", "chunks"])
def test_attention_after_a_cut_is_over_the_kept_tokens(cuda_device, lengths, budget, bt, width):
    rng = np.random.default_rng(62)
    pages = sum(-(-n // bt) for n in lengths) + 1
    pool = make_pool(rng, pages, bt, 2, 64, 32, 4)
    table = make_table(rng, lengths, bt, width, pages)
    slots = (len(lengths), width * bt)
    w = np.exp(2 * rng.standard_normal(slots)).astype(np.float32)
    pos = np.tile(np.arange(slots[1], dtype=np.int32), (len(lengths), 1))
    batch = paged(cuda_device, pool, table, lengths, 4, 32, w, pos)
    new_lengths, new_w, new_p = evict_tokens(batch, budget, sink=2, recent=50)
    batch.lengths.copy_(new_lengths)
    q = torch.from_numpy(rng.standard_normal((len(lengths), 4, 64))).half().to(cuda_device)
    out, lse = HipAttentionBackend().run_paged(q, batch, 0.125)
    # the kept slots' rows of the pool as it was, a page a token
    kept = [evict(w[b], pos[b], n, budget, 2, 50) for b, n in enumerate(lengths)]
    rows = np.full((len(lengths), max(map(len, kept))), -1)
    for b, source in enumerate(kept):
        rows[b, :len(source)] = [table[b, s // bt] * bt + s % bt for s in source]
        assert new_p[b, :len(source)].tolist() == source and new_w[b, :len(source)].tolist() == w[b, source].tolist()
    loose = [a.reshape(pages * bt, 1, *a.shape[2:]) for a in pool]
    want = attend(as_double(q), loose, rows, [len(s) for s in kept], 4, 0.125)
    check_attention(out, lse, want, 64, max(map(len, kept)), torch.float32, True)


@pytest.mark.parametrize(("bits", "d", "g"), [(4, 128, 32), (4, 128, 128), (4, 64, 32), (4, 256, 32), (2, 128, 32),
                                              (2, 128, 64), (2, 256, 256), (2, 96, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scores_are_sums_of_what_the_codes_stand_for(cuda_device, bits, d, g, dtype):
    """Keys of zeros but for one dim: the score is one product.  Were the codes' offset part of the sum, its rounding
    would show: the query's values add up to a thousand times that product's last places."""
    rng = np.random.default_rng(63)
    mid, lengths = 1 << (bits - 1), [1, 40, 200]
    pool = make_pool(rng, 12, 32, 2, d, g, bits)
    codes = np.full((12, 32, 2, d), mid, np.uint8)
    one = rng.integers(0, d, (12, 32, 2, 1))
    np.put_along_axis(codes, one, mid + rng.choice([-1, 1], one.shape).astype(np.uint8), -1)
    pool[0][...] = sum(codes[..., i::8 // bits] << (bits * i) for i in range(8 // bits))
    pool[2][...] = 1.0
    table = make_table(rng, lengths, 32, 7, 12)
    batch = paged(cuda_device, pool, table, lengths, bits, g)
    q = torch.from_numpy(rng.uniform(500, 2000, (3, 8, d))).to(dtype).to(cuda_device)
    scale = 2.0 ** -8
    want = attend(as_double(q), pool, table, lengths, bits, scale)
    for out_dtype in (dtype, torch.float32):
        _, lse = HipAttentionBackend().run_paged(q, batch, scale, out_dtype=out_dtype)
        # scores exact but for their factor's two roundings; lse's own terms as elsewhere
        err = np.abs(as_double(lse) - want["lse"])
        assert (err <= (np.abs(want["lse"]) + 40) * 4 * 2.0 ** -24).all(), float(err.max())
