"""The paged packed cache on the GPU: append, attention, eviction, and a run of them together, against 64-bit oracles.

Tolerances of attention.  Let A = sum_t p_t |v_t| (per output value), u = 2^-24.
* A score is a 32-bit sum of head_dim products plus an offset's share, whose terms add up to at most ``reach``
  (returned by the oracle; per scale group the sum of |q| times twice the largest number a code enters as), then a
  product per group and their sum: off by at most E = (head_dim + 16) u reach.  Softmax weights are then off by at most
  a factor e^(2E) ~ 1 + 2E + ..., lse by E, and 2^x and the logarithm add a few u.
* With 16-bit results each weight times its value scale is rounded to fp16 (2^-11 of it; below fp16's normal range,
  2^-24 times less than the tile's largest, an absolute 2^-25 of what the largest is scaled to, 2^8 or more: nothing
  beside it); with 32-bit ones it is a sum of two fp16 parts (2^-22).
* Sums over n slots in 32 bits: at most n u A.
* The result's rounding: eps/2 of the value.
"""

from __future__ import annotations

import dataclasses
import math

import numpy as np
import pytest
import torch

from kvssd import PagedKVCache, Rotary, append_tokens, evict_tokens
from kvssd.backends import PackedBatch, PagedBatch
from kvssd.backends.hip import HipAttentionBackend
from kvssd.backends.reference import ReferenceAttentionBackend
from kvssd.records_hip import quantize
from paged_oracle import as_double, attend, evict, frequencies, make_pool, make_table, rotate

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def paged(dev, pool, table, lengths, bits, g, weights=None, positions=None) -> PagedBatch:
    t = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return PagedBatch(*(t(a) for a in pool), t(table.astype(np.int32)), t(np.asarray(lengths, np.int32)), bits, g,
                      t(weights), t(positions))


def check_attention(out, lse, want, d, longest, dtype, precise):
    e = (d + 16) * U * want["reach"] + 8 * U
    weight = 2 * e + (2.0 ** -22 if precise else 2.0 ** -11) + (longest + 8) * U
    tol = want["size"] * weight * (1 + weight) + np.abs(want["out"]) * torch.finfo(dtype).eps / 2
    tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    err = np.abs(as_double(out) - want["out"])
    assert (err <= tol).all(), f"out: largest error over its bound {np.nanmax(err / np.maximum(tol, 1e-300))}"
    got = as_double(lse)
    empty = np.isinf(want["lse"])
    assert (got[empty] == -np.inf).all()
    lerr = np.abs(got[~empty] - want["lse"][~empty])
    ltol = e + (np.abs(want["lse"][~empty]) + 40) * 4 * U  # (its terms: a maximum and up to 2^40 in the sum)
    assert (lerr <= ltol).all(), f"lse: {(lerr / ltol).max()}"
    if precise and err.size and np.linalg.norm(want["out"]):
        assert np.linalg.norm(err) <= 1e-5 * np.linalg.norm(want["out"])  # 32-bit grade overall


# bits, query heads, kv heads, head_dim, group, page_tokens, lengths, query dtype
SHAPES = [
    (4, 1, 1, 32, 32, 16, [1], torch.float16),
    (4, 32, 8, 128, 32, 64, [1, 0, 31, 32, 33, 64, 65, 1000], torch.bfloat16),
    (4, 32, 8, 128, 32, 128, [4096], torch.float16),
    (2, 32, 8, 128, 32, 32, [777, 2050, 1], torch.bfloat16),
    (4, 8, 8, 128, 128, 96, [500, 96, 97], torch.float16),
    (4, 24, 8, 128, 64, 24, [23, 24, 25, 300], torch.bfloat16),   # pages that end inside a tile
    (2, 64, 4, 128, 32, 1, [40, 3], torch.float16),               # a page a token
    (4, 10, 2, 96, 32, 16, [333, 8], torch.bfloat16),             # three groups in four columns
    (2, 6, 3, 96, 32, 40, [121, 90], torch.float32),
    (4, 16, 1, 64, 32, 64, [700, 5], torch.float16),
    (4, 40, 1, 64, 64, 7, [129, 64], torch.bfloat16),             # several head tiles and sets
    (2, 4, 2, 64, 32, 128, [1000], torch.float32),
    (4, 12, 12, 64, 32, 32, [65, 64, 63], torch.float16),         # two workgroups over the kv heads
    (4, 18, 9, 256, 32, 64, [100, 260], torch.bfloat16),          # eight groups, an idle wave
    (2, 32, 2, 256, 64, 48, [513], torch.float16),
    (4, 4, 1, 256, 256, 64, [2000, 1], torch.float32),
    (4, 10, 5, 160, 32, 32, [200, 31], torch.bfloat16),           # five groups, half a granule idle
    (2, 2, 1, 224, 32, 56, [111], torch.float16),
    (4, 2, 2, 192, 64, 64, [70], torch.bfloat16),
    (4, 128, 1, 128, 32, 64, [300], torch.bfloat16),              # one kv head, 128 query heads
    (2, 16, 16, 32, 32, 20, [41, 60, 19], torch.bfloat16),
]


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:6])) + f"-{len(s[6])}")
def test_attention_matches_the_oracle(cuda_device, shape, out32):
    bits, qh, kvh, d, g, bt, lengths, dtype = shape
    rng = np.random.default_rng(sum(shape[:6]))
    width = max(-(-n // bt) for n in lengths) + 1
    pages = sum(-(-n // bt) for n in lengths) + 2
    pool = make_pool(rng, pages, bt, kvh, d, g, bits)
    table = make_table(rng, lengths, bt, width, pages)
    weights = rng.uniform(0, 3, (len(lengths), width * bt)).astype(np.float32)
    batch = paged(cuda_device, pool, table, lengths, bits, g, weights)
    q = torch.from_numpy(rng.standard_normal((len(lengths), qh, d))).to(dtype).to(cuda_device)
    scale = 1 / math.sqrt(d)
    want = attend(as_double(q), pool, table, lengths, bits, scale, weights)
    out_dtype = torch.float32 if out32 else dtype
    precise = out_dtype == torch.float32 or dtype == torch.float32
    backend = HipAttentionBackend()
    for hints in ({}, dict(max_length=max(lengths), total_tokens=sum(lengths)), dict(max_length=1, total_tokens=1)):
        out, lse = backend.run_paged(q, batch, scale, out_dtype=out_dtype, **hints)
        assert out.dtype == out_dtype
        check_attention(out, lse, want, d, max(lengths), out_dtype, precise)
    # summed weights: p is off as lse and the score are, and rounds a few times per head
    run = backend.prepare_paged(q, batch, scale, out_dtype=out_dtype, accumulate=True)
    again, _ = run(q)
    e = 2 * (d + 16) * U * want["reach"] + (np.abs(want["lse"][np.isfinite(want["lse"])]).max() + 60) * 8 * U
    got = as_double(batch.weights)
    added = want["weights"] - weights
    assert (np.abs(got - want["weights"]) <= added * (e + qh * U) * 2 + np.abs(want["weights"]) * U * 2).all()
    plain, _ = backend.run_paged(q, batch, scale, out_dtype=out_dtype)
    assert torch.equal(again, plain)


def test_the_portable_backend_computes_the_same(cuda_device):
    rng = np.random.default_rng(5)
    lengths = [70, 0, 33]
    pool = make_pool(rng, 12, 16, 2, 64, 32, 4)
    table = make_table(rng, lengths, 16, 6, 12)
    weights = np.zeros((3, 96), np.float32)
    a, b = (paged(cuda_device, pool, table, lengths, 4, 32, weights) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((3, 8, 64))).half().to(cuda_device)
    out, lse = HipAttentionBackend().run_paged(q, a, 0.125, accumulate=True)
    ref, ref_lse = ReferenceAttentionBackend().run_paged(q, b, 0.125, accumulate=True)
    # both 32-bit grade: 2e-5 is the tolerance of the packed decodes' 32-bit kernels
    torch.testing.assert_close(out, ref, atol=2e-5, rtol=2e-5)
    torch.testing.assert_close(lse, ref_lse, atol=2e-5, rtol=2e-5)
    torch.testing.assert_close(a.weights, b.weights, atol=2e-5, rtol=2e-5)


def test_garbage_outside_the_sequences_has_no_part(cuda_device):
    # unused slots of used pages, unused pages and table entries behind the last page: infinities and NaN as scales,
    # ids far outside the pool; and one sequence's entry in the middle that names no page: its slots are skipped
    rng = np.random.default_rng(6)
    lengths = [45, 130, 64]
    for bt in (32, 20):
        width = 8
        pages = 24
        pool = make_pool(rng, pages, bt, 2, 64, 32, 4)
        table = make_table(rng, lengths, bt, width, pages)
        used = np.zeros((pages, bt), bool)
        for b, n in enumerate(lengths):
            for s in range(n):
                used[table[b, s // bt], s % bt] = True
        for t, bad in ((pool[2], np.nan), (pool[3], np.inf)):
            t[~used] = bad
        table[table < 0] = 1 << 30
        table[1, 1] = -5
        batch = paged(cuda_device, pool, table, lengths, 4, 32, np.zeros((3, width * bt), np.float32))
        q = torch.from_numpy(rng.standard_normal((3, 4, 64))).half().to(cuda_device)
        want = attend(as_double(q), pool, table, lengths, 4, 0.125, as_double(batch.weights))
        out, lse = HipAttentionBackend().run_paged(q, batch, 0.125, accumulate=True)
        check_attention(out, lse, want, 64, 130, torch.float32, True)
        got = as_double(batch.weights)
        assert np.isfinite(got).all() and (got[want["weights"] == 0] == 0).all()
        np.testing.assert_allclose(got, want["weights"], rtol=1e-4, atol=1e-30)


def test_lengths_outside_the_table_are_clamped(cuda_device):
    rng = np.random.default_rng(7)
    pool = make_pool(rng, 8, 32, 2, 64, 32, 4)
    table = np.arange(8, dtype=np.int32).reshape(2, 4)
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).half().to(cuda_device)
    got = HipAttentionBackend().run_paged(q, paged(cuda_device, pool, table, [-7, 1 << 30], 4, 32), 0.125)
    want = HipAttentionBackend().run_paged(q, paged(cuda_device, pool, table, [0, 128], 4, 32), 0.125)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize(("k_scale", "v_scale", "q_scale"), [
    ((1e-6, 6e-5), (1e-6, 6e-5), 3e4), ((100.0, 9000.0), (100.0, 60000.0), 1e-4), ((0.2, 0.5), (6e-8, 6e4), 1.0),
    ((0.2, 0.5), (0.0, 0.0), 1e-20),
], ids=["tiny", "huge", "mixed", "zero"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_scales_over_the_whole_range(cuda_device, k_scale, v_scale, q_scale, dtype):
    rng = np.random.default_rng(12)
    lengths = [300]
    pool = make_pool(rng, 10, 32, 2, 64, 32, 4)
    for t, (lo, hi) in ((pool[2], k_scale), (pool[3], v_scale)):
        t[...] = np.exp(rng.uniform(math.log(max(lo, 1e-30)), math.log(max(hi, 1e-30)), t.shape)).astype(np.float16)
    # small scales first, so that the reference exponent has to grow on the way
    order = np.sort(pool[3].reshape(-1))
    table = np.arange(10, dtype=np.int32).reshape(1, 10)
    pool[3].reshape(-1)[:] = order
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    q = torch.from_numpy(q_scale * rng.standard_normal((1, 8, 64))).to(dtype).to(cuda_device)
    scale = 0.125
    with np.errstate(invalid="ignore"):  # (fp16 holds some of the largest queries as infinities)
        want = attend(as_double(q), pool, table, lengths, 4, scale)
    out, lse = HipAttentionBackend().run_paged(q, batch, scale)
    rows = torch.isfinite(q).all(-1).cpu().numpy()
    assert (rows.any() or dtype == torch.float16) and not np.isfinite(as_double(out)[~rows]).any() and not np.isfinite(as_double(lse)[~rows]).any()
    out, lse = out[torch.from_numpy(rows)], lse[torch.from_numpy(rows)]
    want = {k: v if k == "reach" or v is None else v[rows] for k, v in want.items()}
    e = (64 + 16) * U * want["reach"] + 8 * U
    weight = 2 * e + 2.0 ** -22 + 308 * U
    # weights whose value scale is 2^24 below the largest met are held with an absolute error: 2^-33 of that one's size
    tol = want["size"] * weight * (1 + weight) + np.abs(want["out"]) * U + np.abs(want["size"]).max(initial=0) * 2.0 ** -22
    assert (np.abs(as_double(out) - want["out"]) <= tol + 2.0 ** -149).all()
    assert (np.abs(as_double(lse) - want["lse"]) <= e + (np.abs(want["lse"]) + 40) * 4 * U).all()


def test_scores_that_rise_and_fall_by_thousands(cuda_device):
    # the lazy reference: rising scores move it tile by tile, falling ones never; long runs of equal ones do not
    rng = np.random.default_rng(13)
    lengths = [640, 640, 640]
    pool = make_pool(rng, 60, 32, 1, 32, 32, 4)
    table = np.arange(60, dtype=np.int32).reshape(3, 20)
    pool[0][...] = 0xFF  # every key code 7: the score is 7 scale sum q
    ramp = np.linspace(0.001, 40.0, 640).astype(np.float16)
    for b, r in enumerate((ramp, ramp[::-1], np.full(640, 3.0, np.float16))):
        pool[2][table[b]] = r.reshape(20, 32, 1, 1)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    q = torch.full((3, 2, 32), 0.25, dtype=torch.float16, device=cuda_device)
    q[:, 1] = -0.25
    for hints in (dict(max_length=640, total_tokens=64), {}):
        want = attend(as_double(q), pool, table, lengths, 4, 1.0)
        out, lse = HipAttentionBackend().run_paged(q, batch, 1.0, **hints)
        # the sums here are exact: 32 equal products of a power of two and a whole number; scores round in 32 bits
        s = float(np.abs(want["lse"]).max())
        tol = want["size"] * (8 * s * U + 648 * U + 2.0 ** -22) + np.abs(want["out"]) * U
        assert (np.abs(as_double(out) - want["out"]) <= tol).all()
        assert (np.abs(as_double(lse) - want["lse"]) <= (np.abs(want["lse"]) + 40) * 4 * U).all()


def test_non_finite_inputs_stay_in_their_rows(cuda_device):
    rng = np.random.default_rng(14)
    lengths = [100, 100]
    pool = make_pool(rng, 8, 32, 2, 64, 32, 4)
    table = np.arange(8, dtype=np.int32).reshape(2, 4)
    pool[2][table[1, 0], 3, 1, 0] = np.inf  # a key of sequence 1's second kv head
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    q = rng.standard_normal((2, 8, 64))
    q[0, 1, 5] = np.nan
    q[0, 6, 0] = np.inf
    q = torch.from_numpy(q).half().to(cuda_device)
    out, lse = HipAttentionBackend().run_paged(q, batch, 0.125)
    bad = torch.zeros((2, 8), dtype=torch.bool)
    bad[0, 1] = bad[0, 6] = True
    clean = q.clone()
    clean[0, 1] = clean[0, 6] = 0
    base, base_lse = HipAttentionBackend().run_paged(clean, batch, 0.125)
    assert torch.isnan(out.cpu()[bad]).all() and torch.isnan(lse.cpu()[bad]).all()
    fine = ~bad
    fine[1, 4:] = False  # heads that read the infinite key: a weight of NaN or all of it, as their sign has it
    assert torch.equal(out.cpu()[fine], base.cpu()[fine]) and torch.isfinite(out.cpu()[fine]).all()
    assert torch.equal(lse.cpu()[fine], base_lse.cpu()[fine])


def test_prepared_decode_follows_its_arrays_and_shares_nothing(cuda_device):
    rng = np.random.default_rng(15)
    lengths = [200, 50]
    pool = make_pool(rng, 20, 32, 2, 64, 32, 4)
    table = make_table(rng, [320, 320], 32, 10, 20)
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    backend = HipAttentionBackend()
    q = torch.from_numpy(rng.standard_normal((2, 8, 64))).half().to(cuda_device)
    run = backend.prepare_paged(q, batch, 0.125, max_length=64, total_tokens=64)
    seen = []
    for n in (0, 1, 64, 65, 320):
        batch.lengths.fill_(n)
        out, lse = run(q)
        seen.append((out, lse))
        want = attend(as_double(q), pool, table, [n, n], 4, 0.125)
        check_attention(out, lse, want, 64, 320, torch.float32, True)
    assert len({t.data_ptr() for pair in seen for t in pair}) == 10
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = run(q)
    out, _ = run(q)
    side.synchronize()
    assert torch.equal(other[0], out) and torch.equal(out, seen[-1][0])
    with pytest.raises(ValueError, match="does not match"):
        run(q.float())
    with pytest.raises(ValueError, match="does not match"):
        run(q[:1])
    with pytest.raises(ValueError, match="no backward pass"):
        run(q.clone().requires_grad_())


def test_decode_graphs_replay_as_eager_calls(cuda_device):
    rng = np.random.default_rng(16)
    lengths = [3000, 50, 700]
    pool = make_pool(rng, 140, 32, 4, 128, 32, 4)
    table = make_table(rng, [3200, 640, 640], 32, 100, 140)
    batch = paged(cuda_device, pool, table, lengths, 4, 32, np.zeros((3, 3200), np.float32))
    mirror = dataclasses.replace(batch, weights=batch.weights.clone())
    backend = HipAttentionBackend()
    q = torch.from_numpy(rng.standard_normal((3, 16, 128))).half().to(cuda_device)
    run = backend.prepare_paged(q, batch, 0.09, accumulate=True)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:  # two graphs of one prepared decode
        with torch.cuda.graph(g):
            outs.append(run(q))
    for r in range(4):
        q.copy_(torch.from_numpy(rng.standard_normal((3, 16, 128))).half())
        batch.lengths.copy_(torch.tensor([3000 + r, 50 * r, 700 - r], dtype=torch.int32))
        for g, (out, lse) in zip(graphs, outs):
            g.replay()
            want, want_lse = backend.run_paged(q, mirror, 0.09, accumulate=True)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(batch.weights, mirror.weights)
    del graphs


# ------------------------------------------------------------------------------------------------------------- append

APPENDS = [
    # bits, query heads, kv heads, head_dim, group, page_tokens, rotary_dim, layout, dtype, counts, filled
    (4, 32, 8, 128, 32, 64, 128, "half", torch.bfloat16, None, [0, 1, 63, 64, 65, 127]),
    (4, 0, 8, 128, 32, 128, 128, "half", torch.bfloat16, [130, 0, 1, 70], [0, 5, 127, 100]),
    (2, 16, 4, 64, 32, 24, 32, "interleaved", torch.float32, [30, 3, 100], [0, 23, 24]),
    (2, 4, 4, 128, 64, 32, 128, "half", torch.float16, None, [10]),
    (4, 3, 1, 96, 32, 7, 24, "half", torch.float16, [50, 13], [6, 7]),
    (2, 2, 2, 96, 32, 1, 20, "interleaved", torch.bfloat16, [5, 9], [0, 2]),
    (4, 6, 3, 256, 256, 16, 64, "half", torch.float32, None, [0, 40]),
    (2, 1, 1, 256, 256, 40, 256, "interleaved", torch.float16, [40], [1]),
    (4, 2, 2, 32, 32, 16, 2, "half", torch.bfloat16, [20, 0, 0], [3, 3, 3]),
    (4, 2, 1, 64, 64, 16, 64, "half", torch.bfloat16, [1500, 700], [0, 10]),  # several tokens a workgroup
]


def append_case(case, dev, seed=0):
    bits, qh, kvh, d, g, bt, r, layout, dtype, counts, filled = case
    rng = np.random.default_rng(seed + bits + d + bt)
    n = [1] * len(filled) if counts is None else counts
    after = [a + b for a, b in zip(filled, n)]
    width = max(-(-a // bt) for a in after) + 1
    pages = sum(-(-a // bt) for a in after) + 2
    pool = make_pool(rng, pages, bt, kvh, d, g, bits)
    table = make_table(rng, after, bt, width, pages)
    slots = (len(filled), width * bt)
    batch = paged(dev, pool, table, filled, bits, g, rng.uniform(1, 2, slots).astype(np.float32),
                  rng.integers(0, 9, slots).astype(np.int32))
    total = sum(n)
    made = [torch.from_numpy(rng.standard_normal((total, h, d))).to(dtype).to(dev) for h in (kvh, kvh, max(qh, 1))]
    offsets = None if counts is None else torch.tensor([0, *np.cumsum(n)], dtype=torch.int32, device=dev)
    return pool, table, batch, made, offsets, n, after


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c[:8])))
@pytest.mark.parametrize("rotated", [True, False])
def test_append_writes_what_rotary_and_quantiser_make(cuda_device, case, rotated):
    bits, qh, kvh, d, g, bt, r, layout, dtype, counts, filled = case
    pool, table, batch, (k, v, q), offsets, n, after = append_case(case, cuda_device)
    rot = Rotary(d, rotary_dim=r, layout=layout, device=cuda_device) if rotated else None
    first = torch.tensor([f + 1000 * i for i, f in enumerate(filled)], dtype=torch.int32, device=cuda_device)
    before = [t.clone() for t in (batch.weights, batch.positions, batch.lengths)]
    query = q if rotated and qh else None
    turned, lengths = append_tokens(batch, k, v, offsets=offsets, rotary=rot, query=query, first_positions=first)
    assert lengths.tolist() == after and torch.equal(batch.lengths, before[2])
    seqs = np.repeat(np.arange(len(n)), n)
    nth = np.concatenate([np.arange(c) for c in n])
    position = first.cpu().numpy()[seqs] + nth
    slot = np.array(filled)[seqs] + nth
    page = table[seqs, slot // bt]
    where = page.astype(np.int64) * bt + slot % bt
    # the keys that the rotary operator makes, by the framework's quantiser, bit for bit
    keys = rot(torch.from_numpy(position).to(cuda_device), k) if rotated else k
    want = [torch.from_numpy(a.copy()) for a in pool]
    for x, packed, scales in ((keys, want[0], want[2]), (v, want[1], want[3])):
        coded = quantize(x.reshape(-1, d), bits, g)
        packed.flatten(0, 1)[where] = coded.packed.cpu().view(len(where), kvh, -1)
        scales.flatten(0, 1)[where] = coded.scales.cpu().view(len(where), kvh, -1)
    for name, w in zip(("packed_k", "packed_v", "scales_k", "scales_v"), want):
        got = getattr(batch, name).cpu()
        assert torch.equal(got.view(torch.uint8), w.view(torch.uint8)), name
    if rotated and qh:
        assert torch.equal(turned, rot(torch.from_numpy(position).to(cuda_device), q))
    else:
        assert turned is None
    before[0][torch.from_numpy(seqs), torch.from_numpy(slot)] = 0.0
    before[1][torch.from_numpy(seqs), torch.from_numpy(slot)] = torch.from_numpy(position.astype(np.int32)).to(cuda_device)
    assert torch.equal(batch.weights, before[0]) and torch.equal(batch.positions, before[1])


def test_appended_codes_match_the_64_bit_codec(cuda_device):
    # from the definitions: rotated in 64 bits, rounded to the type, scale max/7 in 32 bits, codes rounded to even
    case = APPENDS[1]
    bits, qh, kvh, d, g, bt, r, layout, dtype, counts, filled = case
    pool, table, batch, (k, v, _), offsets, n, after = append_case(case, cuda_device, 1)
    rot = Rotary(d, device=cuda_device)
    append_tokens(batch, k, v, offsets=offsets, rotary=rot)
    seqs, nth = np.repeat(np.arange(len(n)), n), np.concatenate([np.arange(c) for c in n])
    slot = np.array(filled)[seqs] + nth
    rows = table[seqs, slot // bt].astype(np.int64) * bt + slot % bt
    keys = torch.from_numpy(rotate(as_double(k), slot, frequencies(d), False)).to(dtype).float().numpy()
    top = np.abs(keys.reshape(-1, kvh, d // g, g)).max(-1)
    scale = (np.maximum(top, np.float32(1e-8)) / np.float32(7)).astype(np.float32)
    code = np.rint((keys.reshape(-1, kvh, d // g, g) / scale[..., None]).astype(np.float32)) + 8
    code = code.reshape(-1, kvh, d).astype(np.uint8)
    got = batch.packed_k.cpu().numpy().reshape(-1, kvh, d // 2)[rows]
    assert (got == (code[..., 0::2] | code[..., 1::2] << 4)).all()
    assert (batch.scales_k.cpu().numpy().reshape(-1, kvh, d // g)[rows] == scale.astype(np.float16)).all()


def test_append_of_strided_slices(cuda_device):
    # keys, values and query as slices of one projection, at 16-byte addresses and 2 bytes past them
    rng = np.random.default_rng(20)
    rot = Rotary(64, device=cuda_device)
    for shift in (0, 1):
        fused = torch.from_numpy(rng.standard_normal((3, 8 * 64 + 8))).half().to(cuda_device)
        q = fused[:, shift: shift + 256].unflatten(1, (4, 64))
        k = fused[:, shift + 256: shift + 384].unflatten(1, (2, 64))
        v = fused[:, shift + 384: shift + 512].unflatten(1, (2, 64))
        made = []
        for tensors in ((k, v, q), tuple(t.contiguous() for t in (k, v, q))):
            pool = make_pool(np.random.default_rng(21), 4, 16, 2, 64, 32, 4)
            batch = paged(cuda_device, pool, np.array([[0], [2], [1]]), [3, 4, 5], 4, 32)
            turned, _ = append_tokens(batch, tensors[0], tensors[1], rotary=rot, query=tensors[2])
            made.append((turned, batch.packed_k, batch.packed_v, batch.scales_k, batch.scales_v))
        assert all(torch.equal(a, b) for a, b in zip(*made))


def test_append_drops_what_has_no_place(cuda_device):
    rng = np.random.default_rng(22)
    pool = make_pool(rng, 4, 16, 1, 32, 32, 4)
    table = np.array([[0, -1], [1, 99]])
    batch = paged(cuda_device, pool, table, [14, 30], 4, 32, np.ones((2, 32), np.float32), np.ones((2, 32), np.int32))
    x = torch.from_numpy(rng.standard_normal((9, 1, 32))).half().to(cuda_device)
    # sequence 0: two slots in its page, two where the table names none; sequence 1: two there, three past the end;
    # no token is nobody's
    offsets = torch.tensor([0, 4, 9], dtype=torch.int32, device=cuda_device)
    _, lengths = append_tokens(batch, x, x, offsets=offsets)
    assert lengths.tolist() == [18, 32]
    want = [torch.from_numpy(a.copy()) for a in pool]
    coded = quantize(x[:2].reshape(-1, 32), 4, 32)
    want[0][0, 14:16, 0], want[2][0, 14:16, 0] = coded.packed.cpu(), coded.scales.cpu()
    want[1][0, 14:16, 0], want[3][0, 14:16, 0] = coded.packed.cpu(), coded.scales.cpu()
    for name, w in zip(("packed_k", "packed_v", "scales_k", "scales_v"), want):
        assert torch.equal(getattr(batch, name).cpu(), w), name
    # one token a sequence, lengths advanced in place
    one = torch.cat((x[:1], x[:1]))
    _, same = append_tokens(batch, one, one, lengths_out=batch.lengths)
    assert same is batch.lengths and same.tolist() == [15, 31]
    # no token at all
    none = x[:0]
    _, lengths = append_tokens(batch, none, none, offsets=torch.zeros(3, dtype=torch.int32, device=cuda_device))
    assert lengths.tolist() == [15, 31]


def test_append_of_values_at_the_codecs_edges(cuda_device):
    rng = np.random.default_rng(23)
    x = rng.standard_normal((6, 2, 64)).astype(np.float32)
    x[0] = 0.0
    x[1, 0, :32] = 1e-30
    x[2, 0] = 3e38
    x[3, 1, 5] = np.inf
    x[4, 1, 7] = -np.inf
    x[5, 0, 0] = np.nan
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for bits in (4, 2):
            t = torch.from_numpy(x).to(dtype).to(cuda_device)
            pool = make_pool(np.random.default_rng(24), 2, 8, 2, 64, 32, bits)
            batch = paged(cuda_device, pool, np.array([[1]]), [0], bits, 32)
            append_tokens(batch, t, t, offsets=torch.tensor([0, 6], dtype=torch.int32, device=cuda_device))
            coded = quantize(t.reshape(-1, 64), bits, 32)
            for packed, scales in ((batch.packed_k, batch.scales_k), (batch.packed_v, batch.scales_v)):
                assert torch.equal(packed[1, :6].flatten(0, 1), coded.packed)
                assert torch.equal(scales[1, :6].flatten(0, 1).view(torch.int16), coded.scales.view(torch.int16))


def test_append_graph_advances_lengths(cuda_device):
    rng = np.random.default_rng(25)
    pool = make_pool(rng, 8, 16, 2, 64, 32, 4)
    table = np.arange(8).reshape(2, 4)
    a, b = (paged(cuda_device, pool, table, [3, 14], 4, 32) for _ in range(2))
    rot = Rotary(64, device=cuda_device)
    k = torch.from_numpy(rng.standard_normal((2, 2, 64))).half().to(cuda_device)
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).half().to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, _ = append_tokens(a, k, k, rotary=rot, query=q, lengths_out=a.lengths)
        out, _ = HipAttentionBackend().run_paged(turned, a, 0.125)
    for r in range(5):
        k.copy_(torch.from_numpy(rng.standard_normal((2, 2, 64))).half())
        q.copy_(torch.from_numpy(rng.standard_normal((2, 4, 64))).half())
        graph.replay()
        want, _ = append_tokens(b, k, k, rotary=rot, query=q, lengths_out=b.lengths)
        want_out, _ = HipAttentionBackend().run_paged(want, b, 0.125)
        torch.cuda.synchronize()
        assert a.lengths.tolist() == [4 + r, 15 + r]
        assert torch.equal(turned, want) and torch.equal(out, want_out) and torch.equal(a.packed_k, b.packed_k)
    del graph


# ----------------------------------------------------------------------------------------------------------- eviction

EVICTS = [
    # lengths, budget, sink, recent, page_tokens, kv heads, head_dim, bits, how weights are made
    ([40], 39, 0, 0, 16, 1, 32, 4, "normal"),
    ([100, 64, 65, 1, 0], 64, 4, 16, 24, 2, 64, 4, "zeros"),
    ([3000, 1025, 1024, 2048], 1024, 4, 100, 64, 8, 128, 4, "heavy"),
    ([700, 500], 500, 0, 500, 7, 3, 96, 2, "heavy"),
    ([300, 299], 1, 0, 0, 32, 1, 32, 2, "equal"),
    ([5000], 77, 7, 70, 32, 2, 64, 4, "equal"),
    ([2500, 2500], 2400, 0, 10, 128, 1, 256, 4, "odd"),
    ([20000], 9000, 4, 3000, 128, 1, 64, 4, "heavy"),
    ([33], 4000, 0, 0, 16, 1, 32, 4, "normal"),
]


EVICTS += [  # several chunks of a sequence, chunks without a slot of it, the budget at a chunk's edge
    ([8192, 8191, 1, 0, 5000], 4096, 4, 1000, 128, 1, 32, 4, "zeros"),
    ([8193, 2048, 2049, 0, 1, 8192], 2048, 4, 100, 128, 1, 32, 2, "zeros"),
    ([30000, 12345, 4097], 4096, 0, 50, 100, 1, 32, 2, "equal"),
    ([30000, 16384, 10001], 10000, 3, 0, 64, 1, 32, 2, "odd"),
    ([50000], 49999, 0, 0, 64, 1, 32, 2, "normal"),
    ([50000, 9], 1, 1, 0, 64, 1, 32, 2, "heavy"),
]


@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"{c[0]}-{c[1]}-{c[8]}")
@pytest.mark.parametrize("shuffled", [False, True])
def test_eviction_keeps_and_moves_as_defined(cuda_device, case, shuffled):
    lengths, budget, sink, recent, bt, kvh, d, bits, how = case
    rng = np.random.default_rng(budget)
    width = max(-(-n // bt) for n in lengths) + 1
    pages = sum(-(-n // bt) for n in lengths) + 1
    pool = make_pool(rng, pages, bt, kvh, d, 32, bits)
    table = make_table(rng, lengths, bt, width, pages)
    slots = (len(lengths), width * bt)
    w = np.exp(2 * rng.standard_normal(slots)).astype(np.float32)
    if how == "zeros":
        w[rng.uniform(size=slots) < 0.6] = 0.0
    if how == "equal":
        w[...] = 0.5
    if how == "odd":  # negative ones, both zeros, infinities, NaN, subnormals
        w = np.where(rng.uniform(size=slots) < 0.5, -w, w)
        for x in (np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-42, -1e-42):
            w[rng.uniform(size=slots) < 0.05] = x
    pos = np.tile(np.arange(slots[1], dtype=np.int32), (slots[0], 1))
    if shuffled:
        for b, n in enumerate(lengths):
            pos[b, :n] = 2 * rng.permutation(n) + 1
    batch = paged(cuda_device, pool, table, lengths, bits, 32, w, pos)
    new_lengths, new_w, new_p = evict_tokens(batch, budget, sink=sink, recent=recent)
    assert new_lengths.tolist() == [min(n, budget) for n in lengths]
    assert batch.lengths.tolist() == lengths and np.array_equal(batch.weights.cpu().numpy(), w, equal_nan=True)
    want_w, want_p = np.zeros(slots, np.float32), np.full(slots, -1, np.int32)
    flat = [a.copy().reshape(pages * bt, -1) for a in pool]
    for b, n in enumerate(lengths):
        source = evict(w[b], pos[b], n, budget, sink, recent)
        want_w[b, :len(source)], want_p[b, :len(source)] = w[b, source], pos[b, source]
        for t, f in enumerate(source):
            if t != f:
                for a in flat:
                    a[table[b, t // bt] * bt + t % bt] = a[table[b, f // bt] * bt + f % bt]
    assert np.array_equal(new_p.cpu().numpy(), want_p)
    assert np.array_equal(new_w.cpu().numpy().view(np.int32), want_w.view(np.int32))
    for name, a in zip(("packed_k", "packed_v", "scales_k", "scales_v"), flat):
        got = getattr(batch, name).cpu().numpy().reshape(a.shape)
        assert (got.view(np.uint8) == a.view(np.uint8)).all(), name  # rows of other slots and pages as they were
    # the same again: nothing that the first call wrote is an input of the second
    again = evict_tokens(batch, budget, sink=sink, recent=recent)
    assert torch.equal(again[0], new_lengths) and torch.equal(again[2], new_p)
    assert np.array_equal(again[1].cpu().numpy().view(np.int32), want_w.view(np.int32))
    for name, a in zip(("packed_k", "packed_v", "scales_k", "scales_v"), flat):
        assert (getattr(batch, name).cpu().numpy().reshape(a.shape).view(np.uint8) == a.view(np.uint8)).all(), name


def test_eviction_skips_pages_that_are_not_there(cuda_device):
    rng = np.random.default_rng(30)
    pool = make_pool(rng, 4, 16, 1, 32, 32, 4)
    table = np.array([[0, 7, -1, 2]])
    w = np.arange(64, dtype=np.float32)[None]
    batch = paged(cuda_device, pool, table, [64], 4, 32, w, np.arange(64, dtype=np.int32)[None])
    lengths, new_w, _ = evict_tokens(batch, 20)
    assert lengths.tolist() == [20] and new_w[0, :20].tolist() == list(range(44, 64))
    got = batch.packed_k.cpu().numpy()
    want = pool[0].copy()
    want[0, 4:16] = pool[0][2, 0:12]  # slots 44-47 had no page, so that slots 0-3 have nothing to take
    assert (got == want).all()


def test_eviction_past_two_million_slots(cuda_device):
    """More slots than the most chunks of the smallest size hold: two at a time in each."""
    n, bt, budget = 2_200_000, 64, 1_000_001
    rng = np.random.default_rng(32)
    pages = -(-n // bt) + 1
    pool = make_pool(rng, pages, bt, 1, 32, 32, 2)
    table = make_table(rng, [n], bt, pages, pages)
    w = rng.integers(0, 1 << 20, (1, pages * bt)).astype(np.float32)  # with equal ones
    pos = np.arange(pages * bt, dtype=np.int32)[None]
    batch = paged(cuda_device, pool, table, [n], 2, 32, w, pos)
    lengths, new_w, new_p = evict_tokens(batch, budget, sink=5, recent=999)
    held = (pos[0, :n] < 5) | (pos[0, :n] > n - 1 - 999)
    order = np.lexsort((np.arange(n), -w[0, :n], ~held))
    kept = np.zeros(n, bool)
    kept[order[:budget]] = True
    source = np.arange(budget)
    source[~kept[:budget]] = budget + np.flatnonzero(kept[budget:])
    assert lengths.tolist() == [budget]
    assert np.array_equal(new_p.cpu().numpy()[0, :budget], pos[0, source]) and (new_p[0, budget:] == -1).all()
    assert np.array_equal(new_w.cpu().numpy()[0, :budget], w[0, source]) and (new_w[0, budget:] == 0).all()
    at = lambda s: table[0, s // bt].astype(np.int64) * bt + s % bt
    slots = np.arange(n)
    slots[:budget] = source
    for name, a in zip(("packed_k", "packed_v", "scales_k", "scales_v"), pool):
        got = getattr(batch, name).cpu().numpy().reshape(pages * bt, -1)[at(np.arange(n))]
        assert (got.view(np.uint8) == a.reshape(pages * bt, -1)[at(slots)].view(np.uint8)).all(), name


def test_eviction_graph(cuda_device):
    rng = np.random.default_rng(31)
    pool = make_pool(rng, 20, 16, 2, 64, 32, 4)
    table = np.arange(20).reshape(2, 10)
    pos = np.tile(np.arange(160, dtype=np.int32), (2, 1))
    a, b = (paged(cuda_device, pool, table, [150, 90], 4, 32, np.zeros((2, 160), np.float32), pos) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    evict_tokens(a, 80, recent=5)
    evict_tokens(b, 80, recent=5)
    with torch.cuda.graph(graph):
        got = evict_tokens(a, 80, recent=5)
    for r in range(4):
        w = torch.from_numpy(rng.uniform(0, 1, (2, 160)).astype(np.float32))
        a.weights.copy_(w)
        b.weights.copy_(w)
        graph.replay()
        want = evict_tokens(b, 80, recent=5)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a.packed_v, b.packed_v)
    del graph


def test_eviction_of_long_sequences_in_a_graph(cuda_device):
    rng = np.random.default_rng(33)
    pool = make_pool(rng, 300, 128, 1, 32, 32, 2)
    table = np.arange(300).reshape(2, 150)
    pos = np.tile(np.arange(19200, dtype=np.int32), (2, 1))
    a, b = (paged(cuda_device, pool, table, [19000, 9000], 2, 32, np.zeros((2, 19200), np.float32), pos) for _ in "ab")
    evict_tokens(a, 8000, recent=5)
    evict_tokens(b, 8000, recent=5)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got = evict_tokens(a, 8000, recent=5)
    with torch.cuda.graph(second):
        other = evict_tokens(a, 300, recent=5)
    for r in range(4):
        w = torch.from_numpy(rng.integers(0, 999, (2, 19200)).astype(np.float32))
        a.weights.copy_(w)
        b.weights.copy_(w)
        for graph, have, budget in ((first, got, 8000), (second, other, 300)):
            graph.replay()
            want = evict_tokens(b, budget, recent=5)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(have, want)) and torch.equal(a.packed_v, b.packed_v)
    del first, second


# --------------------------------------------------------------------------------------------- the operators together


@pytest.mark.parametrize(("bits", "dtype", "page_tokens"), [(4, torch.bfloat16, 32), (2, torch.float16, 24)])
def test_a_generation_loop(cuda_device, bits, dtype, page_tokens):
    """Prompts of three sequences, then steps of append, attention with summed weights and eviction to a budget, beside
    a model of it that keeps every row on the host."""
    rng = np.random.default_rng(40)
    kvh, qh, d, g, budget, sink, recent = 2, 8, 64, 32, 60, 2, 20
    cache = PagedKVCache(30, page_tokens, kvh, d, bits=bits, group_size=g, sequences=3, max_pages=8, track_weights=True,
                         device=cuda_device)
    rot = Rotary(d, device=cuda_device)
    rows = [[], [], []]  # per sequence and slot: (position, weight, (k codes, v codes, k scales, v scales))
    ends = [0, 0, 0]

    def model_append(keys, values, counts):
        at = 0
        for b, n in enumerate(counts):
            if n:
                position = torch.arange(ends[b], ends[b] + n, device=cuda_device)
                kq = quantize(rot(position, keys[at:at + n]).reshape(-1, d), bits, g)
                vq = quantize(values[at:at + n].reshape(-1, d), bits, g)
                parts = [t.cpu().numpy().reshape(n, kvh, -1) for t in (kq.packed, vq.packed, kq.scales, vq.scales)]
                rows[b] += [[ends[b] + i, 0.0, tuple(p[i] for p in parts)] for i in range(n)]
            ends[b] += n
            at += n

    steps = [[70, 0, 33]] + [[1, 1, 1]] * 3 + [[0, 50, 1]] + [[1, 1, 1]] * 12
    for step, counts in enumerate(steps):
        n = sum(counts)
        k, v, q = (torch.from_numpy(rng.standard_normal((n, h, d))).to(dtype).to(cuda_device) for h in (kvh, kvh, qh))
        turned = cache.append(k, v, counts, rotary=rot, query=q)
        assert turned.shape == q.shape
        model_append(k, v, counts)
        assert cache.lengths == [len(r) for r in rows] == cache.batch.lengths.tolist()
        query = torch.from_numpy(rng.standard_normal((3, qh, d))).to(dtype).to(cuda_device)
        out, lse = cache.attend(query, accumulate=True)
        longest = max(len(r) for r in rows)
        pool = [np.zeros((3, max(longest, 1), *s), t) for s, t in (
            ((kvh, d * bits // 8), np.uint8), ((kvh, d * bits // 8), np.uint8), ((kvh, d // g), np.float16),
            ((kvh, d // g), np.float16))]
        for b, r in enumerate(rows):
            for s, (_, _, parts) in enumerate(r):
                for a, p in zip(pool, parts):
                    a[b, s] = p
        weights = np.zeros((3, longest))
        for b, r in enumerate(rows):
            weights[b, :len(r)] = [x[1] for x in r]
        want = attend(as_double(query), pool, np.arange(3)[:, None], cache.lengths, bits, d ** -0.5, weights)
        check_attention(out, lse, want, d, longest, torch.float32, True)
        held = cache.batch.weights.cpu().numpy()
        for b, r in enumerate(rows):
            # kept from the device: the next cut goes by these, and a tie or two near ones may fall either way
            np.testing.assert_allclose(held[b, :len(r)], want["weights"][b, :len(r)], rtol=1e-4, atol=1e-7)
            for s, x in enumerate(r):
                x[1] = float(held[b, s])
        if max(cache.lengths) > budget:
            pages = cache.free_pages
            cache.evict(budget, sink=sink, recent=recent)
            for b, r in enumerate(rows):
                source = evict(np.array([x[1] for x in r], np.float32), np.array([x[0] for x in r], np.int32), len(r),
                               budget, sink, recent)
                rows[b] = [list(r[i]) for i in source]
            assert cache.free_pages >= pages
            for b, r in enumerate(rows):
                assert cache.batch.positions[b, :len(r)].tolist() == [x[0] for x in r]
    assert cache.next_positions == ends
    used = 30 - cache.free_pages
    assert used == sum(-(-n // page_tokens) for n in cache.lengths)
    cache.clear(0)
    assert cache.lengths[0] == 0 and cache.batch.lengths.tolist()[0] == 0
    assert 30 - cache.free_pages == sum(-(-n // page_tokens) for n in cache.lengths)


def test_a_stored_layer_goes_on_in_pages(cuda_device, tmp_path):
    # a layer of a store, loaded into pages, answers as the packed decode does, and grows from there
    from kvssd import CacheSpec, KVCacheStore, KVSSDPipeline

    rng = np.random.default_rng(50)
    keys = torch.from_numpy(rng.standard_normal((1, 300, 2, 64))).half()
    store = KVCacheStore.create(tmp_path, keys, keys, CacheSpec(1, 2, 64, 32, 4, 32))
    q = torch.from_numpy(rng.standard_normal((8, 64))).half().to(cuda_device)
    with KVSSDPipeline(store, device="cuda", attention_backend="hip") as pipe:
        pipe.load_resident()
        want = pipe.decode(q, 0)
        cache = pipe.paged_cache(0, spare_pages=4)
    assert cache.lengths == [300] and cache.free_pages == 4
    out, _ = cache.attend(q[None], out_dtype=torch.float16)
    # fp16 results: each weight p_t times its value scale is rounded to fp16, which moves the sum by at most
    # 2^-11 sum_t p_t |v_t| <= 2^-11 max |v| (the packed decode of this shape has 32-bit grade, 2e-5), and each of the
    # two results is rounded once, by half a step
    largest = float(keys.abs().max()) * (1 + 1 / 7)  # (a stored value lies within half a code step of its key)
    torch.testing.assert_close(out[0], want, atol=2e-5 + 2.0 ** -11 * largest, rtol=2.0 ** -10)
    exact, _ = cache.attend(q[None])
    torch.testing.assert_close(exact[0], want.float(), atol=4e-5, rtol=2.0 ** -11)
    more = torch.from_numpy(rng.standard_normal((200, 2, 64))).half().to(cuda_device)
    cache.append(more[:100], more[:100], [100])
    assert cache.lengths == [400]
    with pytest.raises(ValueError, match="at most 448 tokens"):
        cache.append(more, more, [200])
    assert cache.lengths == [400]
