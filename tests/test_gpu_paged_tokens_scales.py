"""Value scales of any size beside each other in attention of many tokens and outside a single token's window, on the GPU
against the 64-bit oracle: a large one that a row does not see takes no bits of that row's result, one that it sees takes
its part.

Tolerances: those of test_gpu_paged_tokens, which go by A = sum_t p_t |v_t| of the row itself, and one more.  A weight is
one or two fp16 numbers, of which the row's largest is 2^8 to 2^14 (2^14 to 2^16 with 32-bit results) and the smallest
step 2^-24: it is off by at most 2^-33 (2^-39) of the largest, beside its relative rounding.  Over n slots that a row sees
this adds at most n 2^-33 (2^-39) of its largest |v|, ``most``.  Values have no such term: two scales of one sequence may
differ by all that fp16 has."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kvssd.backends.hip import HipAttentionBackend
from paged_oracle import as_double, dequantise
from test_gpu_paged_tokens import U, ints, paged, problem, random_parents
from tokens_oracle import attend_tokens, visible

pytestmark = pytest.mark.gpu


def largest(pool, table, lengths, offsets, bits, parents, window, sink, heads) -> np.ndarray:
    """[tokens, heads, d]: the largest |v| that a token sees."""
    kvh, bt = pool[0].shape[2], pool[0].shape[1]
    d = pool[0].shape[3] * 8 // bits
    out = np.zeros((int(offsets[-1]), heads, d))
    for b, length in enumerate(lengths):
        begin, end = int(offsets[b]), int(offsets[b + 1])
        slots = np.arange(length)
        rows = table[b][slots // bt].astype(np.int64) * bt + slots % bt
        seen = visible(length, end - begin, None if parents is None else parents[begin:end], window, sink)
        for h in range(kvh):
            v = np.abs(dequantise(*(x.reshape(-1, kvh, x.shape[-1])[rows, h] for x in (pool[1], pool[3])), bits))
            for i in range(end - begin):
                out[begin + i, h * (heads // kvh):(h + 1) * (heads // kvh)] = v[seen[i]].max(0)
    return out


def check(out, lse, want, most, d, longest, dtype):
    precise = dtype == torch.float32
    e = (d + 16) * U * want["reach"] + 8 * U
    weight = 2 * e + (2.0 ** -21 if precise else 2.0 ** -10) + (longest + 8) * U
    tol = want["size"] * weight * (1 + weight) + np.abs(want["out"]) * torch.finfo(dtype).eps / 2
    tol += longest * 2.0 ** (-39 if precise else -33) * most
    tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    if dtype == torch.float16:
        assert np.abs(want["out"]).max() < 60000  # (the type holds them)
    err = np.abs(as_double(out) - want["out"])
    assert (err <= tol).all(), f"out: largest error over its bound {np.nanmax(err / tol)}"
    lerr = np.abs(as_double(lse) - want["lse"])
    assert (lerr <= e + (np.abs(want["lse"]) + 40) * 4 * U).all()


# query heads, kv heads, head_dim, slots before, new tokens: 32 rows of a kv head and sequence, 128, 256, and several runs
FORMS = {
    "few": (8, 2, 128, [700, 90], [8, 5]),
    "few, short heads": (8, 2, 64, [300, 500], [6, 7]),
    "128 rows": (8, 2, 128, [300, 20], [30, 12]),
    "256 rows": (8, 2, 128, [400], [100]),
    "256 rows, short heads": (4, 2, 64, [600, 5], [140, 70]),
    "long heads": (8, 2, 256, [200, 40], [40, 9]),
    "few, several runs": (4, 1, 128, [3000], [4]),
    "several runs": (4, 1, 128, [3000], [20]),
}
# scales of most slots, and of a few others
SCALES = {
    "usual, some hundreds": ((0.2, 0.5), (256.0, 700.0)),
    "usual, below a border": ((0.2, 0.5), (1.0, 255.9)),
    "usual, the largest": ((0.2, 0.5), (2e4, 6.5e4)),
    "small, the largest": ((1e-4, 1e-3), (2e4, 6.5e4)),
    "subnormal, the largest": ((6e-8, 3e-7), (2e4, 6.5e4)),
    "small, some hundreds": ((1e-3, 1e-2), (300.0, 5000.0)),
    "large, few small": ((300.0, 5e4), (1e-4, 0.5)),
}


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("scales", SCALES)
@pytest.mark.parametrize("form", FORMS)
def test_value_scales_of_any_size_beside_each_other(cuda_device, form, scales, out32):
    qh, kvh, d, before, counts = FORMS[form]
    usual, others = SCALES[scales]
    bits = 2 if form == "256 rows" else 4
    rng, pool, table, lengths, offsets, q = problem(cuda_device, bits, qh, kvh, d, 32, 64, before, counts, torch.bfloat16, 81)
    pool = list(pool)
    plain = np.exp(rng.uniform(*np.log(usual), pool[3].shape)).astype(np.float16)
    parents = random_parents(rng, counts, 0.3)
    scale = 1 / np.sqrt(d)
    dtype = torch.float32 if out32 else torch.bfloat16
    # where the others lie, and what is seen: all of the context's, or those above a token, or those of a window
    for place, up, window, sink in (("context", None, 0, 0), ("new", parents, 0, 0), ("new", None, 40, 1),
                                    ("one group", None, 0, 0), ("first", None, 40, 0)):
        values = plain.copy()
        flat = values.reshape(-1, kvh, values.shape[-1])
        for b, (a, n) in enumerate(zip(before, counts)):
            slots = {"context": [a // 2, a // 2 + 1, a - 1], "new": [a + n // 2, a + n - 1], "one group": [a - 2, a + n // 2],
                     "first": [0, 1]}[place]
            for slot in slots:
                row = table[b][slot // 64] * 64 + slot % 64
                new = np.exp(rng.uniform(*np.log(others), flat[row].shape)).astype(np.float16)
                if place == "one group":
                    flat[row, kvh - 1, 1] = new[kvh - 1, 1]
                else:
                    flat[row] = new
        pool[3] = values
        batch = paged(cuda_device, pool, table, lengths, bits, 32)
        want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, scale, up, window, sink)
        most = largest(pool, table, lengths, offsets, bits, up, window, sink, qh)
        out, lse = HipAttentionBackend().run_paged_tokens(
            q, batch, scale, ints(cuda_device, offsets), None if up is None else ints(cuda_device, up), window=window,
            sink=sink, out_dtype=dtype, max_length=max(lengths), total_tokens=sum(lengths))
        check(out, lse, want, most, d, max(lengths), dtype)


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("count", [8, 40, 150])
def test_a_first_slot_with_nearly_all_the_weight(cuda_device, count, out32):
    """One slot has nearly all of the weight and no value, as a sink does: what the others add keeps its bits, down to
    the weights' step."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 64, [2000], [count], torch.bfloat16, 82)
    pool = list(pool)
    row = table[0][0] * 64
    q = torch.ones_like(q) + q / 16
    pool[0].reshape(-1, 2, 64)[row] = 0xFF  # codes of 7 in every dim
    pool[2].reshape(-1, 2, 4)[row] = 0.2
    pool[2].reshape(-1, 2, 4)[np.arange(len(pool[2]) * 64) != row] *= np.float16(0.1)
    pool[1].reshape(-1, 2, 64)[row] = 0x88  # codes of 0
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    dtype = torch.float32 if out32 else torch.bfloat16
    scale = 1 / np.sqrt(128)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, scale)
    most = largest(pool, table, lengths, offsets, 4, None, 0, 0, 8)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, scale, ints(cuda_device, offsets), out_dtype=dtype)
    check(out, lse, want, most, 128, max(lengths), dtype)


@pytest.mark.parametrize(("d", "count"), [(32, 40), (64, 36), (128, 20), (128, 200), (256, 12)])
def test_weights_keep_their_bits_beside_a_large_scale(cuda_device, d, count):
    """A few nearly equal weights, so that errors of scores and sums are small: those of a stage in which one slot, a
    sibling that no other token sees, has a value scale near fp16's largest."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, d, 32, 64, [2, 4], [count, 30], torch.bfloat16, 83)
    pool = list(pool)
    parents = np.full(count + 30, -1, np.int32)
    for b, n in enumerate(lengths):  # the last
        row = table[b][(n - 1) // 64] * 64 + (n - 1) % 64
        pool[3].reshape(-1, 2, d // 32)[row] = 6e4
    batch = paged(cuda_device, pool, table, lengths, 4, 32)
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, 4, 3e-5, parents)
    most = largest(pool, table, lengths, offsets, 4, parents, 0, 0, 8)
    out, lse = HipAttentionBackend().run_paged_tokens(q, batch, 3e-5, ints(cuda_device, offsets), ints(cuda_device, parents))
    check(out, lse, want, most, d, 5, torch.float32)  # (a token sees the 2 or 4 slots before, and itself)


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("count", [6, 40, 200])
def test_large_scales_beside_pages_that_are_gone_and_scales_that_are_not_finite(cuda_device, count, out32):
    """The second round of the stages: slots without a page take no part in it, what is infinite or NaN makes its group of
    the rows that see it NaN and no other; keys that are NaN make whole rows so."""
    rng, pool, table, lengths, offsets, q = problem(cuda_device, 4, 8, 2, 128, 32, 16, [500, 90], [count, 5], torch.float16, 84)
    pool = tuple(x.copy() for x in pool)
    table[0, [3, 11]] = -1

    def scales(which, b, slot):
        return pool[which].reshape(-1, 2, 4)[table[b][slot // 16] * 16 + slot % 16]

    for slot in (20, 333, 500 + count // 2):
        scales(3, 0, slot)[:] = 1e4
    scales(3, 1, 92)[:, 2] = 300.0
    clean = tuple(x.copy() for x in pool)
    scales(3, 0, 500 + count - 2)[0, 1] = np.inf
    scales(3, 1, 93)[1, 3] = np.nan
    scales(2, 0, 500 + count - 1)[1, 0] = np.nan
    most = largest(clean, np.maximum(table, 0), lengths, offsets, 4, None, 0, 0, 8)
    dtype = torch.float32 if out32 else torch.float16
    for window in (0, 200):
        want = attend_tokens(as_double(q), clean, table, lengths, offsets, 4, 0.09, None, window)
        out, lse = HipAttentionBackend().run_paged_tokens(q, paged(cuda_device, pool, table, lengths, 4, 32), 0.09,
                                                          ints(cuda_device, offsets), window=window, out_dtype=dtype)
        bad = np.zeros(out.shape, bool)
        bad[count - 2:count, :4, 32:64] = True
        bad[count + 3:, 4:, 96:] = True
        bad[count - 1, 4:] = True
        got = as_double(out)
        assert np.array_equal(np.isnan(got), bad)
        assert np.isnan(as_double(lse)[count - 1, 4:]).all() and np.isnan(as_double(lse)).sum() == 4
        got[bad], lse[count - 1, 4:] = want["out"][bad], torch.from_numpy(want["lse"][count - 1, 4:]).to(lse)
        check(torch.from_numpy(got), lse, want, most, 128, max(lengths), dtype)


@pytest.mark.parametrize("out32", [False, True], ids=["own", "f32"])
@pytest.mark.parametrize("value", [np.nan, np.inf, 6.5e4], ids=str)
@pytest.mark.parametrize(("qh", "kvh", "d", "bt", "bits"), [(32, 8, 128, 64, 4), (8, 2, 64, 20, 4), (10, 5, 96, 32, 2), (16, 2, 256, 128, 4)])
def test_slots_outside_a_single_tokens_window_have_no_part(cuda_device, qh, kvh, d, bt, bits, value, out32):
    """Keys' and values' scales of slots behind the sinks and before the window, in stages of which others are seen: the
    same bits as with scales like all others there."""
    lengths = [300, 77, 1000, 64]
    rng, pool, table, _, offsets, q = problem(cuda_device, bits, qh, kvh, d, 32, bt, [n - 1 for n in lengths], [1] * 4,
                                              torch.float16, 85, (1e-3, 1e-2))
    dirty = tuple(x.copy() for x in pool)
    window, sink = 50, 5
    for b, length in enumerate(lengths):
        for slot in range(sink, length - window):
            row = table[b][slot // bt] * bt + slot % bt
            dirty[3].reshape(-1, kvh, d // 32)[row] = value
            if not np.isfinite(value):
                dirty[2].reshape(-1, kvh, d // 32)[row] = value
    dtype = torch.float32 if out32 else torch.float16
    results = [
        HipAttentionBackend().run_paged(q, paged(cuda_device, x, table, lengths, bits, 32), 3.0, window=window, sink=sink, out_dtype=dtype)
        for x in (pool, dirty)
    ]
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    want = attend_tokens(as_double(q), pool, table, lengths, offsets, bits, 3.0, None, window, sink)
    most = largest(pool, table, lengths, offsets, bits, None, window, sink, qh)
    check(*results[1], want, most, d, window + sink, dtype)
