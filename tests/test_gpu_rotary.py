"""Rotary positions on the GPU against their definition in 64 bits.

Tolerance.  The kernel works in 64 bits and rounds to 32 and then to the type: eps/2 of the type and 2^-24 of the
value.  In 64 bits an angle of a radians is off by at most a 2^-53 (its product's rounding) and the sine of it by a few
2^-53 more, which moves a value by at most |pair| (a + 8) 2^-52, |pair| = |x_i| + |x_j|; the oracle's own angles are off
by as much again.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kvssd import Rotary, RotaryScaling
from paged_oracle import as_double, frequencies, rotate

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def check(got: torch.Tensor, x: torch.Tensor, positions, freq, interleaved, magnitude=1.0, inverse=False):
    want = rotate(as_double(x), positions, freq, interleaved, magnitude, inverse)
    d, r = x.shape[2], 2 * len(freq)
    ax = np.abs(as_double(x))
    pair = np.zeros_like(ax)
    low, high = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    pair[..., low] = pair[..., high] = (ax[..., low] + ax[..., high]) * magnitude
    angle = float(np.abs(positions).max(initial=0)) * float(freq.max())
    tol = np.abs(want) * (torch.finfo(x.dtype).eps / 2 + 2.0 ** -24) + pair * (angle + 8) * 2.0 ** -51
    tol += torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # a step among the subnormals
    err = np.abs(as_double(got) - want)
    assert got.shape == x.shape and got.dtype == x.dtype
    assert (err <= tol).all(), f"largest error over its bound: {(err / np.maximum(tol, 1e-300)).max()}"
    if r < d:
        assert torch.equal(got[..., r:], x[..., r:])


SHAPES = [
    # tokens, query heads, key heads, head_dim, rotary_dim
    (1, 1, 1, 2, 2),
    (1, 32, 8, 128, 128),
    (3, 5, 1, 64, 20),
    (7, 4, 2, 96, 24),
    (64, 16, 4, 256, 64),
    (33, 3, 3, 80, 80),
    (2049, 3, 1, 64, 64),   # several tokens a workgroup, the last one alone
    (2055, 2, 1, 1024, 1024),
    (5, 7, 2, 13, 6),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotary_matches_its_definition(cuda_device, shape, layout, dtype):
    tokens, qh, kvh, d, r = shape
    rng = np.random.default_rng(tokens + d)
    positions = rng.integers(0, 1 << 20, tokens)
    q = torch.from_numpy(rng.standard_normal((tokens, qh, d))).to(dtype).to(cuda_device)
    k = torch.from_numpy(rng.standard_normal((tokens, kvh, d))).to(dtype).to(cuda_device)
    rot = Rotary(d, rotary_dim=r, layout=layout, device=cuda_device)
    pos = torch.from_numpy(positions).to(cuda_device)
    tq, tk = rot(pos, q, k)
    freq = frequencies(r)
    check(tq, q, positions, freq, layout == "interleaved")
    check(tk, k, positions, freq, layout == "interleaved")
    # the same through int32 positions, one tensor, and in place
    assert torch.equal(rot(pos.int(), q), tq)
    same = k.clone()
    assert rot(pos, same, inplace=True) is same and torch.equal(same, tk)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_slices_of_a_fused_projection_and_other_strides(cuda_device, layout, dtype):
    # query, key and value side by side in one tensor, at a start and with strides that no 16-byte load fits, and
    # tokens and heads exchanged
    rng = np.random.default_rng(3)
    freq = frequencies(32)
    rot = Rotary(64, rotary_dim=32, layout=layout, device=cuda_device)
    positions = np.array([5, 0, 100000, 7, 1])
    pos = torch.from_numpy(positions).to(cuda_device)
    for shift in (0, 1):
        fused = torch.from_numpy(rng.standard_normal((5, 9 * 64 + 3))).to(dtype).to(cuda_device)
        q = fused[:, shift: shift + 6 * 64].unflatten(1, (6, 64))
        k = fused[:, shift + 6 * 64: shift + 8 * 64].unflatten(1, (2, 64))
        rest = fused[:, shift + 8 * 64:].clone()
        tq, tk = rot(pos, q, k)
        check(tq, q, positions, freq, layout == "interleaved")
        check(tk, k, positions, freq, layout == "interleaved")
        rot(pos, q, k, inplace=True)
        assert torch.equal(q, tq) and torch.equal(k, tk)
        assert torch.equal(fused[:, shift + 8 * 64:], rest)
    heads_first = torch.from_numpy(rng.standard_normal((6, 5, 64))).to(dtype).to(cuda_device).transpose(0, 1)
    check(rot(pos, heads_first), heads_first, positions, freq, layout == "interleaved")
    wide = torch.from_numpy(rng.standard_normal((5, 6, 128))).to(dtype).to(cuda_device)[..., ::2]
    check(rot(pos, wide), wide, positions, freq, layout == "interleaved")
    one = torch.from_numpy(rng.standard_normal((5, 1, 64))).to(dtype).to(cuda_device).expand(5, 3, 64)
    check(rot(pos, one), one, positions, freq, layout == "interleaved")


@pytest.mark.parametrize("scaling", [
    RotaryScaling("linear", 8.0), RotaryScaling("ntk", 4.0), RotaryScaling("yarn", 4.0, 4096),
    RotaryScaling("wavelength", 32.0),
], ids=lambda s: s.kind)
def test_scaled_frequencies_and_magnitude(cuda_device, scaling):
    rng = np.random.default_rng(8)
    rot = Rotary(128, base=500000.0, scaling=scaling, device=cuda_device)
    x = torch.from_numpy(rng.standard_normal((9, 4, 128))).float().to(cuda_device)
    positions = rng.integers(0, 1 << 24, 9)
    freq = rot.frequencies.cpu().numpy()
    check(rot(torch.from_numpy(positions).to(cuda_device), x), x, positions, freq, False, rot.magnitude)


def test_positions_past_32_bits_and_below_zero(cuda_device):
    rng = np.random.default_rng(9)
    rot = Rotary(64, device=cuda_device)
    x = torch.from_numpy(rng.standard_normal((4, 2, 64))).float().to(cuda_device)
    positions = np.array([0, -1, (1 << 33) + 5, -(1 << 31)])
    check(rot(torch.from_numpy(positions).to(cuda_device), x), x, positions, frequencies(64), False)


def test_inverse_is_the_transpose_and_the_gradient(cuda_device):
    # <g, R x> = <R^T g, x>: both sums of 2,560 products of values rounded once (2^-24 of each, |products| sum to S)
    rng = np.random.default_rng(10)
    scaling = RotaryScaling("yarn", 4.0, 4096)
    rot = Rotary(128, layout="interleaved", scaling=scaling, device=cuda_device)
    pos = torch.arange(10, device=cuda_device) * 997
    x = torch.from_numpy(rng.standard_normal((10, 2, 128))).float().to(cuda_device)
    g = torch.from_numpy(rng.standard_normal((10, 2, 128))).float().to(cuda_device)
    left, right = as_double(g) * as_double(rot(pos, x)), as_double(rot(pos, g, inverse=True)) * as_double(x)
    assert abs(left.sum() - right.sum()) <= 2.0 ** -24 * (np.abs(left).sum() + np.abs(right).sum())
    check(rot(pos, g, inverse=True), g, np.arange(10) * 997, rot.frequencies.cpu().numpy(), True, rot.magnitude, True)
    # and against differences: rotation is linear, so f(x + h) - f(x) is the gradient's product with h up to the
    # three results' roundings (2^-24 of each value)
    h = torch.from_numpy(rng.standard_normal((10, 2, 128))).float().to(cuda_device)
    f = lambda t: as_double(g) * as_double(rot(pos, t))  # noqa: E731
    xs = (x + h)
    step = as_double(xs) - as_double(x)
    diff = f(xs) - f(x)
    slope = as_double(rot(pos, g, inverse=True)) * step
    bound = 2.0 ** -24 * (np.abs(f(xs)).sum() + np.abs(f(x)).sum() + np.abs(slope).sum())
    assert abs(diff.sum() - slope.sum()) <= bound


def test_nothing_to_do_other_streams_and_captured(cuda_device):
    rng = np.random.default_rng(11)
    rot = Rotary(64, device=cuda_device)
    none = torch.empty((0, 4, 64), device=cuda_device)
    assert rot(torch.empty(0, dtype=torch.int64, device=cuda_device), none).shape == none.shape
    x = torch.from_numpy(rng.standard_normal((5, 4, 64))).to(torch.bfloat16).to(cuda_device)
    empty_key = torch.empty((5, 0, 64), dtype=torch.bfloat16, device=cuda_device)
    pos = torch.arange(5, device=cuda_device)
    want = rot(pos, x)
    got = rot(pos, x, empty_key)
    assert torch.equal(got[0], want) and got[1].shape == (5, 0, 64)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = rot(pos, x)
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    assert torch.equal(other, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rot(pos, x)
    for r in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal((5, 4, 64))).to(torch.bfloat16))
        pos.copy_(torch.arange(5) * (r + 3))
        graph.replay()
        eager = rot(pos, x)
        torch.cuda.synchronize()
        assert torch.equal(captured, eager), r
    del graph


def test_inplace_rotation_of_overlapping_slices_is_refused(cuda_device):
    rng = np.random.default_rng(12)
    rot = Rotary(32, device=cuda_device)
    pos = torch.arange(6, device=cuda_device)
    x = torch.from_numpy(rng.standard_normal((6, 8, 32))).half().to(cuda_device)
    before = x.clone()
    for q, k in ((x[:, :5], x[:, 3:]), (x[:, 3:], x[:, :5]), (x[:, :3], x[:, 2:]), (x[:, ::2], x[:, 2:3])):
        with pytest.raises(ValueError, match="share no element"):
            rot(pos, q, k, inplace=True)
    with pytest.raises(ValueError, match="share no element"):
        rot(pos[:4], x[:4], x[2:], inplace=True)
    assert torch.equal(x, before)
    want = rot(pos, x)
    for q, k in ((x[:, :5], x[:, 5:]), (x[:, 1::2], x[:, ::2])):  # slices that lie among each other
        x.copy_(before)
        rot(pos, q, k, inplace=True)
        assert torch.equal(x, want)


def test_a_graph_sees_that_its_tensor_was_rotated_in_place(cuda_device):
    rot = Rotary(32, device=cuda_device)
    pos = torch.arange(3, device=cuda_device)
    w = torch.ones((3, 2, 32), device=cuda_device, requires_grad=True)
    x, key = torch.randn((2, 3, 2, 32), device=cuda_device)
    for tensors in ((x,), (key, x)):
        y = (w * x).sum()  # (saves x)
        rot(pos, *tensors, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    y = (w * x).sum()
    rot(pos, x)
    y.backward()
    assert torch.equal(w.grad, x)
    with torch.inference_mode():
        z = torch.randn((3, 2, 32), device=cuda_device)
        want = rot(pos, z)
        assert torch.equal(rot(pos, z, inplace=True), want)
