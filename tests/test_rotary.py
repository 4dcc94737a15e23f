"""Rotary frequencies, and what the operator refuses (no GPU)."""

from __future__ import annotations

import math
import random

import pytest
import torch

from kvssd import Rotary, RotaryScaling
from kvssd.rotary import _overlaps_itself, _share_elements, refuse_grad, rotary_frequencies


def test_plain_frequencies():
    f = rotary_frequencies(8, 10000.0)
    assert f == [1.0, 10000.0 ** -0.25, 10000.0 ** -0.5, 10000.0 ** -0.75]


def test_scaled_frequencies():
    plain = rotary_frequencies(128, 500000.0)
    assert rotary_frequencies(128, 500000.0, RotaryScaling("linear", 4.0)) == [f / 4.0 for f in plain]
    ntk = rotary_frequencies(128, 500000.0, RotaryScaling("ntk", 4.0))
    # the first pair stays, the last is divided by the factor (64 bits: pow is good to a few 2^-53)
    assert ntk[0] == plain[0] and ntk[-1] == pytest.approx(plain[-1] / 4.0, rel=1e-13)
    for kind, low, high in (("yarn", 1.0, 32.0), ("wavelength", 1.0, 4.0)):
        s = RotaryScaling(kind, 8.0, 8192)
        got = rotary_frequencies(128, 500000.0, s)
        assert s.bounds == (low, high)
        turns = [8192 * f / (2 * math.pi) for f in plain]
        for f, g, n in zip(plain, got, turns):
            assert f / 8.0 * (1 - 1e-12) <= g <= f * (1 + 1e-12)
            if n > high * 1.3:
                assert g == pytest.approx(f, rel=1e-15)
            if n < low / 1.3:
                assert g == pytest.approx(f / 8.0, rel=1e-15)
        assert all(a > b for a, b in zip(got, got[1:]))
    assert RotaryScaling("yarn", 4.0).magnitude == 0.1 * math.log(4.0) + 1.0
    assert RotaryScaling("linear", 4.0).magnitude == 1.0


def test_a_ramp_that_is_a_step():
    # a context so short that the ramp's ends meet: still a frequency per pair, all within a factor of 8
    f = rotary_frequencies(4, 10000.0, RotaryScaling("yarn", 8.0, 1))
    assert len(f) == 2 and all(0 < x <= 1 for x in f)


@pytest.mark.parametrize(("args", "kwargs", "match"), [
    ((64,), dict(rotary_dim=0), "even and between"),
    ((64,), dict(rotary_dim=7), "even and between"),
    ((64,), dict(rotary_dim=66), "even and between"),
    ((63,), dict(), "even and between"),
    ((2048,), dict(), "<= 1024"),
    ((64,), dict(layout="pairs"), "unknown rotary layout"),
    ((64,), dict(base=1.0), "base"),
    ((64,), dict(base=float("nan")), "base"),
    ((2,), dict(scaling=RotaryScaling("ntk", 2.0)), "ntk"),
])
def test_refused_layouts(args, kwargs, match):
    with pytest.raises(ValueError, match=match):
        Rotary(*args, device="cpu", **kwargs)


@pytest.mark.parametrize(("args", "match"), [
    (("cubic", 2.0), "unknown rotary scaling"),
    (("linear", 0.5), "at least 1"),
    (("linear", float("inf")), "at least 1"),
    (("yarn", 2.0, 0), "positive"),
    (("yarn", 2.0, 10, 4.0, 2.0), "low < high"),
    (("yarn", 2.0, 10, 0.0), "low < high"),
])
def test_refused_scalings(args, match):
    with pytest.raises(ValueError, match=match):
        RotaryScaling(*args)


def test_cpu_tensors_are_refused():
    rot = Rotary(8, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        rot(torch.arange(3), torch.zeros(3, 1, 8))


def test_gradients_are_refused_not_cut():
    x = torch.zeros(2, requires_grad=True)
    with pytest.raises(ValueError, match="no backward pass"):
        refuse_grad(None, x)
    with torch.no_grad():
        refuse_grad(x)
    refuse_grad(x.detach(), None)


def test_tensors_that_hold_an_element_twice_are_seen():
    t = torch.zeros(4, 6, 8)
    assert not _overlaps_itself(t) and not _overlaps_itself(t.transpose(0, 1)) and not _overlaps_itself(t[:, ::2])
    assert _overlaps_itself(t[:, :1].expand(4, 3, 8))
    assert _overlaps_itself(torch.zeros(20).as_strided((3, 2, 8), (4, 2, 1)))
    assert not _overlaps_itself(torch.zeros(0, 2, 8)) and not _overlaps_itself(t[:1].expand(1, 6, 8))


def test_tensors_that_share_an_element_are_seen():
    def shared(a, b):  # by the elements themselves
        where = [{t.storage_offset() + i * t.stride(0) + h * t.stride(1) + x
                  for i in range(t.shape[0]) for h in range(t.shape[1]) for x in range(t.shape[2])} for t in (a, b)]
        return bool(where[0] & where[1])

    flat = torch.zeros(4000)
    x = flat[:960].view(5, 6, 32)
    pairs = [
        (x, x), (x[:, :5], x[:, 3:]), (x[:, :3], x[:, 2:]), (x[:, :3], x[:, 3:]), (x[:2], x[2:]), (x[:3], x[2:]),
        (x[::2], x[1::2]), (x[::2], x[1:]), (x[:, ::2], x[:, 1::2]), (x[:, ::2], x[:, 2:3]), (x[:1], x[:1, 5:]),
        (x[1:2, 4:], x[1:3, :4]), (x.transpose(0, 1)[:3], x.transpose(0, 1)[3:]), (x.transpose(0, 1), x[:, 5:]),
        (x[..., :16], x[..., 16:]), (x[..., :17], x[..., 15:]), (x[:0], x), (x, torch.zeros(2, 3, 32)),
        (x[:1].expand(1, 6, 32), x[1:, 2:]),
    ]
    rng = random.Random(3)
    while len(pairs) < 2000:  # strides as they come, of tensors without an element twice
        made = []
        for _ in range(2):
            n, h, d = rng.randint(1, 5), rng.randint(1, 4), 8
            strides = rng.choice([(40, 8, 1), (64, 8, 1), (64, 16, 1), (8, 40, 1), (100, 20, 1), (33, 9, 1), (9, 50, 1)])
            made.append(flat.as_strided((n, h, d), strides, rng.randint(0, 200)))
        if not any(map(_overlaps_itself, made)):
            pairs.append(tuple(made))
    seen = [0, 0]
    for a, b in pairs:
        want = shared(a, b) and a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()
        assert _share_elements(a, b) == _share_elements(b, a) == want, (a.shape, a.stride(), b.shape, b.stride())
        seen[want] += 1
    assert min(seen) > 300
    big = torch.zeros(8 * 48).view(1, 48, 8).expand(1, 48, 8)
    assert not _share_elements(big[:, :40], big[:, 40:]) and _share_elements(big[:, :41], big[:, 40:])


def test_tangents_are_refused_not_dropped():
    from torch.autograd import forward_ad

    x = torch.zeros(2)
    refuse_grad(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(2))
        refuse_grad(x, None)
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), pytest.raises(ValueError, match="no forward derivative"):
                refuse_grad(None, dual)
        refuse_grad(forward_ad.unpack_dual(dual).primal)
    with pytest.raises(ValueError, match="no forward derivative"):
        torch.func.jvp(lambda t: refuse_grad(t) or t, (x,), (torch.ones(2),))


@pytest.mark.parametrize("scaling", [
    RotaryScaling("yarn", 8.0, 1), RotaryScaling("yarn", 8.0, 6), RotaryScaling("yarn", 4.0, 600, 100.0, 200.0),
])
def test_no_pair_of_a_short_context_makes_the_turns_that_it_would_stay_for(scaling):
    plain = rotary_frequencies(16, 10000.0)
    assert scaling.original_positions * plain[0] / (2 * math.pi) < scaling.bounds[0]
    assert rotary_frequencies(16, 10000.0, scaling) == [f / scaling.factor for f in plain]


def test_every_pair_of_a_long_context_stays_where_all_turn_often_enough():
    scaling = RotaryScaling("yarn", 8.0, 1 << 40)
    assert rotary_frequencies(16, 100.0, scaling) == rotary_frequencies(16, 100.0)
