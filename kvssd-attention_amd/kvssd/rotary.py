"""Rotary positions on the GPU: queries and keys turned by their tokens' positions.

The reference's cache takes keys as they come and its decode takes the query as
it comes; a model with rotary positions has to turn both.  :class:`Rotary` keeps
the frequencies of one layer shape on the device and turns tensors with them;
``append_tokens`` (``kvssd.paged``) takes it to turn keys on their way into a
packed cache.

Pair i of a head -- values i and i + rotary_dim/2 (``layout="half"``) or 2i and
2i + 1 (``"interleaved"``) -- is turned by the angle position * f_i and
multiplied by the scaling's magnitude; values past ``rotary_dim`` stay.  Without
scaling f_i = base^(-2i/rotary_dim).  Angles, sines and products have 64 bits,
so that positions far past 32-bit angles' precision keep theirs; the result is
rounded to 32 bits and then, for 16-bit values, to their type.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _native
from .backends.base import refuse_grad
from .backends.hip import current_stream_handle, on_device

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16, torch.float32: _native.DTYPE_F32}
_KINDS = ("linear", "ntk", "yarn", "wavelength")
_PAIR = _native.Heads * 2


@dataclass(frozen=True)
class RotaryScaling:
    """Frequencies changed for contexts longer than the ``original_positions``
    that they were made for.

    * ``linear``: every frequency divided by ``factor``;
    * ``ntk``: the base multiplied by factor^(R/(R-2)), which divides the lowest
      frequency by ``factor`` and leaves the highest;
    * ``yarn``: frequencies that make more than ``high`` turns (default 32) in the
      original context stay, those below ``low`` (default 1) are divided by
      ``factor``, with a linear ramp over the pairs between; rotated values are
      multiplied by 0.1 ln(factor) + 1;
    * ``wavelength``: as ``yarn`` with the ramp linear in the number of turns
      (defaults 1 and 4) and no multiplication."""

    kind: str
    factor: float
    original_positions: int = 8192
    low: float | None = None
    high: float | None = None

    def __post_init__(self) -> None:
        if self.kind not in _KINDS:
            raise ValueError(f"unknown rotary scaling '{self.kind}'; choose one of: {', '.join(_KINDS)}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError("rotary scaling factor must be finite and at least 1")
        if self.original_positions < 1:
            raise ValueError("original_positions must be positive")
        low, high = self.bounds
        if not 0 < low < high:
            raise ValueError("rotary scaling needs 0 < low < high")

    @property
    def bounds(self) -> tuple[float, float]:
        high = 32.0 if self.kind == "yarn" else 4.0
        return (1.0 if self.low is None else self.low, high if self.high is None else self.high)

    @property
    def magnitude(self) -> float:
        return 0.1 * math.log(self.factor) + 1.0 if self.kind == "yarn" else 1.0


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: RotaryScaling | None = None) -> list[float]:
    """Angle per position of each of the rotary_dim/2 pairs."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and between 2 and head_dim")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError("rotary base must be finite and greater than 1")
    if scaling is not None and scaling.kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of 4 or more")
        base = base * scaling.factor ** (rotary_dim / (rotary_dim - 2))
    plain = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None or scaling.kind == "ntk":
        return plain
    factor = scaling.factor
    if scaling.kind == "linear":
        return [f / factor for f in plain]
    low, high = scaling.bounds
    if scaling.kind == "wavelength":
        kept = [min(max((scaling.original_positions * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for f in plain]
        return [(1.0 - t) * f / factor + t * f for f, t in zip(plain, kept)]

    def pair_turning(turns: float) -> float:
        """The (fractional) pair that makes this many turns in the original context."""
        return rotary_dim * math.log(scaling.original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

    if pair_turning(low) <= 0:  # not even the first pair makes more
        return [f / factor for f in plain]
    first = max(math.floor(pair_turning(high)), 0)
    last = min(math.ceil(pair_turning(low)), rotary_dim - 1)
    if last <= first:  # the ramp is a step
        last = first + 0.001
    divided = [min(max((i - first) / (last - first), 0.0), 1.0) for i in range(rotary_dim // 2)]
    return [f / factor * t + f * (1.0 - t) for f, t in zip(plain, divided)]


def _overlaps_itself(t: torch.Tensor) -> bool:
    extent = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride < extent:
            return True
        extent = stride * size
    return False


def _share_elements(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [tokens, heads, head_dim] tensors of one type, values of a head side by side and none of them there
    twice, have an element in common."""
    if not a.numel() or not b.numel():
        return False
    (n, h, d), (st, sh, _), (bn, bh, _), (bst, bsh, _) = a.shape, a.stride(), b.shape, b.stride()
    size, first, second = a.itemsize, a.data_ptr(), b.data_ptr()
    reach, b_reach = ((h - 1) * sh + d) * size, ((bh - 1) * bsh + d) * size  # bytes of a token, first value to last
    if first + (n - 1) * st * size + reach <= second or second + (bn - 1) * bst * size + b_reach <= first:
        return False
    if st == bst > 0:  # slices of one projection: apart if their heads are, within a token's stride
        ahead = (second - first) % (st * size)
        if reach <= ahead <= st * size - b_reach:
            return False
    def heads_apart(t: torch.Tensor, first: int) -> torch.Tensor:
        return first + torch.arange(t.shape[1], device="cpu") * (t.stride(1) * size)

    # no head of b may begin less than a head (d values) before or behind one of a
    begins, b_begins = heads_apart(a, first), heads_apart(b, second)
    if st == bst or n == 1 or bn == 1:  # of each pair of heads, at the tokens where the two come closest
        step = (bst if n == 1 else st) * size
        ahead = b_begins - begins[:, None]
        for extra in (0, 1):
            tokens = (-ahead // step + extra).clamp(1 - n, bn - 1) if step else 0
            if bool(((ahead + tokens * step).abs() < d * size).any()):
                return True
        return False
    begins, b_begins = (
        (torch.arange(t.shape[0], device="cpu")[:, None] * (t.stride(0) * size) + x).flatten()
        for t, x in ((a, begins), (b, b_begins))
    )
    begins = begins.sort().values
    at = torch.searchsorted(begins, b_begins)  # (begins[at - 1] < b_begins <= begins[at])
    last = begins.numel() - 1
    behind = b_begins - begins[(at - 1).clamp(min=0)] < d * size
    before = begins[at.clamp(max=last)] - b_begins < d * size
    return bool(((at > 0) & behind).any() or ((at <= last) & before).any())


def heads_of(t: torch.Tensor, out: torch.Tensor | None = None) -> tuple:
    """Fields of kvssd_heads of a [tokens, heads, head_dim] tensor (its values of a head side by side)."""
    token, head, _ = t.stride()
    if out is None:
        return t.data_ptr(), None, token, head, 0, 0, t.shape[1], 0
    out_token, out_head, _ = out.stride()
    return t.data_ptr(), out.data_ptr(), token, head, out_token, out_head, t.shape[1], 0


def empty_heads(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def check_heads(t: torch.Tensor, name: str, tokens: int, head_dim: int, dtype: torch.dtype, device: torch.device) -> None:
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim:
        raise ValueError(f"{name} must be [{tokens}, heads, {head_dim}], got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


class Rotary:
    """Rotary positions of heads of ``head_dim`` values, the first ``rotary_dim`` (default: all) of which turn.

    ``rotary(positions, query, key)`` returns the turned query and key, each [tokens, heads, head_dim] in float16,
    bfloat16 or float32 with any token and head strides; ``positions`` is int32 or int64 [tokens].  Without a key it
    returns the query alone.  ``inverse`` turns back (the transpose, which is also the gradient's map);
    ``inplace`` writes into the tensors given, which must share no element.  One launch on the current stream."""

    def __init__(
        self,
        head_dim: int,
        *,
        rotary_dim: int | None = None,
        base: float = 10000.0,
        layout: str = "half",
        scaling: RotaryScaling | None = None,
        device: str | torch.device = "cuda",
    ):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ("half", "interleaved"):
            raise ValueError(f"unknown rotary layout '{layout}'; choose one of: half, interleaved")
        if head_dim > 1024:
            raise ValueError("rotary head_dim must be <= 1024")
        if rotary_dim % 2 or not 2 <= rotary_dim <= head_dim:
            raise ValueError("rotary_dim must be even and between 2 and head_dim")
        self.head_dim, self.rotary_dim, self.base, self.layout, self.scaling = head_dim, rotary_dim, base, layout, scaling
        self.magnitude = 1.0 if scaling is None else scaling.magnitude
        host = torch.tensor(rotary_frequencies(rotary_dim, base, scaling), dtype=torch.float64)
        self.frequencies = host.to(device)
        self._device = self.frequencies.device  # (with its index, on a GPU)
        self._index = self._device.index if self._device.type == "cuda" else None
        self._specs = tuple(
            _native.RotarySpec(self.frequencies.data_ptr(), self.magnitude, head_dim, rotary_dim,
                               int(layout == "interleaved"), inverse)
            for inverse in (0, 1)
        )
        self._addresses = tuple(ctypes.addressof(s) for s in self._specs)

    def spec(self, inverse: bool = False) -> _native.RotarySpec:
        return self._specs[bool(inverse)]

    def __call__(
        self,
        positions: torch.Tensor,
        query: torch.Tensor,
        key: torch.Tensor | None = None,
        *,
        inverse: bool = False,
        inplace: bool = False,
    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        device, index = self._device, self._index
        if index is None:
            raise ValueError(f"rotary positions require ROCm GPU tensors, got {device.type}")
        dtype, tokens = query.dtype, query.shape[0] if query.ndim else 0
        if dtype not in _DTYPES:
            raise ValueError(f"unsupported dtype {dtype}")
        tensors = (query,) if key is None else (query, key)
        for name, t in zip(("query", "key"), tensors):
            check_heads(t, name, tokens, self.head_dim, dtype, device)
        if positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError("positions must be int32 or int64 [tokens]")
        if positions.device != device:
            raise ValueError(f"positions must be on {device}, got {positions.device}")
        refuse_grad(*tensors)
        if inplace:
            for t in tensors:
                if t.stride(2) != 1 or _overlaps_itself(t):
                    raise ValueError("inplace needs values of a head side by side and no element twice")
            if key is not None and _share_elements(query, key):
                raise ValueError("inplace needs a query and a key that share no element")
            outs = tensors
        else:
            tensors = tuple(t if t.stride(2) == 1 else t.contiguous() for t in tensors)
            outs = tuple(map(empty_heads, tensors))
        if tokens:
            positions = positions if positions.is_contiguous() else positions.contiguous()
            heads = _PAIR(*map(heads_of, tensors, outs))
            with on_device(index):
                rc = _native.load().kvssd_hip_rotary(
                    self._addresses[bool(inverse)], positions.data_ptr(), int(positions.dtype is torch.int64), tokens,
                    _DTYPES[dtype], ctypes.addressof(heads), len(tensors), current_stream_handle(index),
                )
            if rc:
                _native.check(rc, "kvssd_hip_rotary")
            if inplace:  # a graph that has saved them finds them changed, as after torch's own in-place operators
                for t in tensors:
                    torch.autograd.graph.increment_version(t)
        return outs[0] if key is None else outs
