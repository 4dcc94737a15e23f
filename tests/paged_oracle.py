"""64-bit restatements of the generation operators, for tests: rotary positions, the codec over rotated keys, paged
attention and eviction, written from their definitions (numpy, one sequence and one token at a time)."""

from __future__ import annotations

import math

import numpy as np
import torch


def frequencies(r: int, base: float = 10000.0) -> np.ndarray:
    return np.array([base ** (-2.0 * i / r) for i in range(r // 2)])


def rotate(x: np.ndarray, positions: np.ndarray, freq: np.ndarray, interleaved: bool, magnitude: float = 1.0,
           inverse: bool = False) -> np.ndarray:
    """x [tokens, heads, d] in 64 bits."""
    y = x.astype(np.float64).copy()
    r = 2 * len(freq)
    angle = positions.astype(np.float64)[:, None] * freq[None, :] * (-1.0 if inverse else 1.0)
    c, s = magnitude * np.cos(angle)[:, None, :], magnitude * np.sin(angle)[:, None, :]
    low, high = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = y[..., low].copy(), y[..., high].copy()
    y[..., low], y[..., high] = a * c - b * s, b * c + a * s
    return y


def dequantise(packed: np.ndarray, scales: np.ndarray, bits: int) -> np.ndarray:
    """[..., d] in 64 bits of codes [..., d*bits/8] and fp16 scales [..., d/g]."""
    codes = np.stack([(packed >> (bits * i)) & ((1 << bits) - 1) for i in range(8 // bits)], axis=-1)
    codes = codes.reshape(*packed.shape[:-1], -1).astype(np.float64) - (1 << (bits - 1))
    return codes * np.repeat(scales.astype(np.float64), codes.shape[-1] // scales.shape[-1], axis=-1)


def rows_of(table: np.ndarray, length: int, page_tokens: int, pages: int) -> tuple[np.ndarray, np.ndarray]:
    """(slots that lie in a page, their rows in the pool)."""
    length = max(0, min(length, len(table) * page_tokens))
    slots = np.arange(length)
    page = table[slots // page_tokens].astype(np.int64)
    ok = (page >= 0) & (page < pages)
    slots, page = slots[ok], page[ok]
    return slots, page * page_tokens + slots % page_tokens


def attend(query: np.ndarray, pool, table, lengths, bits: int, scale: float, weights: np.ndarray | None = None) -> dict:
    """query [sequences, heads, d]; pool (packed_k, packed_v, scales_k, scales_v).  Returns out, lse, weights and what
    tolerances need: size (sum_t p_t |v_t|, as out) and reach (the largest sum_d |q_d k_d| scale of any score)."""
    pk, pv, sk, sv = pool
    pages, page_tokens, kvh = pk.shape[:3]
    n, heads, d = query.shape
    out, size = np.zeros(query.shape), np.zeros(query.shape)
    lse = np.full((n, heads), -np.inf)
    weights = None if weights is None else weights.astype(np.float64).copy()
    reach = 0.0
    for b in range(n):
        slots, rows = rows_of(table[b], int(lengths[b]), page_tokens, pages)
        if not len(slots):
            continue
        k = dequantise(pk.reshape(-1, kvh, pk.shape[-1])[rows], sk.reshape(-1, kvh, sk.shape[-1])[rows], bits)
        v = dequantise(pv.reshape(-1, kvh, pv.shape[-1])[rows], sv.reshape(-1, kvh, sv.shape[-1])[rows], bits)
        for h in range(heads):
            kh, vh = k[:, h // (heads // kvh)], v[:, h // (heads // kvh)]
            q = query[b, h].astype(np.float64)
            s = kh @ q * scale
            top = s.max()
            p = np.exp(s - top)
            lse[b, h] = top + math.log(p.sum())
            p /= p.sum()
            out[b, h], size[b, h] = p @ vh, p @ np.abs(vh)
            # |code offset| + |code| of a 32-bit sum of 1 + c/F numbers: at most 2 F per scale unit
            unit = np.repeat(np.abs(sk.reshape(-1, kvh, sk.shape[-1])[rows][:, h // (heads // kvh)].astype(np.float64)),
                             d // sk.shape[-1], axis=-1)
            if np.isfinite(q).all():
                reach = max(reach, float((2 * (64 if bits == 4 else 4) * unit @ np.abs(q)).max() * scale))
            if weights is not None:
                weights[b, slots] += p
    return dict(out=out, lse=lse, weights=weights, size=size, reach=reach)


def evict(weights: np.ndarray, positions: np.ndarray, length: int, budget: int, sink: int, recent: int) -> list[int]:
    """Source slot of each slot after the cut, for one sequence."""
    w, p = weights[:length].astype(np.float64), positions[:length].astype(np.int64)
    w = np.where(np.isnan(w), -np.inf, w)
    latest = p.max(initial=-(1 << 40))
    held = (p < sink) | (p > latest - recent)
    order = sorted(range(length), key=lambda i: (not held[i], 0.0 if held[i] else -w[i], i))
    kept = set(order[:budget])
    m = min(length, budget)
    free = [i for i in range(m) if i not in kept]
    place = dict(zip(free, sorted(i for i in kept if i >= m)))
    return [place.get(i, i) for i in range(m)]


def make_pool(rng, pages, page_tokens, kvh, d, g, bits, scale=(0.2, 0.5)):
    """Random (packed_k, packed_v, scales_k, scales_v) as numpy arrays."""
    out = []
    for _ in range(2):
        out.append(rng.integers(0, 256, (pages, page_tokens, kvh, d * bits // 8), dtype=np.uint8))
        out.append(rng.uniform(*scale, (pages, page_tokens, kvh, d // g)).astype(np.float16))
    return out[0], out[2], out[1], out[3]


def make_table(rng, lengths, page_tokens, width, pages) -> np.ndarray:
    """int32 [sequences, width]: pages in random order, -1 behind the last."""
    order = rng.permutation(pages)
    table = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, n in enumerate(lengths):
        need = -(-int(n) // page_tokens)
        table[b, :need] = order[at:at + need]
        at += need
    assert at <= pages
    return table


def as_double(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()
