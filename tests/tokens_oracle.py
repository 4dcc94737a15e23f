"""64-bit restatements, for tests, of attention over part of a paged cache -- windows with sinks, many tokens a sequence,
trees of drafted tokens -- and of keeping some of the drafted tokens, written from their definitions."""

from __future__ import annotations

import numpy as np

from paged_oracle import dequantise


def chain(parents, i: int) -> list[int]:
    """Token i and the tokens above it, nearest first."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(int(parents[out[-1]]))
    return out


def visible(length: int, count: int, parents, window: int, sink: int) -> np.ndarray:
    """bool [count, length]: whether a sequence's last `count` tokens see its slots (parents None: causal)."""
    base = length - count
    out = np.zeros((count, max(length, 0)), bool)
    for i in range(count):
        if parents is None:
            where = {t: t for t in range(max(base + i + 1, 0))}
            position = base + i
        else:
            up = chain(parents, i)
            position = base + len(up) - 1
            where = {t: t for t in range(max(base, 0))}
            where.update({base + a: position - k for k, a in enumerate(up) if base + a >= 0})
        for t, at in where.items():
            out[i, t] = not window or at > position - window or at < sink
    return out


def attend_tokens(query, pool, table, lengths, offsets, bits, scale, parents=None, window=0, sink=0) -> dict:
    """query [tokens, heads, d] in 64 bits; as paged_oracle.attend, `out`, `lse`, `size` and `reach`."""
    pk, pv, sk, sv = pool
    pages, page_tokens, kvh = pk.shape[:3]
    tokens, heads, d = query.shape
    gq = heads // kvh
    out, size = np.zeros(query.shape), np.zeros(query.shape)
    lse = np.full((tokens, heads), -np.inf)
    reach = 0.0
    for b, length in enumerate(lengths):
        length = max(0, min(int(length), table.shape[1] * page_tokens))
        begin, end = int(offsets[b]), int(offsets[b + 1])
        count = end - begin
        if count <= 0 or length == 0:
            continue
        seen = visible(length, count, None if parents is None else parents[begin:end], window, sink)
        page = table[b][np.arange(length) // page_tokens].astype(np.int64)
        held = (page >= 0) & (page < pages) & seen.any(0)
        rows = (page * page_tokens + np.arange(length) % page_tokens)[held]
        seen = seen[:, held]
        if not len(rows):
            continue
        for h in range(kvh):
            flat = [x.reshape(-1, kvh, x.shape[-1])[rows, h] for x in (pk, sk, pv, sv)]
            k, v = dequantise(flat[0], flat[1], bits), dequantise(flat[2], flat[3], bits)
            unit = np.repeat(np.abs(flat[1].astype(np.float64)), d // sk.shape[-1], axis=-1)
            for j in range(gq):
                q = query[begin:end, h * gq + j]
                for i in range(count):
                    if not seen[i].any():
                        continue
                    s = k[seen[i]] @ q[i] * scale
                    top = s.max()
                    p = np.exp(s - top)
                    lse[begin + i, h * gq + j] = top + np.log(p.sum())
                    p /= p.sum()
                    out[begin + i, h * gq + j], size[begin + i, h * gq + j] = p @ v[seen[i]], p @ np.abs(v[seen[i]])
                    if np.isfinite(q[i]).all():
                        unit_q = unit[seen[i]] @ np.abs(q[i])
                        reach = max(reach, float(2 * (64 if bits == 4 else 4) * unit_q.max() * abs(scale)))
    return dict(out=out, lse=lse, size=size, reach=reach)


def keep(pool, table, lengths, drafted, kept, weights=None, positions=None):
    """(pool, lengths, weights, positions) after the cut; rows are all taken before any is written."""
    pools = [x.copy() for x in pool]
    weights, positions = (None if x is None else x.copy() for x in (weights, positions))
    pages, page_tokens = pool[0].shape[:2]
    after = []
    for b, length in enumerate(lengths):
        length = max(0, min(int(length), table.shape[1] * page_tokens))
        n = max(0, min(int(drafted[b]), length))
        path = []
        for x in kept[b]:
            if x >= n or x <= (path[-1] if path else -1):
                break
            path.append(int(x))
        base = length - n

        def row(slot, b=b):
            page = int(table[b][slot // page_tokens])
            return page * page_tokens + slot % page_tokens if 0 <= page < pages else None

        for j, x in enumerate(path):
            to, frm = row(base + j), row(base + x)
            if to is not None and frm is not None:
                for new, old in zip(pools, pool):
                    new.reshape(-1, *new.shape[2:])[to] = old.reshape(-1, *old.shape[2:])[frm]
        if path:
            here = base + np.arange(len(path))
            for t in (weights, positions):
                if t is not None:
                    t[b, here] = t[b, base + np.array(path)].copy()
        after.append(base + len(path))
    return pools, np.array(after), weights, positions
