"""Performance cases of the generation operators: rotary positions, the paged packed cache and its upkeep.

Four operators, as a decode loop over many sequences uses them:

* ``rotary`` -- queries and keys rotated by their positions (half or interleaved pairs, all or part of the head,
  frequencies scaled for long contexts);
* ``append`` -- new tokens of every sequence, keys rotated, quantised into the pages that the sequences own (and
  their queries rotated in the same call);
* ``attend`` -- one new token's attention per sequence over its packed pages, ragged lengths, with or without adding
  each cached token's attention weight to a running sum;
* ``evict``  -- every sequence cut to a budget of tokens by that sum, the first and the latest positions kept.

``own`` false: elementary torch operations.  ``own`` true: the package's kernels.  ``exact``: 64 bits, written apart
from both.  Keys, values and queries are Gaussian; page tables name the pool's pages in random order.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / "kvssd-attention_amd") not in sys.path:
    sys.path.insert(0, str(ROOT / "kvssd-attention_amd"))

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# --------------------------------------------------------------------------- cases


def _rotary(name, tokens, qh, kvh, d, rdim, layout, dtype, scaling="none", factor=1.0, base=10000.0, far=0):
    return dict(name=name, kind="rotary", tokens=tokens, qh=qh, kvh=kvh, d=d, rdim=rdim, layout=layout, dtype=dtype,
                scaling=scaling, factor=factor, base=base, far=far)


def _append(name, seqs, total, longest, qh, kvh, d, g, bt, bits, dtype, rdim, layout, filled):
    return dict(name=name, kind="append", seqs=seqs, total=total, longest=longest, qh=qh, kvh=kvh, d=d, g=g, bt=bt,
                bits=bits, dtype=dtype, rdim=rdim, layout=layout, scaling="none", factor=1.0, base=10000.0, filled=filled)


def _attend(name, seqs, shortest, longest, qh, kvh, d, g, bt, bits, dtype, weights=False):
    return dict(name=name, kind="attend", seqs=seqs, shortest=shortest, longest=longest, qh=qh, kvh=kvh, d=d, g=g, bt=bt,
                bits=bits, dtype=dtype, weights=weights)


def _evict(name, seqs, shortest, longest, budget, sink, recent, kvh, d, g, bt, bits, steady):
    return dict(name=name, kind="evict", seqs=seqs, shortest=shortest, longest=longest, budget=budget, sink=sink,
                recent=recent, kvh=kvh, d=d, g=g, bt=bt, bits=bits, steady=steady)


def listed():
    return [
        # one new token of 64 sequences, far into a context whose frequencies are stretched by parts
        _rotary("rotary_step", 64, 32, 8, 128, 128, "half", "bf16", "yarn", 4.0, 10000.0, 120000),
        # a prompt of the benchmark's model shape
        _rotary("rotary_prompt_8k", 8192 - 5, 32, 8, 128, 128, "half", "bf16", "none", 1.0, 500000.0, 0),
        # interleaved pairs over a quarter of a large head, an odd number of tokens, linear scaling, far positions
        _rotary("rotary_part_d256", 4099, 24, 4, 256, 64, "interleaved", "f16", "linear", 8.0, 10000.0, 1000000),
        # one new token of 64 sequences into INT4 pages of 64 tokens, its query rotated along
        _append("append_step", 64, 64, 1, 32, 8, 128, 32, 64, 4, "bf16", 128, "half", 4000),
        # four prompts of different lengths into fresh pages of 128 tokens
        _append("append_prompt_16k", 4, 16384 - 3, 8000, 0, 8, 128, 32, 128, 4, "bf16", 128, "half", 0),
        # a chunk of each of 8 sequences in INT2, small heads, pages that end inside a tile, 32-bit inputs
        _append("append_int2_d64", 8, 4097, 1024, 16, 4, 64, 32, 24, 2, "f32", 32, "interleaved", 1000),
        # the shortest context of the benchmark, one sequence: launches and round trips
        _attend("attend_4k", 1, 4096, 4096, 32, 8, 128, 32, 128, 4, "f16"),
        # a serving batch of ragged lengths in pages of 64 tokens
        _attend("attend_batch64", 64, 1, 16384, 32, 8, 128, 32, 64, 4, "bf16"),
        # four long contexts
        _attend("attend_long", 4, 131072 - 77, 262144, 32, 8, 128, 32, 128, 4, "f16"),
        # INT2, 8 query heads per kv head, weights summed for eviction
        _attend("attend_int2_weights", 16, 2000, 16384, 64, 8, 128, 32, 32, 2, "bf16", True),
        # the regular cut of a running batch: one page's worth of tokens over the budget
        _evict("evict_step", 64, 4096 + 1, 4096 + 64, 4096, 4, 512, 8, 128, 32, 64, 4, True),
        # long prompts cut to an eighth
        _evict("evict_prompt", 4, 65536 + 9, 131072, 16384, 4, 2048, 8, 128, 32, 128, 4, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "evict"])
    d = rng.choice([64, 96, 128, 128, 128, 256])
    g = rng.choice([x for x in (32, 32, 64, 128) if d % x == 0])
    kvh = rng.choice([1, 2, 3, 4, 8, 8, 8, 16])
    qh = kvh * rng.choice([1, 2, 4, 4, 5, 8, 16])
    bits = rng.choice([4, 4, 2])
    bt = rng.choice([16, 24, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    layout = rng.choice(["half", "interleaved"])
    rdim = rng.choice([d, d, d // 2, d // 4, 20])
    if kind == "rotary":
        tokens = _log_int(rng, 1, max(2, min(16384, (1 << 26) // ((qh + kvh) * d))))
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "wavelength"])
        return dict(kind=kind, tokens=tokens, qh=qh, kvh=kvh, d=d, rdim=rdim, layout=layout, dtype=dtype, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                    base=rng.choice([10000.0, 500000.0]), far=_log_int(rng, 1, 1 << 20))
    if kind == "append":
        seqs = _log_int(rng, 1, 128)
        total = seqs if rng.random() < 0.5 else max(seqs, _log_int(rng, 16, max(32, min(16384, (1 << 24) // (kvh * d)))))
        return dict(kind=kind, seqs=seqs, total=total, longest=max(1, min(total, 3 * total // seqs + 1)),
                    qh=rng.choice([0, qh]), kvh=kvh, d=d, g=g, bt=bt, bits=bits, dtype=dtype, rdim=rdim, layout=layout,
                    scaling="none", factor=1.0, base=10000.0, filled=rng.choice([0, rng.randint(1, 3000)]))
    if kind == "attend":
        # at most a quarter of the largest listed case's cache, whatever the shape
        room = 150000000 // (kvh * (2 * d * bits // 8 + 4 * d // g))
        longest = _log_int(rng, 1, min(131072, room))
        seqs = _log_int(rng, 1, max(2, min(128, room // longest)))
        return dict(kind=kind, seqs=seqs, shortest=rng.choice([0, 1, longest]), longest=longest, qh=qh, kvh=kvh, d=d, g=g,
                    bt=bt, bits=bits, dtype=dtype, weights=rng.choice([False, True]))
    longest = _log_int(rng, 40, 65536)
    seqs = _log_int(rng, 1, max(2, min(64, 131072 // longest)))
    budget = rng.randint(max(8, longest // 8), longest)
    return dict(kind=kind, seqs=seqs, shortest=rng.choice([0, budget, longest]), longest=longest, budget=budget, sink=rng.choice([0, 4]),
                recent=rng.randint(0, budget - 4), kvh=kvh, d=d, g=g, bt=bt, bits=bits, steady=rng.choice([False, True]))


# --------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 11)


def _host_generator(seed):
    return torch.Generator().manual_seed(1000003 * seed + 17)


def _normal(gen, shape, dtype, factor=1.0):
    return (factor * torch.randn(shape, generator=gen, device="cuda")).to(dtype)


def _frequencies(case):
    """(angle per position of each pair, factor of the rotated values), as Python floats."""
    r, base, factor = case["rdim"], case["base"], case["factor"]
    original = 8192  # positions that the unscaled frequencies were made for
    kind = case["scaling"]
    if kind == "ntk":
        base = base * factor ** (r / (r - 2))
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    magnitude = 1.0
    if kind == "linear":
        f = [x / factor for x in f]
    if kind == "yarn":
        def pair_of(turns):
            return r * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), r - 1)
        high = high if high > low else low + 0.001
        ramp = [min(max((i - low) / (high - low), 0.0), 1.0) for i in range(r // 2)]
        f = [x / factor * t + x * (1.0 - t) for x, t in zip(f, ramp)]
        magnitude = 0.1 * math.log(factor) + 1.0
    if kind == "wavelength":
        low, high, scaled = 1.0, 4.0, []
        for x in f:
            turns = original * x / (2 * math.pi)
            t = min(max((turns - low) / (high - low), 0.0), 1.0)
            scaled.append((1.0 - t) * x / factor + t * x)
        f = scaled
    return f, magnitude


def _lengths(case, gen):
    """Lengths from ``shortest`` to ``longest``, spread over their logarithm; both ends occur."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    u = torch.rand((n,), generator=gen, dtype=torch.float64)
    at = torch.exp(math.log(max(lo, 1)) + u * (math.log(max(hi, 1)) - math.log(max(lo, 1)))).round().long()
    at[0] = hi
    if n > 1:
        at[1] = lo
    return at[torch.randperm(n, generator=gen)].clamp(0, hi)


def _page_table(pages_of, width, pool, gen):
    """int32 [seqs, width]: each sequence's pages, drawn from the pool in random order; -1 behind them."""
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    owned = torch.arange(width)[None, :] < pages_of[:, None]
    table = torch.full(owned.shape, -1, dtype=torch.int32)
    table[owned] = order[: int(owned.sum())]
    return table


def _pool(case, gen, pool):
    """Packed keys and values of every page, with scales of Gaussian values' size."""
    bt, kvh, d, g, bits = case["bt"], case["kvh"], case["d"], case["g"], case["bits"]
    out = []
    for _ in range(2):
        codes = torch.randint(0, 256, (pool, bt, kvh, d * bits // 8), generator=gen, device="cuda", dtype=torch.uint8)
        spread = torch.rand((pool, bt, kvh, d // g), generator=gen, device="cuda")
        out += [codes, ((0.25 + 0.15 * spread) * (1.0 if bits == 4 else 4.0)).to(torch.float16)]
    return out[0], out[2], out[1], out[3]


def _inputs(case, seed):
    """Every tensor of a case, on the GPU, and the lengths that a user's program knows on the host."""
    gen, host = _generator(seed), _host_generator(seed)
    kind = case["kind"]
    s = dict(case=case)
    if kind in ("rotary", "append"):
        f, s["magnitude"] = _frequencies(case)
        s["frequencies"] = torch.tensor(f, dtype=torch.float64).cuda()
    if kind == "rotary":
        dtype = DTYPES[case["dtype"]]
        s["query"] = _normal(gen, (case["tokens"], case["qh"], case["d"]), dtype)
        s["key"] = _normal(gen, (case["tokens"], case["kvh"], case["d"]), dtype)
        s["positions"] = (case["far"] + torch.randperm(case["tokens"], generator=host)).cuda()
        return s
    bt = case["bt"]
    if kind == "append":
        dtype = DTYPES[case["dtype"]]
        n, total = case["seqs"], case["total"]
        if total == n:
            counts = torch.ones(n, dtype=torch.long)
            s["offsets"] = None
        else:
            counts = (torch.rand(n, generator=host) * case["longest"]).long()
            counts = (counts * total // max(int(counts.sum()), 1)).clamp(0, total)
            counts[-1] += total - int(counts.sum())
            s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32).cuda()
        lengths = (torch.rand(n, generator=host) * (case["filled"] + 1)).long()
        after = lengths + counts
        first = lengths + torch.randint(0, 100, (n,), generator=host)  # tokens before these were evicted
        s["key"] = _normal(gen, (total, case["kvh"], case["d"]), dtype)
        s["value"] = _normal(gen, (total, case["kvh"], case["d"]), dtype)
        s["query"] = _normal(gen, (total, case["qh"], case["d"]), dtype) if case["qh"] else None
        s["first"] = first.to(torch.int32).cuda()
    else:
        lengths = after = _lengths(case, host)
    pages_of = (after + bt - 1) // bt
    # as many pages whatever the seed: outputs hold the whole pool where it is written
    width = int(pages_of.max().clamp(min=1))
    pool = int(pages_of.sum()) + 3
    if kind == "append":
        width = (case["filled"] + case["total"]) // bt + 1
        pool = (case["seqs"] * case["filled"] + case["total"]) // bt + case["seqs"] + 3
    if kind == "evict":
        pool = case["seqs"] * width + 3
    s["table"] = _page_table(pages_of, width, pool, host).cuda()
    s["lengths"] = lengths.to(torch.int32).cuda()
    s["longest"], s["all_tokens"] = int(lengths.max()), int(lengths.sum())
    s["pk"], s["pv"], s["sk"], s["sv"] = _pool(case, gen, pool)
    capacity = width * bt
    if kind == "attend":
        # scaled scores of standard deviation about 2: attention that picks out some tokens
        s["query"] = _normal(gen, (case["seqs"], case["qh"], case["d"]), DTYPES[case["dtype"]], 1.5)
        s["weights"] = torch.rand((case["seqs"], capacity), generator=gen, device="cuda") if case["weights"] else None
    if kind == "evict":
        # sums of attention weights: heavy-tailed, some exactly zero
        w = torch.exp(2 * torch.randn((case["seqs"], capacity), generator=gen, device="cuda"))
        s["weights"] = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.1, 0.0, w)
        slots = torch.arange(capacity, device="cuda").expand(case["seqs"], -1)
        if case["steady"]:  # after earlier cuts: positions with gaps, in no order
            used = slots < s["lengths"][:, None]
            keys = torch.where(used, torch.rand(w.shape, generator=gen, device="cuda"), 2.0)
            slots = 3 * keys.argsort(dim=1).argsort(dim=1)
        s["positions"] = slots.to(torch.int32).contiguous()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from kvssd.backends import PagedBatch, resolve_attention_backend
        from kvssd.rotary import Rotary, RotaryScaling

        if "frequencies" in s:
            scaling = None
            if case["scaling"] != "none":
                scaling = RotaryScaling(case["scaling"], case["factor"], original_positions=8192)
            s["rotary"] = Rotary(case["d"], rotary_dim=case["rdim"], base=case["base"], layout=case["layout"],
                                 scaling=scaling, device="cuda")
        if "table" in s:
            s["batch"] = PagedBatch(s["pk"], s["pv"], s["sk"], s["sv"], s["table"], s["lengths"], case["bits"], case["g"],
                                    weights=s.get("weights"), positions=s.get("positions"))
        if case["kind"] == "attend":
            backend = resolve_attention_backend("hip", s["query"].device)
            s["decode"] = backend.prepare_paged(s["query"], s["batch"], _scale(case), out_dtype=s["query"].dtype,
                                                accumulate=case["weights"], max_length=s["longest"],
                                                total_tokens=s["all_tokens"])
    return s


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


# --------------------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "attend": _own_attend, "evict": _own_evict}[kind](state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[kind](state)


def _own_rotary(s):
    return s["rotary"](s["positions"], s["query"], s["key"])


def _own_append(s):
    from kvssd.paged import append_tokens

    query, lengths = append_tokens(s["batch"], s["key"], s["value"], offsets=s["offsets"], rotary=s["rotary"],
                                   query=s["query"], first_positions=s["first"])
    return dict(query=query, lengths=lengths, pk=s["pk"], pv=s["pv"], sk=s["sk"], sv=s["sv"])


def _own_attend(s):
    out, lse = s["decode"](s["query"])
    return dict(out=out, lse=lse, weights=s["weights"])


def _own_evict(s):
    from kvssd.paged import evict_tokens

    c = s["case"]
    lengths, weights, positions = evict_tokens(s["batch"], c["budget"], sink=c["sink"], recent=c["recent"])
    return dict(lengths=lengths, weights=weights, positions=positions, pk=s["pk"], pv=s["pv"], sk=s["sk"], sv=s["sv"])


def _turn(x, positions, s):
    """``x`` [tokens, heads, d] rotated: in 64 bits, since the angles of far positions and keys next to the border
    of two codes need them, rounded once to x's type."""
    c = s["case"]
    r = c["rdim"]
    angle = positions.double()[:, None] * s["frequencies"]
    cos, sin = (s["magnitude"] * torch.cos(angle))[:, None], (s["magnitude"] * torch.sin(angle))[:, None]
    y = x.double()
    a, b = (y[..., : r // 2], y[..., r // 2:r]) if c["layout"] == "half" else (y[..., 0:r:2], y[..., 1:r:2])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((lo, hi), -1) if c["layout"] == "half" else torch.stack((lo, hi), -1).flatten(-2)
    return torch.cat((turned, y[..., r:]), -1).to(x.dtype)


def _plain_rotary(s):
    return _turn(s["query"], s["positions"], s), _turn(s["key"], s["positions"], s)


def _coded(x, bits, g):
    """(codes packed low bits first, fp16 scales) of groups of ``g`` values: scale = max|x| / (2^(bits-1) - 1)."""
    mid = 1 << (bits - 1)
    groups = x.float().unflatten(-1, (-1, g))
    amax = groups.abs().amax(-1).clamp_min(1e-8)
    scale = amax / torch.full_like(amax, mid - 1)
    codes = (torch.round(groups / scale[..., None]).clamp(-mid, mid - 1) + mid).to(torch.uint8).flatten(-2)
    lanes = codes.unflatten(-1, (-1, 8 // bits)).long() << torch.arange(0, 8, bits, device=x.device)
    return lanes.sum(-1).to(torch.uint8), scale.to(torch.float16)


def _places(s):
    """(flat row of the pool that each new token goes to, its position, lengths after)."""
    c = s["case"]
    n, total, bt = c["seqs"], c["total"], c["bt"]
    token = torch.arange(total, device="cuda")
    if s["offsets"] is None:
        seq, nth, after = token, torch.zeros_like(token), s["lengths"] + 1
    else:
        seq = torch.searchsorted(s["offsets"].long(), token, right=True) - 1
        nth, after = token - s["offsets"].long()[seq], s["lengths"] + s["offsets"].diff()
    slot = s["lengths"].long()[seq] + nth
    row = s["table"].long()[seq, slot // bt] * bt + slot % bt
    return row, s["first"].long()[seq] + nth, after


def _plain_append(s):
    c = s["case"]
    row, position, after = _places(s)
    key = _turn(s["key"], position, s)
    for x, packed, scales in ((key, s["pk"], s["sk"]), (s["value"], s["pv"], s["sv"])):
        codes, scale = _coded(x, c["bits"], c["g"])
        packed.flatten(0, 1)[row] = codes
        scales.flatten(0, 1)[row] = scale
    query = None if s["query"] is None else _turn(s["query"], position, s)
    return dict(query=query, lengths=after, pk=s["pk"], pv=s["pv"], sk=s["sk"], sv=s["sv"])


def _values_of(packed, scales, pages, c):
    """fp32 [seqs, tokens, kvh, d] of the pages [seqs, n]."""
    bits = c["bits"]
    bytes_of = packed[pages].flatten(1, 2)
    codes = (bytes_of[..., None] >> torch.arange(0, 8, bits, device="cuda", dtype=torch.uint8)) & ((1 << bits) - 1)
    codes = codes.flatten(-2).float() - (1 << (bits - 1))
    return (codes.unflatten(-1, (-1, c["g"])) * scales[pages].flatten(1, 2).float()[..., None]).flatten(-2)


def _plain_attend(s):
    c = s["case"]
    n, kvh, d = c["seqs"], c["kvh"], c["d"]
    pages = s["table"].clamp(min=0).long()
    query = s["query"].float().view(n, kvh, -1, d)
    k = _values_of(s["pk"], s["sk"], pages, c).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(query, k) * _scale(c)  # [seqs, kvh, heads, tokens]
    del k
    used = torch.arange(scores.shape[-1], device="cuda") < s["lengths"][:, None]
    scores = scores.masked_fill(~used[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    v = _values_of(s["pv"], s["sv"], pages, c).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(p, v).reshape(n, -1, d).to(s["query"].dtype)
    lse = (torch.log(total) + top).reshape(n, -1)
    if s["weights"] is not None:
        s["weights"] += p.sum((1, 2))
    return dict(out=out, lse=lse, weights=s["weights"])


def _plain_evict(s):
    c = s["case"]
    bt, budget = c["bt"], c["budget"]
    weights, positions, lengths = s["weights"], s["positions"], s["lengths"].long()[:, None]
    slots = torch.arange(weights.shape[1], device="cuda").expand_as(weights)
    used = slots < lengths
    latest = positions.masked_fill(~used, -1).amax(1, keepdim=True)
    held = (positions < c["sink"]) | (positions > latest - c["recent"])
    order = torch.where(held, math.inf, weights).masked_fill(~used, -math.inf)
    rank = order.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    kept = (rank < budget) & used
    after = lengths.clamp(max=budget)
    # the n-th kept token behind the budget goes to the n-th free slot before it
    behind, free = kept & (slots >= budget), ~kept & (slots < after)
    nth = torch.where(free, free.cumsum(1) - 1, 0)
    source = torch.where(behind, slots, weights.shape[1]).sort(dim=1).values
    source = torch.where(free, source.gather(1, nth), slots)
    live = slots < after
    new_weights = torch.where(live, weights.gather(1, source), 0.0)
    new_positions = torch.where(live, positions.gather(1, source), -1)
    seq, to = free.nonzero(as_tuple=True)
    frm = source[seq, to]
    page = s["table"].long()
    row_to = page[seq, to // bt] * bt + to % bt
    row_from = page[seq, frm // bt] * bt + frm % bt
    for pool in (s["pk"], s["pv"], s["sk"], s["sv"]):
        flat = pool.flatten(0, 1)
        flat[row_to] = flat[row_from]
    return dict(lengths=after[:, 0].to(torch.int32), weights=new_weights, positions=new_positions, pk=s["pk"], pv=s["pv"],
                sk=s["sk"], sv=s["sv"])


# --------------------------------------------------------------------------- work, exact results


def work(case):
    kind = case["kind"]
    item = 4 if case.get("dtype") == "f32" else 2
    if kind == "rotary":
        n = case["tokens"] * (case["qh"] + case["kvh"])
        return {"bytes": 2 * n * case["d"] * item + 8 * case["tokens"], "flops": 3 * n * case["rdim"]}
    kvh, d = case["kvh"], case["d"]
    per_token = kvh * (2 * d * case["bits"] // 8 + 4 * (d // case["g"]))  # packed K and V with their scales
    if kind == "append":
        n = case["total"]
        return {"bytes": n * (2 * (kvh + case["qh"]) * d * item + per_token),
                "flops": n * (3 * (kvh + case["qh"]) * case["rdim"] + 6 * kvh * d)}
    if kind == "attend":
        # the mean of lengths spread over their logarithm
        lo, hi = max(case["shortest"], 1), max(case["longest"], 1)
        n = case["seqs"] * (hi if hi == lo else (hi - lo) / math.log(hi / lo))
        n += 0 if case["seqs"] > 1 else hi - n
        return {"bytes": n * (per_token + (8 if case["weights"] else 0)) + case["seqs"] * case["qh"] * (2 * d * item + 4),
                "flops": 4 * n * case["qh"] * d}
    lo, hi, budget = max(case["shortest"], 1), max(case["longest"], 1), case["budget"]
    n = hi if hi == lo or case["seqs"] == 1 else (hi - lo) / math.log(hi / lo)
    moved = budget * max(n - budget, 0) / max(n, 1)  # kept tokens that lie behind the budget, of evenly spread ones
    return {"bytes": case["seqs"] * (16 * n + 2 * moved * per_token), "flops": case["seqs"] * n}


def _exact_turn(x, positions, s):
    """Pairs as complex numbers times unit ones, in 64 bits."""
    c = s["case"]
    r = c["rdim"]
    unit = torch.polar(torch.full_like(positions.double()[:, None] * s["frequencies"], s["magnitude"]),
                       positions.double()[:, None] * s["frequencies"])[:, None]
    y = x.double().clone()
    if c["layout"] == "half":
        z = torch.complex(y[..., : r // 2].contiguous(), y[..., r // 2:r].contiguous()) * unit
        y[..., : r // 2], y[..., r // 2:r] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:r:2].contiguous(), y[..., 1:r:2].contiguous()) * unit
        y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
    return y


def _exact_append(s):
    """Sequence by sequence; the cache's scales in 64 bits, its codes from them as they are defined (keys are coded
    in their own type, scales with 24 bits)."""
    c = s["case"]
    lengths = s["lengths"].tolist()
    ends = list(range(c["seqs"] + 1)) if s["offsets"] is None else s["offsets"].tolist()
    first, table = s["first"].tolist(), s["table"].tolist()
    mid, bits, g, bt = 1 << (c["bits"] - 1), c["bits"], c["g"], c["bt"]
    pools = [t.clone() for t in (s["pk"], s["pv"])] + [t.double() for t in (s["sk"], s["sv"])]
    queries = []
    for b in range(c["seqs"]):
        count = ends[b + 1] - ends[b]
        if not count:
            continue
        span = slice(ends[b], ends[b + 1])
        position = first[b] + torch.arange(count, device="cuda")
        if s["query"] is not None:
            queries.append(_exact_turn(s["query"][span], position, s))
        key = _exact_turn(s["key"][span], position, s).to(s["key"].dtype)
        rows = torch.tensor([table[b][t // bt] * bt + t % bt for t in range(lengths[b], lengths[b] + count)], device="cuda")
        for x, packed, scales in ((key, pools[0], pools[2]), (s["value"][span], pools[1], pools[3])):
            groups = x.double().reshape(count, c["kvh"], -1, g)
            top = groups.abs().amax(-1).clamp_min(float(torch.tensor(1e-8)))
            step = (top / (mid - 1)).float().double()
            code = (groups / step[..., None]).float().double().round().clamp(-mid, mid - 1) + mid
            code = code.reshape(count, c["kvh"], -1, 8 // bits).long()
            byte = sum(code[..., i] << (bits * i) for i in range(8 // bits))
            packed.view(-1, *packed.shape[2:])[rows] = byte.to(torch.uint8)
            scales.view(-1, *scales.shape[2:])[rows] = top / (mid - 1)
    after = s["lengths"] + (torch.ones_like(s["lengths"]) if s["offsets"] is None else s["offsets"].diff())
    return dict(query=torch.cat(queries) if queries else None, lengths=after, pk=pools[0], pv=pools[1], sk=pools[2], sv=pools[3])


def _exact_attend(s, chunk=16384):
    c = s["case"]
    kvh, d, g, bits, bt = c["kvh"], c["d"], c["g"], c["bits"], c["bt"]
    shift = torch.arange(0, 8, bits, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    outs, lses = [], []

    def rows_of(packed, scales, rows):
        byte = packed.view(-1, kvh, d * bits // 8)[rows].long()
        code = ((byte[..., None] >> shift) % (1 << bits)).reshape(len(rows), kvh, d // g, g).double() - (1 << (bits - 1))
        return (code * scales.view(-1, kvh, d // g)[rows].double()[..., None]).reshape(len(rows), kvh, d)

    for b, length in enumerate(s["lengths"].tolist()):
        q = s["query"][b].double().view(kvh, -1, d)
        if not length:
            outs.append(torch.zeros_like(q).view(-1, d))
            lses.append(torch.full((q.shape[0] * q.shape[1],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        slot = torch.arange(length, device="cuda")
        rows = s["table"][b].long()[slot // bt] * bt + slot % bt
        spans = rows.split(chunk)
        score = [torch.matmul(q, rows_of(s["pk"], s["sk"], r).permute(1, 2, 0).contiguous()) for r in spans]
        score = torch.cat(score, -1) / math.sqrt(d)
        lse = torch.logsumexp(score, -1)
        p = torch.exp(score - lse[..., None])
        out = torch.zeros_like(q)
        for r, w in zip(spans, p.split(chunk, -1)):
            out += torch.matmul(w.contiguous(), rows_of(s["pv"], s["sv"], r).permute(1, 0, 2).contiguous())
        if weights is not None:
            weights[b, :length] += p.sum((0, 1))
        outs.append(out.view(-1, d))
        lses.append(lse.view(-1))
    return dict(out=torch.stack(outs), lse=torch.stack(lses), weights=weights)


def _exact_evict(s):
    """Sequence by sequence, on the host."""
    c = s["case"]
    lengths, table = s["lengths"].tolist(), s["table"].tolist()
    weights, positions = s["weights"].cpu(), s["positions"].cpu()
    new_weights, new_positions = torch.zeros_like(weights, dtype=torch.float64), torch.full_like(positions, -1)
    pools = [t.clone().flatten(0, 1) for t in (s["pk"], s["pv"], s["sk"], s["sv"])]
    after, bt = [], c["bt"]
    for b, n in enumerate(lengths):
        w, p = weights[b, :n].tolist(), positions[b, :n].tolist()
        latest = max(p, default=-1)
        order = sorted(range(n), key=lambda i: (not (p[i] < c["sink"] or p[i] > latest - c["recent"]), 0.0 if (
            p[i] < c["sink"] or p[i] > latest - c["recent"]) else -w[i], i))
        kept = set(order[: c["budget"]])
        m = min(n, c["budget"])
        place = {i: i for i in kept if i < m}
        free = [i for i in range(m) if i not in kept]
        place.update(zip(free, sorted(i for i in kept if i >= m)))
        at = [place[i] for i in range(m)]
        new_weights[b, :m] = weights[b, :n].double()[at]
        new_positions[b, :m] = positions[b, :n][at]
        if free:
            to = torch.tensor([table[b][i // bt] * bt + i % bt for i in free], device="cuda")
            frm = torch.tensor([table[b][place[i] // bt] * bt + place[i] % bt for i in free], device="cuda")
            for pool in pools:
                pool[to] = pool[frm]
        after.append(m)
    shape = s["pk"].shape[:2]
    pools = [t.unflatten(0, shape) for t in pools]
    return dict(lengths=torch.tensor(after, dtype=torch.int32), weights=new_weights, positions=new_positions, pk=pools[0],
                pv=pools[1], sk=pools[2].double(), sv=pools[3].double())


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _exact_turn(s["query"], s["positions"], s), _exact_turn(s["key"], s["positions"], s)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["kind"]](s)
