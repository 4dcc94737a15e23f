"""Performance cases of attention over part of a paged packed cache, and of drafted tokens in it.

Four kinds, as a serving loop with long contexts and speculative decoding uses them:

* ``step``   -- one new token's attention per sequence over the last ``window`` slots and the first ``sink``;
* ``prompt`` -- many new tokens of each sequence at once (whole prompts, or chunks behind a context), causal, with or
  without a window and sinks;
* ``tree``   -- drafted tokens, each of which sees its sequence's context and its own ancestors among them;
* ``keep``   -- the accepted ones of the drafted tokens moved together, the others dropped.

``own`` false: elementary torch operations.  ``own`` true: the package's kernels.  ``exact``: 64 bits, written apart
from both.  Keys, values and queries are Gaussian; page tables name the pool's pages in random order; the new tokens'
keys and values lie in the cache already.
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


def _step(name, seqs, shortest, longest, window, sink, qh, kvh, d, g, bt, bits, dtype):
    return dict(name=name, kind="step", seqs=seqs, shortest=shortest, longest=longest, window=window, sink=sink, qh=qh,
                kvh=kvh, d=d, g=g, bt=bt, bits=bits, dtype=dtype)


def _prompt(name, seqs, total, shortest, longest, window, sink, qh, kvh, d, g, bt, bits, dtype):
    return dict(name=name, kind="prompt", seqs=seqs, total=total, shortest=shortest, longest=longest, window=window,
                sink=sink, qh=qh, kvh=kvh, d=d, g=g, bt=bt, bits=bits, dtype=dtype)


def _tree(name, seqs, nodes, ragged, shortest, longest, window, sink, qh, kvh, d, g, bt, bits, dtype):
    return dict(name=name, kind="tree", seqs=seqs, nodes=nodes, ragged=ragged, shortest=shortest, longest=longest,
                window=window, sink=sink, qh=qh, kvh=kvh, d=d, g=g, bt=bt, bits=bits, dtype=dtype)


def _keep(name, seqs, nodes, ragged, deepest, shortest, longest, kvh, d, g, bt, bits, tracked):
    return dict(name=name, kind="keep", seqs=seqs, nodes=nodes, ragged=ragged, deepest=deepest, shortest=shortest,
                longest=longest, kvh=kvh, d=d, g=g, bt=bt, bits=bits, tracked=tracked)


def listed():
    return [
        # one sequence, a short window: launches and round trips
        _step("step_one", 1, 16384, 16384, 1024, 4, 32, 8, 128, 32, 128, 4, "f16"),
        # a serving batch of ragged lengths, some shorter than the window
        _step("step_batch64", 64, 1, 16384, 4096, 4, 32, 8, 128, 32, 64, 4, "bf16"),
        # long contexts of which an eighth stays visible, INT2, sinks of a whole page
        _step("step_long_int2", 32, 65536 + 9, 131072, 16384, 64, 32, 8, 128, 32, 64, 2, "f16"),
        # a prompt of the benchmark's model shape through a layer with a window
        _prompt("prompt_window_8k", 1, 8192 - 5, 0, 0, 1024, 4, 32, 8, 128, 32, 64, 4, "bf16"),
        # chunks of four prompts behind contexts of up to 32,768 tokens, everything visible
        _prompt("prompt_chunks", 4, 4096, 2000, 32768, 0, 0, 32, 8, 128, 32, 128, 4, "bf16"),
        # short prompts, INT2, small heads, pages that end inside a tile, 32-bit inputs
        _prompt("prompt_int2_d64", 8, 1003, 0, 1000, 300, 2, 16, 4, 64, 32, 24, 2, "f32"),
        # large heads, six query heads a kv head, an odd number of tokens
        _prompt("prompt_d256", 2, 2049, 0, 3000, 0, 0, 24, 4, 256, 64, 32, 4, "f16"),
        # eight drafted tokens of one sequence: launches and round trips
        _tree("tree_one", 1, 8, False, 4096, 4096, 0, 0, 32, 8, 128, 32, 128, 4, "f16"),
        # a serving batch, trees of up to 32 drafted tokens
        _tree("tree_batch16", 16, 32, True, 500, 16384, 0, 0, 32, 8, 128, 32, 64, 4, "bf16"),
        # wide trees over long contexts
        _tree("tree_long", 4, 64, False, 65536 - 77, 131072, 0, 0, 32, 8, 128, 32, 128, 4, "f16"),
        # what a batch's trees leave: a few of 32 drafted tokens each
        _keep("keep_batch64", 64, 32, True, 8, 100, 1000, 8, 128, 32, 64, 4, False),
        # wide trees of many sequences with deep paths, in a cache that tracks weights and positions
        _keep("keep_batch256", 256, 64, False, 32, 64, 512, 8, 128, 32, 32, 4, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "prompt", "prompt", "tree", "tree", "keep"])
    d = rng.choice([32, 64, 96, 128, 128, 128, 192, 256])
    g = rng.choice([x for x in (32, 32, 64, 128) if d % x == 0])
    kvh = rng.choice([1, 2, 3, 4, 8, 8, 8, 16])
    qh = kvh * rng.choice([1, 2, 4, 4, 5, 8, 16])
    bits = rng.choice([4, 4, 2])
    bt = rng.choice([16, 24, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    shape = dict(kvh=kvh, d=d, g=g, bt=bt, bits=bits)
    slot = kvh * (2 * d * bits // 8 + 4 * d // g)
    if kind == "keep":
        seqs, nodes = _log_int(rng, 1, 256), _log_int(rng, 1, 128)
        longest = rng.randint(0, max(1, min(1000, 500000000 // (seqs * slot) - nodes)))
        return dict(kind=kind, seqs=seqs, nodes=nodes, ragged=rng.choice([False, True]), deepest=rng.randint(1, nodes),
                    shortest=rng.choice([0, longest]), longest=longest, tracked=rng.choice([False, True]), **shape)
    sink = rng.choice([0, 1, 4, 100])
    if kind == "step":
        # at most half of the largest listed case's cache, whatever the shape
        room = 600000000 // slot
        longest = _log_int(rng, 1, min(131072, room))
        seqs = _log_int(rng, 1, max(2, min(128, room // longest)))
        return dict(kind=kind, seqs=seqs, shortest=rng.choice([0, 1, longest]), longest=longest,
                    window=_log_int(rng, 1, max(2, longest)), sink=sink, qh=qh, dtype=dtype, **shape)
    # products of (token, slot) pairs: a sixteenth of the largest listed case's at most
    pairs = 3000000 * 4096 // (qh * d)
    if kind == "prompt":
        total = _log_int(rng, 1, 4096)
        longest = rng.choice([0, _log_int(rng, 1, 32768)])
        total = max(1, min(total, int(math.sqrt(pairs)), pairs // max(longest, 1)))
        seqs = _log_int(rng, 1, max(2, min(16, total)))
        longest = min(longest, 300000000 // (slot * seqs))
        window = rng.choice([0, _log_int(rng, 1, max(2, longest + total))])
        return dict(kind=kind, seqs=seqs, total=total, shortest=rng.choice([0, longest]), longest=longest, window=window,
                    sink=sink if window else 0, qh=qh, dtype=dtype, **shape)
    nodes = _log_int(rng, 1, 128)
    longest = _log_int(rng, 1, min(65536, max(2, pairs // nodes), 300000000 // slot))
    seqs = _log_int(rng, 1, max(2, min(32, pairs // (nodes * longest), 300000000 // (slot * longest))))
    window = rng.choice([0, 0, _log_int(rng, 1, max(2, longest))])
    return dict(kind=kind, seqs=seqs, nodes=nodes, ragged=rng.choice([False, True]), shortest=rng.choice([0, 1, longest]),
                longest=longest, window=window, sink=sink if window else 0, qh=qh, dtype=dtype, **shape)


# --------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * seed + 23)


def _host_generator(seed):
    return torch.Generator().manual_seed(1000003 * seed + 29)


def _lengths(case, gen):
    """Lengths from ``shortest`` to ``longest``, spread over their logarithm; both ends occur."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    u = torch.rand((n,), generator=gen, dtype=torch.float64)
    at = torch.exp(math.log(max(lo, 1)) + u * (math.log(max(hi, 1)) - math.log(max(lo, 1)))).round().long()
    at[0] = hi
    if n > 1:
        at[1] = lo
    return at[torch.randperm(n, generator=gen)].clamp(0, hi)


def _counts(case, gen):
    """New tokens of each sequence."""
    n = case["seqs"]
    if case["kind"] == "step":
        return torch.ones(n, dtype=torch.long)
    if case["kind"] == "prompt":
        part = torch.rand((n,), generator=gen, dtype=torch.float64) + 0.1
        counts = (part * case["total"] / part.sum()).long()
        counts[0] += case["total"] - int(counts.sum())
        return counts
    if not case["ragged"]:
        return torch.full((n,), case["nodes"])
    # as many in all whatever the seed, so that outputs of every seed have one shape
    counts = 1 + torch.arange(n) * case["nodes"] // max(n, 1)
    return counts[torch.randperm(n, generator=gen)].clamp(1, case["nodes"])


def _parents(counts, gen):
    """A random tree of each sequence's tokens: node 0 a root, the others children of an earlier one (now and then of
    the context), of the nearer ones more often."""
    out = []
    for n in counts.tolist():
        u = torch.rand((n, 2), generator=gen).tolist()
        out += [-1 if i == 0 or u[i][0] < 0.02 else i - 1 - int(min(i, 12) * u[i][1] ** 2) for i in range(n)]
    return out


def _paths(parents, counts, deepest, gen):
    """One root-to-node path of each sequence's tree, of at most ``deepest`` nodes."""
    out, at = [], 0
    for n in counts.tolist():
        node = int(torch.randint(0, max(n, 1), (1,), generator=gen)) if n else -1
        path = []
        while node >= 0:
            path.append(node)
            node = parents[at + node]
        out.append(path[::-1][:deepest])
        at += n
    return out


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
    """Every tensor of a case, on the GPU, and what a user's program knows on the host."""
    gen, host = _generator(seed), _host_generator(seed)
    kind, bt, seqs = case["kind"], case["bt"], case["seqs"]
    s = dict(case=case)
    counts = _counts(case, host)
    before = _lengths(case, host)
    if kind == "step":
        before = (before - 1).clamp(min=-1)  # (a sequence of length 0 has no token to see)
        lengths = before + 1
    else:
        lengths = before + counts
    ends = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    s["counts"], s["before"] = counts.tolist(), before.tolist()
    s["ends"] = ends.tolist()
    s["lengths"] = lengths.to(torch.int32).cuda()
    s["longest"], s["all_slots"] = int(lengths.max()), int(lengths.sum())
    s["offsets"] = ends.to(torch.int32).cuda()
    pages_of = (lengths + bt - 1) // bt
    width = int(pages_of.max().clamp(min=1))
    pool = int(pages_of.sum()) + 3
    if kind == "keep":  # outputs hold the whole pool: as many pages whatever the seed
        width = (case["longest"] + case["nodes"] + bt - 1) // bt
        pool = seqs * width + 3
    s["table"] = _page_table(pages_of, width, pool, host).cuda()
    s["pk"], s["pv"], s["sk"], s["sv"] = _pool(case, gen, pool)
    if kind in ("tree", "keep"):
        parents = _parents(counts, host)
        s["parents"] = torch.tensor(parents, dtype=torch.int32).cuda()
    if kind == "keep":
        paths = _paths(parents, counts, case["deepest"], host)
        widest = case["deepest"]
        s["kept"] = torch.tensor([p + [-1] * (widest - len(p)) for p in paths], dtype=torch.int32).cuda()
        s["drafted"] = counts.to(torch.int32).cuda()
        s["weights"] = s["positions"] = None
        if case["tracked"]:
            shape = (seqs, width * bt)
            s["weights"] = torch.rand(shape, generator=gen, device="cuda")
            s["positions"] = torch.randint(0, 1 << 20, shape, generator=gen, device="cuda", dtype=torch.int32)
        return s
    tokens = seqs if kind == "step" else int(ends[-1])
    # scaled scores of standard deviation about 2: attention that picks out some tokens
    query = 1.5 * torch.randn((tokens, case["qh"], case["d"]), generator=gen, device="cuda")
    s["query"] = query.to(DTYPES[case["dtype"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from kvssd.backends import PagedBatch, resolve_attention_backend

        s["batch"] = PagedBatch(s["pk"], s["pv"], s["sk"], s["sv"], s["table"], s["lengths"], case["bits"], case["g"],
                                weights=s.get("weights"), positions=s.get("positions"))
        if case["kind"] == "keep":
            return s
        s["backend"] = backend = resolve_attention_backend("hip", s["query"].device)
        visible = dict(window=case["window"], sink=case["sink"])
        known = dict(max_length=s["longest"], total_tokens=s["all_slots"])
        if case["kind"] == "step":
            s["decode"] = backend.prepare_paged(s["query"], s["batch"], _scale(case), out_dtype=s["query"].dtype, **known,
                                                **visible)
        if case["kind"] == "tree":  # a step's trees are of one size again and again
            s["decode"] = backend.prepare_paged_tokens(s["query"], s["batch"], _scale(case), out_dtype=s["query"].dtype,
                                                       **known, **visible)
    return s


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


# --------------------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"step": _own_step, "prompt": _own_prompt, "tree": _own_tree, "keep": _own_keep}[kind](state)
    return {"step": _plain_step, "prompt": _plain_tokens, "tree": _plain_tokens, "keep": _plain_keep}[kind](state)


def _own_step(s):
    out, lse = s["decode"](s["query"])
    return dict(out=out, lse=lse)


def _own_prompt(s):
    c = s["case"]
    out, lse = s["backend"].run_paged_tokens(s["query"], s["batch"], _scale(c), s["offsets"], window=c["window"],
                                             sink=c["sink"], out_dtype=s["query"].dtype, max_length=s["longest"],
                                             total_tokens=s["all_slots"])
    return dict(out=out, lse=lse)


def _own_tree(s):
    out, lse = s["decode"](s["query"], s["offsets"], s["parents"])
    return dict(out=out, lse=lse)


def _own_keep(s):
    from kvssd.paged import keep_tokens

    lengths = keep_tokens(s["batch"], s["drafted"], s["kept"])
    return dict(lengths=lengths, weights=s["weights"], positions=s["positions"], pk=s["pk"], pv=s["pv"], sk=s["sk"],
                sv=s["sv"])


def _values_of(packed, scales, rows, c):
    """fp32 [..., kvh, d] of the pool's rows [...]."""
    bits = c["bits"]
    bytes_of = packed.flatten(0, 1)[rows]
    codes = (bytes_of[..., None] >> torch.arange(0, 8, bits, device="cuda", dtype=torch.uint8)) & ((1 << bits) - 1)
    codes = codes.flatten(-2).float() - (1 << (bits - 1))
    return (codes.unflatten(-1, (-1, c["g"])) * scales.flatten(0, 1)[rows].float()[..., None]).flatten(-2)


def _softmax_sums(scores, seen):
    """(weights, lse) of scores [..., slots] over the slots that are seen; 0 and -inf where none is."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total)), (torch.log(total) + top)[..., 0]


def _plain_step(s):
    c = s["case"]
    n, kvh, d, bt = c["seqs"], c["kvh"], c["d"], c["bt"]
    lengths = s["lengths"].long()[:, None]
    first = (lengths - c["window"]).clamp(min=0)
    # the sinks before the window, then the window
    reach = min(c["window"], max(s["longest"], 1))
    sinks = torch.arange(min(c["sink"], max(s["longest"], 1)), device="cuda").expand(n, -1)
    recent = first + torch.arange(reach, device="cuda")
    slots = torch.cat((sinks, recent), 1)
    seen = torch.cat((sinks < first, recent < lengths), 1)
    slots = torch.where(seen, slots, 0)
    rows = s["table"].clamp(min=0).long().gather(1, slots // bt) * bt + slots % bt
    query = s["query"].float().view(n, kvh, -1, d)
    k = _values_of(s["pk"], s["sk"], rows, c).permute(0, 2, 3, 1).contiguous()
    scores = torch.matmul(query, k) * _scale(c)
    del k
    p, lse = _softmax_sums(scores, seen[:, None, None])
    v = _values_of(s["pv"], s["sv"], rows, c).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(p, v).reshape(n, -1, d).to(s["query"].dtype)
    return dict(out=out, lse=lse.reshape(n, -1))


def _ancestors(parents):
    """bool [nodes, nodes]: whether node t is node i or above it."""
    n = parents.shape[0]
    eye = torch.eye(n, device="cuda")
    up = (parents.long()[:, None] == torch.arange(n, device="cuda")).float() + eye
    for _ in range(max(n - 1, 1).bit_length()):
        up = (torch.matmul(up, up) > 0).float()
    return up > 0


def _plain_tokens(s, most=1 << 28):
    c = s["case"]
    kvh, d, bt = c["kvh"], c["d"], c["bt"]
    window, sink = c["window"], c["sink"]
    outs, lses = [torch.empty((0, c["qh"], d), device="cuda")], [torch.empty((0, c["qh"]), device="cuda")]
    for b, (count, before) in enumerate(zip(s["counts"], s["before"])):
        if not count:
            continue
        query = s["query"][s["ends"][b]:s["ends"][b + 1]].float().view(count, kvh, -1, d)
        length = before + count
        slot = torch.arange(length, device="cuda")
        position = slot.clone()
        above = None
        if c["kind"] == "tree":
            above = _ancestors(s["parents"][s["ends"][b]:s["ends"][b + 1]])
            position[before:] = before + above.sum(1) - 1
        step = max(1, min(count, most // (c["qh"] * length)))
        for i0 in range(0, count, step):
            i1 = min(count, i0 + step)
            # what none of these tokens sees is left out
            use = slot[: length if above is not None else before + i1]
            mine = position[before + i0:before + i1, None]
            if window:
                use = use[(use < sink) | (use >= before) | (use > before + (0 if above is not None else i0) - window)]
            seen = use <= before + torch.arange(i0, i1, device="cuda")[:, None]
            if above is not None:
                tree = torch.zeros((i1 - i0, length), dtype=torch.bool, device="cuda")
                tree[:, :before] = True
                tree[:, before:] = above[i0:i1]
                seen = tree[:, use]
            if window:
                seen = seen & ((position[use] > mine - window) | (position[use] < sink))
            rows = s["table"][b].long()[use // bt] * bt + use % bt
            k = _values_of(s["pk"], s["sk"], rows, c).permute(1, 2, 0).contiguous()
            q = query[i0:i1].permute(1, 2, 0, 3).reshape(kvh, -1, d)  # (head, token)
            scores = (torch.matmul(q, k) * _scale(c)).view(kvh, -1, i1 - i0, len(use))
            del k
            p, lse = _softmax_sums(scores, seen)
            v = _values_of(s["pv"], s["sv"], rows, c).permute(1, 0, 2).contiguous()
            out = torch.matmul(p.view(kvh, -1, len(use)), v).view(kvh, -1, i1 - i0, d)
            outs.append(out.permute(2, 0, 1, 3).reshape(i1 - i0, -1, d))
            lses.append(lse.permute(2, 0, 1).reshape(i1 - i0, -1))
    return dict(out=torch.cat(outs).to(s["query"].dtype), lse=torch.cat(lses))


def _plain_keep(s):
    c = s["case"]
    bt = c["bt"]
    kept = s["kept"].long()
    base = (s["lengths"] - s["drafted"]).long()[:, None]
    used = kept >= 0
    lengths = base[:, 0] + used.sum(1)
    seq, nth = used.nonzero(as_tuple=True)
    frm, to = base[seq, 0] + kept[seq, nth], base[seq, 0] + nth
    page = s["table"].long()
    row_to = page[seq, to // bt] * bt + to % bt
    row_from = page[seq, frm // bt] * bt + frm % bt
    for pool in (s["pk"], s["pv"], s["sk"], s["sv"]):
        flat = pool.flatten(0, 1)
        flat[row_to] = flat[row_from]
    for per_slot in (s["weights"], s["positions"]):
        if per_slot is not None:
            per_slot[seq, to] = per_slot[seq, frm]
    return dict(lengths=lengths.to(torch.int32), weights=s["weights"], positions=s["positions"], pk=s["pk"], pv=s["pv"],
                sk=s["sk"], sv=s["sv"])


# --------------------------------------------------------------------------- work, exact results


def _mean_length(case):
    """The mean of lengths spread over their logarithm."""
    lo, hi = max(case["shortest"], 1), max(case["longest"], 1)
    if hi == lo or case["seqs"] == 1:
        return float(case["longest"])
    return (hi - lo) / math.log(hi / lo)


def work(case):
    kind, kvh, d, seqs = case["kind"], case["kvh"], case["d"], case["seqs"]
    per_slot = kvh * (2 * d * case["bits"] // 8 + 4 * (d // case["g"]))  # packed K and V with their scales
    mean = _mean_length(case)
    if kind == "keep":
        moved = seqs * min(case["deepest"], 1 + math.log(max(case["nodes"], 1)))
        return {"bytes": moved * 2 * per_slot + 8 * seqs, "flops": moved}
    item = 4 if case["dtype"] == "f32" else 2
    qh, window, sink = case["qh"], case["window"], case["sink"]
    if kind == "step":
        slots = seqs * max(1.0, min(mean, window + sink))
        return {"bytes": slots * per_slot + seqs * qh * (2 * d * item + 4), "flops": 4 * slots * qh * d}
    if kind == "prompt":
        tokens = case["total"]
        each = tokens / seqs
    else:
        each = (case["nodes"] + 1) / 2 if case["ragged"] else case["nodes"]
        tokens = seqs * each
    # slots that a token sees, on average, and that a sequence's tokens see together
    if kind == "prompt":
        reach = window + sink if window else mean + each
        grown = min(max(reach - mean, 0.0), each)  # tokens whose view still grows
        seen = (grown * (mean + grown / 2) + (each - grown) * min(reach, mean + each)) / max(each, 1e-9)
        shared = min(mean, reach) + each
    else:
        seen = min(mean, window + sink) if window else mean
        shared = seen + each
    return {"bytes": seqs * shared * per_slot + tokens * qh * (2 * d * item + 4), "flops": 4 * tokens * max(seen, 1.0) * qh * d}


def _exact_rows(packed, scales, rows, c):
    """fp64 [slots, kvh, d]"""
    kvh, d, g, bits = c["kvh"], c["d"], c["g"], c["bits"]
    byte = packed.view(-1, kvh, d * bits // 8)[rows].long()
    code = (byte[..., None] >> torch.arange(0, 8, bits, device="cuda")) % (1 << bits)
    code = code.reshape(len(rows), kvh, d // g, g).double() - (1 << (bits - 1))
    return (code * scales.view(-1, kvh, d // g)[rows].double()[..., None]).reshape(len(rows), kvh, d)


def _exact_attention(s, most=1 << 27):
    """Sequence by sequence, a kv head at a time; what a token sees from its own chain of parents."""
    c = s["case"]
    kvh, d, bt, window, sink = c["kvh"], c["d"], c["bt"], c["window"], c["sink"]
    gq = c["qh"] // kvh
    tokens = s["query"].shape[0]
    out = torch.zeros((tokens, c["qh"], d), dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, c["qh"]), -math.inf, dtype=torch.float64, device="cuda")
    lengths = s["lengths"].tolist()
    parents = s["parents"].tolist() if c["kind"] == "tree" else None
    for b, length in enumerate(lengths):
        count = s["counts"][b]
        if not count or not length:
            continue
        at, before = s["ends"][b], length - count
        chains = [[i] for i in range(count)]
        if parents is not None:
            for i in range(count):
                up = parents[at + i]
                if up >= 0:
                    chains[i] = chains[up] + [i]
        place = torch.arange(length, device="cuda")
        if parents is not None:
            place[before:] = torch.tensor([before + len(chain) - 1 for chain in chains], device="cuda")
        step = max(1, min(count, most // (gq * length)))
        rows = s["table"][b].long()[torch.arange(length, device="cuda") // bt] * bt + torch.arange(length, device="cuda") % bt
        for h in range(kvh):
            k = torch.cat([_exact_rows(s["pk"], s["sk"], r, c)[:, h] for r in rows.split(16384)]).T.contiguous()
            v = torch.cat([_exact_rows(s["pv"], s["sv"], r, c)[:, h] for r in rows.split(16384)])
            for i0 in range(0, count, step):
                i1 = min(count, i0 + step)
                if parents is None:
                    hidden = torch.arange(length, device="cuda") > before + torch.arange(i0, i1, device="cuda")[:, None]
                else:
                    hidden = torch.ones((i1 - i0, length), dtype=torch.bool)
                    hidden[:, :before] = False
                    for i in range(i0, i1):
                        hidden[i - i0, [before + a for a in chains[i]]] = False
                    hidden = hidden.cuda()
                if window:
                    hidden |= (place <= place[before + i0:before + i1, None] - window) & (place >= sink)
                q = s["query"][at + i0:at + i1, h * gq:(h + 1) * gq].double().reshape(-1, d)
                score = torch.matmul(q, k).view(i1 - i0, gq, length) / math.sqrt(d)
                score.masked_fill_(hidden[:, None], -math.inf)
                total = torch.logsumexp(score, -1)
                p = torch.exp(score - total[..., None]).view(-1, length)
                out[at + i0:at + i1, h * gq:(h + 1) * gq] = torch.matmul(p, v).view(i1 - i0, gq, d)
                lse[at + i0:at + i1, h * gq:(h + 1) * gq] = total
    return dict(out=out, lse=lse)


def _exact_keep(s):
    """Sequence by sequence, row by row, on the host's lists."""
    c = s["case"]
    bt, table = c["bt"], s["table"].tolist()
    pools = [t.clone().flatten(0, 1) for t in (s["pk"], s["pv"], s["sk"], s["sv"])]
    weights = None if s["weights"] is None else s["weights"].double()
    positions = None if s["positions"] is None else s["positions"].clone()
    after, frm, to, seq, old, new = [], [], [], [], [], []
    for b, (length, count, kept) in enumerate(zip(s["lengths"].tolist(), s["drafted"].tolist(), s["kept"].tolist())):
        base = length - count
        path = [node for node in kept if node >= 0]
        for j, node in enumerate(path):
            seq.append(b)
            old.append(base + node)
            new.append(base + j)
            frm.append(table[b][(base + node) // bt] * bt + (base + node) % bt)
            to.append(table[b][(base + j) // bt] * bt + (base + j) % bt)
        after.append(base + len(path))
    # every row is taken from where it was before any of them moved
    frm, to, seq, old, new = (torch.tensor(x, dtype=torch.long, device="cuda") for x in (frm, to, seq, old, new))
    for pool in pools:
        pool[to] = pool[frm].clone()
    for t in (weights, positions):
        if t is not None:
            t[seq, new] = t[seq, old].clone()
    pools = [t.unflatten(0, s["pk"].shape[:2]) for t in pools]
    return dict(lengths=torch.tensor(after, dtype=torch.int32, device="cuda"), weights=weights, positions=positions,
                pk=pools[0], pv=pools[1], sk=pools[2].double(), sv=pools[3].double())


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_keep(s) if case["kind"] == "keep" else _exact_attention(s)
