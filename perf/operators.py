"""The key/value cache in 4 bits, the attention over it and its pages: the cases that are timed.

`run` computes an operator in plain torch (own = False) or through
libpktito_b200's entry points (own = True), on the same state. The cache's
bytes are laid out as include/pktito_b200.h documents them (pkb_cache4):
units of 16 tokens of one head, K's and V's codes in the order the tensor
cores take them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = 16  # tokens of one head that lie together
BLOCK = 32  # values of one scale


def listed():
    return [
        # One new token of each of 256 running streams, 8 heads of 128 as the encoder has them: launch latency counts.
        {"name": "append-step", "op": "append", "dtype": "bf16", "seqs": 256, "rows": 1, "ragged": False, "context": 700,
         "heads": 8, "dk": 128, "page": 16, "layers": 2},
        # The frames of 24 segments of up to 20 s each, the products' float rows, taken into the cache at once.
        {"name": "append-frames", "op": "append", "dtype": "f32", "seqs": 24, "rows": 1499, "ragged": True, "context": 1499,
         "heads": 8, "dk": 128, "page": 64, "layers": 1},
        # One stream's next token: the least work, nothing but latency.
        {"name": "decode-one", "op": "attention", "dtype": "f32", "seqs": 1, "queries": 1, "ragged": False, "context": 377,
         "heads": 8, "group": 1, "dk": 128, "page": 16, "causal": True, "window": 0},
        # A server's ordinary step: 64 sequences of uneven length, four query heads to a cached head.
        {"name": "decode-batch", "op": "attention", "dtype": "bf16", "seqs": 64, "queries": 1, "ragged": True,
         "context": 4099, "heads": 8, "group": 4, "dk": 128, "page": 16, "causal": True, "window": 0},
        # Hours of history: few rows over a long axis.
        {"name": "decode-long", "op": "attention", "dtype": "bf16", "seqs": 3, "queries": 1, "ragged": True,
         "context": 120001, "heads": 8, "group": 8, "dk": 128, "page": 64, "causal": True, "window": 0},
        # Streaming with limited left context: 4 frames a chunk, 200 streams, smaller heads, half precision.
        {"name": "stream-window", "op": "attention", "dtype": "f16", "seqs": 200, "queries": 4, "ragged": True,
         "context": 1499, "heads": 8, "group": 1, "dk": 64, "page": 32, "causal": True, "window": 250},
        # A decoder's tokens over the encoder's frames (not causal), float rows as the products write them.
        {"name": "cross-frames", "op": "attention", "dtype": "f32", "seqs": 32, "queries": 23, "ragged": True,
         "context": 750, "heads": 8, "group": 1, "dk": 128, "page": 32, "causal": False, "window": 0},
        # Two long prompts: the largest products.
        {"name": "prompt-long", "op": "attention", "dtype": "bf16", "seqs": 2, "queries": 8191, "ragged": False,
         "context": 8191, "heads": 8, "group": 4, "dk": 128, "page": 64, "causal": True, "window": 0},
        # A step of beam search over 4 segments with 8 hypotheses: drop some, fork others, one more token for all.
        {"name": "beam-small", "op": "beam", "segments": 4, "beams": 8, "context": 61, "heads": 8, "dk": 64, "page": 16,
         "layers": 4},
        # The same over 64 segments and 24 layers.
        {"name": "beam-large", "op": "beam", "segments": 64, "beams": 8, "context": 211, "heads": 8, "dk": 128, "page": 16,
         "layers": 24},
        # Housekeeping between requests: ended sequences are freed, the pool compacted, a few sessions handed over to another pool.
        {"name": "move-small", "op": "move", "seqs": 24, "context": 150, "heads": 8, "dk": 128, "page": 16, "layers": 2},
        # The same over a large pool with long sessions.
        {"name": "move-large", "op": "move", "seqs": 192, "context": 4001, "heads": 8, "dk": 128, "page": 64, "layers": 6},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "beam", "move"])
    page = rng.choice([16, 32, 64, 128])
    dk = rng.choice([32, 64, 96, 128, 128, 256])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "append":
        seqs = _log(rng, 1, 256)
        rows = _log(rng, 1, max(1, 30000 // seqs))
        return {"op": op, "dtype": dtype, "seqs": seqs, "rows": rows, "ragged": rng.random() < 0.5,
                "context": rows + _log(rng, 1, 1000) - 1, "heads": rng.choice([1, 2, 4, 8]), "dk": min(dk, 128), "page": page,
                "layers": rng.choice([1, 2])}
    if op == "attention":
        heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
        if rng.random() < 0.6:  # single tokens and a few
            seqs, queries = _log(rng, 1, 100), rng.choice([1, 1, 1, 2, 5])
            context = _log(rng, queries, 150000 // seqs)
        else:  # chunks and whole prompts
            seqs = _log(rng, 1, 24)
            context = _log(rng, 16, 8000 // seqs)
            queries = _log(rng, 2, context)
            queries = max(1, min(queries, 10**12 // (4 * seqs * context * heads * group * dk)))
        return {"op": op, "dtype": dtype, "seqs": seqs, "queries": queries, "ragged": rng.random() < 0.7, "context": context,
                "heads": heads, "group": group, "dk": dk, "page": page, "causal": rng.random() < 0.7,
                "window": rng.choice([0, 0, _log(rng, 1, 2000)])}
    if op == "beam":
        return {"op": op, "segments": _log(rng, 1, 48), "beams": rng.choice([2, 3, 4, 8]), "context": _log(rng, 1, 200),
                "heads": rng.choice([1, 2, 4, 8]), "dk": min(dk, 128), "page": page, "layers": rng.choice([1, 3, 6])}
    return {"op": op, "seqs": _log(rng, 2, 128), "context": _log(rng, 1, 3000), "heads": rng.choice([1, 2, 4, 8]),
            "dk": min(dk, 128), "page": page, "layers": rng.choice([1, 2, 4])}


# ------------------------------------------------------------------ inputs --

def _spread(n, least, most):
    """n lengths up to `most`, uneven, the same for every seed: a seed sets their order alone."""
    part = torch.rand(n, generator=torch.Generator().manual_seed(n))
    part[0] = 1
    return (most * (least + (1 - least) * part)).long().clamp(1, most)


def _lengths(case, cpu):
    """(tokens a sequence holds, its rows in this call), on the host: the longest is `context`, ragged ones go down to 1."""
    n, context, most = case["seqs"], case["context"], case.get("queries") or case["rows"]
    if not case["ragged"]:
        return torch.full((n,), context), torch.full((n,), min(most, context))
    lens, rows = _spread(n, 0.02, context), _spread(n + 1, 0.3, most)[:n]
    if case["op"] == "append" or case["causal"]:
        rows = torch.minimum(rows, lens)
    order = torch.randperm(n, generator=cpu)
    return lens[order], rows[order]


def _pool(case, n_pages, layers, gen):
    """The bytes of a cache's pages: every token of every page quantized from rows with a few wide channels, as K and V have."""
    heads, dk, groups = case["heads"], case["dk"], case["page"] // UNIT
    shape = (layers, n_pages, heads, groups, UNIT, dk)
    wide = 0.5 + 1.5 * torch.rand((heads, 1, 1, dk), generator=gen, device="cuda")
    k = torch.randn(shape, generator=gen, device="cuda") * wide
    kn, ks = _quantize(k)
    del k
    v = torch.randn(shape, generator=gen, device="cuda")
    vn, vs = _quantize(v)
    del v
    return _pack(kn, ks, vn, vs).reshape(layers, n_pages, -1)


def _table(lens, page, n_pages, max_pages, cpu):
    """Pages in no order for sequences of these lengths: (table, refs), on the host."""
    need = (lens + page - 1) // page
    table = torch.full((len(lens), max_pages), -1, dtype=torch.int32)
    held = torch.arange(max_pages)[None] < need[:, None]
    table[held] = torch.randperm(n_pages, generator=cpu)[:int(need.sum())].int()
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs[table[held].long()] = 1
    return table, refs


def prepare(case, seed):
    cpu, gen = torch.Generator().manual_seed(seed), torch.Generator("cuda").manual_seed(seed)
    page, heads, dk = case["page"], case["heads"], case["dk"]
    state = {"case": dict(case)}
    if case["op"] in ("append", "attention"):
        lens, rows = _lengths(case, cpu)
        max_pages = -(-case["context"] // page) + 1
        n_pages = int(((lens + page - 1) // page).sum()) + 5
        table, refs = _table(lens, page, n_pages, max_pages, cpu)
        layers = case.get("layers", 1)
        starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
        starts[1:] = rows.cumsum(0)
        state |= {"table": table.cuda(), "refs": refs.cuda(), "lens": lens.int().cuda(), "layer": layers - 1,
                  "seqs": torch.randperm(len(lens), generator=cpu).int().cuda(), "n_rows": int(starts[-1]), "max_rows": int(rows.max())}
        order = state["seqs"].cpu().long()  # the call lists the sequences in an order of its own
        starts[1:] = rows[order].cumsum(0)
        state["starts"] = starts.cuda()
        if case["op"] == "append":
            state["pages"] = torch.zeros((layers, n_pages, heads * page * dk * 9 // 8), dtype=torch.uint8, device="cuda")
            state |= {x: torch.randn((state["n_rows"], heads * dk), generator=gen, device="cuda").mul_(2).to(DTYPES[case["dtype"]]) for x in "kv"}
        else:
            state["pages"] = _pool(case, n_pages, layers, gen)
            state["q"] = torch.randn((state["n_rows"], heads * case["group"] * dk), generator=gen, device="cuda").to(DTYPES[case["dtype"]])
        return state
    if case["op"] == "beam":
        # each segment's hypotheses share all but their last two pages; a third of them end and give way to forks of others
        nseg, beams, context = case["segments"], case["beams"], case["context"]
        n = nseg * beams
        lens = _spread(nseg, 0.3, context)[torch.randperm(nseg, generator=cpu)].repeat_interleave(beams)
        need = (lens + page - 1) // page
        max_pages = -(-(context + 1) // page) + 1
        n_pages = int(need.sum()) + n + 3
        table, _ = _table(lens, page, n_pages, max_pages, cpu)
        at = torch.arange(max_pages)[None]
        shared = at < (need - 2)[:, None]
        table = torch.where(shared, table.view(nseg, beams, -1)[:, :1].expand(-1, beams, -1).reshape(n, -1), table)
        refs = torch.bincount(table[table >= 0].long(), minlength=n_pages).int()
        drop = max(1, beams // 3)
        order = torch.rand((nseg, beams), generator=cpu).argsort(1) + beams * torch.arange(nseg)[:, None]
        dst = order[:, :drop].reshape(-1)
        src = order[:, drop:][:, torch.randint(0, beams - drop, (drop,), generator=cpu)].reshape(-1)
        state |= {"dst": dst.int().cuda(), "src": src.int().cuda(), "fork_lens": lens[src].int().cuda(),
                  "all": torch.arange(n).int().cuda(), "add": torch.ones(n).int().cuda()}
    else:
        n = case["seqs"]
        lens = _spread(n, 0.1, case["context"])
        max_pages = -(-case["context"] // page)
        n_pages = int(((lens + page - 1) // page).sum() * 1.15) + 7
        table, refs = _table(lens, page, n_pages, max_pages, cpu)
        # every third sequence has ended, every eighth goes over; the seed sets the order in which they are listed
        slot = torch.arange(n)
        ended, moved = slot[slot % 3 == 0], slot[(slot % 3 > 0) & (slot % 8 == 1)]
        ended, moved = (x[torch.randperm(len(x), generator=cpu)] for x in (ended, moved))
        other = int(((lens[moved] + page - 1) // page).sum()) + 4
        state |= {"ended": ended.int().cuda(), "moved": moved.int().cuda(), "moved_lens": lens[moved].int().cuda(),
                  "slots": torch.randperm(len(moved) + 2, generator=cpu)[:len(moved)].int().cuda(),
                  "other_pages": torch.zeros((case["layers"], other, heads * page * dk * 9 // 8), dtype=torch.uint8, device="cuda"),
                  "other_table": torch.full((len(moved) + 2, max_pages), -1, dtype=torch.int32, device="cuda"),
                  "other_lens": torch.zeros(len(moved) + 2, dtype=torch.int32, device="cuda"),
                  "other_refs": torch.zeros(other, dtype=torch.int32, device="cuda")}
    # pages are moved as they are, so any bytes will do here
    state["pages"] = torch.randint(-2**63, 2**63 - 1, (case["layers"], n_pages, heads * page * dk * 9 // 64), generator=gen, device="cuda").view(torch.uint8)
    state |= {"table": table.cuda(), "refs": refs.cuda(), "lens": lens.int().cuda()}
    # the pages' books as they are before a pass, which each pass starts from
    state |= {name + "0": state[name].clone() for name in ("table", "refs", "lens")}
    return state


# ---------------------------------------------------------------- the format --

def _quantize(x):
    """(codes + 8, scales) of rows of blocks of 32: the scale is amax / 7 cut to 5 significant bits."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    good = b.isfinite().all(-1, keepdim=True) & (amax >= 2.0 ** -121)
    s = ((amax / 7).view(torch.int32) & -(1 << 19)).view(torch.float32)
    n = torch.where(good, torch.round(b / torch.where(good, s, 1)), 0).add_(8).to(torch.uint8)
    return n.flatten(-2), torch.where(good, s, 0).squeeze(-1)


def _nibbles(n):
    """Eight codes (last axis) to four bytes, the first in the low bits."""
    return (n[..., 0::2] | n[..., 1::2] << 4).flatten(-2)


def _pack(kn, ks, vn, vs):
    """Units [..., 18 dk] bytes of codes [..., 16, dk] and scales [..., 16, dk / 32]."""
    lead, nb = kn.shape[:-2], kn.shape[-1] // BLOCK
    d = len(lead)
    axes = lambda *a: list(range(d)) + [d + i for i in a]  # noqa: E731
    # K: token, a fourth of each block, block; a word's 8 values even ones first
    k = kn.view(*lead, UNIT, nb, 4, 4, 2).permute(axes(0, 2, 1, 4, 3)).reshape(*lead, -1, 8)
    # V: block, 8 rows, 4 token pairs, halves of the block; then in a word: token of the pair, tokens 8 on, values 8 on
    v = vn.view(*lead, 2, 4, 2, nb, 2, 2, 8).permute(axes(3, 6, 1, 4, 2, 0, 5)).reshape(*lead, -1, 8)
    scales = torch.cat([ks.reshape(*lead, -1), vs.transpose(-1, -2).reshape(*lead, -1)], -1)
    return torch.cat([_nibbles(k), _nibbles(v), scales.to(torch.bfloat16).view(torch.uint8)], -1)


def _codes(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _unpack(u, dk):
    """K and V [..., 16, dk] in float32 of units [..., 18 dk]."""
    lead, nb = u.shape[:-1], dk // BLOCK
    d = len(lead)
    axes = lambda *a: list(range(d)) + [d + i for i in a]  # noqa: E731
    k, v, ks, vs = u.split([8 * dk, 8 * dk, dk, dk], -1)
    ks = ks.contiguous().view(torch.bfloat16).view(*lead, UNIT, nb, 1)
    vs = vs.contiguous().view(torch.bfloat16).view(*lead, nb, UNIT).transpose(-1, -2).unsqueeze(-1)
    k = _codes(k).view(*lead, UNIT, 4, nb, 2, 4).permute(axes(0, 2, 1, 4, 3)).reshape(*lead, UNIT, nb, BLOCK)
    v = _codes(v).view(*lead, nb, 8, 4, 2, 2, 2, 2).permute(axes(5, 2, 4, 0, 3, 6, 1)).reshape(*lead, UNIT, nb, BLOCK)
    return ((k.float() - 8) * ks.float()).flatten(-2), ((v.float() - 8) * vs.float()).flatten(-2)


# ------------------------------------------------------------ the plain forms --

def _units(state):
    case = state["case"]
    return state["pages"][state["layer"]].view(-1, case["heads"], case["page"] // UNIT, 18 * case["dk"])


def _last_rows(state):
    """For each row of the call: its sequence, and its token's place in it (the call's rows are a sequence's last)."""
    starts, seqs = state["starts"].long(), state["seqs"].long()
    row = torch.arange(state["n_rows"], device="cuda")
    i = torch.searchsorted(starts[1:], row, right=True)
    return seqs[i], state["lens"].long()[seqs[i]] - (starts[i + 1] - row)


def _append_plain(state):
    case, units = state["case"], _units(state)
    page, dk = case["page"], case["dk"]
    seq, pos = _last_rows(state)
    at = state["table"][seq, pos // page].long()
    kn, ks = _quantize(state["k"].unflatten(-1, (-1, dk)))
    vn, vs = _quantize(state["v"].unflatten(-1, (-1, dk)))
    # the units that the rows fall in, with the rows' tokens replaced
    spot = at * (page // UNIT) + pos % page // UNIT
    which, inverse = spot.unique(return_inverse=True)
    p, g = which // (page // UNIT), which % (page // UNIT)
    old = units[p, :, g]
    lead = old.shape[:2]
    ok, ov, oks, ovs = old.split([8 * dk, 8 * dk, dk, dk], -1)
    nb = dk // BLOCK
    ok = _codes(ok).view(*lead, UNIT, 4, nb, 2, 4).permute(0, 1, 2, 4, 3, 6, 5).reshape(*lead, UNIT, dk)
    ov = _codes(ov).view(*lead, nb, 8, 4, 2, 2, 2, 2).permute(0, 1, 7, 4, 6, 2, 5, 8, 3).reshape(*lead, UNIT, dk)
    oks = oks.contiguous().view(torch.bfloat16).view(*lead, UNIT, nb).float()
    ovs = ovs.contiguous().view(torch.bfloat16).view(*lead, nb, UNIT).transpose(-1, -2).float().contiguous()
    token = pos % UNIT
    ok[inverse, :, token], ov[inverse, :, token], oks[inverse, :, token], ovs[inverse, :, token] = kn, vn, ks, vs
    units[p, :, g] = _pack(ok, oks, ov, ovs)
    # and what the new tokens stand for, read back from the pages
    k, v = _unpack(units[p, :, g], dk)
    kind = DTYPES[case["dtype"]]
    return k[inverse, :, token].flatten(1).to(kind), v[inverse, :, token].flatten(1).to(kind)


def _attention_plain(state):
    case, units = state["case"], _units(state)
    page, dk, heads, group = case["page"], case["dk"], case["heads"], case["group"]
    seqs, starts = state["seqs"].long(), state["starts"].long()
    n, lens, rows = len(seqs), state["lens"].long()[seqs], starts[1:] - starts[:-1]
    longest = -(-case["context"] // UNIT) * UNIT
    # each sequence's tokens side by side, as long as the longest
    at = torch.arange(longest // UNIT, device="cuda")
    pages = state["table"][seqs][:, at * UNIT // page].long().clamp_min(0)
    k, v = _unpack(units[pages, :, at % (page // UNIT)], dk)  # [n, units, heads, 16, dk]
    k, v = (x.permute(0, 2, 1, 3, 4).reshape(n, heads, longest, dk) for x in (k, v))
    # and its queries
    most = state["max_rows"]
    row = (starts[:-1, None] + torch.arange(most, device="cuda")).clamp_max(state["n_rows"] - 1)
    q = state["q"].float()[row].view(n, most, heads, group, dk).permute(0, 2, 3, 1, 4).reshape(n, heads, group * most, dk)
    s = q @ k.transpose(-1, -2)
    s = s.mul_(1 / math.sqrt(dk)).view(n, heads, group, most, longest)
    del k, q
    j, pos = torch.arange(longest, device="cuda"), (lens - rows)[:, None] + torch.arange(most, device="cuda")
    hidden = (j >= lens[:, None, None]).expand(n, most, longest)
    if case["causal"]:
        hidden = hidden | (j > pos[..., None])
    if case["window"]:
        hidden = hidden | (j <= pos[..., None] - case["window"])
    s.masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = s.sum(-1).view(n, heads, group * most, 1)
    o = s.view(n, heads, group * most, longest) @ v
    o = torch.where(total > 0, o / total, 0).view(n, heads, group, most, dk).permute(0, 3, 1, 2, 4).reshape(n, most, -1)
    return o[torch.arange(most, device="cuda") < rows[:, None]].to(DTYPES[case["dtype"]])


def _free_plain(table, lens, refs, seqs):
    held = table[seqs]
    refs.sub_(torch.bincount(held[held >= 0].long(), minlength=len(refs)).int())
    table[seqs], lens[seqs] = -1, 0


def _take_plain(table, refs, seqs, wanted):
    """The lowest free pages into the wanted places of the sequences' table rows, sequence by sequence: the pages."""
    pages = (refs == 0).nonzero()[:, 0][:int(wanted.sum())]
    rows = table[seqs]
    rows[wanted] = pages.int()
    table[seqs], refs[pages] = rows, 1
    return pages


def _at(table):
    return torch.arange(table.shape[1], device="cuda")


def _beam_plain(state):
    page, table, lens, refs = state["case"]["page"], state["table"], state["lens"], state["refs"]
    dst, src, n = state["dst"].long(), state["src"].long(), state["fork_lens"].long()
    _free_plain(table, lens, refs, dst)
    shared, last = _at(table) < (n // page)[:, None], _at(table) == torch.where(n % page > 0, n // page, -1)[:, None]
    old = table[src]
    table[dst] = torch.where(shared, old, -1)
    refs.add_(torch.bincount(old[shared].long(), minlength=len(refs)).int())
    new = _take_plain(table, refs, dst, last)
    state["pages"][:, new] = state["pages"][:, old[last].long()]
    lens[dst] = n.int()
    live = state["all"].long()
    before, after = lens[live], lens[live] + state["add"]
    _take_plain(table, refs, live, (_at(table) >= (before + page - 1)[:, None] // page) & (_at(table) < (after + page - 1)[:, None] // page))
    lens[live] = after


def _move_plain(state):
    page, table, lens, refs = state["case"]["page"], state["table"], state["lens"], state["refs"]
    _free_plain(table, lens, refs, state["ended"].long())
    used = refs > 0
    count = used.sum()
    at = torch.arange(len(refs), device="cuda")
    above, holes = (used & (at >= count)).nonzero()[:, 0], (~used & (at < count)).nonzero()[:, 0]
    to = at.clone()
    to[above] = holes
    state["pages"][:, holes] = state["pages"][:, above]
    refs[holes], refs[above] = refs[above], 0
    table.copy_(torch.where(table >= 0, to[table.long().clamp_min(0)].int(), table))
    # the sessions that go over: all of their pages
    slots, moved, n = state["slots"].long(), state["moved"].long(), state["moved_lens"].long()
    wanted = _at(table) < ((n + page - 1) // page)[:, None]
    new = _take_plain(state["other_table"], state["other_refs"], slots, wanted)
    state["other_pages"][:, new] = state["pages"][:, table[moved][wanted].long()]
    state["other_lens"][slots] = n.int()
    return count.int().reshape(1)


# ---------------------------------------------------------------------- a pass --

def _own(state):
    """The library, and the descriptors and workspaces that a program keeps beside its caches."""
    import libpktito_b200 as P
    if "own" not in state:
        case = state["case"]
        shape = (case["page"], case["heads"], case["dk"])
        kept = {"cache": P.Cache4.of(state["pages"], state["table"], state["lens"], state["refs"], *shape),
                "status": torch.zeros(4, dtype=torch.int32, device="cuda")}
        if case["op"] == "attention":
            size = P.attention_cache4_work_bytes(kept["cache"], case["heads"] * case["group"], state["n_rows"], len(state["seqs"]))
        elif case["op"] == "move":
            kept["other"] = P.Cache4.of(state["other_pages"], state["other_table"], state["other_lens"], state["other_refs"], *shape)
            size = P.cache4_work_bytes(kept["cache"])
        else:
            size = P.cache4_work_bytes(kept["cache"])
        kept["work"] = torch.empty(max(256, size), dtype=torch.uint8, device="cuda")
        state["own"] = kept
    return P, state["own"]


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "append":
        if not own:
            return _append_plain(state)
        P, kept = _own(state)
        k, v, width = torch.empty_like(state["k"]), torch.empty_like(state["v"]), state["k"].shape[1]
        rows = (state["seqs"], state["starts"], len(state["seqs"]), state["n_rows"])
        P.cache4_append_dev(kept["cache"], state["layer"], state["k"], width, state["v"], width, *rows)
        P.cache4_read_dev(kept["cache"], state["layer"], k, width, v, width, *rows)
        return k, v
    if op == "attention":
        if not own:
            return _attention_plain(state)
        P, kept = _own(state)
        q = state["q"]
        o, width = torch.empty_like(q), q.shape[1]
        P.attention_cache4_dev(o, width, q, width, case["heads"] * case["group"], kept["cache"], state["layer"], state["seqs"],
                               state["starts"], len(state["seqs"]), state["n_rows"], state["max_rows"], 1 / math.sqrt(case["dk"]),
                               case["causal"], case["window"], kept["work"])
        return o
    # the books as they were, so that a pass can be made again
    for name in ("table", "refs", "lens"):
        state[name].copy_(state[name + "0"])
    if op == "beam":
        if not own:
            _beam_plain(state)
            status = torch.zeros(3, dtype=torch.int32, device="cuda")
        else:
            P, kept = _own(state)
            cache, status, work = kept["cache"], kept["status"][:3], kept["work"]
            P.cache4_free_dev(cache, state["dst"], len(state["dst"]), status[0:], work)
            P.cache4_fork_dev(cache, state["src"], state["dst"], state["fork_lens"], len(state["dst"]), status[1:], work)
            P.cache4_grow_dev(cache, state["all"], state["add"], len(state["all"]), status[2:], work)
        return state["table"], state["lens"], state["refs"], state["pages"].view(torch.int64), status
    state["other_table"].fill_(-1)
    state["other_refs"].zero_()
    state["other_lens"].zero_()
    if not own:
        used = _move_plain(state)
        status = torch.zeros(3, dtype=torch.int32, device="cuda")
    else:
        P, kept = _own(state)
        cache, status, used, work = kept["cache"], kept["status"][:3], kept["status"][3:], kept["work"]
        P.cache4_free_dev(cache, state["ended"], len(state["ended"]), status[0:], work)
        P.cache4_compact_dev(cache, used, status[1:], work)
        P.cache4_copy_dev(kept["other"], cache, state["moved"], state["slots"], state["moved_lens"], len(state["moved"]), status[2:], work)
    return (state["table"], state["lens"], state["refs"], state["pages"].view(torch.int64), state["other_table"],
            state["other_lens"], state["other_refs"], state["other_pages"].view(torch.int64), used, status)


# ------------------------------------------------------------------ its measure --

def _spans(case):
    """(visible keys summed over the rows, tokens read, rows)."""
    lens, rows = _lengths(case, torch.Generator())
    pairs = tokens = 0
    for n, r in zip(lens.tolist(), rows.tolist()):
        pos = torch.arange(n - r, n)
        hi = (pos + 1).clamp(0, n) if case["causal"] else torch.full_like(pos, n)
        lo = (pos - case["window"] + 1).clamp_min(0) if case["window"] else torch.zeros_like(pos)
        lo = torch.minimum(lo, hi)
        pairs += int((hi - lo).sum())
        tokens += int(hi.max() - lo[hi > lo].min()) if bool((hi > lo).any()) else 0
    return pairs, tokens, int(rows.sum())


def work(case):
    heads, dk, page = case["heads"], case["dk"], case["page"]
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("dtype"), 1)
    if case["op"] == "append":
        _, rows = _lengths(case, torch.Generator())
        values = int(rows.sum()) * heads * dk * 2
        # rows in, 4.5 bits a value to the pages and back, rows out
        return {"bytes": values * (2 * size + 2 * 0.5625), "flops": 6 * values}
    if case["op"] == "attention":
        pairs, tokens, rows = _spans(case)
        width = heads * case["group"] * dk
        return {"bytes": tokens * heads * dk * 1.125 + 2 * rows * width * size, "flops": 4 * pairs * width}
    page_bytes = heads * page * dk * 9 // 8
    if case["op"] == "beam":
        n = case["segments"] * case["beams"]
        forks = case["segments"] * max(1, case["beams"] // 3)
        pages = n * (case["context"] * 0.65 / page + 1)
        return {"bytes": 2 * forks * case["layers"] * page_bytes * (page - 1) / page + 8 * pages, "flops": 0}
    pages = case["seqs"] * (case["context"] * 0.55 / page + 0.5)
    ended, moved = -(-case["seqs"] // 3), max(1, case["seqs"] // 12)
    # a third of the pages is free afterwards, and that share of the rest lies above the count of those in use
    share = moved / case["seqs"] + (1 - ended / case["seqs"]) * (1 - (1 - ended / case["seqs"]) / 1.15)
    return {"bytes": 2 * share * pages * case["layers"] * page_bytes + 8 * pages, "flops": 0}


# ------------------------------------------------------------------- in 64 bits --

def _exact_block(x):
    """What a row's blocks of 32 stand for, from the definition."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().max(-1, keepdim=True).values
    m, e = torch.frexp(amax / 7)
    s = torch.ldexp(torch.floor(m * 32) / 32, e)
    held = torch.round(b / s) * s
    return torch.where(b.isfinite().all(-1, keepdim=True) & (amax >= 2.0 ** -121), held, 0.0).flatten(-2)


def _exact_rows(pages, dk, page, heads, which, n):
    """K and V [heads, n, dk] of a sequence's n tokens in the pages `which`, value by value where the format says it lies."""
    j, d = torch.arange(n, device="cuda")[:, None], torch.arange(dk, device="cuda")[None]
    nb, r = dk // 32, j % 16
    flat = pages.reshape(-1)
    base = which.long()[j // page] * pages.shape[-1] + j % page // 16 * 18 * dk
    head = torch.arange(heads, device="cuda")[:, None, None] * (page // 16 * 18 * dk)
    w = d % 32
    k_nibble = r * dk + ((w // 8) * nb + d // 32) * 8 + (w % 8) // 2 + 4 * (w % 2)
    v_nibble = ((((d // 32) * 8 + d % 8) * 4 + r % 8 // 2) * 2 + w // 16) * 8 + (r % 2) * 4 + r // 8 * 2 + w % 16 // 8
    out = []
    for first, nibble, scale in ((0, k_nibble, 16 * dk + 2 * (r * nb + d // 32)), (8 * dk, v_nibble, 17 * dk + 2 * (d // 32 * 16 + r))):
        code = (flat[head + base + first + nibble // 2].long() >> (4 * (nibble % 2))) & 15
        bits = flat[head + base + scale].int() << 16 | flat[head + base + scale + 1].int() << 24
        out.append((code - 8).double() * bits.view(torch.float32).double())
    return out


def exact(case, seed):
    if case["op"] not in ("append", "attention"):
        return None
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_block(state["k"].unflatten(-1, (-1, case["dk"]))).flatten(1), _exact_block(state["v"].unflatten(-1, (-1, case["dk"]))).flatten(1)
    dk, heads, group = case["dk"], case["heads"], case["group"]
    q = state["q"].double().view(-1, heads, group, dk)
    o = torch.zeros_like(q)
    starts, lens = state["starts"].tolist(), state["lens"].tolist()
    for i, seq in enumerate(state["seqs"].tolist()):
        n, rows = lens[seq], starts[i + 1] - starts[i]
        k, v = _exact_rows(state["pages"][state["layer"]], dk, case["page"], heads, state["table"][seq], n)
        j = torch.arange(n, device="cuda")
        step = max(1, (1 << 28) // (n * heads * group))
        for a in range(0, rows, step):
            part = q[starts[i] + a:starts[i] + min(rows, a + step)]
            pos = n - rows + a + torch.arange(len(part), device="cuda")[:, None]
            seen = torch.ones((len(part), n), dtype=torch.bool, device="cuda")
            if case["causal"]:
                seen &= j <= pos
            if case["window"]:
                seen &= j > pos - case["window"]
            s = torch.einsum("rhgd,hjd->hgrj", part, k) / math.sqrt(dk)
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            o[starts[i] + a:starts[i] + min(rows, a + step)] = torch.einsum("hgrj,hjd->rhgd", p, v)
    return o.flatten(1)
