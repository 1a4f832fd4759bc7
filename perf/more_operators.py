"""Attention over a cache of keys and values held in 4 bits, and eviction from it by accumulated attention weight, as programs call them.

Five operators:

* ``append4``: rows of keys and values are rounded to 4 bits and enter the pages of a cache: x = n s, n in -8 .. 7, s (bfloat16) the
  largest |x| of a group of 32, 64 or 128 values of a head's row, divided by 7.  The case reads the rows back as a program would
  (``cache4_values``), so that its result is what the cache stands for.
* ``decode_attention4``: attention of one new token a request over its pages, where asked for with what each key gained in attention
  weight, added to what it had (``mass`` into ``total``).
* ``prefill_attention4``: the same for portions of several tokens a request, under the causal mask.
* ``evict4``: a request and key/value head keeps its newest keys and, of the others, those with the most accumulated weight; they go to
  fresh pages (the old ones may be shared with other requests) in their order, their weights with them.

A state holds what a program holds: the cache and its block tables, the queries, output buffers.
"""
from __future__ import annotations

import math

import torch

own = False


# ---- the cases ---------------------------------------------------------------------------------------------

def _append(tokens, kv, dim, group, page=16):
    return dict(op="append4", tokens=tokens, kv=kv, dim=dim, group=group, page=page)


def _decode(seqs, keys, heads, kv, dim, group, page=16, ragged=False, mass=False, window=0, sink=False, cap=0.0, idle=False):
    return dict(op="decode_attention4", seqs=seqs, keys=keys, heads=heads, kv=kv, dim=dim, group=group, page=page, ragged=ragged, mass=mass, window=window, sink=sink,
                cap=cap, idle=idle)


def _prefill(seqs, new, past, heads, kv, dim, group, page=16, ragged=False, mass=False, window=0, sink=False, cap=0.0):
    return dict(op="prefill_attention4", seqs=seqs, new=new, past=past, heads=heads, kv=kv, dim=dim, group=group, page=page, ragged=ragged, mass=mass, window=window,
                sink=sink, cap=cap)


def _evict(seqs, keys, keep, recent, kv, dim, group, page=16, ragged=False):
    return dict(op="evict4", seqs=seqs, keys=keys, keep=keep, recent=recent, kv=kv, dim=dim, group=group, page=page, ragged=ragged)


def listed():
    named = {
        # A busy server's decode step: the new token's key and value of each request.
        "append_64": _append(64, 8, 128, 64),
        # The prompts of a step.
        "append_4096": _append(4096, 8, 128, 32),
        # One user's next token, GPT-2 XL's heads (a key/value head each, an odd number of them): nothing but latency.
        "decode_1_512": _decode(1, 512, 25, 25, 64, 64),
        # GPT-2 XL's 64 requests, anywhere up to 1,024 positions.
        "decode_64_1024": _decode(64, 1024, 25, 25, 64, 32, ragged=True),
        # A few long conversations, four heads to a key/value head.
        "decode_8_16384": _decode(8, 16384, 32, 8, 128, 64, page=64),
        # One very long document.
        "decode_1_131072": _decode(1, 131072, 32, 8, 128, 128, page=128),
        # A server that keeps account of what its keys are worth, with sinks.
        "decode_mass_16_4096": _decode(16, 4096, 32, 8, 128, 64, ragged=True, mass=True, sink=True),
        # A draft of four tokens and the one before, checked at once.
        "verify_8x5_2048": _prefill(8, 5, 2048, 32, 8, 128, 64, ragged=True),
        # GPT-2 small's prompts: two of a whole context.
        "prefill_2x1024": _prefill(2, 1024, 0, 12, 12, 64, 64),
        # Portions of long prompts behind what is in the cache already, capped scores.
        "prefill_4x512_8192": _prefill(4, 512, 8192, 32, 8, 128, 64, page=64, cap=50.0),
        # One user's conversation halved.
        "evict_1_2048": _evict(1, 2048, 1024, 64, 12, 64, 64),
        # A server makes room: 8 requests back to a quarter of their length.
        "evict_8_8192": _evict(8, 8192, 2048, 128, 8, 128, 64, page=64, ragged=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


_MOST_FLOPS, _MOST_BYTES, _MOST_SCORES = 3.1e11, 1.45e8, 7.2e8      # of the largest listed cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """Key/value heads, query heads to each, values a head, group, page."""
    dim = rng.choice([64, 128])
    return _log_int(rng, 1, 32), rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 16]), dim, rng.choice([g for g in (32, 64, 128) if g <= dim]), rng.choice([16, 16, 32, 64, 128])


def draw(rng):
    while True:
        op = rng.choice(["append4", "decode_attention4", "decode_attention4", "prefill_attention4", "prefill_attention4", "evict4"])
        kv, per, dim, group, page = _heads(rng)
        ragged = rng.random() < 0.6
        more = dict(ragged=ragged, mass=rng.random() < 0.3, window=rng.choice([0, 0, 0, 512, 100]), sink=rng.random() < 0.25, cap=rng.choice([0.0, 0.0, 0.0, 50.0]))
        if op == "append4":
            c = _append(_log_int(rng, 1, 8192), kv, dim, group, page)
        elif op == "decode_attention4":
            c = _decode(_log_int(rng, 1, 128), _log_int(rng, 1, 131072), kv * per, kv, dim, group, page, idle=rng.random() < 0.2, **more)
        elif op == "prefill_attention4":
            new = _log_int(rng, 1, 2048)
            if new > 64:
                more["mass"] = False
            c = _prefill(_log_int(rng, 1, 16), new, rng.choice([0, _log_int(rng, 1, 16384)]), kv * per, kv, dim, group, page, **more)
        else:
            keys = _log_int(rng, 32, 32768)
            keep = rng.randint(1, keys)
            c = _evict(_log_int(rng, 1, 16), keys, keep, rng.randint(0, min(keep, 256)), kv, dim, group, page, ragged)
        if op == "decode_attention4" and c["seqs"] == 1:
            c["idle"] = False
        w = work(c)
        rows = c.get("new", 1)
        keys = c.get("past", 0) + rows if op == "prefill_attention4" else c.get("keys", 1)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and c.get("seqs", 1) * (c.get("heads", 1) * rows + 4 * kv * dim) * keys <= _MOST_SCORES:
            return c


def _lengths(c):
    """The keys of each request (with its new tokens), and its new tokens; the sizes of a case are the same for every seed."""
    n = c["seqs"]
    spread = [1.0 - 0.83 * ((7 * i + 3) % n) / n if c["ragged"] else 1.0 for i in range(n)]
    if c["op"] == "prefill_attention4":
        new = [max(1, int(c["new"] * (1.0 - 0.5 * ((5 * i + 1) % n) / n))) if c["ragged"] and c["new"] > 8 else c["new"] for i in range(n)]
        return [int(c["past"] * f) + m for f, m in zip(spread, new)], new
    keys = [max(1, int(c["keys"] * f)) for f in spread]
    if c.get("idle"):
        keys[n // 2] = 0                # a place of the batch that no request has
    return keys, [1] * n


def _seen(c, keys, new):
    """Query-key pairs, and keys that any of a request's queries sees."""
    pairs = seen = 0
    for n, m in zip(keys, new):
        if n == 0:
            continue
        w = c["window"] if c["window"] > 0 else n
        seen += min(n, w + m - 1)
        pairs += sum(min(w, n - m + i + 1) for i in range(m))
    return pairs, seen


def work(case):
    c = case
    row = c["kv"] * (c["dim"] + 4 * c["dim"] // c["group"])             # bytes of a key and its value, scales included
    if c["op"] == "append4":
        n = c["tokens"]
        # The rows, the cache's bytes twice (written, read back), the values.
        return {"bytes": n * (2 * row + 8 * c["kv"] * c["dim"] + 8), "flops": 6 * n * c["kv"] * c["dim"]}
    keys, new = _lengths(c)
    if c["op"] == "evict4":
        kept = sum(min(n, c["keep"]) for n in keys)
        # The weights read; the kept keys' rows read, written and read back; their values, weights and numbers.
        return {"bytes": 4 * c["kv"] * sum(keys) + kept * (3 * row + 4 * c["kv"] * c["dim"] + 8 * c["kv"]), "flops": c["kv"] * (sum(keys) + 2 * kept * c["dim"])}
    pairs, seen = _seen(c, keys, new)
    q = sum(new) * c["heads"] * c["dim"]
    return {"bytes": seen * row + 4 * q + (8 * c["kv"] * sum(keys) if c["mass"] else 0), "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---- what a program has in hand ----------------------------------------------------------------------------

def _kv_rows(gen, n, kv, dim):
    """Key and value rows of a trained model: keys have channels of their own size and offset, rows differ in size."""
    spread = torch.exp(0.5 * torch.randn(1, kv * dim, generator=gen, device="cuda"))
    offset = torch.randn(1, kv * dim, generator=gen, device="cuda")
    k = (torch.randn(n, kv * dim, generator=gen, device="cuda") * spread + offset).to(torch.bfloat16)
    v = (torch.randn(n, kv * dim, generator=gen, device="cuda") * torch.exp(0.3 * torch.randn(n, 1, generator=gen, device="cuda"))).to(torch.bfloat16)
    return k, v


def _tables(gen, lengths, page, room=0):
    """Block tables of requests with this many keys, their pages anywhere in the cache; (table [seqs, most pages], pages)."""
    pages = [max(1, -(-n // page)) for n in lengths]
    order = torch.randperm(sum(pages) + room, generator=gen, device="cuda").to(torch.int32)
    at = torch.tensor([0] + pages[:-1], device="cuda").cumsum(0)
    column = torch.arange(max(pages), device="cuda")
    index = at[:, None] + torch.minimum(column[None, :], torch.tensor(pages, device="cuda")[:, None] - 1)
    return order[index].contiguous(), order, sum(pages) + room


def _slots(table, lengths, page):
    """The slots of all keys of all requests, one request after the other."""
    parts = [table[i, torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda", dtype=torch.int32) % page for i, n in enumerate(lengths) if n > 0]
    return torch.cat(parts).to(torch.int32)


def _round4(x, kv, dim, group):
    """Rows to 4 bits: (n int8 [rows, kv, dim], s bfloat16 [rows, kv, dim / group])."""
    g = x.float().view(x.shape[0], kv, dim // group, group)
    s = (g.abs().amax(3) / torch.full((), 7.0, device=x.device)).to(torch.bfloat16)      # (a divisor on the GPU: a number on the host would become a product with its reciprocal)
    t = s.float()[..., None]
    n = torch.where(t > 0, (g / torch.where(t > 0, t, torch.ones_like(t))).round().clamp(-8, 7), torch.zeros_like(g))
    return n.view(-1, kv, dim).to(torch.int8), s


def _fill(c, slots, k, v, pages):
    """A cache with these rows at these slots: the framework's, or the plain form's (n, s) by slot."""
    if own:
        from liyab_b200 import ops
        cache = ops.Cache4(pages, c["kv"], c["dim"], c["page"], c["group"])
        ops.append4(k, v, slots, cache, slots.numel())
        return cache
    cache = dict(n=torch.zeros(2, pages * c["page"], c["kv"], c["dim"], dtype=torch.int8, device="cuda"),
                 s=torch.zeros(2, pages * c["page"], c["kv"], c["dim"] // c["group"], dtype=torch.bfloat16, device="cuda"))
    for half, rows in enumerate((k, v)):
        for at in range(0, rows.shape[0], 32768):
            n, s = _round4(rows[at:at + 32768], c["kv"], c["dim"], c["group"])
            cache["n"][half, slots[at:at + 32768].long()], cache["s"][half, slots[at:at + 32768].long()] = n, s
    return cache


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev, bf16 = "cuda", torch.bfloat16
    if c["op"] == "append4":
        n, width = c["tokens"], c["kv"] * c["dim"]
        k, v = _kv_rows(gen, n, c["kv"], c["dim"])
        pages = -(-n // c["page"]) + 3
        slots = torch.randperm(pages * c["page"], generator=gen, device=dev)[:n].to(torch.int32)
        cache = _fill(c, slots[:0], k[:0], v[:0], pages)
        return dict(c=c, k=k, v=v, slots=slots, cache=cache, k_out=torch.empty(n, width, dtype=bf16, device=dev), v_out=torch.empty(n, width, dtype=bf16, device=dev))
    keys, new = _lengths(c)
    page = c["page"]
    room = c["seqs"] * -(-c["keep"] // page) if c["op"] == "evict4" else 0
    table, order, pages = _tables(gen, keys, page, room)
    slots = _slots(table, keys, page)
    k, v = _kv_rows(gen, slots.numel(), c["kv"], c["dim"])
    s = dict(c=c, cache=_fill(c, slots, k, v, pages), table=table, n_keys=torch.tensor(keys, dtype=torch.int32, device=dev))
    most = table.shape[1] * page
    if c["op"] == "evict4":
        # Weights gathered over many steps: a few keys have most of it, many nothing at all.
        mass = torch.exp(2.5 * torch.randn(c["seqs"], c["kv"], most, generator=gen, device=dev))
        s["mass"] = torch.where(torch.rand(c["seqs"], c["kv"], most, generator=gen, device=dev) < 0.2, torch.zeros_like(mass), mass)
        s["dest"] = order[pages - room:].view(c["seqs"], -1).contiguous()
        s["dest_mass"] = torch.zeros(c["seqs"], c["kv"], c["keep"], device=dev)
        s["kept"] = torch.full((c["seqs"], c["kv"], c["keep"]), -1, dtype=torch.int32, device=dev)
        at = torch.arange(c["keep"], device=dev)
        slot = s["dest"].long()[:, at // page] * page + at % page
        s["slots"] = torch.where(at[None, :] < s["n_keys"][:, None], slot, -1).to(torch.int32).view(-1)
        s["k_out"], s["v_out"] = (torch.zeros(c["seqs"] * c["keep"], c["kv"] * c["dim"], dtype=bf16, device=dev) for _ in range(2))
        return s
    # Scores of a spread of about one and a half, as trained heads have: a few keys take most of a token's weight.
    row_size = k[:2048].float().view(-1, c["kv"], c["dim"]).square().sum(2).mean().sqrt()
    tokens = sum(new)
    s["q"] = (torch.randn(tokens, c["heads"] * c["dim"], generator=gen, device=dev) * (1.5 * math.sqrt(c["dim"]) / row_size)).to(bf16)
    s["out"] = torch.zeros(tokens, c["heads"] * c["dim"], dtype=bf16, device=dev)
    s["sink"] = torch.randn(c["heads"], generator=gen, device=dev) if c["sink"] else None
    s["mass"] = torch.rand(c["seqs"], c["kv"], most, generator=gen, device=dev) if c["mass"] else None
    s["total"] = torch.zeros_like(s["mass"]) if c["mass"] else None
    s["new"] = new
    s["max_keys"] = max(keys)
    if c["op"] == "decode_attention4":
        s["positions"] = s["n_keys"] - 1
    else:
        s["q_start"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
        s["n_past"] = (s["n_keys"] - torch.tensor(new, device=dev)).to(torch.int32)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------

def _plain_append(s):
    c = s["c"]
    at = s["slots"].long()
    for half, rows in enumerate((s["k"], s["v"])):
        s["cache"]["n"][half, at], s["cache"]["s"][half, at] = _round4(rows, c["kv"], c["dim"], c["group"])
    return _plain_values(c, s["cache"], at)


def _plain_values(c, cache, at):
    n, step = cache["n"][:, at].float(), cache["s"][:, at].float()
    x = (n.unflatten(3, (-1, c["group"])) * step[..., None]).to(torch.bfloat16).view(2, at.numel(), -1)
    return x[0], x[1]


def _plain_attention(s):
    """All requests at once, their keys padded to the longest's."""
    c, page = s["c"], s["c"]["page"]
    n_seq, kv, per, dim = c["seqs"], c["kv"], c["heads"] // c["kv"], c["dim"]
    most, new = s["max_keys"], max(s["new"])
    key = torch.arange(most, device="cuda")
    at = s["table"].long()[:, key // page] * page + key % page                                            # [seqs, keys]
    k, v = ((s["cache"]["n"][half][at].float().unflatten(3, (-1, c["group"])) * s["cache"]["s"][half][at].float()[..., None]).flatten(3).permute(0, 2, 1, 3) for half in (0, 1))
    if c["op"] == "decode_attention4":
        token = torch.arange(n_seq, device="cuda")[:, None]
        there = torch.ones_like(token, dtype=torch.bool)
        pos = s["positions"].long()[:, None]
    else:
        start, step = s["q_start"].long(), torch.arange(new, device="cuda")[None, :]
        there = step < (start[1:] - start[:-1])[:, None]
        token = torch.where(there, start[:-1, None] + step, 0)
        pos = s["n_past"].long()[:, None] + step
    q = s["q"].float()[token].view(n_seq, new, kv, per, dim).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, per * new, dim)
    score = (q @ k.transpose(2, 3)).view(n_seq, kv, per, new, most) / math.sqrt(dim)
    if c["cap"] > 0:
        score = c["cap"] * torch.tanh(score / c["cap"])
    seen = (key <= pos[..., None]) & there[..., None]
    if c["window"] > 0:
        seen = seen & (key > pos[..., None] - c["window"])
    seen = seen[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, -1e30))
    top = score.amax(4, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(kv, per, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.where(seen, torch.exp(score - top), torch.zeros_like(score))
    below = p.sum(4, keepdim=True)
    if s["sink"] is not None:
        below = below + torch.exp(sink - top)
    p = p / torch.where(below > 0, below, torch.ones_like(below))
    o = (p.view(n_seq, kv, per * new, most) @ v).view(n_seq, kv, per, new, dim).permute(0, 3, 1, 2, 4).reshape(n_seq, new, -1)
    out = torch.zeros(s["q"].shape, dtype=torch.bfloat16, device="cuda")
    out[token[there]] = o[there].to(torch.bfloat16)
    if s["mass"] is None:
        return out
    total = torch.zeros_like(s["mass"])
    total[:, :, :most] = torch.where(key < s["n_keys"][:, None, None], s["mass"][:, :, :most] + p.sum((2, 3)), torch.zeros_like(s["mass"][:, :, :most]))
    return out, total


def _plain_evict(s):
    c, page = s["c"], s["c"]["page"]
    n_seq, kv, keep, most = c["seqs"], c["kv"], c["keep"], s["mass"].shape[2]
    key, n = torch.arange(most, device="cuda"), s["n_keys"].long()[:, None, None]
    # The newest first, then by weight (a stable sort: equal weights in the order of their positions), what is not there last.
    rank = torch.where(key >= n - c["recent"], torch.full_like(s["mass"], math.inf), s["mass"])
    rank = torch.where(key < n, rank, torch.full_like(s["mass"], -math.inf))
    kept = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    there = torch.arange(keep, device="cuda") < n
    kept = torch.sort(torch.where(there, kept, most), dim=2).values
    index = torch.where(there, kept, 0)
    from_slot = torch.gather(s["table"].long()[:, None, :].expand(-1, kv, -1), 2, index // page) * page + index % page
    head = torch.arange(kv, device="cuda")[None, :, None]
    n4, s4 = s["cache"]["n"][:, from_slot, head], s["cache"]["s"][:, from_slot, head]                     # [2, seqs, kv, keep, ..]
    row = torch.arange(keep, device="cuda")
    to_slot = (s["dest"].long()[:, row // page] * page + row % page)[:, None, :].expand(-1, kv, -1)
    i, h, _ = torch.nonzero(there.expand(-1, kv, -1), as_tuple=True)
    where = there.expand(-1, kv, -1)
    s["cache"]["n"][:, to_slot[where], h], s["cache"]["s"][:, to_slot[where], h] = n4[:, where], s4[:, where]
    x = (n4.float().unflatten(4, (-1, c["group"])) * s4.float()[..., None]).flatten(4)
    x = torch.where(there[None, ..., None], x, torch.zeros_like(x)).to(torch.bfloat16).permute(0, 1, 3, 2, 4).reshape(2, n_seq * keep, -1)
    mass = torch.where(there, torch.gather(s["mass"], 2, index), torch.zeros((), device="cuda"))
    return torch.where(there, kept, -1).to(torch.int32), mass, x[0], x[1]


def run(state):
    s = state
    c = s["c"]
    if not own:
        return _plain_append(s) if c["op"] == "append4" else _plain_evict(s) if c["op"] == "evict4" else _plain_attention(s)
    from liyab_b200 import ops
    if c["op"] == "append4":
        ops.append4(s["k"], s["v"], s["slots"], s["cache"], c["tokens"])
        return ops.cache4_values(s["cache"], s["slots"], c["tokens"], s["k_out"], s["v_out"])
    if c["op"] == "evict4":
        ops.evict4(s["cache"], s["mass"], s["table"], s["n_keys"], c["seqs"], c["keep"], c["recent"], s["dest"], s["kept"], s["dest_mass"])
        return (s["kept"], s["dest_mass"], *ops.cache4_values(s["cache"], s["slots"], s["slots"].numel(), s["k_out"], s["v_out"]))
    more = dict(window=c["window"], sink=s["sink"], soft_cap=c["cap"], mass=s["mass"], total=s["total"], max_keys=s["max_keys"])
    scale = 1.0 / math.sqrt(c["dim"])
    if c["op"] == "decode_attention4":
        ops.decode_attention4(s["q"], s["cache"], s["positions"], s["table"], s["out"], c["seqs"], c["heads"], scale, **more)
    else:
        ops.prefill_attention4(s["q"], s["cache"], s["q_start"], s["n_past"], s["table"], s["out"], c["seqs"], c["new"], c["heads"], scale, **more)
    return s["out"] if s["mass"] is None else (s["out"], s["total"])


# ---- the definition in 64 bits -----------------------------------------------------------------------------

def _exact_rows(cache, group, slots):
    """Keys and values [keys, kv, dim] of these slots."""
    f64 = torch.float64
    return [cache["n"][half].index_select(0, slots).to(f64).mul(cache["s"][half].index_select(0, slots).to(f64).repeat_interleave(group, dim=2)) for half in (0, 1)]


def exact(case, seed):
    """What the operators' definitions give in 64 bits, one request after the other."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, f64 = case, torch.float64
    kv, dim, group, page = c["kv"], c["dim"], c["group"], c["page"]
    if c["op"] == "append4":
        result = []
        for rows in (s["k"], s["v"]):
            x = rows.to(f64).reshape(-1, kv * dim // group, group)
            step = x.abs().max(dim=2).values.div(7).to(torch.bfloat16).to(f64).unsqueeze(2)
            n = torch.nan_to_num(x.div(step)).round().clamp(min=-8, max=7)
            result.append(n.mul(step).view(rows.shape))
        return tuple(result)
    lengths = s["n_keys"].tolist()
    if c["op"] == "evict4":
        kept, mass = torch.full_like(s["kept"], -1), torch.zeros(s["dest_mass"].shape, dtype=f64, device="cuda")
        out = [torch.zeros(c["seqs"], c["keep"], kv, dim, dtype=f64, device="cuda") for _ in range(2)]
        for i, n in enumerate(lengths):
            old, m = max(0, n - c["recent"]), min(n, c["keep"])
            slots = s["table"][i].long().mul(page).unsqueeze(1).add(torch.arange(page, device="cuda")).view(-1)[:n]
            rows = _exact_rows(s["cache"], group, slots)
            for h in range(kv):
                by_weight = torch.argsort(s["mass"][i, h, :old], descending=True, stable=True)[:m - (n - old)] if m > n - old else slots[:0]
                choice = torch.cat([by_weight, torch.arange(old, n, device="cuda")]).sort().values
                kept[i, h, :m], mass[i, h, :m] = choice.to(torch.int32), s["mass"][i, h, choice].to(f64)
                for half in (0, 1):
                    out[half][i, :m, h] = rows[half][choice, h]
        return kept, mass, out[0].view(-1, kv * dim), out[1].view(-1, kv * dim)
    per, out = c["heads"] // kv, torch.zeros(s["q"].shape, dtype=f64, device="cuda")
    total = torch.zeros(s["total"].shape, dtype=f64, device="cuda") if c["mass"] else None
    token = 0
    for i, n in enumerate(lengths):
        new = s["new"][i]
        if n > 0:
            slots = s["table"][i].long().mul(page).unsqueeze(1).add(torch.arange(page, device="cuda")).view(-1)[:n]
            k, v = _exact_rows(s["cache"], group, slots)
            place, key = torch.arange(n - new, n, device="cuda").unsqueeze(1), torch.arange(n, device="cuda").unsqueeze(0)
            hidden = key.gt(place) if c["window"] <= 0 else key.gt(place) | key.le(place - c["window"])
            for h in range(c["heads"]):
                z = s["q"][token:token + new, h * dim:(h + 1) * dim].to(f64).mm(k[:, h // per].t()).mul(dim ** -0.5)
                if c["cap"] > 0:
                    z = z.div(c["cap"]).tanh().mul(c["cap"])
                z = z.masked_fill(hidden, -math.inf)
                if s["sink"] is not None:
                    z = torch.cat([z, s["sink"][h].to(f64).expand(new, 1)], dim=1)
                p = torch.softmax(z, dim=1)[:, :n]
                out[token:token + new, h * dim:(h + 1) * dim] = p.mm(v[:, h // per])
                if total is not None:
                    total[i, h // per, :n] += p.sum(dim=0)
            if total is not None:
                total[i, :, :n] += s["mass"][i, :, :n].to(f64)
        token += new
    return out if total is None else (out, total)
