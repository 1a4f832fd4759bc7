"""The 4-bit cache: its rounding, attention of single tokens and of portions over it, the weights its keys gather, and eviction by them, against plain forms in 64 bits."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from liyab_b200 import ops
from test_cache4 import AT, _call
from test_kernels_gpu import dev  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# ---- plain forms -------------------------------------------------------------------------------------------

def _rounded(x, kv, dim, group):
    """(n, s) of rows [rows, kv * dim] by the cache's rule: n int8 [rows, kv, dim], s bfloat16 [rows, kv, dim / group]."""
    g = x.float().view(x.shape[0], kv, dim // group, group)
    top = g.abs().amax(3)
    s = (top / torch.full_like(top, 7.0)).to(BF16)
    s = torch.where(top.isfinite(), s, torch.full_like(s, math.nan))
    t = s.float()[..., None].expand_as(g)                    # quotients are rounded to 32 bits
    n = torch.where(t > 0, (g / torch.where(t > 0, t, torch.ones_like(t))).round().clamp(-8, 7), torch.zeros_like(g))
    return n.view(-1, kv, dim).to(torch.int8), s


def _values(n, s, group):
    return n.double() * s.double().repeat_interleave(group, 2)


def _tables(lengths, page, gen, extra=0):
    """Block tables [requests, most pages] of pages in any order, the pages of the cache; entries past a request's pages are far outside."""
    pages = [-(-n // page) for n in lengths]
    total = sum(pages) + extra
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(pages))), 1 << 30, dtype=torch.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table, order[at:], total


def _slots(table, i, n, page):
    key = torch.arange(n)
    return (table[i, key // page].long() * page + key % page).to(torch.int32)


class Filled:
    """A cache with these requests' keys, and their values in 64 bits: k[i], v[i] [keys, kv, dim]."""

    def __init__(self, dev, lengths, kv, dim, group, page=16, seed=0, extra=0, k_size=1.0, v_size=1.0, spread=0.0):
        from liyab_b200 import ops
        gen = torch.Generator().manual_seed(seed)
        self.table, self.spare, self.pages = _tables(lengths, page, gen, extra)
        self.cache = ops.Cache4(max(1, self.pages), kv, dim, page, group)
        self.cache.memory.fill_(255)                       # what no key has been written to: scales that are NaN
        self.k, self.v = [], []
        for i, n in enumerate(lengths):
            k, v = (torch.randn(n, kv * dim, generator=gen) * size * torch.exp(spread * torch.randn(n, 1, generator=gen)) for size in (k_size, v_size))
            k, v = k.to(BF16).to(dev), v.to(BF16).to(dev)
            if n:
                ops.append4(k, v, _slots(self.table, i, n, page).to(dev), self.cache, n)
            self.k.append(_values(*_rounded(k, kv, dim, group), group))
            self.v.append(_values(*_rounded(v, kv, dim, group), group))
        self.lengths, self.dev, self.kv, self.dim, self.table = lengths, dev, kv, dim, self.table.to(dev)


def _attention(q, k, v, places, scale, window=0, distance=None, sink=None, cap=0.0, many=False):
    """(out [tokens, heads, dim], the weights [tokens, heads, keys], the bound on out's error before its rounding, the relative bound on the weights') in 64 bits.
    q [tokens, heads, dim]; k, v [keys, kv, dim]; places: of the tokens."""
    tokens, heads, dim = q.shape
    keys, kv = k.shape[0], k.shape[1]
    per = heads // kv
    key = torch.arange(keys, device=q.device)
    out, weights = torch.zeros(tokens, heads, dim, dtype=F64, device=q.device), torch.zeros(tokens, heads, keys, dtype=F64, device=q.device)
    bound, relative = torch.zeros_like(out), torch.zeros(tokens, heads, device=q.device, dtype=F64)
    for h in range(heads):
        kh, vh = k[:, h // per], v[:, h // per]
        z = q[:, h].double() @ kh.T * scale
        # Sums of 16 products at a time, each with an error below 2^-23 of the sum of the terms' sizes; the scales, the cap and the penalty add a few roundings of their own terms.
        size = (q[:, h].double().abs() @ kh.abs().T * abs(scale)).amax(1) if keys else torch.zeros(tokens, dtype=F64, device=q.device)
        error = (dim / 16 + 16) * 2.0 ** -23 * size
        # A row of queries is rounded to 16 bits in steps of at most 2^-14 of its largest value: what has more of bfloat16's eight bits below that is off by up to half a step.
        if keys:
            large = q[:, h].double().abs().amax(1, keepdim=True)
            error = error + ((q[:, h].double().abs() < large * 2.0 ** -6).double() * large * 2.0 ** -15 @ kh.abs().T * abs(scale)).amax(1)
        # The kernel for many rows multiplies n s (4 bits by 8) as float16, off by up to 2^-12.
        if many:
            error = error + 2.0 ** -12 * size
        if cap > 0:
            z = cap * torch.tanh(z / cap)
            error = error + 16 * 2.0 ** -23 * cap
        if distance is not None:
            d = (places[:, None] - key[None, :]).clamp(min=0).double()
            r1, r2 = float(distance[h]), float(distance[heads + h])
            z = z - (r1 * d if r2 < 0 else r1 * torch.log1p(r2 * d))
            error = error + 2.0 ** -20 * abs(r1) * (1.0 + (d.amax(1) if r2 < 0 else math.log1p(r2 * max(1, keys))))
        seen = key[None, :] <= places[:, None]
        if window > 0:
            seen &= key[None, :] > places[:, None] - window
        elif window < 0:
            seen &= key[None, :] >= places[:, None].clamp(min=0) // -window * -window
        z = z.masked_fill(~seen, -math.inf)
        if sink is not None:
            z = torch.cat([z, sink[h].double().expand(tokens, 1)], 1)
        none = ~seen.any(1) & (sink is None)
        p = torch.softmax(z.masked_fill(none[:, None], 0.0), 1)[:, :keys].masked_fill(~seen, 0.0)
        out[:, h], weights[:, h] = p @ vh, p
        # A weight is off by its score's error (twice: in the sum as well) and 2^-20 of exponentials; times a scale it is rounded to float16 (2^-11), and the sums over the keys add theirs.
        relative[:, h] = 2 * error + 2.0 ** -20
        bound[:, h] = (p @ vh.abs()) * (2.0 ** -11 + (keys / 16 + 16) * 2.0 ** -23 + 2 * relative[:, h, None])
        # Products p s below float16's normal numbers are off by up to half its smallest number, 2^-25.  They are in units of f, at least 2^-6 of the largest scale's exponent's power of
        # two, so 2^-30 of the largest scale; a value is at most 8 scales, and a scale a seventh of the largest value or little more: 8 / 6.9 2^-30 of that, each key.
        if keys:
            bound[:, h] += keys * 2.0 ** -29 * vh.abs().max()
    return out, weights, bound, relative


def _close(got, want, bound):
    """got (bfloat16) within the bound and its own rounding."""
    error = (got.double() - want).abs()
    allowed = bound + (want.abs() + bound) * 2.0 ** -8 + 2.0 ** -133
    worst = (error - allowed).max().item() if error.numel() else 0.0
    assert not error.isnan().any() and worst <= 0, f"off by {worst} more than allowed"


def _queries(f, tokens, heads, seed, size=1.0):
    gen = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(tokens, heads * f.dim, generator=gen) * size).to(BF16).to(f.dev)


# ---- rows in and out ---------------------------------------------------------------------------------------

FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("kv,page,n", [(1, 16, 1), (3, 16, 50), (2, 64, 200), (25, 32, 33)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_in_and_out(dev, dim, group, kv, page, n, dtype):
    from liyab_b200 import ops
    gen = torch.Generator().manual_seed(n)
    k, v = ((torch.randn(n, kv * dim, generator=gen) * torch.exp(2 * torch.randn(n, 1, generator=gen))).to(dtype).to(dev) for _ in range(2))
    k[0, :group] = 0.0                                    # a group of zeros
    v[n // 2, group - 1] = 1e30 if dtype is F32 else 1e20
    pages = -(-n // page) + 2
    cache = ops.Cache4(pages, kv, dim, page, group)
    cache.memory.fill_(255)
    slots = torch.randperm(pages * page, generator=gen)[:n].to(torch.int32)
    slots[n // 3] = -1 if n > 1 else slots[0]
    ops.append4(k, v, slots.to(dev), cache, n)
    for out_type in (F32, BF16):
        ko, vo = (torch.full((n, kv * dim), 7.5, dtype=out_type, device=dev) for _ in range(2))
        ops.cache4_values(cache, slots.to(dev), n, ko, vo)
        for got, rows in ((ko, k), (vo, v)):
            want = _values(*_rounded(rows, kv, dim, group), group).to(F32).to(out_type).view(n, -1)       # n s is exact in 32 bits
            if n > 1:
                want[n // 3] = 7.5                        # a skipped row is left alone
            assert torch.equal(got, want)


@pytest.mark.parametrize("dim,group", FORMS)
def test_rows_of_any_place(dev, dim, group):
    """Rows off the 16 bytes, of other strides for keys and values, values as results of a wider buffer."""
    from liyab_b200 import ops
    n, kv = 37, 3
    wide = torch.randn(n, 3 * kv * dim + 5, generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    other = torch.randn(n, kv * dim + 1, generator=torch.Generator().manual_seed(4)).to(BF16).to(dev)
    k, v = wide[:, 3:3 + kv * dim], other[:, 1:]
    cache, slots = ops.Cache4(3, kv, dim, 16, group), torch.arange(47, 47 - n, -1, dtype=torch.int32, device=dev)
    ops.append4(k, v, slots, cache, n)
    back = torch.full((n, 2 * kv * dim + 3), 7.5, device=dev)
    ops.cache4_values(cache, slots, n, back[:, 1:1 + kv * dim], back[:, 2 + kv * dim:2 + 2 * kv * dim])
    assert torch.equal(back[:, 1:1 + kv * dim], _values(*_rounded(k, kv, dim, group), group).float().view(n, -1))
    assert torch.equal(back[:, 2 + kv * dim:2 + 2 * kv * dim], _values(*_rounded(v, kv, dim, group), group).float().view(n, -1))
    assert (back[:, 0] == 7.5).all() and (back[:, 1 + kv * dim] == 7.5).all() and (back[:, -1] == 7.5).all()


def test_rows_that_are_not_finite_and_rows_of_all_sizes(dev):
    from liyab_b200 import ops
    kv, dim, group = 2, 128, 32
    k = torch.randn(9, kv * dim, generator=torch.Generator().manual_seed(5)).to(dev)
    k[0, 5], k[1, 40], k[2, 100] = math.inf, -math.inf, math.nan
    k[3] *= 3e38 / k[3].abs().max()
    k[4] *= 1e-37
    k[5] *= 1e-44
    k[6] = 1e-45
    k[7] = 0.0
    cache, slots = ops.Cache4(1, kv, dim, 16, group), torch.arange(9, dtype=torch.int32, device=dev)
    ops.append4(k, -k, slots, cache, 9)
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    ops.cache4_values(cache, slots, 9, ko, vo)
    n, s = _rounded(k, kv, dim, group)
    want = (n.float() * s.float().repeat_interleave(group, 2)).view(9, -1)
    assert torch.equal(ko.isnan(), want.isnan()) and ko.isnan().sum() == 3 * group
    assert torch.equal(ko.nan_to_num(0.0), want.nan_to_num(0.0))
    # Half steps round to the even number on both sides of zero, so that -x becomes minus what x becomes.
    assert torch.equal(vo.nan_to_num(0.0), -want.nan_to_num(0.0))


def test_slots_outside_the_cache_are_skipped(dev):
    from liyab_b200 import ops
    cache = ops.Cache4(2, 1, 64, 16, 64)
    cache.memory.zero_()
    rows = torch.randn(4, 64, device=dev)
    ops.append4(rows, rows, torch.tensor([-1, 32, 1 << 30, -(1 << 31)], dtype=torch.int32, device=dev), cache, 4)
    assert not cache.memory.any()
    out = torch.full((4, 64), 7.5, device=dev)
    ops.cache4_values(cache, torch.tensor([-5, 32, 1 << 30, -(1 << 31)], dtype=torch.int32, device=dev), 4, out, out.clone())
    assert (out == 7.5).all()


# ---- single tokens -----------------------------------------------------------------------------------------

def _decode(f, heads, seed=0, scale=None, size=1.0, places=None, mass=False, max_keys=0, **more):
    """decode_attention4 beside the plain form, for every request; returns (out, total)."""
    from liyab_b200 import ops
    n, scale = len(f.lengths), 1 / math.sqrt(f.dim) if scale is None else scale
    q = _queries(f, n, heads, seed, size)
    places = [m - 1 for m in f.lengths] if places is None else places
    positions = torch.tensor(places, dtype=torch.int32, device=f.dev)
    out = torch.full((n, heads * f.dim), 7.5, dtype=BF16, device=f.dev)
    cells = f.table.shape[1] * f.cache.page_size
    before = torch.rand(n, f.kv, cells, generator=torch.Generator().manual_seed(seed)).to(f.dev) if mass else None
    total = torch.full_like(before, 7.5) if mass else None
    ops.decode_attention4(q, f.cache, positions, f.table, out, n, heads, scale, mass=before, total=total, max_keys=max_keys, **more)
    plain = {k: v for k, v in more.items() if k in ("window", "distance", "sink")} | dict(cap=more.get("soft_cap", 0.0))
    for i in range(n):
        m = places[i] + 1
        want, weights, bound, relative = _attention(q[i:i + 1].view(1, heads, f.dim), f.k[i][:m], f.v[i][:m], torch.tensor([places[i]], device=f.dev), scale, **plain)
        _close(out[i].view(1, heads, f.dim), want, bound)
        if mass:
            gained = weights.view(f.kv, heads // f.kv, m).sum(1)
            allowed = gained * (3 * relative.max() + (heads // f.kv + 2) * 2.0 ** -23) + (before[i, :, :m].double() + gained) * 2.0 ** -23
            assert ((total[i, :, :m].double() - before[i, :, :m].double() - gained).abs() <= allowed).all()
            assert (total[i, :, m:] == 7.5).all()            # behind the request's newest key
    return out, total


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (25, 25), (8, 2), (15, 3), (16, 1), (24, 2), (40, 2)])
def test_decode_forms(dev, dim, group, heads, kv):
    f = Filled(dev, [1, 15, 16, 17, 100, 333], kv, dim, group, seed=heads)
    _decode(f, heads, seed=dim)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("lengths", [[1], [5000], [2, 3000, 0, 129], [700] * 40])
def test_decode_lengths_and_pages(dev, page, lengths):
    _decode(Filled(dev, lengths, 2, 64, 32, page, seed=page), 6)
    _decode(Filled(dev, lengths, 1, 128, 64, page, seed=page + 1), 8)


@pytest.mark.parametrize("dim,group,kv,heads", [(128, 64, 1, 4), (64, 64, 2, 2), (128, 32, 1, 12)])
def test_decode_ranges_of_one_long_request(dev, dim, group, kv, heads):
    """Keys shared by clusters of up to sixteen blocks, and by more, whose states meet in memory."""
    for n in (130, 600, 1100, 2100, 4500, 20000):
        _decode(Filled(dev, [n], kv, dim, group, 64, seed=n), heads, seed=n)


@pytest.mark.parametrize("window", [1, 15, 16, 100, 513, -1, -16, -100])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_windows(dev, window, dim):
    _decode(Filled(dev, [1, 16, 90, 300, 1000, 2500], 2, dim, 64, 32, seed=5), 8, window=window, mass=True)


@pytest.mark.parametrize("dim,group", FORMS)
def test_decode_sinks_caps_and_distances(dev, dim, group):
    heads, kv = 12, 3
    f = Filled(dev, [1, 40, 700, 1500], kv, dim, group, seed=9)
    gen = torch.Generator().manual_seed(2)
    sink = torch.randn(heads, generator=gen).to(dev) * 3
    distance = torch.cat([torch.rand(heads, generator=gen), torch.where(torch.arange(heads) % 3 == 0, -1.0, 0.3)]).to(dev)
    distance[0] = 0.01
    _decode(f, heads, sink=sink)
    _decode(f, heads, soft_cap=5.0, size=4.0)
    _decode(f, heads, distance=distance)
    _decode(f, heads, sink=sink, soft_cap=20.0, distance=distance, window=300, mass=True, size=3.0)


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 1), (12, 1), (48, 2)])
def test_decode_weights(dev, heads, kv):
    """The keys' weights, of one tile of rows and of several, and back into mass."""
    from liyab_b200 import ops
    f = Filled(dev, [1, 31, 400, 0, 1800], kv, 128, 64, seed=heads)
    out, total = _decode(f, heads, mass=True, sink=torch.randn(heads, device=dev))
    # The weights in place, and in rows of another order; other rows stay as they were.
    positions = torch.tensor([n - 1 for n in f.lengths], dtype=torch.int32, device=dev)
    q, cells = _queries(f, 5, heads, 0), f.table.shape[1] * 16
    scale = 1 / math.sqrt(128)
    plain = torch.zeros(5, kv, cells, device=dev)
    ops.decode_attention4(q, f.cache, positions, f.table, torch.empty_like(out), 5, heads, scale, mass=plain)
    rows = torch.tensor([6, 0, 3, 2, 4], dtype=torch.int32, device=dev)
    mass = torch.full((8, kv, cells + 3), 2.0, device=dev)
    ops.decode_attention4(q, f.cache, positions, f.table, torch.empty_like(out), 5, heads, scale, mass=mass, mass_rows=rows)
    for i, r in enumerate(rows.tolist()):
        m = f.lengths[i]
        assert torch.equal(mass[r, :, :m], 2.0 + plain[i, :, :m]) and (mass[r, :, m:] == 2.0).all()
    assert (mass[[1, 5, 7]] == 2.0).all()
    assert torch.allclose(plain.sum((1, 2)), torch.tensor([0.0 if n == 0 else float(heads) for n in f.lengths], device=dev), rtol=1e-5)


def test_decode_is_the_same_every_time(dev):
    f = Filled(dev, [3000, 20, 900], 2, 128, 32, seed=4)
    a, b = _decode(f, 8, mass=True), _decode(f, 8, mass=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_of_requests_without_keys_or_pages(dev):
    """A place of the batch without keys, alone and beside others, with a sink and without; keys on pages outside the cache are not there."""
    from liyab_b200 import ops
    f = Filled(dev, [40, 0, 0, 300], 2, 64, 64, seed=1)
    for sink in (None, torch.zeros(4, device=dev)):
        out, total = _decode(f, 4, mass=True, sink=sink)
        assert not out[1:3].any()
    q, out = _queries(f, 4, 4, 0), torch.full((4, 256), 7.5, dtype=BF16, device=dev)
    table = f.table.clone()
    table[3, 5], table[0, :] = -1, 1 << 29
    ops.decode_attention4(q, f.cache, torch.tensor([39, -1, -7, 299], dtype=torch.int32, device=dev), table, out, 4, 4, 0.125)
    assert not out[:3].any()
    there = torch.tensor([k for k in range(300) if not 80 <= k < 96], device=dev)
    want, _, bound, _ = _attention(q[3:].view(1, 4, 64), f.k[3][there], f.v[3][there], torch.tensor([299], device=dev), 0.125)
    _close(out[3].view(1, 4, 64), want, bound)


def test_decode_reads_no_key_past_the_most(dev):
    """Positions past max_keys, or past the block table, are taken as the last key there."""
    from liyab_b200 import ops
    f = Filled(dev, [320], 1, 64, 64, seed=1)
    q, scale = _queries(f, 1, 2, 0), 0.125
    outs = []
    for place, most in ((99, 0), (5000, 100), (99, 100), (319, 0), (1 << 30, 0)):
        out = torch.empty(1, 128, dtype=BF16, device=dev)
        outs.append(ops.decode_attention4(q, f.cache, torch.tensor([place], dtype=torch.int32, device=dev), f.table, out, 1, 2, scale, max_keys=most))
    want, _, bound, _ = _attention(q.view(1, 2, 64), f.k[0][:100], f.v[0][:100], torch.tensor([99], device=dev), scale)
    for out in outs[:3]:
        _close(out.view(1, 2, 64), want, bound)
    assert torch.equal(outs[3], outs[4])


@pytest.mark.parametrize("k_size,v_size,q_size", [(1e-3, 1e3, 1e3), (1e4, 1e-6, 1e-4), (1e-15, 1e15, 1e15), (1.0, 1e-20, 1.0), (1.0, 1e30, 1e-30), (1e30, 1.0, 1e-30)])
def test_decode_of_all_sizes(dev, k_size, v_size, q_size):
    """Queries, keys and values that float16 does not hold, and values of sizes that differ by key."""
    for spread in (0.0, 1.5):
        f = Filled(dev, [200, 1000], 2, 128, 32, seed=8, k_size=k_size, v_size=v_size, spread=spread)
        _decode(f, 8, size=q_size, mass=True)


def test_decode_of_peaked_scores(dev):
    """Scores that grow from key to key, and differ by hundreds: every tile moves the reference."""
    for k_size in (1.0, 30.0, 300.0):
        _decode(Filled(dev, [900], 2, 64, 32, seed=3, k_size=k_size), 4, size=3.0)


def test_keys_that_are_not_finite(dev):
    """A key with a NaN makes its heads' rows NaN where it is seen, and changes nothing where it is not."""
    from liyab_b200 import ops
    f = Filled(dev, [200], 2, 64, 32, seed=2)
    q, out = _queries(f, 1, 4, 0), torch.empty(1, 256, dtype=BF16, device=dev)
    place = torch.tensor([199], dtype=torch.int32, device=dev)
    clean = ops.decode_attention4(q, f.cache, place, f.table, out.clone(), 1, 4, 0.125, window=50)
    for which in range(2):
        bad = [torch.randn(1, 128, device=dev) for _ in range(2)]
        bad[which][0, 3] = math.nan
        ops.append4(*bad, _slots(f.table.cpu(), 0, 101, 16)[100:].to(dev), f.cache, 1)
        seen = ops.decode_attention4(q, f.cache, place, f.table, out.clone(), 1, 4, 0.125)
        if which == 0:
            assert seen[:, :128].isnan().all() and not seen[:, 128:].isnan().any()
        else:
            assert seen[:, :32].isnan().all() and not seen[:, 128:].isnan().any()
        assert torch.equal(ops.decode_attention4(q, f.cache, place, f.table, out.clone(), 1, 4, 0.125, window=50), clean)
        assert torch.equal(ops.decode_attention4(q, f.cache, torch.tensor([99], dtype=torch.int32, device=dev), f.table, out.clone(), 1, 4, 0.125).isnan().any(), torch.tensor(False, device=dev))


# ---- portions ----------------------------------------------------------------------------------------------

def _way(f, n, heads, most, window=0, mass=False):
    """How the library runs such a call: (1 for the kernel for many rows, rows a tile, blocks that share keys, ..)."""
    got = (C.c_int * 4)()
    width, keys = heads * f.dim, f.table.shape[1] * f.cache.page_size
    call = _call(f.cache.ref, n_head=heads, n_seq=n, n_tokens=n * most, max_keys=keys, table_stride=f.table.shape[1], q_stride=width, out_stride=width, q_start=AT, max_q_len=most, window=window,
                 **(dict(mass=AT, total=AT) if mass else {}))
    assert ops.lib().lb_attention4_plan(call, got) == 0
    return tuple(got)


def _portions(f, new, heads, seed=0, size=1.0, mass=False, max_q=None, **more):
    """prefill_attention4 beside the plain form; new[i] tokens of request i, its last ones."""
    from liyab_b200 import ops
    n, scale = len(f.lengths), 1 / math.sqrt(f.dim)
    q = _queries(f, sum(new), heads, seed, size)
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(f.dev)
    past = torch.tensor([a - b for a, b in zip(f.lengths, new)], dtype=torch.int32, device=f.dev)
    out = torch.full((sum(new) + 2, heads * f.dim), 7.5, dtype=BF16, device=f.dev)
    before = torch.rand(n, f.kv, f.table.shape[1] * f.cache.page_size, generator=torch.Generator().manual_seed(seed)).to(f.dev) if mass else None
    total = torch.full_like(before, 7.5) if mass else None
    most = max(new) if max_q is None else max_q
    ops.prefill_attention4(q, f.cache, start, past, f.table, out, n, most, heads, scale, mass=before, total=total, **more)
    plain = {k: v for k, v in more.items() if k in ("window", "distance", "sink")} | dict(cap=more.get("soft_cap", 0.0))
    token = 0
    for i in range(n):
        places = torch.arange(f.lengths[i] - new[i], f.lengths[i], device=f.dev)
        m = f.lengths[i]
        want, weights, bound, relative = _attention(q[token:token + new[i]].view(-1, heads, f.dim), f.k[i], f.v[i], places, scale, many=_way(f, n, heads, most, more.get("window", 0), mass)[0] == 1, **plain)
        _close(out[token:token + new[i]].view(-1, heads, f.dim), want, bound)
        if mass and new[i]:
            gained = weights.sum(0).view(f.kv, heads // f.kv, m).sum(1)
            allowed = gained * (3 * relative.max() + (new[i] * heads // f.kv + 2) * 2.0 ** -23) + (before[i, :, :m].double() + gained) * 2.0 ** -23
            assert ((total[i, :, :m].double() - before[i, :, :m].double() - gained).abs() <= allowed).all()
            assert (total[i, :, m:] == 7.5).all()
        token += new[i]
    assert (out[sum(new):] == 7.5).all()                     # rows behind the last request
    return out


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 2), (15, 3), (32, 2)])
def test_portions_of_a_few_tokens(dev, dim, group, heads, kv):
    _portions(Filled(dev, [1, 5, 40, 17, 300], kv, dim, group, seed=heads), [1, 5, 3, 0, 4], heads)


@pytest.mark.parametrize("window", [0, 1, 7, 100, -16, -100])
def test_portions_under_windows_with_weights(dev, window):
    _portions(Filled(dev, [64, 200, 33, 1000], 2, 64, 64, 32, seed=2), [64, 17, 33, 2], 6, window=window, mass=True)
    _portions(Filled(dev, [20, 500], 1, 128, 32, seed=3), [16, 16], 4, window=window, mass=True, sink=torch.randn(4, device=dev), soft_cap=15.0)


@pytest.mark.parametrize("lengths,new", [([300], [300]), ([129, 1000, 64], [129, 200, 1]), ([2000], [130]), ([16, 4000], [16, 257])])
@pytest.mark.parametrize("dim,group,heads,kv", [(64, 64, 4, 4), (64, 32, 12, 2), (128, 64, 8, 2), (128, 128, 5, 1), (128, 32, 16, 1)])
def test_portions_of_prompts(dev, lengths, new, dim, group, heads, kv):
    _portions(Filled(dev, lengths, kv, dim, group, 32, seed=dim + heads), new, heads)


def test_portions_longer_than_named_are_cut(dev):
    """Tokens past max_q_len are left alone, and nothing is read or written for them."""
    from liyab_b200 import ops
    f = Filled(dev, [40], 1, 64, 64)
    q, out = _queries(f, 12, 2, 0), torch.full((12, 128), 7.5, dtype=BF16, device=dev)
    mass = torch.zeros(1, 1, f.table.shape[1] * 16, device=dev)
    ops.prefill_attention4(q, f.cache, torch.tensor([0, 12], dtype=torch.int32, device=dev), torch.tensor([28], dtype=torch.int32, device=dev), f.table, out, 1, 8, 2, 0.125, mass=mass)
    want, _, bound, _ = _attention(q[:8].view(8, 2, 64), f.k[0], f.v[0], torch.arange(28, 36, device=dev), 0.125)
    _close(out[:8].view(8, 2, 64), want, bound)
    assert (out[8:] == 7.5).all() and not mass[0, 0, 36:].any() and abs(mass.sum().item() - 16) < 1e-3


def _forms_of_many(dev, heads):
    """Options beside each other, with scores that stay far below the cap and some that pass it."""
    gen = torch.Generator().manual_seed(heads)
    sink = torch.randn(heads, generator=gen).to(dev)
    slopes = torch.rand(heads, generator=gen)
    line = torch.cat([slopes * 0.1, torch.full((heads,), -1.0)]).to(dev)
    log = torch.cat([slopes, slopes * 0.3]).to(dev)
    return [(1.0, dict(sink=sink)), (1.0, dict(soft_cap=50.0)), (4.0, dict(soft_cap=3.0, sink=sink)), (1.0, dict(distance=line)), (1.0, dict(distance=log, sink=sink))]


@pytest.mark.parametrize("form", range(5))
@pytest.mark.parametrize("dim,group,heads,kv,window", [(64, 32, 8, 2, 0), (128, 64, 6, 2, 200), (128, 32, 4, 4, -96), (128, 32, 32, 2, -96), (64, 64, 16, 1, 7)])
def test_portions_of_many_rows_with_sinks_caps_and_distances(dev, form, dim, group, heads, kv, window):
    size, more = _forms_of_many(dev, heads)[form]
    f = Filled(dev, [300, 900, 129], kv, dim, group, 32, seed=form)
    assert _way(f, 3, heads, 300, window)[0] == (heads > kv)           # (few rows and keys: the other kernel)
    _portions(f, [300, 260, 128], heads, seed=form, size=size, window=window, **more)


@pytest.mark.parametrize("window", [0, 1000, -1024, 100, 1])
@pytest.mark.parametrize("dim,group,heads,kv,new", [(128, 64, 8, 2, [64, 60, 9]), (64, 64, 4, 4, [150, 1, 129]), (128, 128, 16, 1, [200, 70, 0])])
def test_portions_of_many_rows_whose_keys_blocks_share(dev, dim, group, heads, kv, new, window):
    """One request behind many keys, and requests of all lengths beside each other: blocks of the short ones find no keys."""
    f = Filled(dev, [6000, 90, 2000], kv, dim, group, 64, seed=window % 97)
    assert window != 0 or (_way(f, 3, heads, max(new))[0] == 1 and _way(f, 3, heads, max(new))[2] > 1)
    _portions(f, new, heads, window=window)
    one = Filled(dev, [5000], kv, dim, group, 16, seed=5)
    _portions(one, [max(new)], heads, window=window, sink=torch.randn(heads, device=dev))


def test_portions_of_many_rows_of_any_place(dev):
    """Rows of q and out that no wide load reaches, in the middle of wider rows; what lies between them is left alone."""
    f = Filled(dev, [400, 300], 1, 128, 32, 16, seed=3)
    assert _way(f, 2, 16, 300)[:3] == (1, 256, 1)
    q = _queries(f, 600, 16, 3)
    start, past = torch.tensor([0, 300, 600], dtype=torch.int32, device=dev), torch.tensor([100, 0], dtype=torch.int32, device=dev)
    want = ops.prefill_attention4(q, f.cache, start, past, f.table, torch.empty_like(q), 2, 300, 16, 0.125)
    for pad in (1, 8):
        wide = torch.zeros(600, 2048 + 2 * pad + 1, dtype=BF16, device=dev)
        wide[:, pad:pad + 2048] = q
        out = torch.full((601, 2048 + 2 * pad), 7.5, dtype=BF16, device=dev)
        ops.prefill_attention4(wide[:, pad:pad + 2048], f.cache, start, past, f.table, out[:600, pad:pad + 2048], 2, 300, 16, 0.125)
        assert torch.equal(out[:600, pad:pad + 2048], want) and (out[:, :pad] == 7.5).all() and (out[:, pad + 2048:] == 7.5).all() and (out[600] == 7.5).all()


def test_portions_of_many_rows_on_pages_that_are_not_there(dev):
    """Keys on pages outside the cache are not there; a request without any has rows of zeros; a place of the batch without tokens changes nothing."""
    f = Filled(dev, [400, 300, 260], 2, 128, 64, 16, seed=4)
    assert _way(f, 3, 8, 400)[0] == 1
    table = f.table.clone()
    table[0, 3], table[0, 20], table[1, :] = -1, 1 << 29, -5
    q, out = _queries(f, 700, 8, 1), torch.full((702, 1024), 7.5, dtype=BF16, device=dev)
    start, past = torch.tensor([0, 400, 700, 700], dtype=torch.int32, device=dev), torch.tensor([0, 0, 260], dtype=torch.int32, device=dev)
    ops.prefill_attention4(q, f.cache, start, past, table, out, 3, 400, 8, 0.1)
    keys = torch.tensor([k for k in range(400) if k // 16 not in (3, 20)], device=dev)
    k, v = f.k[0].clone(), f.v[0].clone()
    # The plain form for each token over the keys that are there: those up to its place.
    for place in (47, 48, 63, 64, 255, 256, 319, 340, 399):
        there = keys[keys <= place]
        want, _, bound, _ = _attention(q[place:place + 1].view(1, 8, 128), k[there], v[there], torch.tensor([1 << 20], device=dev), 0.1, many=True)
        _close(out[place].view(1, 8, 128), want, bound)
    assert not out[400:700].any() and (out[700:] == 7.5).all()


@pytest.mark.parametrize("past", [0, 4000])
def test_portions_of_many_rows_and_keys_that_are_not_finite(dev, past):
    """A key with a NaN, or a value's group: the rows that see it are NaN there, and the others are as they were."""
    f = Filled(dev, [past + 300], 2, 64, 32, 16, seed=6)
    assert _way(f, 1, 32, 300)[0] == 1
    q, start, n_past = _queries(f, 300, 32, 0), torch.tensor([0, 300], dtype=torch.int32, device=dev), torch.tensor([past], dtype=torch.int32, device=dev)
    run = lambda **more: ops.prefill_attention4(q, f.cache, start, n_past, f.table, torch.empty_like(q), 1, 300, 32, 0.125, **more)  # noqa: E731
    clean, narrow = run(), run(window=40)
    place = past + 130
    for which in range(2):
        rows = [_values_as_rows(x[0][place:place + 1]) for x in (f.k, f.v)]
        rows[which][0, 3] = math.nan
        ops.append4(*rows, _slots(f.table.cpu(), 0, place + 1, 16)[place:].to(dev), f.cache, 1)
        got, got_narrow = run(), run(window=40)
        assert torch.equal(got[:130], clean[:130]) and torch.equal(got_narrow[:130], narrow[:130]) and torch.equal(got_narrow[170:], narrow[170:])
        columns = [c for h in range(16) for c in range(64 * h, 64 * h + (64 if which == 0 else 32))]
        others = [c for c in range(2048) if c not in columns]
        assert got[130:, columns].isnan().all() and got_narrow[130:170, columns].isnan().all()
        assert torch.equal(got[:, others], clean[:, others]) and torch.equal(got_narrow[:, others], narrow[:, others])
        rows = [_values_as_rows(x[0][place:place + 1]) for x in (f.k, f.v)]
        ops.append4(*rows, _slots(f.table.cpu(), 0, place + 1, 16)[place:].to(dev), f.cache, 1)
    q[7] = math.nan
    got = run()
    assert got[7].isnan().all() and torch.equal(got[:7], clean[:7]) and torch.equal(got[8:], clean[8:])


def _values_as_rows(x):
    """Rows whose rounding is these values again: n s, its largest |n| being 7 (7 s / 7 is s; a bfloat16 scale of values that float32 holds exactly)."""
    return x.reshape(1, -1).float().contiguous()


@pytest.mark.parametrize("k_size,v_size,q_size", [(1e-3, 1e3, 1e3), (1e4, 1e-6, 1e-4), (1e-15, 1e15, 1e15), (1.0, 1e-20, 1.0), (1.0, 1e30, 1e-30), (1e30, 1.0, 1e-30)])
def test_portions_of_many_rows_of_all_sizes(dev, k_size, v_size, q_size):
    f = Filled(dev, [700, 300], 2, 128, 32, seed=9, k_size=k_size, v_size=v_size)
    assert _way(f, 2, 16, 300)[0] == 1
    _portions(f, [300, 257], 16, size=q_size)


def test_portions_are_the_same_every_time(dev):
    f = Filled(dev, [3000, 20, 900], 2, 128, 32, seed=4)
    for new in ([300, 20, 257], [64, 3, 50], [2, 3, 1]):
        assert torch.equal(_portions(f, new, 8), _portions(f, new, 8))


def test_decode_of_more_requests_than_a_launch_row(dev):
    """Requests of one block each and requests whose keys all warps share give what each gives alone."""
    f = Filled(dev, [(i * 37) % 90 for i in range(290)], 1, 64, 64, seed=2)
    ways = set()
    for most in (0, 96, 1 << 20):
        table = torch.nn.functional.pad(f.table, (0, 4096 if most > 96 else 0), value=-1)
        q, positions = _queries(f, 290, 2, 0), torch.tensor([n - 1 for n in f.lengths], dtype=torch.int32, device=dev)
        out = torch.full((290, 128), 7.5, dtype=BF16, device=dev)
        ops.decode_attention4(q, f.cache, positions, table, out, 290, 2, 0.125, max_keys=most)
        got = (C.c_int * 4)()
        call = _call(f.cache.ref, n_head=2, n_seq=290, n_tokens=290, max_keys=table.shape[1] * 16 if most != 96 else 96, table_stride=table.shape[1], q_stride=128, out_stride=128)
        assert ops.lib().lb_attention4_plan(call, got) == 0
        ways.add(got[3] > 1)
        for i in range(0, 290, 7):
            want, _, bound, _ = _attention(q[i:i + 1].view(1, 2, 64), f.k[i], f.v[i], torch.tensor([f.lengths[i] - 1], device=dev), 0.125)
            _close(out[i].view(1, 2, 64), want, bound)
    assert ways == {False, True}


@pytest.mark.parametrize("heads,new,many", [(4, 6, 0), (32, 300, 1)])
@pytest.mark.parametrize("window", [0, 50, -64])
def test_portions_read_no_key_past_the_most(dev, heads, new, many, window):
    """Places past max_keys are taken as the last key there, in the kernel for few rows and the one for many."""
    f = Filled(dev, [700, 400], 2, 64, 32, 16, seed=5)
    q = _queries(f, 2 * new, heads, 1)
    start, past = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=dev), torch.tensor([700 - new, 400 - new], dtype=torch.int32, device=dev)
    most = 700 - new // 2
    got = (C.c_int * 4)()
    call = _call(f.cache.ref, n_head=heads, n_seq=2, n_tokens=2 * new, max_keys=most, table_stride=f.table.shape[1], q_stride=64 * heads, out_stride=64 * heads, q_start=AT, max_q_len=new,
                 window=window)
    assert ops.lib().lb_attention4_plan(call, got) == 0 and got[0] == many
    out = ops.prefill_attention4(q, f.cache, start, past, f.table, torch.empty_like(q), 2, new, heads, 0.125, window=window, max_keys=most)
    for i, n in enumerate((700, 400)):
        places = torch.arange(n - new, n, device=dev).clamp(max=most - 1)
        want, _, bound, _ = _attention(q[i * new:(i + 1) * new].view(new, heads, 64), f.k[i][:most], f.v[i][:most], places, 0.125, window=window, many=many == 1)
        _close(out[i * new:(i + 1) * new].view(new, heads, 64), want, bound)


def test_requests_that_share_pages_and_weights_of_other_rows(dev):
    """Two requests over the same pages; the keys' weights on rows of any order, others left alone, rows outside skipped."""
    f = Filled(dev, [300, 100], 2, 64, 64, 16, seed=2)
    table = torch.stack([f.table[0], f.table[0], f.table[1]])
    q, places = _queries(f, 3, 4, 0), torch.tensor([299, 120, 99], dtype=torch.int32, device=dev)
    mass = torch.full((4, 2, table.shape[1] * 16), 0.5, device=dev)
    rows = torch.tensor([3, 7, 0], dtype=torch.int32, device=dev)
    out = ops.decode_attention4(q, f.cache, places, table, torch.empty_like(q), 3, 4, 0.125, mass=mass, mass_rows=rows)
    for i, (of, n, r) in enumerate(((0, 300, 3), (0, 121, None), (1, 100, 0))):
        want, weights, bound, relative = _attention(q[i:i + 1].view(1, 4, 64), f.k[of][:n], f.v[of][:n], torch.tensor([n - 1], device=dev), 0.125)
        _close(out[i].view(1, 4, 64), want, bound)
        if r is not None:
            gained = weights.view(2, 2, n).sum(1)
            assert ((mass[r, :, :n].double() - 0.5 - gained).abs() <= gained * (3 * relative.max() + 2.0 ** -21) + (0.5 + gained) * 2.0 ** -23).all() and (mass[r, :, n:] == 0.5).all()
    assert (mass[1:3] == 0.5).all()


def test_calls_of_nothing(dev):
    f = Filled(dev, [40], 2, 64, 64, seed=1)
    none, i32 = torch.empty(0, 256, dtype=BF16, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    before = f.cache.memory.clone()
    ops.append4(none[:, :128], none[:, :128], i32, f.cache, 0)
    ops.cache4_values(f.cache, i32, 0, none[:, :128], none[:, :128])
    ops.decode_attention4(none, f.cache, i32[:0], f.table, none, 0, 4, 0.125)
    ops.prefill_attention4(none, f.cache, i32, i32[:0], f.table, none, 0, 5, 4, 0.125)
    ops.evict4(f.cache, torch.zeros(1, 2, 48, device=dev), f.table, i32, 0, 4, 2, f.table, torch.empty(0, 2, 4, dtype=torch.int32, device=dev))
    assert torch.equal(f.cache.memory, before)


# ---- eviction ----------------------------------------------------------------------------------------------

def _evict(f, mass, keep, recent, mass_rows=None):
    from liyab_b200 import ops
    n, page = len(f.lengths), f.cache.page_size
    per = -(-keep // page)
    dest = f.spare[:n * per].view(n, per).to(f.dev)
    kept = torch.full((n, f.kv, keep), 77, dtype=torch.int32, device=f.dev)
    dest_mass = torch.full((mass.shape[0], f.kv, keep + 2), 7.5, device=f.dev)
    n_keys = torch.tensor(f.lengths, dtype=torch.int32, device=f.dev)
    before = f.cache.memory.clone()
    got = ops.evict4(f.cache, mass, f.table, n_keys, n, keep, recent, dest, kept, dest_mass, mass_rows=mass_rows)
    assert got is kept
    k, v = (torch.full((n * keep, f.kv * f.dim), 7.5, device=f.dev) for _ in range(2))
    slots = torch.cat([_slots(dest.cpu(), i, keep, page) for i in range(n)]).view(n, keep)
    for i, m in enumerate(f.lengths):
        slots[i, min(m, keep):] = -1
    ops.cache4_values(f.cache, slots.view(-1).to(f.dev), n * keep, k, v)
    for i, m in enumerate(f.lengths):
        stay, r = min(m, keep), i if mass_rows is None else int(mass_rows[i])
        old = m - min(recent, m)
        for h in range(f.kv):
            w = mass[r, h, :old].double()
            w = torch.where(w.isnan(), torch.full_like(w, math.inf), w) if not w.isinf().any() else w
            order = torch.sort(w, descending=True, stable=True).indices[:stay - (m - old)]
            want = torch.cat([order, torch.arange(old, m, device=f.dev)]).sort().values
            assert torch.equal(kept[i, h, :stay].long(), want) and (kept[i, h, stay:] == -1).all()
            assert torch.equal(dest_mass[r, h, :stay], mass[r, h][want]) or mass[r, h][want].isnan().any()
            assert (dest_mass[r, h, stay:keep] == 0).all() and (dest_mass[r, h, keep:] == 7.5).all()
            at = i * keep
            assert torch.equal(k[at:at + stay].view(stay, f.kv, f.dim)[:, h], f.k[i][want, h].float())
            assert torch.equal(v[at:at + stay].view(stay, f.kv, f.dim)[:, h], f.v[i][want, h].float())
    # The pages that were there before are as they were.
    size = before.numel() // f.cache.n_pages
    untouched = torch.ones(f.cache.n_pages, dtype=torch.bool)
    untouched[dest.cpu().long().view(-1)] = False
    assert torch.equal(f.cache.memory.view(-1, size)[untouched], before.view(-1, size)[untouched])
    return dest, dest_mass


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("lengths,keep,recent", [([50], 20, 5), ([1, 30, 200, 0], 32, 32), ([500, 2000, 33], 100, 0), ([40, 64], 64, 3), ([3000], 1, 1), ([5000], 2500, 100)])
def test_evict(dev, dim, group, lengths, keep, recent):
    f = Filled(dev, lengths, 3, dim, group, 16, seed=keep, extra=len(lengths) * -(-keep // 16))
    mass = torch.exp(3 * torch.randn(len(lengths), 3, f.table.shape[1] * 16, generator=torch.Generator().manual_seed(keep))).to(dev)
    _evict(f, mass, keep, recent)


@pytest.mark.parametrize("kind", ["equal", "few values", "zeros", "negative", "special"])
def test_evict_by_equal_and_special_weights(dev, kind):
    lengths, keep, recent = [700, 90, 2100], 80, 11
    f = Filled(dev, lengths, 2, 64, 32, 32, seed=1, extra=9)
    gen = torch.Generator().manual_seed(6)
    mass = torch.zeros(3, 2, f.table.shape[1] * 32)
    if kind == "few values":
        mass = torch.randint(0, 3, mass.shape, generator=gen).float()
    elif kind == "zeros":
        mass = torch.where(torch.rand(mass.shape, generator=gen) < 0.5, 0.0, -0.0)
    elif kind == "negative":
        mass = torch.randn(mass.shape, generator=gen) * 1e-38
    elif kind == "special":
        mass = torch.randn(mass.shape, generator=gen)
        mass[:, 0, ::50] = math.nan
        mass[:, 1, ::50], mass[:, 1, 1::50] = math.inf, -math.inf
    _evict(f, mass.to(dev), keep, recent)


def test_evict_rows_of_another_order(dev):
    f = Filled(dev, [100, 300], 2, 128, 64, 16, seed=1, extra=8)
    mass = torch.rand(5, 2, 320, generator=torch.Generator().manual_seed(1)).to(dev)
    _evict(f, mass, 50, 10, torch.tensor([4, 1], dtype=torch.int32, device=dev))


@pytest.mark.parametrize("keep,recent", [(1000, 10), (50000, 49990), (59999, 0)])
def test_evict_of_more_keys_than_a_block_holds(dev, keep, recent):
    f = Filled(dev, [60000], 1, 64, 64, 64, seed=1, extra=-(-keep // 64))
    mass = torch.rand(1, 1, f.table.shape[1] * 64, generator=torch.Generator().manual_seed(2)).to(dev)
    _evict(f, mass, keep, recent)
    _evict(f, (mass * 4).floor(), keep, recent)              # equal weights on both sides of what the block holds


@pytest.mark.parametrize("kv,n,keep,recent", [(2, 8193, 100, 3), (1, 20000, 19000, 0), (3, 70001, 333, 40), (40, 9000, 4500, 32), (1, 8200, 8200, 8200)])
def test_evict_of_keys_that_blocks_share(dev, kv, n, keep, recent):
    """Two to eight blocks a head, and one where there are many heads; other requests beside them with none and one of their keys to drop."""
    lengths = [n, 0, keep + 1] if kv < 40 else [n]
    f = Filled(dev, lengths, kv, 64, 64, 64, seed=1, extra=len(lengths) * -(-keep // 64))
    mass = torch.rand(len(lengths), kv, f.table.shape[1] * 64, generator=torch.Generator().manual_seed(2)).to(dev)
    _evict(f, mass, keep, recent)
    _evict(f, (mass * 3).floor(), keep, recent)
    _evict(f, torch.zeros_like(mass), keep, recent)


# ---- together ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_them_together(dev, captured):
    """A prompt, tokens one by one with their keys' weights, an eviction, more tokens over what is left; eagerly, and every step replayed from a graph, on a stream of its own."""
    from liyab_b200 import ops
    kv, heads, dim, group, page, keep, recent = 2, 8, 64, 32, 16, 48, 16
    lengths = [70, 131]
    gen = torch.Generator().manual_seed(12)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        f = Filled(dev, lengths, kv, dim, group, page, seed=7, extra=40)
        spare = f.spare.to(dev)
        table = torch.cat([f.table, torch.full((2, 3), -1, dtype=torch.int32, device=dev)], 1)
        for i, n in enumerate(lengths):                       # pages for the tokens to come
            table[i, -(-n // page):-(-n // page) + 2] = spare[2 * i:2 * i + 2]
        mass = torch.zeros(2, kv, table.shape[1] * page, device=dev)
        ks, vs = [x.clone() for x in f.k], [x.clone() for x in f.v]
        width, scale = kv * dim, 1 / math.sqrt(dim)
        k, v = (torch.zeros(2, width, dtype=BF16, device=dev) for _ in range(2))
        q, out = torch.zeros(2, heads * dim, dtype=BF16, device=dev), torch.zeros(2, heads * dim, dtype=BF16, device=dev)
        slots, positions = (torch.zeros(2, dtype=torch.int32, device=dev) for _ in range(2))

        def step():
            ops.append4(k, v, slots, f.cache, 2)
            ops.decode_attention4(q, f.cache, positions, table, out, 2, heads, scale, mass=mass, max_keys=mass.shape[2])
        graph = None
        if captured:
            slots.fill_(-1)
            positions.fill_(-1)
            step()
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            mass.zero_()
        place = [n - 1 for n in lengths]

        def tokens(count):
            for _ in range(count):
                for dst in (k, v, q):
                    dst.copy_(torch.randn(dst.shape, generator=gen).to(BF16).to(dev))
                for i in range(2):
                    place[i] += 1
                    slots[i] = table[i, place[i] // page] * page + place[i] % page
                    positions[i] = place[i]
                    for rows, new in ((ks, k), (vs, v)):
                        rows[i] = torch.cat([rows[i], _values(*_rounded(new[i:i + 1], kv, dim, group), group)])
                graph.replay() if captured else step()
                for i in range(2):
                    want, weights, bound, _ = _attention(q[i:i + 1].view(1, heads, dim), ks[i], vs[i], torch.tensor([place[i]], device=dev), scale)
                    _close(out[i].view(1, heads, dim), want, bound)
                    gathered[i][:, :place[i] + 1] += weights.view(kv, heads // kv, place[i] + 1).sum(1)
        gathered = [torch.zeros(kv, mass.shape[2], dtype=F64, device=dev) for _ in range(2)]
        tokens(6)
        for i in range(2):
            assert torch.allclose(mass[i].double(), gathered[i], rtol=1e-4, atol=1e-6)
        dest = spare[10:16].view(2, 3)
        kept = torch.empty(2, kv, keep, dtype=torch.int32, device=dev)
        new_mass = torch.zeros_like(mass)
        ops.evict4(f.cache, mass, table, torch.tensor([p + 1 for p in place], dtype=torch.int32, device=dev), 2, keep, recent, dest, kept, new_mass)
        for i in range(2):
            for rows in (ks, vs):
                rows[i] = torch.stack([rows[i][kept[i, h].long(), h] for h in range(kv)], 1)
            gathered[i] = torch.nn.functional.pad(torch.stack([gathered[i][h, kept[i, h].long()] for h in range(kv)]), (0, mass.shape[2] - keep))
            place[i] = keep - 1
            table[i, :3], table[i, 3:5] = dest[i], spare[20 + 2 * i:22 + 2 * i]
        mass.copy_(new_mass)
        tokens(5)
        for i in range(2):
            assert torch.allclose(mass[i].double(), gathered[i], rtol=1e-4, atol=1e-6)
    stream.synchronize()


def test_two_streams_and_graphs_beside_each_other(dev):
    """Calls under way on two streams at once, eager ones and graphs' replays, with inputs that change between replays, give what they give alone."""
    kv, heads, dim = 2, 8, 128
    f = Filled(dev, [4000, 100, 1500], kv, dim, 64, 16, seed=8, extra=120)
    mass = torch.rand(3, kv, f.table.shape[1] * 16, generator=torch.Generator().manual_seed(3)).to(dev)
    n_keys = torch.tensor(f.lengths, dtype=torch.int32, device=dev)
    dest = f.spare[:60].view(3, 20).to(dev)
    dest2 = f.spare[60:120].view(3, 20).to(dev)
    positions = n_keys - 1
    new = [200, 64, 130]
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
    past = n_keys - torch.tensor(new, dtype=torch.int32, device=dev)

    class Work:
        def __init__(self, dest):
            self.q, self.p = torch.empty(3, heads * dim, dtype=BF16, device=dev), torch.empty(sum(new), heads * dim, dtype=BF16, device=dev)
            self.out, self.outp, self.total = torch.empty_like(self.q), torch.empty_like(self.p), torch.zeros_like(mass)          # (behind the newest key nothing is written)
            self.kept, self.dest = torch.empty(3, kv, 320, dtype=torch.int32, device=dev), dest
            self.few = torch.empty(9, heads * dim, dtype=BF16, device=dev)

        def load(self, seed):
            gen = torch.Generator().manual_seed(seed)
            for t in (self.q, self.p):
                t.copy_(torch.randn(t.shape, generator=gen).to(BF16))

        def run(self):
            ops.decode_attention4(self.q, f.cache, positions, f.table, self.out, 3, heads, 0.09, mass=mass, total=self.total)
            ops.prefill_attention4(self.p, f.cache, start, past, f.table, self.outp, 3, 200, heads, 0.09)
            ops.prefill_attention4(self.p[:9], f.cache, self.three, n_keys - 3, f.table, self.few, 3, 3, heads, 0.09)
            ops.evict4(f.cache, self.total, f.table, n_keys, 3, 320, 20, self.dest, self.kept)

        three = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device=dev)

        def results(self):
            return [t.clone() for t in (self.out, self.outp, self.total, self.kept, self.few)]

    a, b = Work(dest), Work(dest2)
    want = {}
    for seed in range(4):
        a.load(seed)
        a.run()
        want[seed] = a.results()
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for w, s in zip((a, b), streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            w.run()
        graphs.append(graph)
    torch.cuda.synchronize()
    for first, second in ((0, 1), (2, 3), (1, 1)):
        for replayed in (True, False):
            for w, seed in ((a, first), (b, second)):
                w.load(seed)
            torch.cuda.synchronize()
            for _ in range(5):
                for w, s, g in zip((a, b), streams, graphs):
                    with torch.cuda.stream(s):
                        g.replay() if replayed else w.run()
            torch.cuda.synchronize()
            for w, seed in ((a, first), (b, second)):
                assert all(torch.equal(x, y) for x, y in zip(w.results(), want[seed]))
    del graphs
