"""The 4-bit cache where single values are not finite or of the largest and smallest sizes, against plain forms in 64 bits."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from liyab_b200 import ops
from test_cache4 import _call
from test_cache4_gpu import BF16, FORMS, Filled, _attention, _close, _decode, _portions, _queries, _rounded, _slots, _values, _values_as_rows
from test_kernels_gpu import dev  # noqa: F401

pytestmark = pytest.mark.gpu


def _shared(f, n, heads, most, **more):
    """Whether all warps of a launch share the keys (a launch joins their states), or a block has a request's row tile and key/value head to itself; None: the kernel for many rows."""
    got = (C.c_int * 4)()
    width, keys = heads * f.dim, f.table.shape[1] * f.cache.page_size
    portions = dict(q_start=1 << 20, max_q_len=most) if most > 1 else {}
    call = _call(f.cache.ref, n_head=heads, n_seq=n, n_tokens=n * most, max_keys=keys, table_stride=f.table.shape[1], q_stride=width, out_stride=width, **portions, **more)
    assert ops.lib().lb_attention4_plan(call, got) == 0
    return None if got[0] == 1 else got[2] > 1 or got[3] > 1


def _spoil(f, i, place, head, group):
    """A value of request i's key at `place` becomes NaN: the group of this head's that has it is not finite."""
    rows = [_values_as_rows(x[i][place:place + 1]) for x in (f.k, f.v)]
    rows[1][0, head * f.dim + group * f.cache.group + 3] = math.nan
    ops.append4(*rows, _slots(f.table.cpu(), i, place + 1, f.cache.page_size)[place:].to(f.dev), f.cache, 1)
    f.v[i][place, head, group * f.cache.group:(group + 1) * f.cache.group] = math.nan


def _beside(f, new, heads, seed=0, mass=False, window=0, sink=None):
    """Attention of the last new[i] tokens of each request beside the plain form, whose values that are NaN are 0: a row that sees such a group is NaN there, all else is within its bound."""
    n, scale = len(f.lengths), 1 / math.sqrt(f.dim)
    q, out = _queries(f, sum(new), heads, seed), torch.full((sum(new), heads * f.dim), 7.5, dtype=BF16, device=f.dev)
    cells = f.table.shape[1] * f.cache.page_size
    before = torch.rand(n, f.kv, cells, generator=torch.Generator().manual_seed(seed)).to(f.dev) if mass else None
    total = torch.full_like(before, 7.5) if mass else None
    more = dict(mass=before, total=total, window=window, sink=sink)
    past = torch.tensor([a - b for a, b in zip(f.lengths, new)], dtype=torch.int32, device=f.dev)
    if max(new) == 1:
        ops.decode_attention4(q, f.cache, past, f.table, out, n, heads, scale, **more)
    else:
        ops.prefill_attention4(q, f.cache, torch.tensor([0] + new).cumsum(0).to(torch.int32).to(f.dev), past, f.table, out, n, max(new), heads, scale, **more)
    token = 0
    for i, (m, count) in enumerate(zip(f.lengths, new)):
        places, key = torch.arange(m - count, m, device=f.dev)[:, None], torch.arange(m, device=f.dev)[None, :]
        want, weights, bound, relative = _attention(q[token:token + count].view(-1, heads, f.dim), f.k[i], f.v[i].nan_to_num(0.0), places[:, 0], scale, window=window, sink=sink)
        sees = (key <= places) & (key > places - (window if window > 0 else 1 << 30))
        nan = (sees.double() @ f.v[i].isnan().double().view(m, -1) > 0).view(count, f.kv, 1, f.dim).expand(-1, -1, heads // f.kv, -1).reshape(count, heads, f.dim)
        got = out[token:token + count].view(-1, heads, f.dim)
        assert torch.equal(got.isnan(), nan)
        _close(torch.where(nan, torch.zeros_like(got), got), want.masked_fill(nan, 0.0), bound)
        if mass:
            gained = weights.sum(0).view(f.kv, heads // f.kv, m).sum(1)
            allowed = gained * (3 * relative.max() + (count * heads // f.kv + 2) * 2.0 ** -23) + (before[i, :, :m].double() + gained) * 2.0 ** -23
            assert ((total[i, :, :m].double() - before[i, :, :m].double() - gained).abs() <= allowed).all()
        token += count


@pytest.mark.parametrize("dim,group", FORMS)
@pytest.mark.parametrize("heads", [2, 4, 16])
@pytest.mark.parametrize("lengths,shared", [([200, 90], False), ([9000, 40], True)])
def test_a_value_that_is_not_finite_changes_nothing_but_its_group(dev, dim, group, heads, lengths, shared):  # noqa: F811
    """Single tokens: the other groups of the head, the other heads, and the weights that the keys got are what they are without it."""
    f = Filled(dev, lengths, 2, dim, group, seed=heads)
    assert _shared(f, 2, heads, 1) == shared
    _spoil(f, 0, 101, 0, 0)
    _spoil(f, 0, lengths[0] - 1, 1, dim // group - 1)
    _spoil(f, 1, 0, 1, 0)
    for more in (dict(), dict(mass=True), dict(window=120), dict(sink=torch.randn(heads, generator=torch.Generator().manual_seed(1)).to(dev), mass=True)):
        _beside(f, [1, 1], heads, **more)


@pytest.mark.parametrize("dim,group", [(64, 64), (64, 32), (128, 64), (128, 32)])
@pytest.mark.parametrize("heads", [2, 4, 10])
@pytest.mark.parametrize("lengths,shared", [([60, 45, 8], False), ([9000, 45, 8], True)])
def test_a_later_token_that_is_not_finite_does_not_reach_the_ones_before(dev, dim, group, heads, lengths, shared):  # noqa: F811
    """Drafts: the last token's value is NaN; under a window, that of a key which only the first tokens see."""
    f = Filled(dev, lengths, 2, dim, group, seed=heads)
    assert _shared(f, 3, heads, 5) == shared
    _spoil(f, 0, lengths[0] - 1, 0, 0)
    _spoil(f, 1, 43, 1, dim // group - 1)
    for mass in (False, True):
        _beside(f, [5, 4, 3], heads, mass=mass)
    _spoil(f, 0, lengths[0] - 23, 1, 0)
    for mass in (False, True):
        _beside(f, [5, 4, 3], heads, mass=mass, window=20)


@pytest.mark.parametrize("v_size", [3e37, 1e-34])
@pytest.mark.parametrize("dim,group,heads", [(64, 64, 2), (64, 32, 10), (128, 32, 8), (128, 128, 2)])
@pytest.mark.parametrize("lengths", [[200, 90], [9000, 40]])
def test_values_of_the_largest_and_the_smallest_sizes(dev, lengths, dim, group, heads, v_size):  # noqa: F811
    """The weights and their sums do not depend on the values' size, nor do the results' relative errors."""
    f = Filled(dev, lengths, 2, dim, group, seed=heads, v_size=v_size)
    _decode(f, heads, mass=True)
    _decode(f, heads, window=150, sink=torch.zeros(heads, device=dev))
    _portions(f, [5, 3], heads, mass=True)


def _resize_values(f, i, power):
    """Request i's values times 2^power[key]."""
    f.v[i] = f.v[i] * torch.exp2(power.double())[:, None, None]
    m = f.lengths[i]
    ops.append4(*(_values_as_rows(x[i].flatten()).view(m, -1) for x in (f.k, f.v)), _slots(f.table.cpu(), i, m, f.cache.page_size).to(f.dev), f.cache, m)


@pytest.mark.parametrize("dim,group,heads", [(64, 32, 2), (64, 64, 10), (128, 64, 8), (128, 32, 4)])
@pytest.mark.parametrize("lengths", [[200, 90], [9000, 40]])
@pytest.mark.parametrize("low,high", [(0, 122), (-110, 0), (-100, 120)])
def test_values_of_sizes_far_apart(dev, lengths, dim, group, heads, low, high):  # noqa: F811
    """Keys whose values are near the ends of float32's range beside others: states of very different units meet, and every key keeps its weight."""
    f = Filled(dev, lengths, 2, dim, group, seed=heads, k_size=2.0)
    gen = torch.Generator().manual_seed(heads)
    for i, m in enumerate(lengths):
        _resize_values(f, i, torch.where((torch.rand(m // 8 + 1, generator=gen) < 0.3).repeat_interleave(8)[:m], float(high), float(low)).to(dev))
    _decode(f, heads, mass=True)
    _portions(f, [5, 3], heads, mass=True)


@pytest.mark.parametrize("k_size,q_size", [(1e34, 1e-34), (1e-36, 1e36)])
@pytest.mark.parametrize("dim,group,heads", [(64, 64, 2), (64, 32, 10), (128, 32, 8), (128, 128, 2)])
def test_keys_of_the_largest_and_the_smallest_sizes(dev, dim, group, heads, k_size, q_size):  # noqa: F811
    """Keys far from 1 whose scores are ordinary numbers, in the kernel for few rows, both ways, and in the one for many."""
    for lengths in ([200, 90], [9000, 40]):
        f = Filled(dev, lengths, 2, dim, group, seed=heads, k_size=k_size)
        _decode(f, heads, mass=True, size=q_size)
        _portions(f, [5, 3], heads, size=q_size)
    f = Filled(dev, [400, 300], 1, dim, group, seed=heads, k_size=k_size)
    assert _shared(f, 2, 16, 300) is None
    _portions(f, [300, 257], 16, size=q_size)


def _evict_with_holes(f, table, mass, keep, recent, mass_rows=None):
    """evict4 of requests some of whose pages are not in the cache beside what api.h says: of the keys that are there the last `recent` places' and then those with the largest weights; nothing else is
    named as kept, and nothing else's destination is written."""
    n, page, dev = len(f.lengths), f.cache.page_size, f.dev  # noqa: F811
    per = -(-keep // page)
    dest = f.spare[:n * per].view(n, per).to(dev)
    kept, dest_mass = torch.full((n, f.kv, keep), 77, dtype=torch.int32, device=dev), torch.full((mass.shape[0], f.kv, keep), 7.5, device=dev)
    size = f.cache.memory.numel() // f.cache.n_pages
    f.cache.memory.view(-1, size)[dest.long().view(-1)] = 255                    # scales that are NaN
    before = f.cache.memory.clone()
    n_keys = torch.tensor(f.lengths, dtype=torch.int32, device=dev)
    ops.evict4(f.cache, mass, table, n_keys, n, keep, recent, dest, kept, dest_mass, mass_rows=mass_rows)
    stays = torch.zeros(n, dtype=torch.int32)
    for i, m in enumerate(f.lengths):
        key, r = torch.arange(m, device=dev), i if mass_rows is None else int(mass_rows[i])
        pages = table[i, key // page]
        there = (pages >= 0) & (pages < f.cache.n_pages)
        for h in range(f.kv):
            new = key[there & (key >= m - recent)]
            old = key[there & (key < m - recent)]
            w = mass[r, h][old].double()
            first = old[torch.sort(w, descending=True, stable=True).indices[:keep - len(new)]]
            want = torch.cat([first, new]).sort().values
            stay = len(want)
            assert torch.equal(kept[i, h, :stay].long(), want) and (kept[i, h, stay:] == -1).all()
            assert torch.equal(dest_mass[r, h, :stay], mass[r, h][want]) and (dest_mass[r, h, stay:] == 0).all()
            stays[i] = stay
            slots = _slots(dest.cpu(), i, keep, page)[:stay].to(dev)
            k, v = (torch.zeros(stay, f.kv * f.dim, device=dev) for _ in range(2))
            ops.cache4_values(f.cache, slots, stay, k, v)
            assert torch.equal(k.view(stay, f.kv, f.dim)[:, h], f.k[i][want, h].float()) and torch.equal(v.view(stay, f.kv, f.dim)[:, h], f.v[i][want, h].float())
    untouched = torch.ones(f.cache.n_pages, dtype=torch.bool)
    untouched[dest.cpu().long().view(-1)] = False
    assert torch.equal(f.cache.memory.view(-1, size)[untouched], before.view(-1, size)[untouched])
    return dest, stays


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths,keep,recent", [([400, 330, 70], 100, 30), ([500, 64, 0], 64, 64), ([900, 40, 333], 300, 0), ([20000], 300, 100), ([20000, 9000], 12000, 11000), ([70001], 4000, 17)])
def test_evict_of_requests_with_pages_that_are_not_there(dev, lengths, keep, recent, page):  # noqa: F811
    """Keys on pages outside the cache do not stay, in what blocks of one and of several share, past what a block holds, among the newest and the others; attention over what stayed is attention over those
    keys."""
    n = len(lengths)
    f = Filled(dev, lengths, 2, 64, 32, page, seed=keep, extra=n * -(-keep // page))
    gen = torch.Generator().manual_seed(keep)
    mass = torch.exp(2 * torch.randn(n, 2, f.table.shape[1] * page, generator=gen)).to(dev)
    for holes in (0.0, 0.1, 0.9, 1.0):
        table = torch.where(torch.rand(f.table.shape, generator=gen).to(dev) < holes, torch.tensor([-1, 1 << 29, f.pages, -(1 << 31)], dtype=torch.int32)[torch.randint(0, 4, f.table.shape, generator=gen)].to(dev), f.table)
        dest, stays = _evict_with_holes(f, table, mass, keep, recent)
        _evict_with_holes(f, table, (mass * 2).floor(), keep, recent)
        _evict_with_holes(f, table, torch.full_like(mass, -math.inf), keep, recent)
    for i, m in enumerate(lengths):                       # one page of the newest keys, one of the first
        if m:
            table = f.table.clone()
            table[:, 0] = -1
            table[i, (m - 1) // page] = f.pages
            _evict_with_holes(f, table, mass, keep, recent)


def test_a_whole_prompt_that_the_kernel_for_few_rows_does_not_number(dev):  # noqa: F811
    n, kv, heads = 131072, 4, 16
    f = Filled(dev, [n], kv, 64, 64, 128, seed=1)
    q = _queries(f, n, heads, 0)
    out = torch.full((n + 1, heads * 64), 7.5, dtype=BF16, device=dev)
    start, past = torch.tensor([0, n], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    ops.prefill_attention4(q, f.cache, start, past, f.table, out, 1, n, heads, 0.125)
    tokens = torch.tensor([0, 1, 255, 256, 40000, 65535, 65536, 100001, n - 1], device=dev)
    want, _, bound, _ = _attention(q[tokens].view(-1, heads, 64), f.k[0], f.v[0], tokens, 0.125, many=True)
    _close(out[tokens].view(-1, heads, 64), want, bound)
    assert not out.isnan().any() and (out[n] == 7.5).all()


def test_weights_in_memory_that_is_shared(dev):  # noqa: F811
    """Rows of weights that lie between another tensor's give what rows of their own do; rows that overlap are refused, and nothing is written."""
    from liyab_b200.status import LiyabError
    kv, heads, n = 2, 4, 3
    f = Filled(dev, [100, 40, 77], kv, 64, 64, seed=1, extra=3 * 4)
    cells, keep, q = f.table.shape[1] * 16, 50, _queries(f, n, heads, 0)
    places, out = torch.tensor([m - 1 for m in f.lengths], dtype=torch.int32, device=dev), torch.empty(n, heads * 64, dtype=BF16, device=dev)
    n_keys, dest, kept = places + 1, f.spare[:12].view(3, 4).to(dev), torch.empty(n, kv, keep, dtype=torch.int32, device=dev)
    mass = torch.rand(n, kv, cells, generator=torch.Generator().manual_seed(2)).to(dev)

    def run(mass, total, dest_mass):
        ops.decode_attention4(q, f.cache, places, f.table, out, n, heads, 0.125, mass=mass, total=total)
        ops.evict4(f.cache, mass if total is None else total, f.table, n_keys, n, keep, 5, dest, kept, dest_mass)

    total, dest_mass = torch.zeros_like(mass), torch.zeros(n, kv, keep, device=dev)
    run(mass, total, dest_mass)
    for shape, pick in (((2, n, kv, cells), 0), ((n, 2, kv, cells), 1), ((n, kv, 2, cells), 2)):
        buffer = torch.zeros(shape, device=dev)
        a, b = buffer.select(pick, 0), buffer.select(pick, 1)
        a.copy_(mass)
        run(a, b, dest_mass_2 := torch.zeros(n, kv, keep, device=dev))
        assert torch.equal(b, total) and torch.equal(a, mass) and torch.equal(dest_mass_2, dest_mass)
        ops.evict4(f.cache, b, f.table, n_keys, n, keep, 5, dest, kept, a[:, :, :keep])
        assert torch.equal(a[:, :, :keep], dest_mass)
    wide = torch.zeros(n, kv, cells + 1, device=dev)
    wide[:, :, :cells] = mass
    before = wide.clone()
    shared = torch.zeros(1, kv, cells, device=dev)
    for bad in (lambda: run(mass, shared.expand(n, -1, -1), dest_mass), lambda: run(mass, torch.zeros(n, 1, cells, device=dev).expand(-1, kv, -1), dest_mass),
                lambda: run(shared.expand(n, -1, -1), None, dest_mass), lambda: run(wide[:, :, :cells], wide[:, :, 1:], dest_mass), lambda: run(wide[:, :, 1:], wide[:, :, :cells], dest_mass),
                lambda: ops.evict4(f.cache, wide, f.table, n_keys, n, keep, 5, dest, kept, wide[:, :, 1:1 + keep]),
                lambda: ops.evict4(f.cache, wide, f.table, n_keys, n, keep, 5, dest, kept, torch.zeros(1, kv, keep, device=dev).expand(n, -1, -1))):
        with pytest.raises(LiyabError):
            bad()
    assert torch.equal(wide, before) and not shared.any()


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32)])
@pytest.mark.parametrize("requests,new", [(1, 1), (160, 1), (160, 16)])
def test_a_key_of_little_value_that_takes_most_weight(dev, dim, group, requests, new):  # noqa: F811
    """The first key takes most of the weight and has values of zero; what comes out is made of 2^17 equal weights of 2^-20.5 of its: they do not lose bits beside it, in the kernels for few rows and for many.
    (Requests over the same pages, so many that none shares its keys out.)"""
    n, heads = 1 << 17, 16
    f = Filled(dev, [16], 1, dim, group, 128, seed=1, extra=n // 128)
    table = torch.cat([f.table[0], f.spare.to(dev)])[None, :n // 128].expand(requests, -1).contiguous()
    k, v = torch.zeros(n, dim, device=dev), torch.ones(n, dim, device=dev)
    k[1:, 0], v[0] = -7.109375, 0.0
    slot = torch.arange(n, device=dev)
    ops.append4(k, v, (table[0, slot // 128] * 128 + slot % 128).to(torch.int32), f.cache, n)
    (kn, ks), (vn, vs) = _rounded(k, 1, dim, group), _rounded(v, 1, dim, group)
    q = torch.zeros(requests * new, heads * dim, dtype=BF16, device=dev)
    q.view(-1, heads, dim)[:, :, 0] = 16.0
    out, past = torch.empty_like(q), torch.full((requests,), n - new, dtype=torch.int32, device=dev)
    f.table = table
    if new == 1:
        ops.decode_attention4(q, f.cache, past, table, out, requests, heads, 0.125)
    else:
        assert _shared(f, requests, heads, new) is None
        ops.prefill_attention4(q, f.cache, torch.arange(0, requests * new + 1, new, dtype=torch.int32, device=dev), past, table, out, requests, new, heads, 0.125)
    want, _, bound, _ = _attention(q[:1].view(1, heads, dim), _values(kn, ks, group), _values(vn, vs, group), torch.tensor([n - new], device=dev), 0.125)
    assert 0.05 < want.min() and want.max() < 0.1
    _close(out[::new][:1].view(1, heads, dim), want, bound)
    assert torch.equal(out[::new], out[:1].expand(requests, -1))
