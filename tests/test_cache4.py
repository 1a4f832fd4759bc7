"""The 4-bit cache, what the host decides without a GPU: its size, how attention is cut, scratch, and refusals at the C entries and in `ops`."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from liyab_b200 import ops
from liyab_b200.status import LiyabError

AT = 1 << 20                 # an address that is never read


def _bytes(*sizes):
    n = C.c_int64(-1)
    return ops.lib().lb_cache4_bytes(*sizes, C.byref(n)), n.value


@pytest.mark.parametrize("pages,kv,dim,page,group", [(1, 1, 64, 16, 32), (7, 25, 64, 16, 64), (100, 8, 128, 128, 32), (100000, 8, 128, 64, 128), (0, 1, 64, 16, 64), (1 << 19, 32, 128, 1024, 64)])
def test_sizes(pages, kv, dim, page, group):
    assert _bytes(pages, kv, dim, page, group) == (0, pages * kv * page * (dim + 4 * dim // group))


@pytest.mark.parametrize("sizes", [(-1, 1, 64, 16, 32), (1, 0, 64, 16, 32), (1, 1, 96, 16, 32), (1, 1, 64, 8, 32), (1, 1, 64, 48, 32), (1, 1, 64, 0, 32), (1, 1, 64, 16, 16), (1, 1, 64, 16, 128),
                                   (1, 1, 64, 16, 0), (1 << 27, 1, 64, 16, 32), (1 << 20, 32, 128, 1024, 64), (1, 70000, 64, 16, 32)])
def test_sizes_refused(sizes):
    assert _bytes(*sizes)[0] != 0 and ops.lib().lb_last_error()


def test_arguments_are_as_long_as_the_library_reads_them():
    length = ops.lib().lb_struct_bytes
    assert len(ops._attention4_args(*[0] * 27, 0.0, 0.0)) == length(7)
    assert len(ops._evict4_args(*[0] * 21)) == length(8)
    assert C.sizeof(ops.Cache4Args) == length(9)


def _cache(pages=64, kv=2, dim=64, page=16, group=64, memory=AT, device=0):
    c = ops.Cache4Args(memory, pages, kv, dim, page, group, device)
    return c, C.addressof(c)


def _call(ref, **change):
    a = dict(cache=ref, q=AT, q_start=0, last=AT, table=AT, out=AT, mass=0, total=0, rows=0, distance=0, sink=0, scratch=0, stream=0, q_stride=512, out_stride=512, mass_stride=0,
             mass_head=0, total_stride=0, total_head=0, table_stride=64, n_seq=4, n_tokens=4, n_head=8, max_q_len=1, max_keys=1024, n_mass=0, window=0, scale=0.125, soft_cap=0.0)
    assert not set(change) - set(a)
    return ops._attention4_args(*(a | change).values())


@pytest.mark.parametrize("change", [dict(n_head=7), dict(n_head=0), dict(n_seq=-1), dict(n_seq=70000, n_tokens=70000), dict(n_tokens=-1), dict(n_tokens=3), dict(max_q_len=0), dict(max_q_len=2),
                                    dict(max_keys=0), dict(table_stride=0), dict(table_stride=1 << 28), dict(q=0), dict(last=0), dict(table=0), dict(out=0), dict(q=AT + 1), dict(out=AT + 1),
                                    dict(q_stride=511), dict(out_stride=500), dict(total=AT), dict(total=AT, mass=AT, scratch=0), dict(total=AT, mass=AT, scratch=AT + 4),
                                    dict(total=AT, mass=AT, scratch=AT, q_start=AT, max_q_len=65), dict(total=AT, mass=AT, scratch=AT, mass_stride=-1), dict(q_start=AT, max_q_len=1 << 24)])
def test_attention_refused(change):
    c, ref = _cache()
    assert ops.lib().lb_attention4(_call(ref, **change)) != 0 and ops.lib().lb_last_error()


@pytest.mark.parametrize("change", [dict(memory=0), dict(memory=AT + 8), dict(dim=32), dict(page=24), dict(group=48), dict(kv=3)])
def test_caches_refused(change):
    c, ref = _cache(**change)
    assert ops.lib().lb_attention4(_call(ref)) != 0
    if "kv" not in change:
        assert ops.lib().lb_append4(1, AT, 128, AT, 128, AT, ref, 3, 0) != 0
        assert ops.lib().lb_cache4_values(1, ref, AT, 3, AT, 128, AT, 128, 0) != 0
    assert ops.lib().lb_attention4(_call(0)) != 0 and ops.lib().lb_append4(1, AT, 128, AT, 128, AT, None, 3, 0) != 0


@pytest.mark.parametrize("args", [(2, AT, 128, AT, 128, AT, 3), (1, 0, 128, AT, 128, AT, 3), (1, AT, 128, 0, 128, AT, 3), (1, AT, 128, AT, 128, 0, 3), (1, AT, 127, AT, 128, AT, 3),
                                  (1, AT, 128, AT, 64, AT, 3), (1, AT, 128, AT, 128, AT, -1), (1, AT + 1, 128, AT, 128, AT, 3), (0, AT, 128, AT + 2, 128, AT, 3), (1, AT, 128, AT, 128, AT + 2, 3)])
def test_rows_refused(args):
    c, ref = _cache()
    code, k, ldk, v, ldv, slots, n = args
    assert ops.lib().lb_append4(code, k, ldk, v, ldv, slots, ref, n, 0) != 0 and ops.lib().lb_last_error()
    assert ops.lib().lb_cache4_values(code, ref, slots, n, k, ldk, v, ldv, 0) != 0


def test_nothing_to_do_is_not_refused():
    c, ref = _cache()
    assert ops.lib().lb_append4(1, 0, 0, 0, 0, 0, ref, 0, 0) == 0 and ops.lib().lb_cache4_values(0, ref, 0, 0, 0, 0, 0, 0, 0) == 0
    assert ops.lib().lb_attention4(_call(ref, n_seq=0, n_tokens=0, q=0, out=0, last=0, table=0)) == 0
    assert ops.lib().lb_evict4(_evict(ref, n_seq=0)) == 0


def _evict(ref, **change):
    a = dict(cache=ref, mass=AT, rows=0, table=AT, n_keys=AT, dest=AT, kept=AT, dest_mass=0, stream=0, mass_stride=0, mass_head=0, dest_stride=0, dest_head=0, table_stride=64,
             dest_table_stride=8, n_seq=2, keep=128, recent=16, max_keys=1024, n_mass=2, n_dest=0)
    assert not set(change) - set(a)
    return ops._evict4_args(*(a | change).values())


@pytest.mark.parametrize("change", [dict(mass=0), dict(table=0), dict(n_keys=0), dict(dest=0), dict(kept=0), dict(n_seq=-1), dict(n_seq=70000), dict(keep=0), dict(keep=129), dict(recent=-1),
                                    dict(recent=129), dict(max_keys=1025), dict(max_keys=-1), dict(dest_mass=AT), dict(n_mass=-1), dict(mass_stride=-4)])
def test_eviction_refused(change):
    c, ref = _cache()
    assert ops.lib().lb_evict4(_evict(ref, **change)) != 0 and ops.lib().lb_last_error()


@pytest.mark.parametrize("change", [dict(max_keys=(1 << 30) + 1, table_stride=1 << 27), dict(keep=(1 << 30) + 1, dest_table_stride=1 << 27)])
def test_evictions_too_long_are_refused(change):
    c, ref = _cache()
    assert ops.lib().lb_evict4(_evict(ref, **change)) != 0 and b"more than one launch" in ops.lib().lb_last_error()


def _plan(kv, heads, n_seq, keys, q_len=1, dim=64):
    c, ref = _cache(kv=kv, dim=dim)
    got = (C.c_int * 4)()
    more = dict(q_start=AT, max_q_len=q_len) if q_len > 1 else {}
    call = _call(ref, n_head=heads, n_seq=n_seq, n_tokens=n_seq * q_len, max_keys=keys, table_stride=-(-keys // 16), q_stride=heads * dim, out_stride=heads * dim, **more)
    assert ops.lib().lb_attention4_plan(call, got) == 0
    return tuple(got), ops.lib().lb_attention4_scratch(call)


def test_how_attention_is_cut():
    """Rows a tile, blocks, and requests that share them, by the requests, heads, tokens and keys alone."""
    assert _plan(25, 25, 64, 1024)[0] == (0, 4, 2 * 148, 64) and _plan(8, 128, 64, 1024, dim=128)[0] == (0, 8, 3 * 148, 64)
    assert _plan(8, 32, 1, 16)[0][2] == 1                      # eight tiles of keys, two warps' work
    assert _plan(1, 1, 65535, 1024)[0][3] == 256              # requests in rows of the launch
    assert _plan(32, 32, 100, 1 << 27)[0][3] == 4              # a row numbers its tiles in 30 bits
    c, ref = _cache()
    assert ops.lib().lb_attention4_plan(_call(ref), None) != 0
    assert ops.lib().lb_attention4(_call(ref, n_head=8, max_keys=1 << 30, table_stride=1 << 26, q_start=AT, max_q_len=1 << 14)) != 0


def test_scratch():
    """States of all runs (a run more than warps and units together has), where requests' tiles start, and the keys' weights."""
    (_, rows, blocks, per), got = _plan(8, 32, 4, 4096, dim=128)
    states, starts = (8 * blocks + 4 * 8) * rows * 132 * 4, 5 * 4
    assert got == states + -(-starts // 16) * 16
    assert _plan(8, 32, 4, 1024, dim=128) == ((0, 4, 1, 1), 0)          # few keys: a block for each request and key/value head, whose warps' states meet in it
    c, ref = _cache(kv=8, dim=128)
    scratch = ops.lib().lb_attention4_scratch
    assert scratch(_call(ref, n_head=32, mass=AT, total=AT)) - scratch(_call(ref, n_head=32)) == 4 * 32 * 1024 * 4 + 4 * 32 * 4
    assert scratch(_call(ref, n_head=7)) == 0                  # a call that is refused


def test_ops_refuse_memory_that_is_not_on_a_gpu():
    class Sizes:
        n_kv_head, head_dim, page_size, group, index, device, n_pages, ref = 2, 64, 16, 64, 0, torch.device("cuda:0"), 4, 0
    cache, i32 = Sizes(), torch.int32
    rows, slots = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=i32)
    table, weights = torch.zeros(3, 4, dtype=i32), torch.zeros(3, 2, 64)
    for call in (lambda: ops.append4(rows, rows, slots, cache, 3), lambda: ops.append4(rows, rows.float(), slots, cache, 3), lambda: ops.append4(rows, rows, slots, cache, 4),
                 lambda: ops.append4(rows[:, :64], rows, slots, cache, 3), lambda: ops.append4(rows, rows, slots.long(), cache, 3), lambda: ops.cache4_values(cache, slots, 3, rows, rows),
                 lambda: ops.decode_attention4(rows, cache, slots, table, rows, 3, 2, 0.1), lambda: ops.decode_attention4(rows, cache, slots, table, rows, 4, 2, 0.1),
                 lambda: ops.prefill_attention4(rows, cache, slots, slots, table, rows, 2, 3, 2, 0.1), lambda: ops.evict4(cache, weights, table, slots, 3, 16, 4, table, slots),
                 lambda: ops.Cache4(4, 2, 64, device="cpu"), lambda: ops.Cache4(4, 2, 80, device="cpu")):
        with pytest.raises(LiyabError):
            call()
