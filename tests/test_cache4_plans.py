"""How attention over a 4-bit cache is cut, and what of its arguments is refused, without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from liyab_b200 import ops
from liyab_b200.status import LiyabError
from test_cache4 import AT, _cache, _call, _evict


def _plan(kv, heads, n_seq, keys, q_len, dim=128, **more):
    c, ref = _cache(kv=kv, dim=dim)
    got = (C.c_int * 4)()
    call = _call(ref, n_head=heads, n_seq=n_seq, n_tokens=n_seq * q_len, max_keys=keys, table_stride=-(-keys // 16), q_stride=heads * dim, out_stride=heads * dim, q_start=AT, max_q_len=q_len, **more)
    return tuple(got) if ops.lib().lb_attention4_plan(call, got) == 0 else None


def test_long_prompts_are_the_kernel_for_many_rows_s():
    """What the kernel for few rows does not number is the other's, up to what a launch gets through in seconds; the keys' weights come from the one for few rows alone."""
    assert _plan(8, 32, 1, 131072, 131072)[0] == 1             # 2^32 steps of eight rows and sixteen keys
    assert _plan(8, 32, 1, 1 << 19, 1 << 18)[0] == 1
    assert _plan(8, 32, 1, 1 << 20, 1 << 19) is None and b"more than one launch" in ops.lib().lb_last_error()
    assert _plan(8, 32, 1, 1 << 20, 1 << 19, window=4096)[0] == 1
    assert _plan(1, 4096, 1, 1 << 20, 64)[0] == 1
    assert _plan(1, 4096, 1, 1 << 20, 64, mass=AT, total=AT) is None and b"more than one launch" in ops.lib().lb_last_error()
    assert _plan(1, 4096, 1, 1 << 18, 64, mass=AT, total=AT)[0] == 0


def test_the_kernel_is_chosen_by_the_time_of_the_way_that_runs():
    """Calls whose keys all warps share out although a block to a row tile is estimated to be a bit shorter: it is the time of what would run that the other kernel's is compared with."""
    assert _plan(2, 8, 8, 4096, 16, dim=64)[:2] == (1, 256) and _plan(12, 12, 2, 4096, 48)[:2] == (1, 256)
    assert _plan(2, 8, 8, 4096, 4, dim=64)[0] == 0


def _overlap(a, b=None):
    """By listing them: whether two rows of a share a number, or one of a's and one of b's.  Rows: (place, row stride, head stride, rows, heads, width)."""
    def places(at, row, head, n, heads, width):
        return [at + r * row + h * head + i for r in range(n) for h in range(heads) for i in range(width)]
    x = places(*a)
    return len(set(x)) < len(x) if b is None else bool(set(x) & set(places(*b)))


# (row stride, head stride) of three rows of two heads of 64 numbers.
STRIDES = [(128, 64), (200, 64), (64, 192), (70, 300), (0, 64), (128, 0), (127, 64), (128, 63), (64, 191), (64, 64), (1000, 100)]


@pytest.mark.parametrize("row,head", STRIDES)
def test_rows_of_weights_that_overlap_are_refused(row, head):
    """Weights that go to the same numbers twice, by the strides of total and of dest_mass: three requests, two key/value heads, 64 keys (48 of which stay)."""
    c, ref = _cache(kv=2, device=99)                       # (what is not refused for its weights is for its device)
    weights = dict(mass=AT, mass_stride=128, mass_head=64, total=2 * AT, total_stride=row, total_head=head, n_mass=3)
    rc = ops.lib().lb_attention4(_call(ref, n_head=4, n_seq=3, n_tokens=3, max_keys=64, scratch=AT, **weights))
    assert rc != 0 and (b"overlap" in ops.lib().lb_last_error()) == _overlap((0, row, head, 3, 2, 64))
    rc = ops.lib().lb_evict4(_evict(ref, n_seq=3, keep=48, max_keys=64, n_mass=3, mass_stride=128, mass_head=64, dest_mass=2 * AT, dest_stride=row, dest_head=head, n_dest=3))
    assert rc != 0 and (b"overlap" in ops.lib().lb_last_error()) == _overlap((0, row, head, 3, 2, 48))


@pytest.mark.parametrize("mass,total", [((0, 128, 64), (0, 128, 64)), ((0, 128, 64), (384, 128, 64)), ((0, 128, 64), (383, 128, 64)), ((0, 256, 64), (128, 256, 64)), ((0, 256, 64), (127, 256, 64)),
                                        ((0, 256, 128), (64, 256, 128)), ((0, 256, 128), (65, 256, 128)), ((64, 256, 128), (0, 256, 128)), ((0, 256, 128), (-64, 256, 128)), ((1, 128, 64), (0, 128, 64)),
                                        ((0, 128, 64), (0, 256, 64)), ((0, 64, 192), (0, 128, 64)), ((0, 128, 64), (640, 128, 64)), ((700, 128, 64), (0, 256, 64)), ((0, 64, 400), (192, 64, 400))])
def test_weights_that_overlap_where_they_come_from_are_refused(mass, total):
    c, ref = _cache(kv=2, device=99)                       # (what is not refused for its weights is for its device)
    at = 2 * AT
    weights = dict(mass=at + 4 * mass[0], mass_stride=mass[1], mass_head=mass[2], total=at + 4 * total[0], total_stride=total[1], total_head=total[2], n_mass=3)
    rc = ops.lib().lb_attention4(_call(ref, n_head=4, n_seq=3, n_tokens=3, max_keys=64, scratch=AT, **weights))
    shared = mass != total and _overlap((*mass, 3, 2, 64), (*total, 3, 2, 64))
    assert rc != 0 and (b"overlap" in ops.lib().lb_last_error()) == shared
    # Of eviction's destinations the first 48 numbers of a row are written, and none may be one of mass's.
    rc = ops.lib().lb_evict4(_evict(ref, n_seq=3, keep=48, max_keys=64, n_mass=3, mass=at + 4 * mass[0], mass_stride=mass[1], mass_head=mass[2], dest_mass=at + 4 * total[0], dest_stride=total[1],
                                    dest_head=total[2], n_dest=3))
    assert rc != 0 and (b"memory of their own" in ops.lib().lb_last_error()) == _overlap((*mass, 3, 2, 64), (*total, 3, 2, 48))


def test_weights_of_single_rows_have_any_stride():
    c, ref = _cache(kv=1, device=99)
    for strides in ((0, 0), (7, 9)):
        weights = dict(mass=AT, mass_stride=1, mass_head=5, total=AT, total_stride=strides[0], total_head=strides[1], n_mass=1)
        rc = ops.lib().lb_attention4(_call(ref, n_head=4, n_seq=1, n_tokens=1, max_keys=64, scratch=AT, **weights))
        assert rc != 0 and b"overlap" not in ops.lib().lb_last_error()


def test_numbers_that_no_call_holds_are_refused(monkeypatch):
    """Sizes past 32 bits and negative ones are refused as the other arguments are, by `ops`, before the library is asked."""
    class Sizes:
        n_kv_head, head_dim, page_size, group, index, device, n_pages, ref, scratch = 2, 64, 1 << 20, 64, -1, torch.device("cpu"), 4, 0, {}
    monkeypatch.setattr(ops, "stream_of", lambda index: 0)
    monkeypatch.setattr(ops, "lib", lambda: pytest.fail("the library was asked"))
    cache, i32 = Sizes(), torch.int32
    rows, places, table = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(4, dtype=i32), torch.zeros(3, 4, dtype=i32)
    wide = torch.zeros(3, 1, dtype=i32).expand(3, 2048)                                        # 2^31 keys
    weights, kept = torch.zeros(3, 2, 64), torch.zeros(3, 2, 16, dtype=i32)
    for call in (lambda: ops.decode_attention4(rows, cache, places, table, rows, 3, 2, 0.1, max_keys=-1), lambda: ops.decode_attention4(rows, cache, places, table, rows, 3, 2, 0.1, window=1 << 40),
                 lambda: ops.decode_attention4(rows, cache, places, table, rows, 3, 2, 0.1, window=-(1 << 31)),
                 lambda: ops.decode_attention4(rows, cache, places, wide.contiguous(), rows, 3, 2, 0.1),
                 lambda: ops.prefill_attention4(rows, cache, places, places, table, rows, 3, 1 << 31, 2, 0.1),
                 lambda: ops.evict4(cache, weights, table, places, 3, 0, 0, table, kept[:, :, :0]), lambda: ops.evict4(cache, weights, table, places, 3, 16, -1, table, kept),
                 lambda: ops.evict4(cache, weights, table, places, 3, 16, 17, table, kept), lambda: ops.evict4(cache, weights, table, places, 3, 16, 1 << 32, table, kept),
                 lambda: ops.Cache4((1 << 32) + 1, 2, 64), lambda: ops.Cache4(4, 2, 64 + (1 << 32)), lambda: ops.Cache4(-1, 2, 64)):
        with pytest.raises(LiyabError):
            call()
