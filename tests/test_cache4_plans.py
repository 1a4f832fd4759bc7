"""How attention over a 4-bit cache is cut, and what of its arguments is refused, without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from liyab_b200 import ops
from test_cache4 import AT, _cache, _call


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
