"""Attention over a 4-bit cache whose keys or scores are never announced runs its waits to the limit, reports it and returns.

The failure is made on the host's order and faults nothing: one call's kernel leaves barriers unsignalled (a warp's second tile of a pair is not asked for; a group's scores are computed and
not announced).  Whoever waits for them polls to the limit of about two seconds, writes the status word and goes to the kernel's end; the next calls are right."""
from __future__ import annotations

import pytest
import torch

from liyab_b200 import ops
from test_cache4_gpu import Filled, _decode, _portions, _queries, _way
from test_kernels_gpu import dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_order_left_behind():
    from liyab_b200.engine import device_status
    yield
    ops.lib().lb_attention4_withhold_next(0)
    device_status()


@pytest.mark.parametrize("lengths,heads,new", [([300, 40], 4, 1),              # a block for each request and key/value head
                                               ([9000, 40], 4, 1),             # warps that share the keys, and states joined
                                               ([400, 300], 32, 300),          # many rows
                                               ([6000, 90], 32, 60)])          # many rows whose keys blocks share
def test_keys_that_are_never_announced_and_the_next_calls_are_right(dev, lengths, heads, new):  # noqa: F811
    from liyab_b200.engine import device_status
    f = Filled(dev, lengths, 2, 64, 32, 16, seed=3)
    news = [min(new, n) for n in lengths]
    assert new == 1 or _way(f, 2, heads, new)[0] == 1

    def call():
        _decode(f, heads) if new == 1 else _portions(f, news, heads)

    call()
    assert device_status() == (0, 0)
    ops.lib().lb_attention4_withhold_next(1)
    q, out = _queries(f, sum(news), heads, 0), torch.empty(sum(news), heads * 64, dtype=torch.bfloat16, device=dev)
    if new == 1:
        ops.decode_attention4(q, f.cache, torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device=dev), f.table, out, 2, heads, 0.125)
    else:
        start, past = torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device=dev), torch.tensor([a - b for a, b in zip(lengths, news)], dtype=torch.int32, device=dev)
        ops.prefill_attention4(q, f.cache, start, past, f.table, out, 2, new, heads, 0.125)
    torch.cuda.synchronize()
    word, barrier = device_status()
    assert word >> 12 == 0xC and 1 <= (word & 0xFFF) <= 6 and barrier == 0, f"a role reports itself: {word:#x}"
    for _ in range(3):
        call()
    assert device_status() == (0, 0)
