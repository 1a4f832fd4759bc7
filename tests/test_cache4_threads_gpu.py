"""Attention over a 4-bit cache called by two threads of a process."""
from __future__ import annotations

import threading

import pytest
import torch

from liyab_b200 import ops
from test_cache4_gpu import Filled, _decode, _queries
from test_kernels_gpu import dev  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_launch_that_one_thread_withholds_is_not_taken_by_another(dev):  # noqa: F811
    """The order to leave a call's barriers unsignalled is its thread's: another thread's call in between is right, and the next one of this thread's runs its waits out."""
    from liyab_b200.engine import device_status
    f = Filled(dev, [300, 40], 2, 64, 32, 16, seed=3)
    q, out = _queries(f, 2, 4, 0), torch.empty(2, 256, dtype=torch.bfloat16, device=dev)
    places = torch.tensor([299, 39], dtype=torch.int32, device=dev)

    def call(to):
        return ops.decode_attention4(q, f.cache, places, f.table, to, 2, 4, 0.125)

    want = call(torch.empty_like(out)).clone()
    torch.cuda.synchronize()
    assert device_status() == (0, 0)
    ops.lib().lb_attention4_withhold_next(1)
    try:
        other = threading.Thread(target=lambda: (torch.cuda.set_device(dev), call(out), torch.cuda.synchronize()))
        other.start()
        other.join()
        status = device_status()
        assert status == (0, 0) and torch.equal(out, want)
        call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert device_status()[0] >> 12 == 0xC
    finally:
        ops.lib().lb_attention4_withhold_next(0)
        device_status()
    _decode(f, 4)
    assert device_status() == (0, 0)
