"""Products with 4-bit weights whose sums are never announced run their waits to the limit, report it and return.

The failure is made on the host's order and faults nothing: one launch leaves its accumulator-ready barriers unsignalled.  Whoever waits for them polls to the limit of about two
seconds, writes the status word and goes to the kernel's end, where tensor memory is given back; the next launches are right."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
FORMS = [(40, 256, 1024, "bfloat16", False),      # small tiles, two blocks an SM
         (16, 256, 1024, "e4m3", False),          # e4m3 that becomes float16 on its way
         (24, 512, 8192, "bfloat16", False),      # a reduction cut between the blocks of a cluster
         (100, 256, 1024, "bfloat16", True),      # one block an SM
         (250, 25600, 256, "bfloat16", False)]    # blocks that walk the tiles


@pytest.fixture(autouse=True)
def no_order_left_behind():
    from liyab_b200 import ops
    from liyab_b200.engine import device_status
    yield
    ops.lib().lb_linear4_withhold_next(0)
    device_status()


@pytest.mark.parametrize("M,N,K,rows,gated", FORMS)
def test_product_whose_sums_are_never_announced_gives_up_and_the_next_one_is_right(M, N, K, rows, gated):
    from liyab_b200 import ops
    from liyab_b200.engine import device_status
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(9)
    a, scale = torch.randn((M, K), generator=g).to(torch.bfloat16).to(dev), None
    if rows == "e4m3":
        a, scale = a.to(torch.float8_e4m3fn), torch.ones(M, device=dev)
    w = ops.quantise_weights4((torch.randn((N, K), generator=g) * 0.05).to(dev), 64, paired=gated)
    want = a.double() @ ops.weights4_values(w).double().t()
    if gated:
        want = want[:, :N // 2].clamp(min=0) * want[:, N // 2:]
    out = torch.zeros((M, N // 2 if gated else N), device=dev)

    def call():
        if gated:
            ops.gated4(a, w, out, M, gate="relu", a_scale=scale)
        else:
            ops.linear4(a, w, None, out, M, a_scale=scale)
        torch.cuda.synchronize()

    assert device_status() == (0, 0)
    ops.lib().lb_linear4_withhold_next(1)
    call()
    word, barrier = device_status()
    assert word >> 12 == 0xB and (word >> 8 & 0xF) in (1, 3, 4, 5) and barrier == 0, f"a role of the product reports itself: {word:#x}"
    for _ in range(3):
        out.fill_(float("nan"))
        call()
        # Sums of K products in 32 bits: K 2^-24 of their sizes, here below 1e-4 for values of a few units.
        assert (out.double() - want).abs().max().item() <= 1e-4 * max(1.0, want.abs().max().item())
    assert device_status() == (0, 0)
