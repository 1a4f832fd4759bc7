"""The bounded waits of products with 4-bit weights whose reduction is several chains of additions (float32 results over long reductions): as in test_weights4_waits_gpu.py, which describes
the failure that the host makes."""
from __future__ import annotations

import pytest

import test_weights4_waits_gpu as waits

pytestmark = pytest.mark.gpu
no_order_left_behind = waits.no_order_left_behind
FORMS = [(64, 300, 16384, "bfloat16", False),     # small tiles, an accumulator a chain
         (250, 2048, 9000, "e4m3", True),         # and large ones
         (100, 6400, 16384, "bfloat16", False),   # finishing warps that move a chain's sums, blocks that share a reduction
         (250, 25600, 1700, "bfloat16", False)]   # and blocks that walk the tiles


@pytest.mark.parametrize("M,N,K,rows,gated", FORMS)
def test_chained_product_whose_sums_are_never_announced_gives_up_and_the_next_one_is_right(M, N, K, rows, gated):
    waits.test_product_whose_sums_are_never_announced_gives_up_and_the_next_one_is_right(M, N, K, rows, gated)
