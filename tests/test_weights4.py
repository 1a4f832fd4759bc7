"""4-bit weights, what the host decides without a GPU: sizes of the memory they take, scratch that a product asks for, and refusals at the C entries."""
from __future__ import annotations

import ctypes as C

import pytest

from liyab_b200 import ops


def _sizes(n, k, group, paired):
    nibbles, scales, rows = C.c_int64(0), C.c_int64(0), C.c_int(0)
    status = ops.lib().lb_weights4_sizes(n, k, group, paired, C.byref(nibbles), C.byref(scales), C.byref(rows))
    return status, nibbles.value, scales.value, rows.value


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (128, 128, 128), (129, 127, 64), (50257, 1600, 128), (5003, 4104, 32), (2 * 5461, 2048, 64), (1 << 20, 16384, 128)])
@pytest.mark.parametrize("paired", [0, 1])
def test_sizes(n, k, group, paired):
    if paired and n % 2:
        assert _sizes(n, k, group, paired)[0] != 0
        return
    rows = 2 * (-(-(n // 2) // 8) * 8) if paired else n
    padded, wide = -(-rows // 128) * 128, -(-k // 128) * 128
    assert _sizes(n, k, group, paired) == (0, padded * wide // 2, padded * wide // group, padded)


@pytest.mark.parametrize("n,k,group,paired", [(0, 8, 32, 0), (8, 0, 32, 0), (-1, 8, 32, 0), (8, 8, 16, 0), (8, 8, 0, 0), (7, 8, 32, 1), (1 << 27, 8, 32, 0)])
def test_sizes_refused(n, k, group, paired):
    assert _sizes(n, k, group, paired)[0] != 0 and ops.lib().lb_last_error()


def test_arguments_are_as_long_as_the_library_reads_them():
    """Both products and the norm copy their arguments as one struct: a shorter one here would be read past its end."""
    length = ops.lib().lb_struct_bytes
    assert len(ops._linear4_args(*[0] * 15, 0.0, 0.0)) == length(4)
    assert len(ops._rms_add_args(*[0] * 17, 0.0, 0.0)) == length(5)
    assert C.sizeof(ops.Weights4Args) == length(6)


def _weights(n, k, group=128, paired=0, nibbles=1 << 20):
    w = ops.Weights4Args(nibbles, 1 << 20, 1 << 20, n, k, group, paired)
    return w, C.addressof(w)


def test_scratch_for_rows_that_are_not_read_as_they_are():
    scratch, at = ops.lib().lb_linear4_scratch, 1 << 20
    w, ref = _weights(4096, 4096)
    BF16, E4M3 = ops.BF16, ops.E4M3
    assert scratch(ref, BF16, at, 4096, 1) == scratch(ref, BF16, at + 2, 4096, 8) == scratch(ref, E4M3, at + 1, 4097, 8) == 0      # up to eight tokens: any rows
    assert scratch(ref, BF16, at, 4096, 100) == 0                              # rows that TMA takes
    assert scratch(ref, BF16, at + 2, 4096, 100) == scratch(ref, BF16, at, 4097, 100) == 100 * 4096 * 2
    assert scratch(ref, E4M3, at, 4096, 16) == 0                               # e4m3 that becomes float16 on its way
    assert scratch(ref, E4M3, at + 1, 4096, 16) == 16 * 4096 * 2
    assert scratch(ref, E4M3, at, 4096, 300) == 300 * 4096 * 2
    w, ref = _weights(64, 131)
    assert scratch(ref, BF16, at, 131, 9) == 9 * 136 * 2                       # rows filled up to eights
    assert scratch(ref, BF16, at, 136, 0) == scratch(None, BF16, at, 136, 9) == 0


def test_how_a_product_is_cut():
    """One token to many: the kernel for few, tiles with a block each, reductions that blocks share, blocks that walk the tiles."""
    def plan(n, k, m, paired=0, out=ops.BF16):
        w, ref = _weights(n, k, paired=paired)
        got = (C.c_int * 4)()
        assert ops.lib().lb_linear4_plan(ref, m, out, got) == 0
        return tuple(got)
    assert plan(1600, 1600, 1) == (0, 1, 1, 100) and plan(1600, 1600, 8)[0] == 0 and plan(1600, 1600, 9)[0] == 1
    assert plan(4096, 16384, 8)[::2] == (0, 2)                                 # activations of a whole reduction do not fit a block
    for n, k, m, paired in ((8192, 8192, 2048, 0), (7002, 200, 600, 0), (7002, 200, 600, 1)):
        which, tokens, splits, tiles = plan(n, k, m, paired)
        assert which == 2 and splits == 1 and tokens % 16 == 0 and 16 <= tokens <= 256 and tiles == -(-m // tokens) * -(-n // 128) > 148
    assert plan(512, 8192, 24)[2] > 1
    w, ref = _weights(64, 64)
    assert ops.lib().lb_linear4_plan(ref, 0, ops.BF16, (C.c_int * 4)()) != 0 and ops.lib().lb_linear4_plan(ref, 1, ops.F32, None) != 0 and ops.lib().lb_linear4_plan(ref, 1, 5, (C.c_int * 4)()) != 0


@pytest.mark.parametrize("n,k,paired", [(64, 1, False), (1600, 1600, False), (4096, 8192, True), (512, 16384, False), (16, 90000, False), (16, 250000, False), (16, 2000000, False)])
def test_which_products_never_need_scratch(n, k, paired):
    """The number that calls compare their rows with is the library's: as many rows as the kernel for few takes."""
    import torch
    w = ops.Weights4(n, k, 128, paired, torch.device("cpu"))
    kinds = []
    for m in range(1, 12):
        out = (C.c_int * 4)()
        assert ops.lib().lb_linear4_plan(w.ref, m, ops.F32, out) == 0
        kinds.append(out[0] != 0)
    assert w.few == (kinds + [True]).index(True) and all(kinds[w.few:])


def _call(name, ref, a=1 << 20, scale=0, bias=0, residual=0, out=1 << 20, lda=256, ldr=0, ldo=64, code=None, out_code=0, m=0, act=0):
    code = ops.BF16 if code is None else code
    return getattr(ops.lib(), name)(ops._linear4_args(ref or 0, a, scale, bias, residual, out, 0, 0, lda, ldr, ldo, code, out_code, m, act, 0.0, 0.0))


def test_products_refuse_before_they_launch():
    plain, ref = _weights(64, 256)
    pairs, pref = _weights(128, 256, paired=1)
    assert _call("lb_linear4", ref) == 0 and _call("lb_gated4", pref) == 0     # no rows: nothing to do
    assert _call("lb_linear4", ref, a=0, out=0) == 0
    bad = [dict(m=-1), dict(m=1, a=0), dict(m=1, out=0), dict(lda=255), dict(ldo=63), dict(residual=1 << 20, ldr=63), dict(code=7), dict(out_code=ops.E4M3), dict(code=ops.E4M3),
           dict(scale=1 << 20), dict(m=65535 * 16 + 1)]
    for kw in bad:
        assert _call("lb_linear4", ref, **kw) != 0, kw
    for kw in (dict(act=-1), dict(act=99)):
        assert _call("lb_linear4", ref, **kw) != 0 and _call("lb_gated4", pref, **kw) != 0, kw
    assert _call("lb_linear4", pref) != 0 and _call("lb_gated4", ref) != 0     # pairs are for the gated product
    assert _call("lb_gated4", pref, bias=1 << 20) != 0 and _call("lb_gated4", pref, residual=1 << 20, ldr=128) != 0
    odd, oref = _weights(64, 256, group=48)
    assert _call("lb_linear4", oref) != 0
    empty, eref = _weights(64, 256, nibbles=0)
    assert _call("lb_linear4", eref) != 0 and _call("lb_linear4", None) != 0


@pytest.mark.parametrize("change", [dict(n=0), dict(k=0), dict(n=-16), dict(k=-128), dict(n=1 << 27), dict(n=127, paired=1), dict(group=0), dict(nibbles=(1 << 20) + 8), dict(scales=(1 << 20) + 4),
                                    dict(rows=(1 << 20) + 2), dict(scales=0), dict(rows=0)])
def test_weights_that_no_kernel_can_read_are_refused(change):
    """As an invalid argument (1), by whichever entry is given them, with an error and not by a division by zero or a fault in a kernel."""
    w = ops.Weights4Args(**{**dict(nibbles=1 << 20, scales=1 << 20, rows=1 << 20, n=128, k=256, group=128, paired=0), **change})
    ref = C.addressof(w)
    for m in (1, 9):
        assert _call("lb_linear4", ref, m=m, lda=1 << 27, ldo=1 << 27) == 1 and _call("lb_gated4", ref, m=m, lda=1 << 27, ldo=1 << 27) == 1
        assert ops.lib().lb_linear4_scratch(ref, ops.BF16, 1 << 20, 1 << 27, m) == 0 and ops.lib().lb_linear4_plan(ref, m, ops.F32, (C.c_int * 4)()) == 1
    assert ops.lib().lb_weights4_values(ref, 1 << 20, 1 << 27, None) == 1


def test_pointers_off_their_type_are_refused():
    plain, ref = _weights(64, 256)
    at = 1 << 20
    for kw in (dict(a=at + 1), dict(out=at + 1), dict(out=at + 2, out_code=ops.F32), dict(bias=at + 2), dict(residual=at + 1, ldr=64), dict(code=ops.E4M3, scale=at + 2)):
        assert _call("lb_linear4", ref, m=1, **kw) == 1, kw
