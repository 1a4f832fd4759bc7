"""4-bit weights: their layout and rounding, the products that read them and the norm that feeds those, against plain forms in 64 bits."""
from __future__ import annotations

import pytest
import torch

from test_kernels_gpu import _rand, dev  # noqa: F401

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _parts(n, k, group, dev, seed=0):
    """(q, s, r): every value of q and a wide range of scales, among them zeros."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    s = torch.rand((n, -(-k // group)), generator=g) * 448.0
    s = torch.where(torch.rand(s.shape, generator=g) < 0.05, torch.zeros(()), s).to(F8)
    r = torch.exp(torch.randn((n,), generator=g)) * 1e-4
    return q.to(dev), s.to(dev), r.to(dev)


def _matrix(q, s, r, group):
    """The matrix in 64 bits."""
    at = torch.arange(q.shape[1], device=q.device) // group
    return q.double() * s.double()[:, at] * r.double()[:, None]


def _rows8(a):
    scale = a.float().abs().amax(1) / 448.0
    return (a.float() / scale[:, None]).to(F8), scale


def _sum_bound(k):
    """Relative to the sum of the terms' sizes: the tensor core adds 16 products to a 32-bit sum at a time, each time with an error below 2^-23 of the larger of the two
    (truncation); a group's scale, the parts' sums, the row's factor and scale, bias and residual add less than 16 further roundings."""
    return (k / 16 + 16) * 2.0 ** -23


SHAPES = [(1, 1, 32), (8, 31, 64), (16, 128, 128), (17, 129, 64), (100, 200, 32), (250, 1000, 128), (1600, 1600, 64), (1000, 4104, 128), (5003, 768, 128), (129, 16384, 32)]
TOKENS = [1, 2, 7, 8, 9, 16, 17, 31, 64, 65, 130, 300]


# ---- the weights -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("paired", [False, True])
def test_laid_out_and_back(dev, n, k, group, paired):
    from liyab_b200 import ops
    n = 2 * n if paired else n
    q, s, r = _parts(n, k, group, dev)
    w = ops.lay_out_weights4(q, s, r, group, paired)
    at = torch.arange(k, device=dev) // group
    assert torch.equal(ops.weights4_values(w), q.float() * s.float()[:, at] * r[:, None])       # q s is exact: one rounding on both sides


@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rounded_to_four_bits(dev, n, k, group, paired, dtype):
    """The same weights as the definition gives in 32-bit arithmetic on the CPU (whose divisions are rounded correctly, as the kernel's are)."""
    from liyab_b200 import ops
    n = 2 * n if paired else n
    g = torch.Generator().manual_seed(n + k)
    m = torch.randn((n, k + 3), generator=g) * torch.exp(torch.randn((n, 1), generator=g)) * 0.02
    m[0] = 0.0
    m[-1, : k // 2] *= 1e-7                                     # groups far below their row's largest
    m = m.to(dtype)[:, :k]
    groups = -(-k // group)
    padded = torch.nn.functional.pad(m.float(), (0, groups * group - k)).view(n, groups, group)
    t = padded.abs().amax(2) / torch.tensor(7.0)
    r = t.amax(1) / torch.tensor(448.0)
    s = torch.where(r[:, None] > 0, t / r[:, None], torch.zeros(())).clamp(max=448.0).to(F8)
    step = s.float() * r[:, None]
    q = torch.where(step[..., None] > 0, padded / step[..., None], torch.zeros(())).round().clamp(-8, 7)
    want = (q * s.float()[..., None] * r[:, None, None]).reshape(n, -1)[:, :k]
    w = ops.quantise_weights4(m.to(dev), group, paired)
    assert torch.equal(ops.weights4_values(w).cpu(), want)


def test_rounding_of_special_rows(dev):
    """Rows of zeros and of numbers too small for a normal factor become zeros; an infinity or a NaN makes its row NaN and leaves the others alone."""
    from liyab_b200 import ops
    m = torch.randn((24, 256), generator=torch.Generator().manual_seed(3))
    m[1], m[2], m[3, 7], m[4, 200], m[5] = 0.0, 1e-40, float("inf"), float("nan"), 1e30 * m[5]
    got = ops.weights4_values(ops.quantise_weights4(m.to(dev), 64)).cpu()
    assert (got[1:3] == 0).all() and got[3:5].isnan().all() and got[[0, *range(5, 24)]].isfinite().all()
    # The nearest of steps of (largest / 7): half a step off, and a scale in e4m3 is up to 1/16 off and may clamp 7.47 steps to 7.
    step = m[6:].view(18, 4, 64).abs().amax(2, keepdim=True) / 7.0
    assert ((got[6:].view(18, 4, 64) - m[6:].view(18, 4, 64)).abs() <= 0.55 * step).all()


# ---- the products ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", TOKENS)
@pytest.mark.parametrize("n,k,group", SHAPES)
@pytest.mark.parametrize("eight", [False, True])
def test_linear(dev, m, n, k, group, eight):
    """float32 results with a residual in place, bfloat16 ones with bias and activation, both against 64 bits; the same bits on a second call."""
    from liyab_b200 import ops
    q, s, r = _parts(n, k, group, dev, seed=m)
    w, ref_w = ops.lay_out_weights4(q, s, r, group), _matrix(q, s, r, group)
    a, scale = _rand((m, k), 5, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    bias, res = _rand((n,), 6, dev), _rand((m, n + 8), 7, dev)[:, :n]
    ref = rows @ ref_w.T
    bound = _sum_bound(k) * (rows.abs() @ ref_w.abs().T + bias.double().abs() + res.double().abs())
    outs = []
    for _ in range(2):
        out = res.clone()
        ops.linear4(a, w, None, out, m, residual=out, a_scale=scale)
        assert ops.device_status() == 0
        assert ((out.double() - ref - res.double()).abs() <= bound).all()
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    half = torch.full((m, n + 3), float("nan"), dtype=torch.bfloat16, device=dev)
    ops.linear4(a, w, bias, half[:, :n], m, activation="relu2", a_scale=scale)
    z = ref + bias.double()
    want = z.clamp(min=0) ** 2
    assert ((half[:, :n].double() - want).abs() <= 2.0 ** -8 * want + 2 * (z.abs() + bound) * bound).all()
    assert half[:, n:].isnan().all()


@pytest.mark.parametrize("m,n,k", [(8, 76200, 6900), (5, 76200, 700)])
def test_rounds_of_row_tiles(dev, m, n, k):
    """More row tiles than a block takes between two barriers, in blocks that share an SM and in ones whose activations leave no room for a second; every eleventh feature is looked at."""
    from liyab_b200 import ops
    g = torch.Generator(device=dev).manual_seed(k)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device=dev)
    s = (torch.rand((n, -(-k // 128)), generator=g, device=dev) * 448.0).to(F8)
    r = torch.rand((n,), generator=g, device=dev) * 1e-4
    a = _rand((m, k), 16, dev).to(torch.bfloat16)
    out = torch.full((m, n), float("nan"), device=dev)
    ops.linear4(a, ops.lay_out_weights4(q, s, r, 128), None, out, m)
    assert ops.device_status() == 0
    assert out.isfinite().all()
    some = torch.arange(0, n, 11, device=dev)
    ref_w = _matrix(q[some], s[some], r[some], 128)
    assert ((out[:, some].double() - a.double() @ ref_w.T).abs() <= _sum_bound(k) * (a.double().abs() @ ref_w.abs().T)).all()


@pytest.mark.parametrize("m,n,k,splits", [(8, 38505, 14500, 2), (8, 20003, 30000, 4), (5, 10007, 90000, 8)])
def test_shared_reductions_in_rounds(dev, m, n, k, splits):
    """Blocks that share a reduction take more row tiles than fit between two barriers, and the features end inside a warp's; every 37th feature and the last ones are looked at."""
    from liyab_b200 import ops
    g = torch.Generator(device=dev).manual_seed(k)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device=dev)
    s = (torch.rand((n, -(-k // 128)), generator=g, device=dev) * 448.0).to(F8)
    r = torch.rand((n,), generator=g, device=dev) * 1e-4
    w = ops.lay_out_weights4(q, s, r, 128)
    assert ops.linear4_plan(w, m)[0] == "few" and ops.linear4_plan(w, m)[2] == splits
    a, res = _rand((m, k), 17, dev).to(torch.bfloat16), _rand((m, n), 18, dev)
    out = res.clone()
    ops.linear4(a, w, None, out, m, residual=out)
    assert ops.device_status() == 0
    assert out.isfinite().all()
    some = torch.cat([torch.arange(0, n, 37, device=dev), torch.arange(n - 20, n, device=dev)])
    ref_w = _matrix(q[some], s[some], r[some], 128)
    size = a.double().abs() @ ref_w.abs().T + res[:, some].double().abs()
    assert ((out[:, some].double() - a.double() @ ref_w.T - res[:, some].double()).abs() <= _sum_bound(k) * size).all()


@pytest.mark.parametrize("m,n,k,group", [(20, 19100, 160, 32), (33, 25000, 64, 64), (130, 12900, 333, 128), (600, 7001, 200, 64), (2500, 1600, 1100, 128), (257, 19000, 129, 32),
                                         (1, 28446, 200, 64), (8, 30010, 97, 32), (3, 40000, 1290, 128), (4, 152000, 130, 128)])
@pytest.mark.parametrize("eight", [False, True])
def test_many_tiles(dev, m, n, k, group, eight):
    """More tiles than SMs, with remainders of rows, tokens and k tiles; as a gated product too."""
    from liyab_b200 import ops
    q, s, r = _parts(n, k, group, dev, seed=m)
    w, ref_w = ops.lay_out_weights4(q, s, r, group), _matrix(q, s, r, group)
    a, scale = _rand((m, k), 14, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    bias = _rand((n,), 15, dev)
    ref = rows @ ref_w.T
    size = rows.abs() @ ref_w.abs().T
    out = torch.full((m, n), float("nan"), device=dev)
    ops.linear4(a, w, bias, out, m, a_scale=scale)
    assert ops.device_status() == 0
    assert ((out.double() - ref - bias.double()).abs() <= _sum_bound(k) * (size + bias.double().abs())).all()
    if n % 2 == 0:
        f = n // 2
        half = torch.full((m, f), float("nan"), dtype=torch.bfloat16, device=dev)
        ops.gated4(a, ops.lay_out_weights4(q, s, r, group, paired=True), half, m, gate="relu", a_scale=scale)
        assert ops.device_status() == 0
        want, eg, eu = ref[:, :f].clamp(min=0) * ref[:, f:], _sum_bound(k) * size[:, :f], _sum_bound(k) * size[:, f:]
        bound = eg * (ref[:, f:].abs() + eu) + ref[:, :f].abs() * eu
        assert ((half.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


LONG = [(9, 2048, 16384, 64), (24, 512, 9000, 32), (64, 300, 16384, 128), (100, 6400, 16384, 64), (130, 1000, 2177, 64), (300, 2048, 11456, 128), (1711, 2673, 11456, 32), (2048, 4096, 5000, 64),
        (700, 20000, 2300, 128), (250, 136, 16300, 64), (5, 64, 300000, 128)]


@pytest.mark.parametrize("m,n,k,group", LONG)
@pytest.mark.parametrize("eight", [False, True])
def test_long_reductions_keep_float32_results(dev, m, n, k, group, eight):
    """The tensor core truncates every addition: chains of up to 2,048 values, which measure 3.4e-7 of the results (norms), a row's factors and scales a few 2^-24 and the chains' sums less: below 6e-7
    at every length.  One chain over these lengths has 1e-6 to 5e-6."""
    from liyab_b200 import ops
    g = torch.Generator(device=dev).manual_seed(k)
    q = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8, device=dev)
    s = (torch.rand((n, -(-k // group)), generator=g, device=dev) * 448.0).to(F8)
    r = torch.rand((n,), generator=g, device=dev) * 1e-4 + 1e-5
    ref_w, w = _matrix(q, s, r, group), ops.lay_out_weights4(q, s, r, group)
    a, scale = torch.randn((m, k), generator=g, device=dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    want, out, res = rows @ ref_w.T, torch.full((m, n), float("nan"), device=dev), torch.randn((m, n), generator=g, device=dev)
    ops.linear4(a, w, None, out, m, a_scale=scale)
    assert ops.device_status() == 0
    assert ((out.double() - want).norm() / want.norm()).item() <= 6e-7
    assert ((out.double() - want).abs() <= _sum_bound(k) * (rows.abs() @ ref_w.abs().T)).all()
    again = res.clone()
    ops.linear4(a, w, None, again, m, residual=again, a_scale=scale)
    assert torch.equal(again, out + res)                          # the same sums, then one addition
    f = n // 2
    half, both = torch.empty((m, f), device=dev), rows @ ref_w[:2 * f].T
    ops.gated4(a, ops.lay_out_weights4(q[:2 * f], s[:2 * f], r[:2 * f], group, paired=True), half, m, gate="relu", a_scale=scale)
    assert ops.device_status() == 0
    want = both[:, :f].clamp(min=0) * both[:, f:]
    assert ((half.double() - want).norm() / want.norm()).item() <= 1.2e-6                             # two factors


@pytest.mark.parametrize("m", [1, 5, 16, 40, 129])
@pytest.mark.parametrize("activation", ["gelu_tanh", "gelu_erf", "xielu", "relu2", "none"])
def test_activations(dev, m, activation):
    """Beside the product of the 32-bit units on the matrix that the weights stand for."""
    from liyab_b200 import ops
    n, k = 328, 640
    q, s, r = _parts(n, k, 64, dev)
    w = ops.lay_out_weights4(q, s, r * 0.05, 64)
    a, bias = _rand((m, k), 8, dev, torch.bfloat16), _rand((n + 2,), 9, dev)
    bias[n:] = torch.tensor([0.8, 0.4], device=dev)
    want, out = torch.empty((m, n), device=dev), torch.empty((m, n), device=dev)
    values = ops.weights4_values(w)
    ops.gemm_ffma(a.float(), values, bias, want, m, activation)
    ops.linear4(a, w, bias, out, m, activation=activation)
    # Both sums are within the bound of the exact one; the activations' slopes stay below 3 here but for the two squares.
    size = a.double().abs() @ values.double().abs().T + bias[:n].double().abs()
    slope = 3.0 + 4.0 * (size if activation in ("relu2", "xielu") else 0.0)
    assert ((out.double() - want.double()).abs() <= 2.0 * _sum_bound(2 * k) * size * slope).all()


@pytest.mark.parametrize("m", TOKENS)
@pytest.mark.parametrize("f,k,group", [(1, 1, 32), (8, 64, 64), (9, 129, 128), (100, 200, 32), (682, 1600, 64), (1000, 4104, 128), (2731, 2048, 64)])
@pytest.mark.parametrize("eight", [False, True])
def test_gated(dev, m, f, k, group, eight):
    from liyab_b200 import ops
    q, s, r = _parts(2 * f, k, group, dev, seed=m + 1)
    r = r * 0.05
    w, ref_w = ops.lay_out_weights4(q, s, r, group, paired=True), _matrix(q, s, r, group)
    a, scale = _rand((m, k), 10, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    both, size = rows @ ref_w.T, _sum_bound(k) * (rows.abs() @ ref_w.abs().T)
    g, u, eg, eu = both[:, :f], both[:, f:], size[:, :f], size[:, f:]
    for gate in ("silu", "relu", "gelu_tanh", "sigmoid", "capped"):
        if gate == "capped":
            gg, uu = g.clamp(max=2.0), u.clamp(-2.0, 2.0)
            want, uu = gg * torch.sigmoid(1.7 * gg) * (uu + 1.0), uu + 1.0
            slope, act = 1.7, gg * torch.sigmoid(1.7 * gg)
        else:
            act = {"silu": lambda: g * torch.sigmoid(g), "relu": lambda: g.clamp(min=0), "sigmoid": lambda: torch.sigmoid(g),
                   "gelu_tanh": lambda: 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3)))}[gate]()
            want, uu, slope = act * u, u, 1.2
        for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
            out = torch.full((m, f + 1), float("nan"), dtype=dtype, device=dev)
            ops.gated4(a, w, out[:, :f], m, gate=gate, a_scale=scale, alpha=1.7, limit=2.0)
            # The product's rule on both sums' errors, and the gate's own 32-bit arithmetic (under 16 roundings).
            bound = slope * eg * (uu.abs() + eu) + act.abs() * eu + 2.0 ** -19 * (want.abs() + act.abs()) + 1e-30
            assert ((out[:, :f].double() - want).abs() <= bound + rounding * want.abs()).all(), (gate, dtype)
            assert out[:, f:].isnan().all()
    assert ops.device_status() == 0


def _activated(z, kind, a=0.8, b=0.4):
    """(the activation of z in 64 bits, a bound on its slope within e of z as a function of e)"""
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3))), lambda e: 1.2
    if kind == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476)), lambda e: 1.2
    if kind == "xielu":
        a, b = torch.nn.functional.softplus(torch.tensor([a, b], dtype=torch.float64)).tolist()
        return torch.where(z > 0, a * z * z + 0.5 * z, (b + 0.5) * (torch.expm1(z.clamp(max=0)) - z) + 0.5 * z), lambda e: 2 * a * (z.abs() + e) + b + 1.0
    if kind == "relu2":
        return z.clamp(min=0) ** 2, lambda e: 2 * (z.abs() + e)
    return z, lambda e: 1.0


@pytest.mark.parametrize("m,n,k,group", [(1, 328, 640, 64), (7, 1001, 333, 32), (9, 328, 640, 64), (30, 1001, 333, 32), (64, 2000, 1000, 128), (100, 6400, 200, 64), (140, 328, 640, 64),
                                         (24, 512, 8192, 128), (250, 1003, 2000, 64), (600, 3610, 200, 64), (1000, 1001, 4096, 32)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("activation", ["none", "gelu_tanh", "gelu_erf", "xielu", "relu2"])
def test_activations_in_both_results(dev, m, n, k, group, eight, activation):
    """Few tokens, small tiles, whole tiles and reductions that blocks share: float32 with a residual, bfloat16 (whose exponentials are the fast ones) with and without one."""
    from liyab_b200 import ops
    q, s, r = _parts(n, k, group, dev, seed=m + 2)
    r = r * 0.02
    w, ref_w = ops.lay_out_weights4(q, s, r, group), _matrix(q, s, r, group)
    assert ops.linear4_plan(w, m)[0] == ("few" if m <= 8 else "tiles")
    a, scale = _rand((m, k), 44, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    bias, res = _rand((n + 2,), 45, dev), _rand((m, n), 46, dev)
    bias[n:] = torch.tensor([0.8, 0.4], device=dev)
    z = rows @ ref_w.T + bias[:n].double()
    e = _sum_bound(k) * (rows.abs() @ ref_w.abs().T + bias[:n].double().abs())
    want, slope = _activated(z, activation)
    # The bounds of test_walked_tiles.
    bound = e * slope(e) + 2.0 ** -19 * (want.abs() + z.abs()) + 2.0 ** -23 * res.double().abs()
    out = res.clone()
    ops.linear4(a, w, bias, out, m, activation=activation, residual=out, a_scale=scale)
    assert ((out.double() - want - res.double()).abs() <= bound).all()
    half = torch.empty((m, n), dtype=torch.bfloat16, device=dev)
    for residual in (None, res):
        ops.linear4(a, w, bias, half, m, activation=activation, residual=residual, a_scale=scale)
        total = want if residual is None else want + res.double()
        assert ((half.double() - total).abs() <= bound + 2.0 ** -15 * (want.abs() + bound) + 2.0 ** -8 * (total.abs() + bound) + 2.0 ** -19 * z.abs()).all()
    assert ops.device_status() == 0


# Products whose blocks walk the tiles: remainders of rows, tokens and k tiles.
WALKS = [(600, 7002, 200, 64), (1030, 5006, 72, 32), (700, 8010, 1000, 128)]


@pytest.mark.parametrize("m,n,k,group", WALKS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("activation", ["none", "gelu_tanh", "gelu_erf", "xielu", "relu2"])
def test_walked_tiles(dev, m, n, k, group, eight, activation):
    """Blocks that walk the tiles, with a bias, an activation and a residual (float32: in place), in both result types."""
    from liyab_b200 import ops
    q, s, r = _parts(n, k, group, dev, seed=m)
    r = r * 0.02
    w, ref_w = ops.lay_out_weights4(q, s, r, group), _matrix(q, s, r, group)
    assert ops.linear4_plan(w, m)[0] == "walk"
    a, scale = _rand((m, k), 40, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    bias, res = _rand((n + 2,), 41, dev), _rand((m, n), 42, dev)
    bias[n:] = torch.tensor([0.8, 0.4], device=dev)
    z = rows @ ref_w.T + bias[:n].double()
    e = _sum_bound(k) * (rows.abs() @ ref_w.abs().T + bias[:n].double().abs())
    want, slope = _activated(z, activation)
    # The sum's error times the slope; the function's own arithmetic (library calls in 32 bits: under 16 roundings of terms no larger than z and the value); the residual's addition.
    bound = e * slope(e) + 2.0 ** -19 * (want.abs() + z.abs()) + 2.0 ** -23 * res.double().abs()
    out = res.clone()
    ops.linear4(a, w, bias, out, m, activation=activation, residual=out, a_scale=scale)
    assert ops.device_status() == 0
    assert ((out.double() - want - res.double()).abs() <= bound).all()
    half = torch.full((m, n + 1), float("nan"), dtype=torch.bfloat16, device=dev)
    ops.linear4(a, w, bias, half[:, :n], m, activation=activation, a_scale=scale)
    assert ops.device_status() == 0
    # Results in bfloat16: the fast exponential (2 + 1.2 |argument| units of 2^-23, arguments to 90) and division, then the rounding.
    assert ((half[:, :n].double() - want).abs() <= bound + (2.0 ** -8 + 2.0 ** -15) * (want.abs() + bound) + 2.0 ** -19 * z.abs()).all()
    assert half[:, n:].isnan().all()


@pytest.mark.parametrize("m,n,k", [(1, 264, 320), (8, 264, 4096), (12, 264, 320), (40, 264, 320), (100, 264, 320), (24, 512, 8192), (600, 7002, 200)])
def test_bias_that_the_launch_before_wrote(dev, m, n, k):
    """The bias, xIELU's two numbers behind it among them, comes from a product right before, which the launch overlaps; other numbers every time."""
    from liyab_b200 import ops
    q, s, r = _parts(n, k, 64, dev)
    w, ref_w = ops.lay_out_weights4(q, s, r * 0.02, 64), _matrix(q, s, r * 0.02, 64)
    makes = ops.quantise_weights4(_rand((n + 2, 2048), 50, dev, scale=0.02), 128)
    a = _rand((m, k), 51, dev, torch.bfloat16)
    sources, biases, outs = _rand((6, 2048), 52, dev, torch.bfloat16), torch.zeros((1, n + 2), device=dev), torch.empty((6, m, n), device=dev)
    seen = torch.empty((6, n + 2), device=dev)
    for i in range(6):
        ops.linear4(sources[i:i + 1], makes, None, biases, 1)
        ops.linear4(a, w, biases[0], outs[i], m, activation="xielu")
        seen[i].copy_(biases[0])
    assert ops.device_status() == 0 and len({tuple(b.tolist()) for b in seen[:, n:]}) == 6
    for i in range(6):
        z = a.double() @ ref_w.T + seen[i, :n].double()
        e = _sum_bound(k) * (a.double().abs() @ ref_w.abs().T + seen[i, :n].double().abs())
        want, slope = _activated(z, "xielu", seen[i, n].item(), seen[i, n + 1].item())
        assert ((outs[i].double() - want).abs() <= e * slope(e) + 2.0 ** -19 * (want.abs() + z.abs())).all()


@pytest.mark.parametrize("m,n,k,group", WALKS)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("gate", ["silu", "relu", "gelu_tanh", "sigmoid", "capped"])
def test_walked_gates(dev, m, n, k, group, eight, gate):
    from liyab_b200 import ops
    f = n // 2
    q, s, r = _parts(n, k, group, dev, seed=m + 1)
    r = r * 0.02
    w, ref_w = ops.lay_out_weights4(q, s, r, group, paired=True), _matrix(q, s, r, group)
    assert ops.linear4_plan(w, m)[0] == "walk"
    a, scale = _rand((m, k), 43, dev), None
    if eight:
        a, scale = _rows8(a)
        rows = a.double() * scale.double()[:, None]
    else:
        a = a.to(torch.bfloat16)
        rows = a.double()
    both, size = rows @ ref_w.T, _sum_bound(k) * (rows.abs() @ ref_w.abs().T)
    g, u, eg, eu = both[:, :f], both[:, f:], size[:, :f], size[:, f:]
    slope = 1.2
    if gate == "capped":
        g, u, slope = g.clamp(max=2.0), u.clamp(-2.0, 2.0) + 1.0, 1.7
        act = g * torch.sigmoid(1.7 * g)
    else:
        act = {"silu": lambda: g * torch.sigmoid(g), "relu": lambda: g.clamp(min=0), "sigmoid": lambda: torch.sigmoid(g), "gelu_tanh": lambda: _activated(g, "gelu_tanh")[0]}[gate]()
    want = act * u
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8 + 2.0 ** -15)):
        out = torch.full((m, f + 1), float("nan"), dtype=dtype, device=dev)
        ops.gated4(a, w, out[:, :f], m, gate=gate, a_scale=scale, alpha=1.7, limit=2.0)
        assert ops.device_status() == 0
        # As in test_gated: the product's rule on both sums' errors, and the gate's own 32-bit arithmetic.
        bound = slope * eg * (u.abs() + eu) + act.abs() * eu + 2.0 ** -19 * (want.abs() + act.abs()) + 1e-30
        assert ((out[:, :f].double() - want).abs() <= bound + rounding * (want.abs() + bound)).all()
        assert out[:, f:].isnan().all()


@pytest.mark.parametrize("m", [1, 3, 12, 40, 150])
@pytest.mark.parametrize("eight", [False, True])
def test_rows_that_lie_anyhow(dev, m, eight):
    """Strides and starts that are no multiple of 16 bytes, and rows behind the last that are not read."""
    from liyab_b200 import ops
    n, k = 136, 520
    q, s, r = _parts(n, k, 64, dev)
    w = ops.lay_out_weights4(q, s, r, 64)
    for pad, first in ((0, 0), (8, 8), (16, 0), (3, 1), (1, 0), (4, 4)):
        wide = _rand((m, k + pad), 11, dev)
        if eight:
            rows, scale = _rows8(wide)
        else:
            rows, scale = wide.to(torch.bfloat16), None
        a = rows[:, first:first + k] if first + k <= k + pad else rows[:, :k]
        a64 = a.double() if scale is None else a.double() * scale.double()[:, None]
        ref_w = _matrix(q, s, r, 64)
        out = torch.full((m + 2, n + 1), 5.0, device=dev)
        ops.linear4(a, w, None, out[:, :n], m, a_scale=scale)
        assert ((out[:m, :n].double() - a64 @ ref_w.T).abs() <= _sum_bound(k) * (a64.abs() @ ref_w.abs().T)).all()
        assert (out[m:] == 5.0).all() and (out[:, n:] == 5.0).all()


@pytest.mark.parametrize("m", [1, 9, 33, 140])
def test_special_values_stay_in_their_row(dev, m):
    """An infinity or a NaN in a row of activations makes that row's outputs what 64 bits make of them, and no other row's; so does a NaN factor of a feature."""
    from liyab_b200 import ops
    n, k = 200, 384
    q, s, r = _parts(n, k, 128, dev)
    r[5] = float("nan")
    w = ops.lay_out_weights4(q, s, r, 128)
    a = _rand((m, k), 12, dev, torch.bfloat16)
    a[0, 17], a[m // 2, 100], a[m - 1, 380] = float("inf"), float("-inf"), float("nan")
    out = torch.empty((m, n), device=dev)
    ops.linear4(a, w, None, out, m)
    want = a.double() @ _matrix(q, s, r, 128).T
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[out.isinf()], want.float()[out.isinf()]) and torch.equal(out.isinf(), want.isinf())
    a8, scale = _rows8(_rand((m, k), 13, dev))
    scale[0] = float("nan")
    ops.linear4(a8, w, None, out, m, a_scale=scale)
    assert out[0].isnan().all() and out[1:, :5].isfinite().all() and out[:, 5].isnan().all()


# Sums of gates: the ends of the range, values whose exponentials overflow, and ordinary ones.  (Not between -745 and -88: there the sigmoid is a number in 64 bits and 0 in 32.)
GATE_SUMS = [float("inf"), -float("inf"), float("nan"), 0.0, 3e38, -3e38, 1e30, -1e30, 1e20, -1e20, 1e4, -1e4, 87.0, -87.0, 3.0, -3.0, 1e-30, -1e-30]
OTHER_SUMS = [1.5, -2.0, 0.0, 3e38, float("inf"), -float("inf"), float("nan")]


def _special_sums(m, k, sums, eight, paired, dev):
    """(a, a_scale, weights, the sums in 64 bits [m, len(sums)]): a feature's only product is +-1, and its factor the sum."""
    from liyab_b200 import ops
    n = len(sums)
    q, s, r = torch.zeros((n, k), dtype=torch.int8), torch.ones((n, -(-k // 64))).to(F8), torch.tensor(sums)
    q[:, 5] = 1
    sign = torch.where(torch.arange(m) % 3 == 2, -1.0, 1.0)
    a = torch.zeros((m, k))
    a[:, 5] = sign
    a = a.to(F8 if eight else torch.bfloat16).to(dev)
    return a, torch.ones(m, device=dev) if eight else None, ops.lay_out_weights4(q.to(dev), s.to(dev), r.to(dev), 64, paired), sign.to(dev).double()[:, None] * r.to(dev).double()


def _gate64(g, kind, alpha, limit):
    if kind == "gelu_tanh":
        return g * torch.sigmoid(1.5957691216057308 * (g + 0.044715 * g ** 3))
    return {"sigmoid": lambda: torch.sigmoid(g), "silu": lambda: g * torch.sigmoid(g), "relu": lambda: g.clamp(min=0), "capped": lambda: g.clamp(max=limit) * torch.sigmoid(alpha * g.clamp(max=limit))}[kind]()


def _same_specials(out, want, bound):
    """NaN and infinities (numbers past float32's range are) where 64 bits have them, the others within the bound."""
    expected = want.float().to(out.dtype)
    finite = expected.isfinite()
    return torch.equal(out.isnan(), expected.isnan()) and torch.equal(out[expected.isinf()], expected[expected.isinf()]) and bool(((out.double() - want).abs() <= bound)[finite].all())


@pytest.mark.parametrize("m,repeats", [(1, 1), (8, 1), (9, 1), (33, 1), (140, 1), (600, 30)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("gate", ["sigmoid", "silu", "gelu_tanh", "relu", "capped"])
def test_gates_of_special_sums(dev, m, repeats, eight, gate):
    """On both sides of eight tokens, in small tiles, whole ones and walked ones, in both result types: what the definition makes of them in 64 bits."""
    from liyab_b200 import ops
    gates = [g for g in GATE_SUMS for _ in OTHER_SUMS] * repeats
    others = [u for _ in GATE_SUMS for u in OTHER_SUMS] * repeats
    a, scale, w, sums = _special_sums(m, 192, gates + others, eight, True, dev)
    assert ops.linear4_plan(w, m)[0] == ("few" if m <= 8 else "walk" if m == 600 else "tiles")
    f = len(gates)
    g, u = sums[:, :f], sums[:, f:]
    act = _gate64(g, gate, 1.7, 2.0)
    if gate == "capped":
        u = u.clamp(-2.0, 2.0) + 1.0
    # The gate in 32 bits: the fast exponential's 2^-15 at arguments to 90, nothing below 2^-126 (times a gate of up to 88), and where 1 + tanh cancels 2^-22 of the argument.
    off = 2.0 ** -15 * act.abs() + 1e-35 + (2.0 ** -22 * g.abs().clamp(max=20.0) if gate == "gelu_tanh" else 0.0)
    for dtype, rounding in ((torch.float32, 2.0 ** -22), (torch.bfloat16, 2.0 ** -8)):
        out = torch.zeros((m, f), dtype=dtype, device=dev)
        ops.gated4(a, w, out, m, gate=gate, a_scale=scale, alpha=1.7, limit=2.0)
        assert _same_specials(out, act * u, off * u.abs() + rounding * (act * u).abs() + 1e-37), dtype
    assert ops.device_status() == 0


@pytest.mark.parametrize("m,repeats", [(1, 1), (8, 1), (9, 1), (33, 1), (140, 1), (600, 350)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("activation", ["none", "gelu_tanh", "gelu_erf", "xielu", "relu2"])
def test_activations_of_special_sums(dev, m, repeats, eight, activation):
    """As the gates': with xIELU's numbers behind a bias of zeros, the others with and without a bias."""
    from liyab_b200 import ops
    a, scale, w, z = _special_sums(m, 192, GATE_SUMS * repeats, eight, False, dev)
    assert ops.linear4_plan(w, m)[0] == ("few" if m <= 8 else "walk" if m == 600 else "tiles")
    n = len(GATE_SUMS) * repeats
    bias = torch.zeros(n + 2, device=dev)
    bias[n:] = torch.tensor([0.8, 0.4], device=dev)
    want = _gate64(z, "gelu_tanh", 0.0, 0.0) if activation == "gelu_tanh" else z * torch.special.ndtr(z) if activation == "gelu_erf" else _activated(z, activation)[0]
    # As for the gates; where 1 + tanh or 1 + erf cancels, and in xIELU's exponential less 1, 2^-22 of the argument.
    off = 2.0 ** -15 * want.abs() + 1e-35 + 2.0 ** -22 * z.abs().clamp(max=20.0)
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        for b in (bias,) if activation == "xielu" else (bias, None):
            out = torch.zeros((m, n), dtype=dtype, device=dev)
            ops.linear4(a, w, b, out, m, activation=activation, a_scale=scale)
            assert _same_specials(out, want, off + rounding * want.abs()), (dtype, b is None)
    assert ops.device_status() == 0


@pytest.mark.parametrize("m,repeats", [(1, 1), (9, 1), (140, 1), (600, 70)])
def test_xielu_of_small_sums(dev, m, repeats):
    """exp(v) - 1 - v of small v, in both result types: to the results' own rounding, not to that of 1."""
    from liyab_b200 import ops
    sums = [s * d * 10.0 ** -p for p in range(30) for s in (1.0, -1.0) for d in (1.0, 2.7)] * repeats
    a, scale, w, z = _special_sums(m, 192, sums, False, False, dev)
    assert ops.linear4_plan(w, m)[0] == ("few" if m <= 8 else "walk" if m == 600 else "tiles")
    bias = torch.zeros(len(sums) + 2, device=dev)
    bias[-2:] = torch.tensor([0.8, 0.4], device=dev)
    want, size = _activated(z, "xielu")[0], z.abs()
    for dtype, rounding in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = torch.zeros((m, len(sums)), dtype=dtype, device=dev)
        ops.linear4(a, w, bias, out, m, activation="xielu")
        # Terms no larger than twice the argument, each with the fast exponential's 2^-15 (argument below 3) of its own size at the worst where it is not cancelled.
        assert ((out.double() - want).abs() <= rounding * want.abs() + 2.0 ** -14 * size.clamp(max=1.0) + 2.0 ** -15 * want.abs()).all(), dtype
    assert ops.device_status() == 0


@pytest.mark.parametrize("m,n", [(1, 264), (8, 264), (9, 264), (33, 264), (100, 264), (600, 7002)])
def test_small_scales(dev, m, n):
    """Rows that the norm scales by its smallest factors: the row's factor and the weights' meet the sum one after the other (their product is below the smallest normal number)."""
    from liyab_b200 import ops
    k = 256
    q, s, r = _parts(n, k, 64, dev, seed=m)
    a8, _ = _rows8(_rand((m, k), 70, dev))
    scale = torch.full((m,), 1.5e-38, device=dev)
    rows = a8.double() * scale.double()[:, None]
    ref_w = _matrix(q, s, r, 64)
    want, bound = rows @ ref_w.T, _sum_bound(k) * (rows.abs() @ ref_w.abs().T) + 2.0 ** -149
    out = torch.empty((m, n), device=dev)
    ops.linear4(a8, ops.lay_out_weights4(q, s, r, 64), None, out, m, a_scale=scale)
    assert ((out.double() - want).abs() <= bound).all()
    # The gated product: the other half's weights are as large as the row's scale is small.
    r[n // 2:] *= 1e38
    ref_w = _matrix(q, s, r, 64)
    both, size = rows @ ref_w.T, _sum_bound(k) * (rows.abs() @ ref_w.abs().T) + 2.0 ** -149
    g, u, eg, eu = both[:, :n // 2].clamp(min=0), both[:, n // 2:], size[:, :n // 2], size[:, n // 2:]
    half = torch.empty((m, n // 2), device=dev)
    ops.gated4(a8, ops.lay_out_weights4(q, s, r, 64, paired=True), half, m, gate="relu", a_scale=scale)
    assert ((half.double() - g * u).abs() <= eg * (u.abs() + eu) + g * eu + 2.0 ** -23 * (g * u).abs() + 2.0 ** -149).all()
    assert ops.device_status() == 0


def test_no_rows(dev):
    from liyab_b200 import ops
    q, s, r = _parts(32, 64, 32, dev)
    out = torch.full((4, 32), 3.0, device=dev)
    ops.linear4(torch.zeros((4, 64), dtype=torch.bfloat16, device=dev), ops.lay_out_weights4(q, s, r, 32), None, out, 0)
    ops.gated4(torch.zeros((4, 64), dtype=torch.bfloat16, device=dev), ops.lay_out_weights4(q, s, r, 32, paired=True), out[:, :16], 0)
    assert (out == 3.0).all()


# ---- the norm ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("width", [1, 7, 64, 130, 1600, 4096, 5461, 8192, 16384, 57344])
@pytest.mark.parametrize("x_type,delta_type", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_norm(dev, rows, width, x_type, delta_type):
    from liyab_b200 import ops
    x, delta = _rand((rows, width), 20, dev, x_type, 3.0), _rand((rows, width), 21, dev, delta_type)
    gain = 1.0 + 0.3 * _rand((width,), 22, dev)
    t = x.double() + delta.double()
    h = t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * (0.5 + gain.double())
    # t: one rounding in 32 bits (and one to x's type, 2^-8 for bfloat16's eight bits); the mean: errors of a sum of squares, all of one sign, in parts of 32 at least and 64 levels at most: 2^-17 covers it.
    total_bound = (2.0 ** -24 + (2.0 ** -8 if x_type is torch.bfloat16 else 0.0)) * t.abs()
    h_bound = 2.0 ** -17 * h.abs() + 2.0 ** -22 * (0.5 + gain.double()).abs()
    half = torch.empty((rows, width), dtype=torch.bfloat16, device=dev)
    total = torch.empty_like(x)
    ops.rms_add(x, delta, gain, 1e-5, half, total=total, gain_offset=0.5)
    assert ((total.double() - t).abs() <= total_bound).all()
    assert ((half.double() - h).abs() <= 2.0 ** -8 * h.abs() + h_bound).all()
    out, scale = torch.empty((rows, width), dtype=F8, device=dev), torch.empty(rows, device=dev)
    moved = x.clone()
    ops.rms_add(moved, delta, gain, 1e-5, out, scale=scale, gain_offset=0.5)                      # in place
    assert torch.equal(moved, total)
    top = h.abs().amax(1)
    assert ((scale.double() - top / 448.0).abs() <= 2.0 ** -16 * top / 448.0 + 2.0 ** -30).all()
    # e4m3: half a step is 2^-4 of a normal number, 2^-10 below 2^-6.
    got = out.double() * scale.double()[:, None]
    assert ((got - h).abs() <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale.double()[:, None]) + 2 * h_bound).all()
    assert (out.float().abs().amax(1) == 448.0).all()


def test_norm_alone_and_strided(dev):
    """Without a delta nothing is written but the result; without a gain it is one; rows that lie apart, at odd places."""
    from liyab_b200 import ops
    for width, pad, first in ((96, 7, 3), (1600, 8, 0), (1600, 1, 1), (4096, 4, 4)):
        wide = _rand((5, width + pad), 23, dev)
        x = wide[:, first:first + width]
        keep = wide.clone()
        out = torch.full((5, width + pad), float("nan"), dtype=torch.bfloat16, device=dev)
        ops.rms_add(x, None, None, 1e-6, out[:, first:first + width])
        h = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
        assert ((out[:, first:first + width].double() - h).abs() <= (2.0 ** -8 + 2.0 ** -17) * h.abs()).all()
        assert torch.equal(wide, keep) and int(out.isnan().sum()) == 5 * pad
        eight, scale = torch.zeros((5, width + pad), dtype=F8, device=dev), torch.empty(5, device=dev)
        delta = _rand((5, width + 5), 24, dev)[:, 2:2 + width]
        ops.rms_add(x, delta, None, 1e-6, eight[:, first:first + width], scale=scale)
        t = keep[:, first:first + width].double() + delta.double()
        assert ((x.double() - t).abs() <= 2.0 ** -23 * t.abs()).all()
        h = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
        got = eight[:, first:first + width].double() * scale.double()[:, None]
        assert ((got - h).abs() <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale.double()[:, None]) + 2.0 ** -16 * h.abs()).all()


@pytest.mark.parametrize("rows,width,place", [(1, 2, 2), (5, 98, 2), (3, 1602, 6), (40, 8190, 2), (2, 40002, 0), (300, 16386, 0)])
@pytest.mark.parametrize("x_type,delta_type", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_norm_of_rows_in_twos(dev, rows, width, place, x_type, delta_type):
    """Rows whose places are even but no multiple of 16 bytes: they go through shared memory two values at a time."""
    from liyab_b200 import ops
    x, delta = _rand((rows, width + 8), 26, dev, x_type)[:, place:place + width], _rand((rows, width + 2), 27, dev, delta_type)[:, :width]
    out, scale, total = torch.empty((rows, width), dtype=F8, device=dev), torch.empty(rows, device=dev), torch.empty((rows, width), dtype=x_type, device=dev)
    ops.rms_add(x, delta, None, 1e-5, out, scale=scale, total=total)
    t = x.double() + delta.double()
    h = t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt()
    # As in test_norm: one rounding of the sum and one to x's type, a mean's error of 2^-17, half a step of e4m3.
    assert ((total.double() - t).abs() <= (2.0 ** -24 + (2.0 ** -8 if x_type is torch.bfloat16 else 0.0)) * t.abs()).all()
    got = out.double() * scale.double()[:, None]
    assert ((got - h).abs() <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale.double()[:, None]) + 2 * (2.0 ** -17 * h.abs() + 2.0 ** -22)).all()


def test_norm_of_special_rows(dev):
    from liyab_b200 import ops
    for width in (40, 1600, 9000):
        x = _rand((7, width), 25, dev)
        x[1], x[2, 3], x[3, width - 1], x[4] = 0.0, float("inf"), float("nan"), 1e-38
        x[5] = 1e-3 * x[5]
        out, scale, half = torch.ones((7, width), dtype=F8, device=dev), torch.empty(7, device=dev), torch.empty((7, width), dtype=torch.bfloat16, device=dev)
        ops.rms_add(x, None, None, 0.1, out, scale=scale)
        assert (out[1:5].float() == 0).all() and (scale[[1, 4]] == 0).all() and not scale[2:4].isfinite().any() and (scale[[0, 5, 6]] > 0).all()
        ops.rms_add(x, None, None, 0.1, half)
        assert (half[1] == 0).all() and half[3].isnan().all() and half[[0, 1, 4, 5, 6]].isfinite().all()


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("width", [40, 41, 42, 512, 1600, 9000, 9001])
@pytest.mark.parametrize("x_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ends", ["large", "small"])
def test_norm_at_the_ends_of_the_range(dev, rows, width, x_type, ends):
    """Rows whose largest |h| lies above 2^126 (gains of 1.5e38), and rows so small that 448 / |t| is no float32 number, zeros among their values."""
    from liyab_b200 import ops
    g = torch.Generator().manual_seed(width)
    x = (0.5 + 0.5 * torch.rand((rows, width), generator=g)) * (torch.randint(0, 2, (rows, width), generator=g) * 2.0 - 1.0)
    gain = None
    if ends == "large":
        gain = torch.full((width,), 1.5e38, device=dev)
    else:
        x = torch.where(torch.rand((rows, width), generator=g) < 0.2, torch.zeros(()), x * 1e-37)
        x[:, 0] = 1e-37
    x = x.to(x_type).to(dev)
    h = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * (1.0 if gain is None else gain.double())
    top = h.abs().amax(1)
    out, scale, half = torch.empty((rows, width), dtype=F8, device=dev), torch.empty(rows, device=dev), torch.empty((rows, width), dtype=torch.bfloat16, device=dev)
    ops.rms_add(x, None, gain, 1e-6, out, scale=scale)
    ops.rms_add(x, None, gain, 1e-6, half)
    # The bounds of test_norm.
    assert ((scale.double() - top / 448.0).abs() <= 2.0 ** -16 * top / 448.0).all()
    got = out.double() * scale.double()[:, None]
    assert ((got - h).abs() <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale.double()[:, None]) + 2.0 ** -16 * h.abs()).all()
    assert ((half.double() - h).abs() <= (2.0 ** -8 + 2.0 ** -17) * h.abs()).all()


@pytest.mark.parametrize("rows", [295, 296, 297, 1001])
@pytest.mark.parametrize("width", [8, 40, 256, 264, 512, 520, 2048, 2056, 4096, 4104])
@pytest.mark.parametrize("x_type,delta_type", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_norm_of_many_rows(dev, rows, width, x_type, delta_type):
    """Enough rows for a warp a row and for more values a thread, on both sides of where those begin; the sum in place and apart, both outputs; zeros, an infinity and a NaN."""
    from liyab_b200 import ops
    x, delta = _rand((rows, width), 28, dev, x_type, 3.0), _rand((rows, width), 29, dev, delta_type)
    gain = 1.0 + 0.3 * _rand((width,), 30, dev)
    x[7], delta[7] = 0.0, 0.0
    x[rows - 2, width - 1], delta[294, 0] = float("inf"), float("nan")
    odd = torch.zeros(rows, dtype=torch.bool, device=dev)
    odd[rows - 2] = odd[294] = True
    t = x.double() + delta.double()
    h = t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * (0.5 + gain.double())
    # The bounds of test_norm.
    total_bound = (2.0 ** -24 + (2.0 ** -8 if x_type is torch.bfloat16 else 0.0)) * t.abs()
    h_bound = 2.0 ** -17 * h.abs() + 2.0 ** -22 * (0.5 + gain.double()).abs()
    half, total = torch.empty((rows, width), dtype=torch.bfloat16, device=dev), torch.empty_like(x)
    ops.rms_add(x, delta, gain, 1e-5, half, total=total, gain_offset=0.5)
    assert torch.equal(total.isnan(), t.isnan()) and torch.equal(total.isinf(), t.isinf())
    assert ((total.double() - t).abs() <= total_bound)[t.isfinite()].all()
    assert ((half.double() - h).abs() <= 2.0 ** -8 * h.abs() + h_bound)[~odd].all()
    out, scale = torch.ones((rows, width), dtype=F8, device=dev), torch.ones(rows, device=dev)
    moved = x.clone()
    ops.rms_add(moved, delta, gain, 1e-5, out, scale=scale, gain_offset=0.5)                      # in place
    assert torch.equal(moved.nan_to_num(7.0), total.nan_to_num(7.0))
    assert not scale[odd].isfinite().any() and (out[odd].float() == 0).all() and scale[7] == 0 and (out[7].float() == 0).all()
    top, fine = h.abs().amax(1), ~odd
    assert ((scale.double() - top / 448.0).abs() <= 2.0 ** -16 * top / 448.0 + 2.0 ** -30)[fine].all()
    got = out.double() * scale.double()[:, None]
    assert ((got - h).abs() <= torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale.double()[:, None]) + 2 * h_bound)[fine].all()
    fine[7] = False
    assert (out.float().abs().amax(1) == 448.0)[fine].all()


def test_single_rows_and_columns_of_any_stride(dev):
    """A dimension of one has no stride: a column turned over, a broadcast row and columns of one value are rows like any other."""
    from liyab_b200 import ops
    from liyab_b200.status import LiyabError
    n, k = 72, 640
    q, s, r = _parts(n, k, 64, dev)
    ref_w, gate_w = _matrix(q, s, r, 64), _matrix(q, s, r * 0.05, 64)
    w, pairs = ops.lay_out_weights4(q, s, r, 64), ops.lay_out_weights4(q, s, r * 0.05, 64, paired=True)
    a = _rand((k, 1), 60, dev, torch.bfloat16)
    want = a.t().double() @ ref_w.T
    bound = _sum_bound(k) * (a.t().double().abs() @ ref_w.abs().T)
    for row in (a.t(), a[:, 0].expand(1, k)):
        out, res = torch.empty((n, 1), device=dev), _rand((n, 1), 61, dev)
        ops.linear4(row, w, None, out.t(), 1, residual=res.t())
        assert ((out.t().double() - want - res.t().double()).abs() <= bound + 2.0 ** -23 * res.t().abs()).all()
        half = torch.empty((n // 2, 1), device=dev)
        ops.gated4(row, pairs, half.t(), 1, gate="relu")
        both = row.double() @ gate_w.T
        size = _sum_bound(k) * (row.double().abs() @ gate_w.abs().T)
        g, u, eg, eu = both[:, :n // 2].clamp(min=0), both[:, n // 2:], size[:, :n // 2], size[:, n // 2:]
        assert ((half.t().double() - g * u).abs() <= eg * (u.abs() + eu) + g * eu + 2.0 ** -23 * (g * u).abs()).all()
        normed, scale = torch.empty((k, 1), dtype=F8, device=dev), torch.empty(1, device=dev)
        ops.rms_add(row, row.t().t(), None, 1e-6, normed.t(), scale=scale, total=torch.empty((k, 1), dtype=torch.bfloat16, device=dev).t())
        t = 2.0 * row.double()
        h = t / (t.square().mean() + 1e-6).sqrt()
        assert ((normed.t().double() * scale.double() - h).abs() <= 2.0 ** -4 * h.abs() + 2.0 ** -10 * scale.double() + 2.0 ** -16 * h.abs()).all()
    # One column: a product over k = 1, one feature, and norms of one value.
    one, by = _rand((1, 30), 62, dev, torch.bfloat16), ops.lay_out_weights4(q[:, :1], s[:, :1].clone().view(1, n).t(), r, 64)
    out = torch.empty((30, n), device=dev)
    ops.linear4(one.t(), by, None, out, 30)
    want = one.t().double() @ _matrix(q[:, :1], s[:, :1], r, 64).T
    assert ((out.double() - want).abs() <= 2.0 ** -20 * want.abs()).all()
    single = ops.lay_out_weights4(q[:1, :], s[:1], r[:1], 64)
    rows, out = _rand((30, k), 63, dev, torch.bfloat16), torch.empty((1, 30), device=dev)
    ops.linear4(rows, single, None, out.t(), 30)
    assert ((out.t().double() - rows.double() @ ref_w[:1].T).abs() <= _sum_bound(k) * (rows.double().abs() @ ref_w[:1].abs().T)).all()
    assert torch.equal(ops.weights4_values(ops.quantise_weights4(a.t())), ops.weights4_values(ops.quantise_weights4(a.t().clone(memory_format=torch.contiguous_format).view(1, k))))
    out = torch.empty((1, 30), dtype=torch.bfloat16, device=dev)
    ops.rms_add(one.t(), None, None, 1e-6, out.t())
    want = one.double() / (one.double().square() + 1e-6).sqrt()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17 * want.abs()).all()
    # Other shapes are refused for one value a row too.
    x = torch.zeros((1, 1), device=dev)
    for bad in (lambda: ops.rms_add(x, None, None, 1e-6, out), lambda: ops.rms_add(x, out, None, 1e-6, out[:, :1]), lambda: ops.rms_add(x, x, None, 1e-6, out[:, :1], total=x[0]),
                lambda: ops.rms_add(x.expand(3, 1), None, None, 1e-6, torch.empty((3, 1), dtype=torch.bfloat16, device=dev))):
        with pytest.raises(LiyabError):
            bad()


# ---- together, and refusals --------------------------------------------------------------------------------

def test_a_block_on_its_own_stream_and_in_a_graph(dev):
    """Norm, gated half and second half as a feed-forward block: on a stream of its own, then captured and replayed on new rows."""
    from liyab_b200 import ops
    width, f = 640, 1712
    up = ops.quantise_weights4(_rand((2 * f, width), 30, dev, scale=0.04), 64, paired=True)
    down = ops.quantise_weights4(_rand((width, f), 31, dev, torch.bfloat16, 0.03), 128)
    wu, wd = ops.weights4_values(up).double(), ops.weights4_values(down).double()
    gain = 1.0 + 0.1 * _rand((width,), 32, dev)
    for m in (1, 6, 20, 150):
        x, delta = _rand((m, width), 33, dev), _rand((m, width), 34, dev)
        out8, scale = torch.empty((m, width), dtype=F8, device=dev), torch.empty(m, device=dev)
        mid = torch.empty((m, f), dtype=torch.bfloat16, device=dev)

        def block():
            ops.rms_add(x, delta, gain, 1e-6, out8, scale=scale)
            ops.gated4(out8, up, mid, m, a_scale=scale)
            ops.linear4(mid, down, None, x, m, residual=x)

        def check(x0):
            t = x0.double() + delta.double()
            h = out8.double() * scale.double()[:, None]
            z = h @ wu.T
            inner = z[:, :f] * torch.sigmoid(z[:, :f]) * z[:, f:]
            assert ((mid.double() - inner).abs() <= 2.0 ** -8 * inner.abs() + 1e-4).all()
            y = t + mid.double() @ wd.T
            assert ((x.double() - y).abs() <= _sum_bound(f) * (mid.double().abs() @ wd.abs().T + t.abs())).all()

        start = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block()
        torch.cuda.current_stream().wait_stream(side)
        check(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            block()
        x.copy_(_rand((m, width), 35, dev))
        start = x.clone()
        graph.replay()
        check(start)
        assert ops.device_status() == 0


def test_refusals(dev):
    from liyab_b200 import ops
    from liyab_b200.status import LiyabError
    q, s, r = _parts(32, 64, 32, dev)
    w, pw = ops.lay_out_weights4(q, s, r, 32), ops.lay_out_weights4(q, s, r, 32, paired=True)
    a, out = torch.zeros((4, 64), dtype=torch.bfloat16, device=dev), torch.zeros((4, 32), device=dev)
    a8, scale = torch.zeros((4, 64), dtype=F8, device=dev), torch.ones(4, device=dev)
    x = torch.zeros((4, 64), device=dev)
    for bad in (
            lambda: ops.lay_out_weights4(q, s, r, 16), lambda: ops.lay_out_weights4(q, s[:, :1], r, 32), lambda: ops.lay_out_weights4(q.float(), s, r, 32),
            lambda: ops.lay_out_weights4(q[:31], s[:31], r[:31], 32, paired=True), lambda: ops.lay_out_weights4(q.cpu(), s, r, 32), lambda: ops.lay_out_weights4(q, s, r.double(), 32),
            lambda: ops.quantise_weights4(x.half()), lambda: ops.quantise_weights4(x.t()), lambda: ops.quantise_weights4(x, 48), lambda: ops.quantise_weights4(x[:0]),
            lambda: ops.linear4(a, pw, None, out, 4), lambda: ops.gated4(a, w, out[:, :16], 4), lambda: ops.linear4(a, w, None, out, 5), lambda: ops.linear4(a, w, None, out, -1),
            lambda: ops.linear4(a.float(), w, None, out, 4), lambda: ops.linear4(a8, w, None, out, 4), lambda: ops.linear4(a, w, None, out, 4, a_scale=scale),
            lambda: ops.linear4(a8, w, None, out, 4, a_scale=scale[:3]), lambda: ops.linear4(a[:, :60], w, None, out, 4), lambda: ops.linear4(a, w, None, out.half(), 4),
            lambda: ops.linear4(a, w, None, out[:, :31], 4), lambda: ops.linear4(a, w, out[0, :31], out, 4), lambda: ops.linear4(a, w, None, out, 4, activation="xielu"),
            lambda: ops.linear4(a, w, None, out, 4, residual=out[:3]), lambda: ops.linear4(a.t().contiguous().t(), w, None, out, 4), lambda: ops.linear4(a.cpu(), w, None, out, 4),
            lambda: ops.gated4(a, pw, out, 4), lambda: ops.gated4(a, pw, out[:, :16], 4, gate="relu2"), lambda: ops.gated4(a, pw, out[:, :16], 4, gate="tanh"),
            lambda: ops.rms_add(x, None, None, 1e-5, a8), lambda: ops.rms_add(x, None, None, 1e-5, a, scale=scale), lambda: ops.rms_add(x, x[:3], None, 1e-5, a),
            lambda: ops.rms_add(x, None, None, 1e-5, x), lambda: ops.rms_add(x, x, None, 1e-5, a, total=a), lambda: ops.rms_add(x, None, scale, 1e-5, a),
            lambda: ops.rms_add(x, None, None, 1e-5, a8, scale=scale[:2]), lambda: ops.rms_add(x.half(), None, None, 1e-5, a), lambda: ops.rms_add(x.cpu(), None, None, 1e-5, a.cpu())):
        with pytest.raises(LiyabError):
            bad()
    with pytest.raises(KeyError):
        ops.linear4(a, w, None, out, 4, activation="tanh")


def test_memory_of_another_device_is_refused(dev, monkeypatch):
    """Kernels run on the current device: tensors of another one are refused before a launch (the test says that theirs is another)."""
    from liyab_b200 import ops
    from liyab_b200.status import LiyabError
    q, s, r = _parts(32, 64, 32, dev)
    w, pw = ops.lay_out_weights4(q, s, r, 32), ops.lay_out_weights4(q, s, r, 32, paired=True)
    a, out, x = torch.zeros((4, 64), dtype=torch.bfloat16, device=dev), torch.zeros((4, 32), device=dev), torch.zeros((4, 64), device=dev)
    set_up = (lambda: ops.weights4_values(w), lambda: ops.quantise_weights4(x, 32), lambda: ops.lay_out_weights4(q, s, r, 32))
    products = (lambda: ops.linear4(a, w, None, out, 4), lambda: ops.gated4(a, pw, out[:, :16], 4))
    for call in set_up + products:
        call()
    monkeypatch.setattr(ops, "_current_device", lambda: dev.index + 1)
    for call in set_up:
        with pytest.raises(LiyabError, match="current device"):
            call()
    w.args.device = pw.args.device = dev.index + 2
    for call in products:
        with pytest.raises(LiyabError, match="current device"):
            call()
    norm = lambda device: ops.lib().lb_rms_add_rows(ops._rms_add_args(x.data_ptr(), 0, 0, 0, a.data_ptr(), 0, ops.stream_ptr(), 64, 0, 0, 64, ops.F32, 0, ops.BF16, 4, 64, device, 0.0, 1e-6))
    assert norm(dev.index + 1) == norm(0) == 0 and norm(dev.index + 2) == 1
    monkeypatch.undo()
    with pytest.raises(LiyabError):
        ops.lay_out_weights4(q, s.cpu(), r, 32)
    with pytest.raises(LiyabError):
        ops.lay_out_weights4(q, s, r.cpu(), 32)
