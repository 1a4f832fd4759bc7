"""Products with 4-bit weights, and the norm that feeds them, as programs call them.

Three operators:

* ``rms_add``: a sublayer's output joins the residual stream, and the RMS norm of the sum is left in 8 bits (e4m3) with one scale a
  row, or in bfloat16.
* ``linear4``: out = act(a w^T + bias) + residual, where w[n, k] = q[n, k] s[n, k / group] r[n]: q in 4 bits (-8 .. 7), s in e4m3,
  r in 32 bits.  The activations are bfloat16 or e4m3 with a scale a row.
* ``gated4``: out = gate(a w_gate^T) * (a w_up^T) over the same kind of weights.

A state holds what a program holds: activations, the weights as they are read (laid out once), biases and output buffers.
"""
from __future__ import annotations

import math

import torch

own = False


# ---- the cases ---------------------------------------------------------------------------------------------

def _rms(rows, width, x="f32", delta="f32", out="e4m3"):
    return dict(op="rms_add", rows=rows, width=width, x=x, delta=delta, out=out)


def _linear(m, n, k, group, a="bf16", out="bf16", bias=False, act="none", residual=False):
    return dict(op="linear4", m=m, n=n, k=k, group=group, a=a, out=out, bias=bias, act=act, residual=residual)


def _gated(m, f, k, group, a="bf16", gate="silu"):
    return dict(op="gated4", m=m, f=f, k=k, group=group, a=a, gate=gate)


def listed():
    named = {
        # One user's next token between two sublayers of the largest model of the benchmark: nothing but latency.
        "norm_one": _rms(1, 1600, delta="bf16"),
        # A busy server's decode step.
        "norm_64": _rms(64, 4096),
        # A step of long prompts with a bfloat16 residual stream.
        "norm_prefill": _rms(4096, 8192, x="bf16", delta="bf16"),
        # One user's next token: the attention output's projection, summed into the stream.
        "proj_1": _linear(1, 1600, 1600, 64, out="f32", residual=True),
        # A small server's logits: odd number of features.
        "head_4": _linear(4, 50257, 1600, 128, out="f32"),
        # A small server's step: the long reduction of a wide feed-forward's second half.
        "down_8": _linear(8, 4096, 16384, 128, out="f32", residual=True),
        # A server's fused query, key and value projection with 8-bit activations and small groups.
        "qkv_16": _linear(16, 4800, 1600, 32, a="e4m3", bias=True),
        # One short question beside running requests: tokens that fill no tile.
        "mid_100": _linear(100, 6400, 1600, 64, bias=True, act="gelu_tanh"),
        # Two full contexts of a large model: the tensor cores' rate.
        "prefill_2048": _linear(2048, 8192, 8192, 128),
        # One user's next token through a wide feed-forward's first half, from 8-bit activations.
        "gated_1": _gated(1, 10240, 4096, 128, a="e4m3"),
        # A server's step with an odd inner size.
        "gated_24": _gated(24, 5461, 2048, 64, gate="gelu_tanh"),
        # Prompts of several users, 8-bit activations.
        "gated_1024": _gated(1024, 12288, 4096, 128, a="e4m3"),
    }
    return [dict(c, name=n) for n, c in named.items()]


_MOST_FLOPS, _MOST_BYTES = 2.7e11, 2.3e8      # of the largest listed cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _length(rng, lo, hi):
    """A reduction's length: mostly a multiple of 32, as matrices of models are, now and then any number."""
    k = _log_int(rng, lo, hi)
    return k if rng.random() < 0.15 else max(lo, k // 32 * 32)


def draw(rng):
    while True:
        op = rng.choice(["rms_add", "linear4", "linear4", "gated4"])
        if op == "rms_add":
            c = _rms(_log_int(rng, 1, 8192), _log_int(rng, 128, 16384), rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), rng.choice(["e4m3", "e4m3", "bf16"]))
        else:
            m, group, a = _log_int(rng, 1, 2048), rng.choice([32, 64, 128]), rng.choice(["bf16", "bf16", "e4m3"])
            if op == "linear4":
                residual = rng.random() < 0.4
                c = _linear(m, _log_int(rng, 64, 50257), _length(rng, 64, 16384), group, a, "f32" if residual else rng.choice(["bf16", "f32"]), rng.random() < 0.4,
                            rng.choice(["none", "none", "gelu_tanh", "gelu_erf", "relu2"]), residual)
            else:
                c = _gated(m, _log_int(rng, 64, 16384), _length(rng, 64, 8192), group, a, rng.choice(["silu", "gelu_tanh", "sigmoid", "relu"]))
        w = work(c)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return c


_BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}
_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def work(case):
    c = case
    if c["op"] == "rms_add":
        n = c["rows"] * c["width"]
        return {"bytes": n * (2 * _BYTES[c["x"]] + _BYTES[c["delta"]] + _BYTES[c["out"]]) + 4 * c["width"] + (4 * c["rows"] if c["out"] == "e4m3" else 0),
                "flops": 8 * n}
    m, k = c["m"], c["k"]
    n = c["n"] if c["op"] == "linear4" else 2 * c["f"]
    groups = -(-k // c["group"])
    weights = n * (k / 2 + groups + 4)
    rows = m * (k * _BYTES[c["a"]] + (4 if c["a"] == "e4m3" else 0))
    if c["op"] == "linear4":
        more = m * n * (_BYTES[c["out"]] + (4 if c["residual"] else 0)) + (4 * n if c["bias"] else 0)
    else:
        more = m * c["f"] * 2
    return {"bytes": weights + rows + more, "flops": 2 * m * n * k}


# ---- what a program has in hand ----------------------------------------------------------------------------

def _weights(gen, n, k, group):
    """(q int8 [n, k], s e4m3 [n, groups], r float32 [n]): a matrix with the spread of a trained one, rounded to the nearest 4-bit weight."""
    w = torch.randn(n, k, generator=gen, device="cuda") * (0.5 / math.sqrt(k))
    w *= torch.exp(0.3 * torch.randn(n, 1, generator=gen, device="cuda"))
    groups = -(-k // group)
    padded = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
    t = padded.abs().amax(2) / 7.0
    r = t.amax(1) / 448.0
    s = (t / r[:, None]).to(torch.float8_e4m3fn)
    step = s.float() * r[:, None]
    q = torch.where(step[:, :, None] > 0, (padded / step[:, :, None]).round().clamp(-8, 7), torch.zeros_like(padded))
    return q.view(n, groups * group)[:, :k].to(torch.int8).contiguous(), s, r


def _rows8(a):
    """Float rows as e4m3 with a scale a row."""
    scale = a.abs().amax(1) / 448.0
    return (a / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dev = "cuda"
    if c["op"] == "rms_add":
        rows, width = c["rows"], c["width"]
        # A residual stream: a few channels are far larger than the others, and rows differ in size.
        spread = torch.exp(0.7 * torch.randn(1, width, generator=gen, device=dev))
        size = torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device=dev))
        s = dict(c=c, x=(torch.randn(rows, width, generator=gen, device=dev) * spread * size).to(_TYPE[c["x"]]),
                 delta=(0.3 * torch.randn(rows, width, generator=gen, device=dev) * spread).to(_TYPE[c["delta"]]),
                 gain=1.0 + 0.2 * torch.randn(width, generator=gen, device=dev), eps=1e-5)
        s["total"] = torch.empty_like(s["x"])
        s["out"] = torch.empty(rows, width, dtype=_TYPE[c["out"]], device=dev)
        s["scale"] = torch.empty(rows, device=dev) if c["out"] == "e4m3" else None
        return s
    m, k, gated = c["m"], c["k"], c["op"] == "gated4"
    n = 2 * c["f"] if gated else c["n"]
    q, s8, r = _weights(gen, n, k, c["group"])
    a = torch.randn(m, k, generator=gen, device=dev) * torch.exp(0.4 * torch.randn(1, k, generator=gen, device=dev))
    s = dict(c=c, scale=None, bias=None, residual=None)
    if c["a"] == "e4m3":
        s["a"], s["scale"] = _rows8(a)
    else:
        s["a"] = a.to(torch.bfloat16)
    if gated:
        s["out"] = torch.empty(m, c["f"], dtype=torch.bfloat16, device=dev)
    else:
        s["out"] = torch.empty(m, n, dtype=_TYPE[c["out"]], device=dev)
        if c["bias"]:
            s["bias"] = 0.1 * torch.randn(n, generator=gen, device=dev)
        if c["residual"]:
            s["residual"] = torch.randn(m, n, generator=gen, device=dev)
    if own:
        from liyab_b200 import ops
        s["w"] = ops.lay_out_weights4(q, s8, r, c["group"], paired=gated)
    else:
        s["w"] = (q, s8, r)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------

def _gelu_tanh(x):
    return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _act(x, kind):
    if kind == "gelu_tanh":
        return _gelu_tanh(x)
    if kind == "gelu_erf":
        return 0.5 * x * (1.0 + torch.erf(x * 0.7071067811865476))
    if kind == "relu2":
        return torch.relu(x) * torch.relu(x)
    if kind == "silu":
        return x / (1.0 + torch.exp(-x))
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    if kind == "relu":
        return torch.relu(x)
    return x


def _plain_product(s):
    c = s["c"]
    q, s8, r = s["w"]
    k = c["k"]
    w = q.float() * s8.float().repeat_interleave(c["group"], dim=1)[:, :k]
    y = s["a"].float() @ w.T * r
    return y if s["scale"] is None else y * s["scale"][:, None]


def _plain(s):
    c = s["c"]
    if c["op"] == "rms_add":
        t = s["x"].float() + s["delta"].float()
        h = t * torch.rsqrt((t * t).mean(1, keepdim=True) + s["eps"]) * s["gain"]
        if s["scale"] is None:
            return t.to(s["x"].dtype), h.to(s["out"].dtype)
        scale = h.abs().amax(1) / 448.0
        return t.to(s["x"].dtype), (h / scale[:, None]).to(s["out"].dtype), scale
    y = _plain_product(s)
    if c["op"] == "gated4":
        return (_act(y[:, :c["f"]], c["gate"]) * y[:, c["f"]:]).to(s["out"].dtype)
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _act(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"]
    return y.to(s["out"].dtype)


def run(state):
    s = state
    if not own:
        return _plain(s)
    from liyab_b200 import ops
    c = s["c"]
    if c["op"] == "rms_add":
        ops.rms_add(s["x"], s["delta"], s["gain"], s["eps"], s["out"], scale=s["scale"], total=s["total"])
        return (s["total"], s["out"]) if s["scale"] is None else (s["total"], s["out"], s["scale"])
    if c["op"] == "gated4":
        return ops.gated4(s["a"], s["w"], s["out"], c["m"], gate=c["gate"], a_scale=s["scale"])
    return ops.linear4(s["a"], s["w"], s["bias"], s["out"], c["m"], activation=c["act"], residual=s["residual"], a_scale=s["scale"])


# ---- the definition in 64 bits -----------------------------------------------------------------------------

def exact(case, seed):
    """What the operators' definitions give in 64 bits.  Outputs of few bits are given before their rounding."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c, f64 = case, torch.float64
    if c["op"] == "rms_add":
        t = torch.add(s["x"].to(f64), s["delta"].to(f64))
        h = t.div(t.pow(2).mean(dim=-1, keepdim=True).add(s["eps"]).sqrt()).mul(s["gain"].to(f64))
        if c["out"] == "bf16":
            return t, h
        top = h.abs().max(dim=-1).values.div(448)
        return t, h.div(top.unsqueeze(-1)), top
    q, s8, r = s["w"]
    n, k = q.shape
    group = torch.arange(k, device=q.device) // c["group"]
    w = q.to(f64).mul(s8.to(f64).index_select(1, group)).mul(r.to(f64).unsqueeze(1))
    a = s["a"].to(f64)
    if s["scale"] is not None:
        a = a.mul(s["scale"].to(f64).unsqueeze(1))
    y = torch.einsum("mk,nk->mn", a, w)
    kind = c["gate"] if c["op"] == "gated4" else c["act"]
    z = y[:, :c["f"]] if c["op"] == "gated4" else y if s["bias"] is None else y.add(s["bias"].to(f64))
    if kind == "gelu_tanh":
        z = z.mul(torch.sigmoid(z.add(z.pow(3).mul(0.044715)).mul(2.0 * math.sqrt(2.0 / math.pi))))
    elif kind == "gelu_erf":
        z = z.mul(torch.special.ndtr(z))
    elif kind == "relu2":
        z = z.clamp(min=0).pow(2)
    elif kind == "silu":
        z = z.mul(torch.sigmoid(z))
    elif kind == "sigmoid":
        z = torch.sigmoid(z)
    elif kind == "relu":
        z = z.clamp(min=0)
    if c["op"] == "gated4":
        return z.mul(y[:, c["f"]:])
    return z if s["residual"] is None else z.add(s["residual"].to(f64))
