"""Small, self-timed workloads of single kernels and single steps, for profiling.

    python -m liyab_b200.kernel_cases gemm --m 2048 --n 768 --k 3072 --out float32 --reps 20
    python -m liyab_b200.kernel_cases decode-attention --batch 64 --context 768 --reps 20
    python -m liyab_b200.kernel_cases prefill-attention --seqs 2 --length 1024 --reps 20
    python -m liyab_b200.kernel_cases sample --rows 8 --vocab 50257 --temp 0.8 --top-k 40 --top-p 0.95
    python -m liyab_b200.kernel_cases decode-step --batch 8 --layers 12 --reps 20 [--eager]
    python -m liyab_b200.kernel_cases prefill-step --tokens 2048 --layers 12 --reps 3
    python -m liyab_b200.kernel_cases channel-memory --batch 2 --new 1024 --heads 6 --dim 64 --vdim 128 --delta
    python -m liyab_b200.kernel_cases prefill-attention --soft-cap 50 --score-bound 8.2
    python -m liyab_b200.kernel_cases norm-join --rows 2048 --width 768 --experts 16
    python -m liyab_b200.kernel_cases streams --rows 2048 --streams 2 --width 768 --experts 20
    python -m liyab_b200.kernel_cases weights4 --rows 1 --width 4096 --inner 10240 [--e4m3]
    python -m liyab_b200.kernel_cases cache4 --batch 8 --context 8192 --heads 32 --kv 8 --dim 128 --new 512

Each prints one line with the CUDA-event time per repetition and the achieved rate.  The cases are what the
ncu summaries under profiles/ were captured on (one kernel, a few launches, inputs of a few hundred MB at most).
"""
from __future__ import annotations

import argparse
import os
import sys
import tempfile
import numpy as np
import torch

GPT2_SMALL = dict(model_type="gpt2", n_layer=12, n_embd=768, n_head=12, n_inner=3072, vocab_size=50257,
                  n_positions=1024, layer_norm_epsilon=1e-5, activation_function="gelu_new")
GPT2_SIZES = {"small": GPT2_SMALL,
              "medium": dict(GPT2_SMALL, n_layer=24, n_embd=1024, n_head=16, n_inner=4096),
              "large": dict(GPT2_SMALL, n_layer=36, n_embd=1280, n_head=20, n_inner=5120),
              "xl": dict(GPT2_SMALL, n_layer=48, n_embd=1600, n_head=25, n_inner=6400)}


def _timed(fn, reps: int, warmup: int = 2) -> float:
    for _ in range(warmup):
        fn()
    torch.cuda.synchronize()
    s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    s.record()
    for _ in range(reps):
        fn()
    e.record()
    torch.cuda.synchronize()
    return s.elapsed_time(e) / reps


def _graph_timed(launch, reps: int, per_graph: int = 20) -> float:
    """Time per launch with `per_graph` launches captured in one CUDA graph: the kernel without the host's launch cost."""
    launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(per_graph):
            launch()
    return _timed(graph.replay, max(1, reps // per_graph)) / per_graph


class _Scratch:
    """The scratch buffers that ops.linear asks a workspace for (split-K partial sums and counters)."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, {}

    def flat(self, name, n, dtype, zero=False):
        key = (name, dtype)
        if key not in self.bufs or self.bufs[key].numel() < n:
            self.bufs[key] = torch.zeros(n, dtype=dtype, device=self.dev)
        return self.bufs[key][:n]


def case_gemm(args) -> None:
    from . import ops
    dev = torch.device("cuda:0")
    odt = torch.float32 if args.out == "float32" else torch.bfloat16
    a = torch.randn(args.m, args.k, device=dev).to(torch.bfloat16)
    w = (torch.randn(args.n, args.k, device=dev) * 0.05).to(torch.bfloat16)
    bias = torch.randn(args.n, device=dev)
    out = torch.zeros(args.m, args.n, dtype=odt, device=dev)
    res = out if odt == torch.float32 else None
    if args.weights > 1:
        # A chain of the same product over several weight matrices (more bytes than L2 holds: every launch streams
        # its weights from DRAM, as a layer's products do in a step).
        ws, many, turn = _Scratch(dev), [w] + [w.clone() for _ in range(args.weights - 1)], [0]

        def launch():
            wi = many[turn[0] % len(many)]
            turn[0] += 1
            if args.rows:
                ops.gemm_rows(a, wi, bias, out, args.m, args.act, residual=res)
            else:
                ops.linear(a, wi, bias, out, args.m, args.act, residual=res, workspace=ws)
    elif args.rows:
        launch = lambda: ops.gemm_rows(a, w, bias, out, args.m, args.act, residual=res)
    elif args.one_tile:
        launch = lambda: ops.gemm_tcgen05(a, w, bias, out, args.m, args.act, residual=res, token_tile=args.tile)
    elif args.m > 64 and ops.gemm_persistent_tile(a, w, out, args.m, res) > 0:
        launch = lambda: ops.gemm_persistent(a, w, bias, out, args.m, args.act, residual=res, feature_tile=args.tile)
    else:
        ws = _Scratch(dev)
        launch = lambda: ops.linear(a, w, bias, out, args.m, args.act, residual=res, workspace=ws)
    ms = _graph_timed(launch, args.reps) if args.graph else _timed(launch, args.reps)
    print(f"gemm M={args.m} N={args.n} K={args.k} out={args.out}: {ms * 1e3:.1f} us per launch (includes the host's "
          f"launch cost when the kernel is shorter), {2 * args.m * args.n * args.k / ms / 1e9:.1f} TFLOP/s, "
          f"{(args.n * args.k * 2) / ms / 1e6:.1f} GB/s of weights, status {ops.device_status()}")


def case_decode_attention(args) -> None:
    from . import ops
    dev = torch.device("cuda:0")
    B, H, hd, ps, ctx = args.batch, args.heads, args.head_dim, 16, args.context
    pages_per = -(-ctx // ps)
    cache = torch.randn(B * pages_per, 2, H, ps, hd, device=dev).to(torch.bfloat16)
    table = torch.arange(B * pages_per, dtype=torch.int32, device=dev).view(B, pages_per)
    q = torch.randn(B, H * hd, device=dev).to(torch.bfloat16)
    out = torch.empty_like(q)
    positions = torch.full((B,), ctx - 1, dtype=torch.int32, device=dev)
    tensor = ops.decode_attention_kernels(H, H, hd, ps)[1] and not args.scalar
    splits = args.splits or ops.decode_splits(B, H, ctx, tensor_cores=tensor)
    partial = torch.empty(B * H * splits * (hd + 2), device=dev)
    counters = torch.zeros(B * H, dtype=torch.int32, device=dev)
    def launch():
        ops.decode_attention(q, cache, positions, table, out, partial, counters, B, H, H, hd, ps, hd ** -0.5, 0, splits,
                             tensor_cores=tensor)

    ms = _graph_timed(launch, args.reps) if args.graph else _timed(launch, args.reps)
    nbytes = B * ctx * 2 * H * hd * 2
    kind = "tensor-core" if tensor else "scalar"
    print(f"decode-attention ({kind}) batch={B} heads={H} head_dim={hd} context={ctx} splits={splits}: {ms * 1e3:.1f} us, "
          f"{nbytes / ms / 1e6:.1f} GB/s of cache ({nbytes / 1e6:.1f} MB)")


def case_generic_attention(args) -> None:
    """The 32-bit engine's attention: `batch` requests at `context`, each with `new` tokens in this step."""
    from . import ops
    dev = torch.device("cuda:0")
    dt = torch.float32 if args.dtype == "float32" else torch.bfloat16
    B, H, hd, ps, ctx, new = args.batch, args.heads, args.head_dim, 16, args.context, args.new
    pages_per = -(-ctx // ps)
    cache = torch.randn(B * pages_per, 2, H, ps, hd, device=dev).to(dt)
    table = torch.arange(B * pages_per, dtype=torch.int32, device=dev).view(B, pages_per)
    q = torch.randn(B * new, H * hd, device=dev).to(dt)
    out = torch.empty_like(q)
    tok_seq = torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(new)
    positions = torch.arange(ctx - new, ctx, dtype=torch.int32, device=dev).repeat(B)
    launch = lambda: ops.paged_attention_generic(q, cache, tok_seq, positions, table, out, B * new, H, H, hd, ps, hd ** -0.5, 0)
    ms = _graph_timed(launch, args.reps) if args.graph else _timed(launch, args.reps)
    nbytes = B * ctx * 2 * H * hd * cache.element_size()
    print(f"generic-attention {args.dtype} batch={B} new={new} heads={H} head_dim={hd} context={ctx}: {ms * 1e3:.1f} us, "
          f"{nbytes / ms / 1e6:.1f} GB/s of cache ({nbytes / 1e6:.1f} MB)")


def case_gemm_f32(args) -> None:
    """The 32-bit engine's product (FMA pipe, one summation order for every number of tokens)."""
    from . import ops
    dev = torch.device("cuda:0")
    a = torch.randn(args.m, args.k, device=dev)
    w = torch.randn(args.n, args.k, device=dev) * 0.05
    bias = torch.randn(args.n, device=dev)
    out = torch.zeros(args.m, args.n, device=dev)
    launch = lambda: ops.gemm_ffma(a, w, bias, out, args.m, args.act)
    ms = _graph_timed(launch, args.reps) if args.graph else _timed(launch, args.reps)
    print(f"gemm-f32 M={args.m} N={args.n} K={args.k}: {ms * 1e3:.1f} us per launch, {2 * args.m * args.n * args.k / ms / 1e9:.2f} TFLOP/s, "
          f"{(args.n * args.k * 4) / ms / 1e6:.1f} GB/s of weights")


def case_prefill_attention(args) -> None:
    from . import ops
    dev = torch.device("cuda:0")
    S, L, H, hd, ps = args.seqs, args.length, args.heads, args.head_dim, 16
    pages_per = -(-(L + args.past) // ps)
    cache = torch.randn(S * pages_per, 2, H, ps, hd, device=dev).to(torch.bfloat16)
    table = torch.arange(S * pages_per, dtype=torch.int32, device=dev).view(S, pages_per)
    q = torch.randn(S * L, H * hd, device=dev).to(torch.bfloat16)
    out = torch.empty_like(q)
    q_start = torch.arange(0, (S + 1) * L, L, dtype=torch.int32, device=dev)
    n_past = torch.full((S,), args.past, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()

    def launch():
        ops.prefill_attention(q, cache, q_start, n_past, table, out, S, L, H, H, hd, ps, hd ** -0.5, 0,
                              tcgen05=False if args.mma_sync else None, soft_cap=args.soft_cap, score_bound=args.score_bound)

    ms = _graph_timed(launch, args.reps) if args.graph else _timed(launch, args.reps)
    flop = S * H * (L * L / 2 + L * args.past) * hd * 4
    print(f"prefill-attention seqs={S} length={L} heads={H} head_dim={hd}{f" soft cap {args.soft_cap:g}" if args.soft_cap else ""}: {ms * 1e3:.1f} us, {flop / ms / 1e9:.1f} TFLOP/s "
          f"(causal half of the square)")


def case_sample(args) -> None:
    from . import ops
    dev = torch.device("cuda:0")
    R, V = args.rows, args.vocab
    logits = torch.randn(R, V, device=dev) * args.spread
    temp = torch.full((R,), args.temp, device=dev)
    top_k = torch.full((R,), args.top_k, dtype=torch.int32, device=dev)
    top_p = torch.full((R,), args.top_p, device=dev)
    u = torch.rand(R, dtype=torch.float64, device=dev)
    ids = torch.empty(R, dtype=torch.int32, device=dev)
    ms = _graph_timed(lambda: ops.sample(logits, R, temp, top_k, top_p, u, ids), args.reps)
    print(f"sample rows={R} vocab={V} temp={args.temp} top_k={args.top_k} top_p={args.top_p}: {ms * 1e3:.1f} us "
          f"(20 launches per CUDA graph)")


def _model_folder(layers: int, dtype: str, size: str = "small") -> str:
    """A random model of the asked size in a temporary folder that is removed when the process ends."""
    import atexit
    import shutil
    from .weights import write_random_model
    tmp = tempfile.mkdtemp(prefix="liyab_b200_case_")
    atexit.register(shutil.rmtree, tmp, ignore_errors=True)
    return write_random_model(os.path.join(tmp, "m"), dict(GPT2_SIZES[size], n_layer=layers or GPT2_SIZES[size]["n_layer"]), 0, dtype)


def case_decode_step(args) -> None:
    """A few decode steps of the whole model through the library's own measurement (what bench.py times)."""
    from .engine import Replayer
    B = args.batch
    rep = Replayer(_model_folder(args.layers, args.dtype, args.size), args.dtype, max_tokens=B * 1024, max_requests=B,
                   cuda_graphs=not args.eager, fused_decode=args.fused and not args.no_fused, max_step_tokens=1024)
    r = rep.bench_decode(B, args.context, args.reps, 3)
    path = "fused" if r["fused_steps"] else ("graph" if r["graph_steps"] else "parts")
    print(f"decode-step size={args.size} batch={B} layers={len(rep.info['spec']['layers'])} context~{r['mean_context']:.0f} path={path}: "
          f"{r['ms_per_step'] * 1e3:.1f} us per step, {B / r['ms_per_step'] * 1e3:.0f} tokens/s, {r['kernel_launches'] // args.reps} launches a step")
    if args.stamps and r["fused_steps"]:
        # Where the one-kernel step's time goes: the five barriers of layer 5 (numbers 27..31), all blocks' arrivals.
        rep.set("fused_stamps", 1)
        rep.bench_decode(B, args.context, 3, 1)
        t = rep.fused_stamps().astype(np.float64) / 1e3
        n_blocks = int(np.count_nonzero(t[256:256 + 160]))
        last_barrier = int(np.flatnonzero(t[:126]).max())
        print(f"  whole kernel after its first barrier: {t[last_barrier] - t[1]:.1f} us over {last_barrier - 1} barriers; head {t[127] - t[126]:.1f} us; "
              f"from block 0's start to the first barrier's end {t[1] - t[0]:.1f} us")
        names = ["LayerNorm + projection", "attention", "output projection", "LayerNorm + up", "down"]
        for j, name in enumerate(names):
            arrive = np.sort(t[256 + 160 * j:256 + 160 * j + n_blocks])
            before, after = t[26 + j], t[27 + j]
            print(f"  layer 5 {name:>22}: work {arrive[0] - before:5.2f} / {np.median(arrive) - before:5.2f} / {arrive[-1] - before:5.2f} us "
                  f"(first / median / last block to arrive), barrier left {after - arrive[-1]:5.2f} us after the last arrival, phase {after - before:5.2f} us")


def case_prefill_step(args) -> None:
    from .engine import Replayer
    n_seq = max(1, args.tokens // 1024)
    per = args.tokens // n_seq
    rep = Replayer(_model_folder(args.layers, args.dtype, args.size), args.dtype, max_tokens=2 * args.tokens,
                   cuda_graphs=not args.eager, max_step_tokens=args.tokens)
    r = rep.bench_prefill(n_seq, per, args.reps)
    print(f"prefill-step size={args.size} tokens={n_seq}x{per} layers={len(rep.info['spec']['layers'])}: best {r['ms_per_step']:.3f} ms, "
          f"median {r['wall_ms_per_step']:.3f} ms per step, {n_seq * per / r['ms_per_step'] * 1e3:.0f} tokens/s, {r['kernel_launches']} launches")


def case_channel_memory(args) -> None:
    """A memory with a decay per key channel: whole prompts in pieces (`--new` above 15) or rows of a few tokens, over random projections."""
    from . import ops
    dev, H, D, E, B, n = torch.device("cuda:0"), args.heads, args.dim, args.vdim, args.batch, args.new
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    rank, taps = 16 if not args.delta else 32, 4 if args.delta else 0
    cols = 2 * H * D + H * E + rank + (rank + H if args.delta else H * E)
    m = dict(n_head=H, kv_head=H, dim=D, vdim=E, delta=args.delta, taps=taps, unit=args.delta, gate="sigmoid" if args.delta else "silu", z_bias=r(H * D),
             a2=(r(H * D, rank) * rank ** -0.5).bfloat16(), g2=(r(H * E, rank) * rank ** -0.5).bfloat16() if args.delta else None,
             conv=r(2 * H * D + H * E, taps) * 0.5 if args.delta else None, a_log=r(H) - 1 if args.delta else None, tau=16.0, norm=r(E), q_scale=D ** -0.5, eps=1e-5)
    proj = r(B * n, (cols + 7) // 8 * 8)[:, :cols]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    positions, tok_seq = i32(list(range(n)) * B), i32([s for s in range(B) for _ in range(n)])
    q_start, slots = i32([s * n for s in range(B + 1)]), i32(list(range(B)))
    state = torch.zeros(B, H * D * E + taps * (2 * H * D + H * E), device=dev)
    heads = torch.empty(B * n, H * E, dtype=torch.bfloat16, device=dev)
    scratch = torch.empty(ops.channel_memory_floats(B * n, B, H, D, E, args.delta), device=dev)
    ms = _timed(lambda: ops.channel_memory(m, proj, positions, tok_seq, q_start, slots, state, heads, None, pieces=n >= 16, decode_only=n == 1, scratch=scratch),
                args.reps)
    moved = (proj.numel() * 4 + heads.numel() * 2 + 2 * state.numel() * 4) / 1e9
    print(f"channel memory {B} x {n} rows, {H} heads of {D} x {E}{' delta' if args.delta else ''}: {1e3 * ms:.1f} us, {moved / ms * 1e3:.0f} GB/s of rows and state, "
          f"{B * n * H * D * E * (6 if args.delta else 4) / ms / 1e9:.2f} TFLOP/s of the recurrence")


def case_streams(args) -> None:
    """The launch between two sublayers: routed results (or a row) into the streams, the next input, and a router on it with `--experts`."""
    from . import ops
    dev, T, S, W = torch.device("cuda:0"), args.rows, args.streams, args.width
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    x, h = r(T, S * W), torch.empty(T, W, dtype=torch.bfloat16, device=dev)
    mix, to, ls, norm = r(S, S) * 0.5 / S, r(S), r(W), (torch.full((1,), 0.5, device=dev), r(W), r(W))
    router = None
    if args.experts:
        ids, weights = torch.empty(T, 2, dtype=torch.int32, device=dev), torch.empty(T, 2, device=dev)
        router = ops.router_args(r(args.experts, W).bfloat16(), 2, ids, weights, correction=r(args.experts), groups=2, keep=1)
        terms, read = ops.output_terms([r(T, W)], [1.0]), 4 * T * W
    else:
        ids = torch.randint(0, 16, (T, 2), dtype=torch.int32, device=dev, generator=gen)
        place = torch.randperm(2 * T, device=dev, generator=gen).int()
        terms, read = ops.output_terms((), (), r(2 * T, W), place, ids, r(T, 2), 16, h), 8 * T * W
    ms = _timed(lambda: ops.streams_join(x, S, T, terms, mix, to, ls, next_in=to, norm=norm, h=h, router=router), args.reps)
    print(f"streams {T} rows of {S} x {W}{', routed' if router else ''}: {1e3 * ms:.1f} us, {(8 * T * S * W + read + 2 * T * W) / ms / 1e6:.0f} GB/s")


def case_norm_join(args) -> None:
    """The launch between two norms: a row (or, with `--routed`, routed results and a gated row) through its norm into the stream, the next input, and a
    router with a gate on it with `--experts`."""
    from . import ops
    dev, T, W = torch.device("cuda:0"), args.rows, args.width
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    x, y, h, gain, factor = r(T, W), r(T, W), torch.empty(T, W, dtype=torch.bfloat16, device=dev), r(W) * 0.1, r(T)
    terms, read = ops.output_terms([y], [1.0]), 4 * T * W
    if args.routed:
        ids = torch.randint(0, 16, (T, 2), dtype=torch.int32, device=dev, generator=gen)
        place, pairs, weights = torch.randperm(2 * T, device=dev, generator=gen).int(), r(2 * T, W), r(T, 2)
        terms, read = ops.output_terms([y], [1.0], pairs, place, ids, weights, 16, None, factor=(factor,)), 12 * T * W
    router = None
    if args.experts:
        chosen, shares, gate = torch.empty(T, 2, dtype=torch.int32, device=dev), torch.empty(T, 2, device=dev), torch.empty(T, device=dev)
        router = ops.router_args(r(args.experts + 1, W).bfloat16(), 2, chosen, shares, renormalise=True, gate=gate)
    launch = lambda: ops.norm_join(x, terms, (gain, 1.0, 1e-6), T, next_norm=(gain, 1.0, 1e-6), h=h, router=router)
    ms = _graph_timed(launch, args.reps)
    print(f"norm-join {T} rows of {W}{', routed results' if args.routed else ''}{', with a router' if router else ''}: {1e3 * ms:.1f} us, {(10 * T * W + read) / ms / 1e6:.0f} GB/s")


def case_weights4(args) -> None:
    """What stands around attention in a decoder's layer, with 4-bit weights: the output product, the stream's sum and norm, a gated feed-forward and its way back into the stream,
    the sum and norm for the next layer and its joint projection.  Beside it the same with bfloat16 weights, and how far the two streams are apart."""
    from . import ops
    dev, T, W, F = torch.device("cuda:0"), args.rows, args.width, args.inner
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *shape: torch.randn(*shape, device=dev, generator=gen)
    full = [r(W, W) * W ** -0.5, r(2 * F, W) * W ** -0.5, r(W, F) * F ** -0.5, r(3 * W, W) * W ** -0.5]
    w_out, w_gate_up, w_down, w_qkv = (ops.quantise_weights4(w, args.group, paired=i == 1) for i, w in enumerate(full))
    plain = [w.bfloat16() for w in full]
    gains, x0, attended, eps = [1.0 + 0.1 * r(W) for _ in range(2)], r(T, W), r(T, W).bfloat16(), 1e-6
    x, delta, inner, qkv = x0.clone(), torch.empty(T, W, device=dev), torch.empty(T, F, dtype=torch.bfloat16, device=dev), torch.empty(T, 3 * W, dtype=torch.bfloat16, device=dev)
    h = torch.empty(T, W, dtype=torch.float8_e4m3fn if args.e4m3 else torch.bfloat16, device=dev)
    scale = torch.empty(T, device=dev) if args.e4m3 else None

    def layer4():
        ops.linear4(attended, w_out, None, delta, T)
        ops.rms_add(x, delta, gains[0], eps, h, scale=scale)
        ops.gated4(h, w_gate_up, inner, T, gate="silu", a_scale=scale)
        ops.linear4(inner, w_down, None, delta, T)
        ops.rms_add(x, delta, gains[1], eps, h, scale=scale)
        ops.linear4(h, w_qkv, None, qkv, T, a_scale=scale)

    y, rounded, gate_up, room = x0.clone(), torch.empty(T, W, dtype=torch.bfloat16, device=dev), torch.empty(T, 2 * F, device=dev), _Scratch(dev)

    def layer16():
        ops.linear(attended, plain[0], None, y, T, residual=y, workspace=room)
        ops.rms_offset(y, gains[0], 0.0, eps, rounded)
        ops.linear(rounded, plain[1], None, gate_up, T, workspace=room)
        ops.gated_act_kind(gate_up, inner, "silu")
        ops.linear(inner, plain[2], None, y, T, residual=y, workspace=room)
        ops.rms_offset(y, gains[1], 0.0, eps, rounded)
        ops.linear(rounded, plain[3], None, qkv, T, workspace=room)

    layer4()
    layer16()
    torch.cuda.synchronize()
    apart = ((x - y).norm() / (y - x0).norm()).item()
    us4, us16 = 1e3 * _graph_timed(layer4, args.reps), 1e3 * _graph_timed(layer16, args.reps)
    held = sum(w.nbytes for w in (w_out, w_gate_up, w_down, w_qkv))
    print(f"weights4 {T} rows, {W} wide, {F} inner, groups of {args.group}{', e4m3 rows' if args.e4m3 else ''}: {us4:.1f} us, {held / 1e6:.0f} MB of weights; "
          f"bfloat16 {us16:.1f} us, {sum(2 * w.numel() for w in plain) / 1e6:.0f} MB; what the sublayers add differs by {100 * apart:.1f} %")


def case_cache4(args) -> None:
    """A 4-bit cache's calls as serving makes them: a step's rows go in, its tokens attend (with and without the keys' weights), a portion of a prompt does, and the keys that gained least
    are dropped.  Beside them the same tokens and portion over a bfloat16 cache, and how far the tokens' results are apart."""
    from . import ops
    dev, B, C, H, KV, D, N = torch.device("cuda:0"), args.batch, args.context, args.heads, args.kv, args.dim, min(args.new, args.context)
    gen = torch.Generator(device=dev).manual_seed(0)
    r = lambda *shape: torch.randn(*shape, device=dev, generator=gen).bfloat16()
    page, scale, keep = 16, D ** -0.5, max(1, C // 2)
    per, kept_pages = -(-C // page), -(-keep // page)
    table = torch.randperm(B * per, device=dev, generator=gen).to(torch.int32).view(B, per)
    cache = ops.Cache4(B * (per + kept_pages), KV, D, page, args.group)
    dest = torch.arange(B * per, B * (per + kept_pages), dtype=torch.int32, device=dev).view(B, kept_pages)
    plain = torch.empty(B * per, 2, KV, page, D, dtype=torch.bfloat16, device=dev)
    key = torch.arange(C, device=dev)
    for i in range(B):
        k, v = r(C, KV * D), r(C, KV * D)
        ops.append4(k, v, (table[i, key // page] * page + key % page).to(torch.int32), cache, C)
        for of, x in enumerate((k, v)):
            rows = torch.zeros(per * page, KV, D, dtype=torch.bfloat16, device=dev)
            rows[:C] = x.view(C, KV, D)
            plain[table[i].long(), of] = rows.view(per, page, KV, D).transpose(1, 2)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    k1, v1, q1, qn = r(B, KV * D), r(B, KV * D), r(B, H * D), r(B * N, H * D)
    o1, o16, on = torch.empty_like(q1), torch.empty_like(q1), torch.empty_like(qn)
    slots, last, n_keys, start, past = table[:, -1] * page + (C - 1) % page, i32([C - 1] * B), i32([C] * B), i32([N * i for i in range(B + 1)]), i32([C - N] * B)
    mass = torch.zeros(B, KV, per * page, device=dev)
    total, kept = torch.zeros_like(mass), torch.empty(B, KV, keep, dtype=torch.int32, device=dev)
    splits = ops.decode_splits(B, KV, C, tensor_cores=True)
    partial, counters = torch.empty(B * H * splits * (D + 2), device=dev), torch.zeros(B * H, dtype=torch.int32, device=dev)

    def tokens16():
        ops.decode_attention(q1, plain, last, table, o16, partial, counters, B, H, KV, D, page, scale, 0, splits)

    us = lambda fn: 1e3 * _graph_timed(fn, args.reps)
    ops.decode_attention4(q1, cache, last, table, o1, B, H, scale, mass=mass, total=total)
    line = {"tokens": us(lambda: ops.decode_attention4(q1, cache, last, table, o1, B, H, scale)),
            "with weights": us(lambda: ops.decode_attention4(q1, cache, last, table, o1, B, H, scale, mass=mass, total=total)),
            f"portions of {N}": us(lambda: ops.prefill_attention4(qn, cache, start, past, table, on, B, N, H, scale)),
            f"{keep} keys kept": us(lambda: ops.evict4(cache, total, table, n_keys, B, keep, min(keep, 32), dest, kept))}
    if ops.decode_attention_supports(H, KV, D, page):
        line["tokens over bfloat16"] = us(tokens16)
    if ops.prefill_attention_supports(H, KV, D, page):
        line["portions over bfloat16"] = us(lambda: ops.prefill_attention(qn, plain, start, past, table, on, B, N, H, KV, D, page, scale))
    apart = f"; tokens' results differ by {100 * ((o1.float() - o16.float()).norm() / o16.float().norm()).item():.1f} %" if "tokens over bfloat16" in line else ""
    line["rows in"] = us(lambda: ops.append4(k1, v1, slots, cache, B))
    print(f"cache4 {B} x {C} keys, {H} heads over {KV} of {D}, groups of {args.group}: {', '.join(f'{k} {v:.1f} us' for k, v in line.items())}; "
          f"{B * per * page * KV * (D + 4 * D // args.group) / 1e6:.0f} MB of keys and values, bfloat16 {2 * plain.numel() / 1e6:.0f}{apart}")


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="python -m liyab_b200.kernel_cases")
    sub = ap.add_subparsers(dest="case", required=True)
    g = sub.add_parser("gemm")
    g.add_argument("--m", type=int, default=2048)
    g.add_argument("--n", type=int, default=768)
    g.add_argument("--k", type=int, default=3072)
    g.add_argument("--out", default="bfloat16", choices=["bfloat16", "float32"])
    g.add_argument("--act", default="none", choices=["none", "gelu_tanh", "gelu_erf"])
    g.add_argument("--tile", type=int, default=0, help="feature tile of the persistent kernel (token tile with --one-tile)")
    g.add_argument("--graph", action="store_true", help="time 20 launches captured in a CUDA graph")
    g.add_argument("--one-tile", action="store_true", help="the one-tile-per-block kernel also for many tokens")
    g.add_argument("--weights", type=int, default=1, help="cycle through this many copies of the weights (with --graph: 20 per graph)")
    g.add_argument("--rows", action="store_true", help="the one-launch mma.sync product (up to 64 tokens) whatever the size")
    g.add_argument("--reps", type=int, default=20)
    d = sub.add_parser("decode-attention")
    d.add_argument("--batch", type=int, default=64)
    d.add_argument("--heads", type=int, default=12)
    d.add_argument("--head-dim", type=int, default=64)
    d.add_argument("--context", type=int, default=768)
    d.add_argument("--reps", type=int, default=20)
    d.add_argument("--splits", type=int, default=0, help="key ranges per request and head (0: the engine's choice)")
    d.add_argument("--graph", action="store_true", help="time 20 launches captured in a CUDA graph")
    d.add_argument("--scalar", action="store_true", help="the scalar kernel even where the tensor-core one takes the shape")
    ga = sub.add_parser("generic-attention")
    ga.add_argument("--batch", type=int, default=8)
    ga.add_argument("--new", type=int, default=1, help="tokens of each request in this step")
    ga.add_argument("--heads", type=int, default=12)
    ga.add_argument("--head-dim", type=int, default=64)
    ga.add_argument("--context", type=int, default=768)
    ga.add_argument("--dtype", default="float32", choices=["bfloat16", "float32"])
    ga.add_argument("--reps", type=int, default=20)
    ga.add_argument("--graph", action="store_true", help="time 20 launches captured in a CUDA graph")
    gf = sub.add_parser("gemm-f32")
    gf.add_argument("--m", type=int, default=8)
    gf.add_argument("--n", type=int, default=2304)
    gf.add_argument("--k", type=int, default=768)
    gf.add_argument("--act", default="none", choices=["none", "gelu_tanh", "gelu_erf"])
    gf.add_argument("--reps", type=int, default=20)
    gf.add_argument("--graph", action="store_true", help="time 20 launches captured in a CUDA graph")
    a = sub.add_parser("prefill-attention")
    a.add_argument("--seqs", type=int, default=2)
    a.add_argument("--length", type=int, default=1024)
    a.add_argument("--past", type=int, default=0, help="earlier tokens of every request")
    a.add_argument("--heads", type=int, default=12)
    a.add_argument("--head-dim", type=int, default=64)
    a.add_argument("--reps", type=int, default=20)
    a.add_argument("--graph", action="store_true", help="time 20 launches captured in a CUDA graph")
    a.add_argument("--soft-cap", type=float, default=0.0, help="cap on the scores, c tanh(s / c)")
    a.add_argument("--score-bound", type=float, default=0.0, help="the largest |score| that can occur (0: unknown)")
    a.add_argument("--mma-sync", action="store_true", help="the mma.sync kernel even where the tcgen05 one takes the shape")
    sm = sub.add_parser("sample")
    sm.add_argument("--rows", type=int, default=8)
    sm.add_argument("--vocab", type=int, default=50257)
    sm.add_argument("--temp", type=float, default=0.8)
    sm.add_argument("--top-k", type=int, default=40)
    sm.add_argument("--top-p", type=float, default=0.95)
    sm.add_argument("--spread", type=float, default=3.0, help="standard deviation of the random logits (8: peaked like a model's)")
    sm.add_argument("--reps", type=int, default=400)
    cm = sub.add_parser("channel-memory")
    cm.add_argument("--batch", type=int, default=2)
    cm.add_argument("--new", type=int, default=1024, help="rows of each request in this step")
    cm.add_argument("--heads", type=int, default=6)
    cm.add_argument("--dim", type=int, default=64)
    cm.add_argument("--vdim", type=int, default=128)
    cm.add_argument("--delta", action="store_true", help="the delta rule with short convolutions (default: gated linear attention)")
    cm.add_argument("--reps", type=int, default=20)
    nj = sub.add_parser("norm-join")
    nj.add_argument("--rows", type=int, default=2048)
    nj.add_argument("--width", type=int, default=768)
    nj.add_argument("--experts", type=int, default=0)
    nj.add_argument("--routed", action="store_true", help="the sublayer's output is routed experts' results and a gated shared one")
    nj.add_argument("--reps", type=int, default=20)
    st = sub.add_parser("streams")
    st.add_argument("--rows", type=int, default=2048)
    st.add_argument("--streams", type=int, default=2)
    st.add_argument("--width", type=int, default=768)
    st.add_argument("--experts", type=int, default=0)
    st.add_argument("--reps", type=int, default=20)
    w4 = sub.add_parser("weights4")
    w4.add_argument("--rows", type=int, default=1)
    w4.add_argument("--width", type=int, default=4096)
    w4.add_argument("--inner", type=int, default=10240)
    w4.add_argument("--group", type=int, default=128, choices=[32, 64, 128])
    w4.add_argument("--e4m3", action="store_true", help="the norms leave e4m3 rows with a scale each")
    w4.add_argument("--reps", type=int, default=200)
    c4 = sub.add_parser("cache4")
    c4.add_argument("--batch", type=int, default=8)
    c4.add_argument("--context", type=int, default=8192)
    c4.add_argument("--heads", type=int, default=32)
    c4.add_argument("--kv", type=int, default=8)
    c4.add_argument("--dim", type=int, default=128, choices=[64, 128])
    c4.add_argument("--group", type=int, default=64, choices=[32, 64, 128])
    c4.add_argument("--new", type=int, default=512, help="tokens of a portion")
    c4.add_argument("--reps", type=int, default=100)
    for name in ("decode-step", "prefill-step"):
        p = sub.add_parser(name)
        p.add_argument("--batch", type=int, default=8)
        p.add_argument("--tokens", type=int, default=2048)
        p.add_argument("--context", type=int, default=512)
        p.add_argument("--layers", type=int, default=0, help="fewer layers than the size has (0: all)")
        p.add_argument("--size", default="small", choices=sorted(GPT2_SIZES))
        p.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
        p.add_argument("--reps", type=int, default=10)
        p.add_argument("--eager", action="store_true", help="no captured graphs")
        p.add_argument("--no-fused", action="store_true", help="not the one-kernel decode step")
        p.add_argument("--fused", action="store_true", help="decode steps of up to 16 requests as one persistent kernel (default: part by part)")
        p.add_argument("--stamps", action="store_true", help="decode-step: per-phase times from inside the one-kernel step")
    args = ap.parse_args(argv)
    {"gemm": case_gemm, "generic-attention": case_generic_attention, "gemm-f32": case_gemm_f32, "decode-attention": case_decode_attention, "prefill-attention": case_prefill_attention, "sample": case_sample, "decode-step": case_decode_step,
     "prefill-step": case_prefill_step, "channel-memory": case_channel_memory, "streams": case_streams, "norm-join": case_norm_join, "weights4": case_weights4, "cache4": case_cache4}[args.case](args)
    return 0


if __name__ == "__main__":
    sys.exit(main())
