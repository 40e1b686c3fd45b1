"""The dense operators (``ops.fused``: row norm, balance loss, linear layers) on one GPU, each call as a user makes it.

    python -m fast_b200.bench.dense                 the measured cases (perf/operators.py): us a call in a stream of calls, host included, and replayed as a CUDA graph
    python -m fast_b200.bench.dense --host          what torch's autograd costs the host, measured on calls that launch nothing, beside the small training cases
    python -m fast_b200.bench.dense --kernels [N]   a launch of every kernel at the sizes of profiles/dense_operators.md, twice, for a profiler (the second is warm)

CUDA-event timing after warm-up. Streams of calls of one case keep small operands in L2, as a layer's own does not: see the profile for cold ones.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import time

import torch

from ..ops import fused, gemm

BF = torch.bfloat16


def _cases():
    path = os.path.join(os.path.dirname(__file__), "..", "..", "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("operators", path)
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    return ops


def _stream_us(fn, seconds=0.3):
    for _ in range(5):
        fn()
    torch.cuda.synchronize()
    n = 10
    while True:
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(n):
            fn()
        e1.record()
        torch.cuda.synchronize()
        ms = e0.elapsed_time(e1)
        if ms > 1e3 * seconds / 4:
            return 1e3 * ms / n
        n = max(2 * n, int(n * 300 * seconds / max(ms, 1e-3)))


def _graph_us(run, state):
    """``run`` captured ten times over, on leaves of its own (a graph of autograd's holds on to the leaves that it was made of)."""
    state = {k: v.detach().clone().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in state.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            run(state)
    return _stream_us(graph.replay) / 10


def _table(only):
    ops = _cases()
    print(f"{'case':28s} {'stream':>9s} {'graph':>9s}   us a call")
    for case in ops.listed():
        if only and case["name"] not in only:
            continue
        state = ops.prepare(case, 1)
        print(f"{case['name']:28s} {_stream_us(lambda: ops.run(state)):9.2f} {_graph_us(ops.run, state):9.2f}", flush=True)
        del state
        torch.cuda.empty_cache()
    gemm.check()


def _host_us(fn, n=3000):
    for _ in range(300):
        fn()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(n):
        fn()
    host = time.perf_counter() - t0   # the host's own time: nothing is waited for
    torch.cuda.synchronize()
    return 1e6 * host / n


def _host():
    none = torch.empty(0, 64, device="cuda", dtype=BF, requires_grad=True)
    row, w = torch.ones(1, 64, device="cuda", dtype=BF).requires_grad_(), torch.ones(64, 64, device="cuda", dtype=BF)
    d0, d1 = torch.empty_like(none), torch.ones_like(row)
    lines = [("linear of no rows, forward", lambda: fused.linear(none, w)), ("linear of no rows, forward and grad", lambda: torch.autograd.grad(fused.linear(none, w), none, d0)),
             ("torch: x * 2, forward", lambda: row * 2.0), ("torch: x * 2, forward and grad", lambda: torch.autograd.grad(row * 2.0, row, d1)),
             ("linear of one row, forward", lambda: fused.linear(row, w)), ("linear of one row, forward and grad", lambda: torch.autograd.grad(fused.linear(row, w), row, d1))]
    ops = _cases()
    for case in ops.listed():
        if case["name"] in ("norm_train_odd_fp32", "balance_train_32768x8", "balance_train_16384x256"):
            state = ops.prepare(case, 1)
            lines.append((case["name"], lambda state=state: ops.run(state)))
    for name, fn in lines:
        print(f"{name:40s} {_host_us(fn):8.2f} us of the host", flush=True)


def _kernels(times):
    g = torch.Generator(device="cuda").manual_seed(1)

    def t(*shape, std=1.0, dtype=BF):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    def norm(T, H, residual, quantise=False, train=False):
        x, r, w = t(T, H).requires_grad_(train), t(T, H).requires_grad_(train) if residual else None, t(H).requires_grad_(train)
        out = fused.add_rms_norm(x, w, residual=r, quantise=quantise)
        if train:
            torch.autograd.grad([out.y, out.h], [x, w, r], [t(T, H), t(T, H)])

    def linear(T, K, N, act=None, bias=False, residual=False, train=False):
        x, w = t(T, K).requires_grad_(train), t(N, K, std=K**-0.5).requires_grad_(train)
        b, r = t(N) if bias else None, t(T, N) if residual else None
        y = fused.linear(x, w, bias=b, activation=act, residual=r)
        if train:
            torch.autograd.grad(y, [x, w], t(*y.shape))

    logits, idx = t(65536, 256, dtype=torch.float32).requires_grad_(), torch.randint(0, 256, (65536, 8), generator=g, device="cuda").to(torch.int32)
    for run in (lambda: norm(16384, 4096, True, quantise=True), lambda: norm(32768, 4096, True, train=True), lambda: norm(8192, 4097, False),
                lambda: torch.autograd.grad(fused.balance_loss(logits, idx)[0], logits), lambda: linear(1, 4096, 14336), lambda: linear(64, 4096, 14336), lambda: linear(1, 4096, 4096),
                lambda: linear(512, 2048, 4096), lambda: linear(1235, 1000, 2760, "silu", True, True), lambda: linear(2048, 4096, 14336, "gelu"), lambda: linear(8192, 1024, 14336, "gelu", train=True)):
        for _ in range(times):
            run()
    torch.cuda.synchronize()
    gemm.check()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--only", default="", help="comma-separated names of measured cases")
    ap.add_argument("--host", action="store_true")
    ap.add_argument("--kernels", type=int, nargs="?", const=2, default=0, metavar="N")
    a = ap.parse_args()
    if a.host:
        _host()
    elif a.kernels:
        _kernels(a.kernels)
    else:
        _table(set(a.only.split(",")) - {""})


if __name__ == "__main__":
    main()
