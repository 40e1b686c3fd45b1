"""Waits of kernels with warp roles are given up together (sources only: a warp or a group that splits may never return), and launches that give up leave everything usable."""
import os
import re

import pytest
import torch

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "kernels")


def _blocks_around(text, at):
    """What stands in front of every brace that is open at `at`, innermost last."""
    opened, start = [], 0
    for m in re.finditer(r"[{};]", text[:at]):
        if m.group() == "{":
            opened.append(text[start:m.start()].strip())
        elif m.group() == "}" and opened:
            opened.pop()
        start = m.end()
    return opened


def _source(name):
    text = open(os.path.join(KERNELS, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_a_wait_of_one_lane_belongs_to_a_role_of_one_thread():
    """tcgen05.ld, ldmatrix, stmatrix and warp barriers are for whole warps. Lanes that each decide whether a wait gave up can decide differently."""
    files = [f for f in sorted(os.listdir(KERNELS)) if f.endswith((".cu", ".cuh")) and "tmem_" in _source(f) and f != "sm100_ptx.cuh"]
    assert {"grouped_gemm.cu", "grouped_gemm_pair.cu", "grouped_gemm_tokens.cu", "linear_few.cu"} <= set(files)
    bad, single, together = [], 0, 0
    for f in files:
        text = _source(f)
        for m in re.finditer(r"\bmbar_wait_bounded\(", text):
            if any("elect_one()" in b for b in _blocks_around(text, m.start())):
                single += 1
            else:
                bad.append((f, text[:m.start()].count("\n") + 1))
        together += len(re.findall(r"\bmbar_wait_(?:warp|group)\(", text))
    assert not bad, bad
    assert single >= 12 and together >= 7


def test_groups_that_meet_at_a_barrier_without_a_limit_give_up_as_one():
    """Four warps around `bar.sync`: one that has left would be waited for. Their waits end in a vote of the group, or, in kernels with a warp's own stores, in one of the warp."""
    for f in ("grouped_gemm_tokens.cu", "grouped_gemm_pair.cu"):
        text = _source(f)
        for m in re.finditer(r"\bmbar_wait_warp\(", text):
            line = text[text.rfind("\n", 0, m.start()) + 1:text.find("\n", m.start())]
            around = " ".join(_blocks_around(text, m.start())) + line
            voted = "const bool here" in line and "group_all(group, here)" in text[m.start():]
            assert voted or "EPI == GemmEpilogue::kLinear" in around or "constexpr (WIDE)" in around or "q_full" in line, (f, line)


@pytest.mark.gpu
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("counts,N,K", [([40, 0, 61], 512, 512), ([100, 128], 512, 2048), ([700, 0, 1030], 512, 512), ([300, 256], 1024, 8192)])
def test_launches_that_give_up_leave_the_next_as_if_they_had_not_been(counts, N, K, swiglu):
    """Tiles of up to 64, 128 and 256 tokens wait for rows that never come (what they have on its way is there long before 20 ms are over)."""
    from fast_b200 import runtime
    from fast_b200.ops import gemm

    if not gemm.USE_PAIR:
        pytest.skip("belongs to the CTA-pair kernels")
    g = torch.Generator(device="cuda").manual_seed(1)
    off, rows = [0], 0
    for n in counts:
        rows += -(-n // 256) * 256
        off.append(rows)
    a = torch.randn(rows, K, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(len(counts), N, K, generator=g, device="cuda") * K**-0.5).to(torch.bfloat16)
    off, live = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (off, counts))
    target = torch.tensor(counts, dtype=torch.int64, device="cuda")
    out = torch.zeros(rows, N // 2 if swiglu else N, device="cuda", dtype=torch.bfloat16)

    def run(counter, limit):
        gemm.grouped_gemm_fwd(a, w, off, out.zero_(), swiglu=swiglu, live_rows=live, granule=32, gate=(counter.data_ptr(), target), timeout_s=limit, most_rows=max(counts))

    run(target, 5.0)
    gemm.check()
    want = out.clone()
    for short in [i for i, n in enumerate(counts) if n]:
        counter = target.clone()
        counter[short] -= 1
        run(counter, 0.02)
        with pytest.raises(runtime.CollectiveTimeout):
            gemm.check()
        gemm.reset()
        run(target, 5.0)
        gemm.check()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", [(300, 512, 20000), (40, 512, 4096)])
def test_a_limit_does_not_count_the_kernel_in_front(T, K, N):
    """A linear layer that is set up while a longer kernel in front of it still runs (on a few SMs, waiting for a row that never comes) has its own limit from then on."""
    from fast_b200 import runtime
    from fast_b200.ops import fused, gemm

    if not gemm.USE_PAIR:
        pytest.skip("belongs to the CTA-pair kernels")
    C = runtime.ext()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randint(-2, 3, s, generator=g, device="cuda").to(torch.bfloat16) for s in ((T, K), (N, K)))
    want = fused.linear(x, w)
    rows, inner = 256, 512
    a, e = torch.zeros(rows, inner, device="cuda", dtype=torch.bfloat16), torch.zeros(1, 512, inner, device="cuda", dtype=torch.bfloat16)
    off, live = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, rows], [200]))
    target, counter = torch.tensor([200], device="cuda"), torch.tensor([199], device="cuda")
    out = torch.zeros(rows, 512, device="cuda", dtype=torch.bfloat16)
    for _ in range(3):
        gemm.grouped_gemm_fwd(a, e, off, out, live_rows=live, granule=32, gate=(counter.data_ptr(), target), timeout_s=0.06, ctas=4)
        got = C.linear(x, w, None, None, 0, 0.01)
        with pytest.raises(runtime.CollectiveTimeout):
            gemm.check()
        assert C.dense_status().read()[0] == 0 and torch.equal(got, want)
        gemm.reset()


def test_a_kernel_that_gives_up_waits_for_what_is_under_way():
    """Every kernel with a TMA ring: its loads, its products and, with a residual that comes in by TMA, that."""
    for f in ("grouped_gemm.cu", "grouped_gemm_pair.cu", "grouped_gemm_tokens.cu", "linear_few.cu"):
        text = _source(f)
        end = text[text.index("__syncwarp();\n  const bool ok = mbar_wait_warp") if f == "linear_few.cu" else text.rindex("tc_fence_before_sync();\n  __syncthreads();"):]
        told = "if (!ok && warp == 1)" if f == "linear_few.cu" else "*abort_flag)"
        drained = "mbar_drain(&ctl->full" if f == "grouped_gemm_tokens.cu" else "drain_loads(ctl->full"
        assert end.index(told) < end.index(drained) < end.rindex("tmem_dealloc"), f
        assert re.search(r"mma_commit(_pair)?\((ok \? &ctl->done : )?&ctl->products", text) and "mbar_drain(&ctl->products, 0)" in text, f
    assert "mbar_drain(&ctl->epi_load" in _source("grouped_gemm_tokens.cu")


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,kw", [
    (1, 1 << 24, 128, {}), (300, 1 << 22, 256, {"bias": True}),         # few tokens: one tile for a cluster of CTAs, and several
    (2048, 1 << 20, 2048, {"act": 2, "bias": True, "residual": True}),   # tiles of 256 features, a warp's own stores
    (2048, 1 << 20, 2048, {"act": 4}),                                   # ... a group's stores
    (4096, 1 << 19, 7168, {}),                                           # tiles of up to 512 tokens
])
def test_a_linear_layer_whose_limit_ends_in_the_middle(T, K, N, kw):
    """The limit (looked at every 256 polls: about every millisecond) is shorter than the reduction of a tile, 5 ms and more: the launch reports that, ends, and the next one is right."""
    from fast_b200 import runtime
    from fast_b200.ops import gemm

    C = runtime.ext()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randint(-1, 2, s, generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16) for s in ((T, K), (N, K)))
    act = kw.get("act", 0)
    b = torch.ones(N, device="cuda", dtype=torch.bfloat16) if kw.get("bias") else None
    r = torch.ones(T, N, device="cuda", dtype=torch.bfloat16) if kw.get("residual") else None
    want = C.linear(x, w, b, r, act, 5.0)
    gemm.check()
    for _ in range(3):
        C.linear(x, w, b, r, act, 50e-6)
        with pytest.raises(runtime.CollectiveTimeout):
            gemm.check()
        gemm.reset()
        again = C.linear(x, w, b, r, act, 5.0)
        gemm.check()
        assert torch.equal(again, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", [(1 << 23, 64, 1024), (1 << 20, 1024, 4096)])   # rows shared out, and a tile a pair of CTAs
def test_a_weight_gradient_whose_limit_ends_in_the_middle(T, K, N):
    from fast_b200 import runtime
    from fast_b200.ops import gemm

    C = runtime.ext()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randint(-1, 2, s, generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16) for s in ((T, K), (N, K)))
    w.requires_grad_()
    dy = torch.ones(T, N, device="cuda", dtype=torch.bfloat16)
    want = torch.autograd.grad(C.linear(x, w, None, None, 0, 5.0), w, dy)[0]
    gemm.check()
    for _ in range(2):
        y = C.linear(x, w, None, None, 0, 50e-6)
        gemm.check()
        torch.autograd.grad(y, w, dy)
        with pytest.raises(runtime.CollectiveTimeout):
            gemm.check()
        gemm.reset()
        assert torch.equal(torch.autograd.grad(C.linear(x, w, None, None, 0, 5.0), w, dy)[0], want)
        gemm.check()
