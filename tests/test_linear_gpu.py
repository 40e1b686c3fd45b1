"""Linear layers with an epilogue against a plain implementation in 64 bits.

Two kinds of input. Small whole numbers: every product and sum is exact in fp32, so results are the 64-bit ones rounded to bf16, equal bit for bit,
whatever the order of a sum. Normal numbers: half a step of bf16 for the rounding at the end, and for fp32 sums of n terms in blocks of 16 whose
additions may truncate, (n / 16 + 16) 2^-23 of what is added in magnitude."""
import pytest
import torch

from fast_b200.models.moe import interleave_gate_up
from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF = 2.0**-8
SHAPES = [(1, 8, 8), (1, 4096, 256), (2, 72, 136), (31, 64, 264), (33, 1000, 1736), (64, 2048, 7168), (65, 512, 520), (100, 7168, 1032), (129, 136, 72), (257, 1024, 1024), (300, 8, 2000), (513, 4096, 8),
          (1235, 1000, 2760), (2000, 200, 4104), (700, 9000, 328), (50, 136, 20008), (100, 136, 20008),   # narrow tiles in more than a round
          (100, 8192, 8200), (8200, 8200, 3432), (8200, 3432, 8200)]                                      # wide weight gradients, forward and data gradients


def whole(shape, seed, most=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(BF)


def normal(shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


def bf(v):
    return v.to(BF)   # from 64 bits: these values are whole numbers below 2^24, rounded once


ACT = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_whole_numbers_are_exact(T, K, N):
    x, w, b, r, dy = whole((T, K), 1), whole((N, K), 2), whole((N,), 3, 9), whole((T, N), 4, 9), whole((T, N), 5)
    for act, bias, res in ((None, None, None), (None, b, None), ("relu", None, r), ("relu", b, r), (None, None, r)):
        leaves = [t.clone().requires_grad_() for t in (x, w, bias, res) if t is not None]
        it = iter(leaves)
        lx, lw = next(it), next(it)
        lb, lr = next(it) if bias is not None else None, next(it) if res is not None else None
        y = fused.linear(lx, lw, bias=lb, activation=act, residual=lr)
        z = x.double() @ w.double().t() + (bias.double() if bias is not None else 0)
        assert torch.equal(y, bf(ACT[act](z) + (res.double() if res is not None else 0)))
        with torch.no_grad():
            assert torch.equal(fused.linear(x, w, bias=bias, activation=act, residual=res), y)
        grads = iter(torch.autograd.grad(y, leaves, dy))
        dz = dy.double() * (z > 0) if act else dy.double()
        assert torch.equal(next(grads), bf(dz @ w.double()))
        assert torch.equal(next(grads), bf(dz.t() @ x.double()))
        if bias is not None:
            assert torch.equal(next(grads), bf(dz.sum(0)))
        if res is not None:
            assert torch.equal(next(grads), dy)
    gemm.check()


def noise(n, size):
    return (n / 16 + 16) * 2.0**-23 * size


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("T,K,N", [(1, 512, 264), (50, 1000, 1736), (300, 2048, 520), (1500, 264, 1032)])
def test_activations_and_gradients(T, K, N, act):
    x, w, b, r, dy = normal((T, K), 1), normal((N, K), 2, K**-0.5), normal((N,), 3, 0.5), normal((T, N), 4), normal((T, N), 5)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = fused.linear(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3])
    z = (x.double() @ w.double().t() + b.double()).requires_grad_()
    size = x.double().abs() @ w.double().abs().t() + b.double().abs()
    a = ACT[act](z)
    want = (a + r.double()).detach()
    # slopes stay below 1.13; an activation in fp32 is off by a few roundings of z
    off = 1.13 * noise(K, size) + 16 * 2.0**-23 * z.detach().abs()
    assert ((y.double() - want).abs() <= HALF * want.abs() + off).all()
    grads = torch.autograd.grad(y, leaves, dy)
    (slope,) = torch.autograd.grad(a.sum(), z)
    dz = dy.double() * slope
    # z was kept in bf16 (second derivatives below 0.8; a relu's sign may be decided by the product's rounding), dz is rounded to bf16
    near = (z.detach().abs() <= noise(K, size)).double() if act == "relu" else 0.8 * (HALF * z.detach().abs() + noise(K, size)) + 2.0**-18 if act else 0.0
    edz = dy.double().abs() * near + HALF * dz.abs() * (1 + HALF)
    dx, dw, db = dz @ w.double(), dz.t() @ x.double(), dz.sum(0)
    assert ((grads[0].double() - dx).abs() <= HALF * dx.abs() * 1.01 + 1.01 * (edz @ w.double().abs()) + noise(N, dz.abs() @ w.double().abs())).all()
    assert ((grads[1].double() - dw).abs() <= HALF * dw.abs() * 1.01 + 1.01 * (edz.t() @ x.double().abs()) + noise(T, dz.abs().t() @ x.double().abs())).all()
    assert ((grads[2].double() - db).abs() <= HALF * db.abs() * 1.01 + 1.01 * edz.sum(0) + noise(16 * T, dz.abs().sum(0))).all()
    assert torch.equal(grads[3], dy)
    # over all values roundings do not add up: a few of them in the 2-norm
    for got, ref in zip(grads, (dx, dw, db)):
        assert (got.double() - ref).norm() <= 4 * HALF * ref.norm()


@pytest.mark.parametrize("T,K,I", [(1, 512, 128), (7, 1000, 256), (130, 7168, 2048), (600, 264, 384), (1100, 2048, 640), (300, 4104, 52224)])
def test_swiglu(T, K, I):
    x, w1, w3, dy = normal((T, K), 1), normal((I, K), 2, K**-0.5), normal((I, K), 3, K**-0.5), normal((T, I), 4)
    w = interleave_gate_up(w1.unsqueeze(0), w3.unsqueeze(0))[0].requires_grad_()
    leaf = x.clone().requires_grad_()
    y = fused.linear(leaf, w, activation="swiglu")
    g, u = (x.double() @ t.double().t() for t in (w1, w3))
    g.requires_grad_(), u.requires_grad_()
    a = torch.nn.functional.silu(g) * u
    want = a.detach()
    sg, su = (x.double().abs() @ t.double().abs().t() for t in (w1, w3))
    off = 1.1 * noise(K, sg) * u.detach().abs() + noise(K, su) * g.detach().abs() + 2.0**-20 * want.abs() + 2.0**-40
    assert y.shape == (T, I) and ((y.double() - want).abs() <= HALF * want.abs() + 2 * off).all()
    with torch.no_grad():
        assert torch.equal(fused.linear(x, w, activation="swiglu"), y)
    dx, dw = torch.autograd.grad(y, [leaf, w], dy)
    dg, du = torch.autograd.grad(a, [g, u], dy.double())
    ref = dg @ w1.double() + du @ w3.double()
    assert (dx.double() - ref).norm() <= 4 * HALF * ref.norm()
    ref = interleave_gate_up((dg.t() @ x.double()).unsqueeze(0), (du.t() @ x.double()).unsqueeze(0))[0]
    assert (dw.double() - ref).norm() <= 4 * HALF * ref.norm()
    assert ((dw.double() - ref).abs() <= 16 * HALF * (ref.abs() + ref.abs().mean())).all()
    gemm.check()


def test_gradient_against_differences():
    """The result is bf16, so differences are taken of the plain 64-bit formula, at a step that its own roundings allow, and the slope is the kernel's gradient."""
    T, K, N = 20, 64, 72
    for act in ("silu", "gelu", "swiglu"):
        n = 256 if act == "swiglu" else N
        x, w, dy = normal((T, K), 1), normal((n, K), 2, K**-0.5), normal((T, n // 2 if act == "swiglu" else n), 3)
        leaf = x.clone().requires_grad_()
        (g,) = torch.autograd.grad(fused.linear(leaf, w, activation=act), leaf, dy)

        def value(at):
            z = at @ w.double().t()
            if act == "swiglu":
                t = z.view(T, -1, 2, 128)
                v = (torch.nn.functional.silu(t[:, :, 0]) * t[:, :, 1]).reshape(T, -1)
            else:
                v = ACT[act](z)
            return (v * dy.double()).sum()

        d = normal((T, K), 4).double()
        slope = (value(x.double() + 1e-5 * d) - value(x.double() - 1e-5 * d)) / 2e-5
        assert abs(slope - (g.double() * d).sum()) <= 8 * HALF * (g.double() * d).norm()


def test_strides_alignment_and_shapes():
    T, K, N = 45, 136, 264
    w, b, r = whole((N, K), 2), whole((N,), 3), whole((T, N), 4)
    wide, flat = whole((T, 2 * K + 3), 5), whole((T * K + 1,), 6)
    even = whole((2 * T, 2 * K), 7)
    views = [wide[:, :K], wide[:, 3:3 + K], flat[1:].view(T, K), even[::2, 8:8 + K], whole((K, T), 8).t(), whole((1, K), 9).expand(T, K), even[:T, ::2]]
    for v in views:
        leaf = v.detach().requires_grad_()
        y = fused.linear(leaf, w, bias=b, residual=r)
        assert torch.equal(y, bf(v.double() @ w.double().t() + b.double() + r.double()))
        (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert torch.equal(g, bf(torch.ones_like(y).double() @ w.double()))
    x = views[0].contiguous()
    for other in (whole((K, N), 10).t(), whole((N, K + 8), 11)[:, :K], whole((N, K + 1), 12)[:, 1:], whole((2 * N, K), 13)[::2]):
        leaf = other.detach().requires_grad_()
        y = fused.linear(x, leaf)
        assert torch.equal(y, bf(x.double() @ other.double().t()))
        (g,) = torch.autograd.grad(y, leaf, r)
        assert torch.equal(g, bf(r.double().t() @ x.double()))
    late = whole((N + 1,), 18)[1:]         # a bias that starts between two words
    for rows in (x, x.repeat(3, 1)):
        assert torch.equal(fused.linear(rows, w, bias=late), bf(rows.double() @ w.double().t() + late.double()))
    for res in (whole((N, T), 14).t(), whole((T, N + 5), 15)[:, 5:], whole((1, N), 16).expand(T, N)):
        assert torch.equal(fused.linear(x, w, residual=res), bf(x.double() @ w.double().t() + res.double()))
    y = fused.linear(x.view(5, 9, K), w, residual=r.view(5, 9, N))
    assert y.shape == (5, 9, N) and torch.equal(y.view(T, N), fused.linear(x, w, residual=r))
    assert torch.equal(fused.linear(x[0], w), fused.linear(x[:1], w)[0])
    leaf = x.clone().requires_grad_()      # an expanded gradient, and one with rows in strides
    y = fused.linear(leaf, w)
    (g,) = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    assert torch.equal(g, bf(torch.ones(T, N, device="cuda").double() @ w.double()))
    dy = whole((T, 2 * N), 17)[:, N:]
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], bf(dy.double() @ w.double()))


def test_no_rows_and_single_gradients():
    w, b = whole((264, 136), 1).requires_grad_(), whole((264,), 2).requires_grad_()
    x = torch.empty(0, 136, device="cuda", dtype=BF, requires_grad=True)
    y = fused.linear(x, w, bias=b, activation="gelu")
    assert y.shape == (0, 264)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert gx.shape == (0, 136) and not gw.any() and not gb.any()
    x, r = whole((40, 136), 3), whole((40, 264), 4).requires_grad_()
    dy = whole((40, 264), 5)
    only = fused.linear(x, w.detach(), activation="silu", residual=r)
    assert torch.equal(torch.autograd.grad(only, r, dy)[0], dy)
    assert torch.equal(torch.autograd.grad(fused.linear(x, w.detach(), bias=b), b, dy)[0], bf(dy.double().sum(0)))
    assert torch.equal(torch.autograd.grad(fused.linear(x, w), w, dy)[0], bf(dy.double().t() @ x.double()))


def test_infinities_and_nan_stay_in_their_rows():
    x, w = whole((70, 128), 1), whole((256, 128), 2)
    clean = fused.linear(x, w)
    x[3, 5], x[40, 7] = float("nan"), float("inf")
    y = fused.linear(x, w)
    keep = torch.ones(70, dtype=torch.bool)
    keep[[3, 40]] = False
    assert torch.equal(y[keep], clean[keep]) and y[3].isnan().all() and not y[40].isfinite().all()


def test_rows_behind_the_last_stay_as_they_were():
    """The result ends inside a tile: what lies behind it in memory belongs to somebody else."""
    x, w = whole((33, 128), 1), whole((264, 128), 2)
    torch.cuda.empty_cache()
    pool = torch.full((64 * 264 * 4,), 7.0, device="cuda", dtype=BF)
    at = pool.data_ptr()
    del pool
    y = fused.linear(x, w)
    if y.data_ptr() == at:   # the allocator gave the same block back: the rest of it still holds sevens
        rest = torch.as_strided(y, (y.numel() + 31 * 264,), (1,))[y.numel():] if y.untyped_storage().nbytes() >= 2 * (y.numel() + 31 * 264) else None
        assert rest is None or (rest == 7).all()
    assert torch.equal(y, bf(x.double() @ w.double().t()))


@pytest.mark.parametrize("T", [3, 700])
def test_streams_and_graphs(T):
    K, N = 4096, 1032          # cut along the reduction: partial sums and counters of each launch
    x, w, b, r, dy = whole((T, K), 1), whole((N, K), 2), whole((N,), 3), whole((T, N), 4), whole((T, N), 5)

    def step(at):
        leaf, lw = at.detach().requires_grad_(), w.detach().requires_grad_()
        y = fused.linear(leaf, lw, bias=b, activation="relu", residual=r)
        return [y.detach(), *torch.autograd.grad(y, [leaf, lw], dy)]

    want = step(x)
    sides = [torch.cuda.Stream() for _ in range(2)]
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for side in sides:
            with torch.cuda.stream(side):
                got.append(step(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for g in got for a, c in zip(g, want))
    graphs, inputs, outs = [], [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        inputs.append(x.clone())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(inputs[-1]))
    for seed in (20, 21, 22):
        for i in range(2):
            inputs[i].copy_(whole((T, K), seed + 10 * i))
        torch.cuda.synchronize()
        for _ in range(3):                                   # both at once, on streams of their own
            for side, graph in zip(sides, graphs):
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, c) for a, c in zip(outs[i], step(inputs[i])))
    gemm.check()


def test_its_backward_has_no_gradient():
    x, w = whole((3, 64), 1).requires_grad_(), whole((72, 64), 2).requires_grad_()
    (g,) = torch.autograd.grad(fused.linear(x, w, activation="silu").float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        g.float().sum().backward()


# (tokens, reduction, columns): one, two, four and eight CTAs a tile; their sums beside the stages (up to 64 tokens a tile) and in their place; all of an SM's shared memory and
# half of it; the last part of the reduction and the last tile cut off.
FEW = [(1, 4104, 264), (16, 4096, 4736), (13, 8200, 136), (16, 4160, 1000), (17, 4104, 264), (60, 1032, 1000), (64, 520, 4744), (48, 1096, 9480), (100, 2056, 640), (128, 4104, 1288), (90, 1024, 9472),
       (250, 1104, 2056), (500, 1032, 1000), (400, 200, 9480), (600, 528, 4104), (1000, 128, 4096), (1100, 264, 8328), (2, 72, 40008)]


@pytest.mark.parametrize("T,K,N", FEW)
def test_whole_numbers_are_exact_however_few_tokens_are_shared_out(T, K, N):
    test_whole_numbers_are_exact(T, K, N)


@pytest.mark.parametrize("T,K,I", [(1, 4104, 256), (16, 4096, 2048), (60, 1032, 256), (64, 520, 4864), (100, 2056, 384), (128, 4104, 1152), (250, 1032, 1024), (500, 264, 2432)])
def test_swiglu_however_few_tokens_are_shared_out(T, K, I):
    test_swiglu(T, K, I)


@pytest.mark.parametrize("T,K,I", [(60, 512, 1024), (2000, 640, 512), (2000, 128, 4096), (1100, 2048, 2048)])
def test_swiglu_gradients_have_the_error_of_two_roundings(T, K, I):
    """That of dz, which both products take in bf16, and of the result. A gate and an up rounded to bf16 on the way would add a third as large: 1.2 times as much."""
    x, w1, w3, dy = normal((T, K), 1), normal((I, K), 2, K**-0.5), normal((I, K), 3, K**-0.5), normal((T, I), 4)
    w, leaf = interleave_gate_up(w1.unsqueeze(0), w3.unsqueeze(0))[0].requires_grad_(), x.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fused.linear(leaf, w, activation="swiglu"), [leaf, w], dy)
    g, u = (x.double() @ t.double().t() for t in (w1, w3))
    g.requires_grad_(), u.requires_grad_()
    dg, du = torch.autograd.grad(torch.nn.functional.silu(g) * u, [g, u], dy.double())
    rg, ru = dg.to(BF).double(), du.to(BF).double()
    both = lambda a, b: interleave_gate_up((a.t() @ x.double()).unsqueeze(0), (b.t() @ x.double()).unsqueeze(0))[0]
    for got, exact, rounded in ((dx, dg @ w1.double() + du @ w3.double(), rg @ w1.double() + ru @ w3.double()), (dw, both(dg, du), both(rg, ru))):
        # 1.05: the errors are sums of thousands of independent roundings, and gate and up keep 16 bits
        assert (got.double() - exact).norm() <= 1.05 * (rounded.to(BF).double() - exact).norm()
    gemm.check()
