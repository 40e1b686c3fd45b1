"""Linear layers whose tiles are cut along the reduction: sums in scratch memory and counters that belong to one launch. And which way a shape goes, asked of the rules themselves."""
import pytest
import torch

from fast_b200 import runtime
from fast_b200.models.moe import interleave_gate_up
from fast_b200.ops import fused, gemm

BF = torch.bfloat16
# tokens, inputs, outputs: forward cut as a stream of shares (one token tile) and in parts, by 2, 3 and 4 pairs a tile, for several widths of a tile
STREAM = [(100, 8192, 20000, 128), (181, 7304, 4840, 256)]
PARTS = [(781, 7256, 1368, 160), (1552, 6864, 3496, 256), (1552, 7448, 2832, 256)]
SWIGLU = [(129, 7512, 4864, 256), (972, 7256, 1280, 160), (524, 8008, 2048, 256)]


def path(tokens, reduction, features, swiglu=False, plain=False, sectors=True):
    return runtime.ext().dense_path(tokens, features, reduction, swiglu, plain, sectors)


def test_the_shapes_below_are_cut():
    for T, K, N, tile in STREAM + PARTS:
        p = path(T, K, N)
        assert not p["few"] and p["tile"] == tile and p["cut_tiles"] > 0 and p["stream"] == ((T, K, N, tile) in STREAM), (T, K, N, p)
        q = path(T, K, N, sectors=False)
        assert not q["few"]
    assert {path(T, K, N)["shares"] for T, K, N, _ in PARTS} == {2, 3, 4}
    for T, K, N, tile in SWIGLU:
        p = path(T, K, N, swiglu=True)
        assert not p["few"] and p["tile"] == tile and p["cut_tiles"] > 0, (T, K, N, p)
    wide = path(8200, 8200, 3432, plain=True)
    assert wide["tile"] == 512 and wide["cut_tiles"] > 0 and path(8200, 8200, 3432)["tile"] == 256


def test_up_to_64_tokens_are_always_few():
    for T in (1, 33, 64):
        for K in (8, 4096, 1 << 20):
            for N in (8, 4096, 1 << 24):
                assert path(T, K, N)["few"] and path(T, K, N, sectors=False)["few"]


def whole(shape, seed, most=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda", dtype=torch.int8).to(BF)


def _exact(T, K, N, act, bias, residual):
    x, w, b, r = whole((T, K), 1), whole((N, K), 2), whole((N,), 3, 9), whole((T, N), 4, 9)
    z = (x.double() @ w.double().t()) + (b.double() if bias else 0)
    want = ((torch.relu(z) if act else z) + (r.double() if residual else 0)).to(BF)
    return x, w, b if bias else None, r if residual else None, z, want


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,tile", STREAM + PARTS + [(8200, 8200, 3432, 512)])
@pytest.mark.parametrize("act,bias,residual", [("relu", True, True), (None, False, False), (None, True, True)])
def test_cut_products_are_exact(T, K, N, tile, act, bias, residual):
    """Whole numbers: every sum is exact whatever its order. Forward with what a backward pass keeps and without, and the gradients."""
    x, w, b, r, z, want = _exact(T, K, N, act, bias, residual)
    lx, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fused.linear(lx, lw, bias=b, activation=act, residual=r)
    assert torch.equal(y, want)
    with torch.no_grad():
        assert torch.equal(fused.linear(x, w, bias=b, activation=act, residual=r), want)
    dy = whole((T, N), 5)
    dx, dw = torch.autograd.grad(y, [lx, lw], dy)
    dz = dy.double() * (z > 0) if act else dy.double()
    assert torch.equal(dx, (dz @ w.double()).to(BF)) and torch.equal(dw, (dz.t() @ x.double()).to(BF))
    gemm.check()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,tile", STREAM + PARTS)
def test_cut_data_gradients_are_exact(T, K, N, tile):
    """The same shapes the other way round: the data gradient reduces over the outputs."""
    x, w, dy = whole((T, N), 1), whole((K, N), 2), whole((T, K), 3)
    p = path(T, K, N, plain=True)
    assert not p["few"] and p["cut_tiles"] > 0
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(fused.linear(leaf, w), leaf, dy)
    assert torch.equal(dx, (dy.double() @ w.double()).to(BF))
    gemm.check()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,tile", SWIGLU)
def test_cut_swiglu_is_what_uncut_tiles_give(T, K, N, tile):
    """Whole numbers: gate and up are exact either way, and so everything behind them is the same: a cut launch and, token by token, launches of few tokens."""
    I = N // 2
    w = interleave_gate_up(whole((1, I, K), 2, 1), whole((1, I, K), 3, 1))[0]
    x = whole((T, K), 1, 1)
    leaf, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fused.linear(leaf, lw, activation="swiglu")
    z = (x.double() @ w.double().t()).view(T, -1, 2, 128)
    exact = (torch.nn.functional.silu(z[:, :, 0]) * z[:, :, 1]).reshape(T, I)
    # the exponential's argument, up to 128 there, is rounded by 2^-24 of itself; a few roundings more: 2^-15
    assert ((y.double() - exact).abs() <= (2.0**-8 + 2.0**-15) * exact.abs() + 2.0**-100).all()
    with torch.no_grad():
        assert torch.equal(fused.linear(x, w, activation="swiglu"), y)
        assert path(64, K, N, swiglu=True)["few"]
        few = torch.cat([fused.linear(x[i:i + 64], w, activation="swiglu") for i in range(0, T, 64)])
    assert torch.equal(few, y)
    dy = whole((T, I), 4)
    dx, dw = torch.autograd.grad(y, [leaf, lw], dy)
    zz = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad((torch.nn.functional.silu(zz[:, :, 0]) * zz[:, :, 1]).reshape(T, I), zz, dy.double())
    dz = dz.reshape(T, N)
    for got, ref in ((dx, dz @ w.double()), (dw, dz.t() @ x.double())):
        assert (got.double() - ref).norm() <= 4 * 2.0**-8 * ref.norm()
    gemm.check()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,kind", [(100, 8192, 20000, "linear"), (1552, 7448, 2832, "linear"), (129, 7512, 4864, "swiglu"), (524, 8008, 2048, "swiglu"), (8200, 8200, 3432, "plain")])
def test_cut_launches_on_streams_and_in_graphs(T, K, N, kind):
    """Several at once: every launch has scratch and counters of its own, a graph those that it was captured with."""
    p = path(T, K, N, swiglu=kind == "swiglu", plain=kind == "plain")
    assert not p["few"] and p["cut_tiles"] > 0
    w, b = whole((N, K), 2, 1), whole((N,), 3)

    def run(x):
        if kind == "plain":
            return fused.linear(x, w)
        return fused.linear(x, w, activation="swiglu") if kind == "swiglu" else fused.linear(x, w, bias=b, activation="relu")

    xs = [whole((T, K), 10 + i, 1) for i in range(2)]
    with torch.no_grad():
        want = [run(x) for x in xs]
        assert not torch.equal(*want)
        sides = [torch.cuda.Stream() for _ in xs]
        for side in sides:
            side.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(6):
            for i, side in enumerate(sides):
                with torch.cuda.stream(side):
                    got[i].append(run(xs[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])
        del got
        graphs, ins, outs = [], [], []
        for x in xs:
            graphs.append(torch.cuda.CUDAGraph())
            ins.append(torch.empty_like(x))
            with torch.cuda.graph(graphs[-1]):
                outs.append(run(ins[-1]))
        for turn in range(3):
            for i in range(2):
                ins[i].copy_(xs[(i + turn) % 2])
            torch.cuda.synchronize()
            for _ in range(3):
                for side, graph in zip(sides, graphs):
                    with torch.cuda.stream(side):
                        graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(outs[i], want[(i + turn) % 2]) for i in range(2))
    gemm.check()
