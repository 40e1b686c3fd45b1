"""Linear layers on rows with infinities and NaN, and on weights with them, under every activation: what diverged must not come out healthy."""
import pytest
import torch

from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ACT = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}
SHAPES = [(5, 128, 264), (70, 128, 256), (300, 512, 20000)]   # few tokens to a tile of the weight (one and several tokens tiles), and tiles of 256 features


def whole(shape, seed, most=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(1, most + 1, shape, generator=g, device="cuda") * (1 - 2 * torch.randint(0, 2, shape, generator=g, device="cuda"))
    return v.to(BF)   # no zeros: an infinity times a zero would be NaN


def same_kind(y, want):
    w = want.to(BF)
    return torch.equal(y.isnan(), w.isnan()) and torch.equal(y.isposinf(), w.isposinf()) and torch.equal(y.isneginf(), w.isneginf())


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", None])
@pytest.mark.parametrize("T,K,N", SHAPES)
def test_rows_with_infinities_and_nan(T, K, N, act):
    x, w, b, dy = whole((T, K), 1), whole((N, K), 2), whole((N,), 3), whole((T, N), 4)

    def step(at):
        leaves = [t.clone().requires_grad_() for t in (at, w, b)]
        y = fused.linear(leaves[0], leaves[1], bias=leaves[2], activation=act)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    clean = step(x)
    assert all(t.isfinite().all() for t in clean)
    x[1, 5], x[3, 7] = float("nan"), float("inf")
    got = step(x)
    with torch.no_grad():
        assert same_kind(fused.linear(x, w, bias=b, activation=act), got[0])
    keep = torch.ones(T, dtype=torch.bool)
    keep[[1, 3]] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
    z = x.double() @ w.double().t() + b.double()
    assert z[1].isnan().all() and z[3].isinf().all()
    assert same_kind(got[0], ACT[act](z)) and got[0][1].isnan().all()
    if act is None:
        assert torch.equal(got[1], clean[1]) and torch.equal(got[3], clean[3])   # these gradients do not know x
    else:
        assert got[1][1].isnan().all() and got[3].isnan().all()
    assert got[2][:, 5].isnan().all()
    gemm.check()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", None])
@pytest.mark.parametrize("T,K,N", SHAPES)
def test_a_row_of_the_weight_with_nan(T, K, N, act):
    x, w, dy = whole((T, K), 1), whole((N, K), 2), whole((T, N), 4)
    clean = fused.linear(x, w, activation=act)
    w[9, 3] = float("nan")
    leaf, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = fused.linear(leaf, lw, activation=act)
    keep = torch.arange(N) != 9
    assert y[:, 9].isnan().all() and torch.equal(y[:, keep], clean[:, keep])
    dx, dw = torch.autograd.grad(y, [leaf, lw], dy)
    assert dx[:, 3].isnan().all() and dw[9].isnan().all() == (act is not None) and dw[keep].isfinite().all()
    gemm.check()


@pytest.mark.parametrize("T,K,I", [(5, 128, 256), (300, 512, 10240)])
def test_swiglu_on_rows_with_infinities_and_nan(T, K, I):
    x, w = whole((T, K), 1), whole((2 * I, K), 2)
    clean = fused.linear(x, w, activation="swiglu")
    x[1, 5], x[3, 7] = float("nan"), float("inf")
    keep = torch.ones(T, dtype=torch.bool)
    keep[[1, 3]] = False
    leaf = x.clone().requires_grad_()
    y = fused.linear(leaf, w, activation="swiglu")
    z = (x.double() @ w.double().t()).view(T, -1, 2, 128)
    assert torch.equal(y[keep], clean[keep]) and same_kind(y, (torch.nn.functional.silu(z[:, :, 0]) * z[:, :, 1]).reshape(T, I))
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert g[1].isnan().all() and g[keep].isfinite().all()
    gemm.check()
