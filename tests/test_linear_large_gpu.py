"""Linear layers whose results have more elements than 32 bits count."""
import pytest
import torch

from fast_b200.models.moe import interleave_gate_up
from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def whole(shape, seed, most=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda", dtype=torch.int8).to(BF)


def parts(T):
    """Rows at both ends, around 2^31 / 520 and 2^32 / 1040, and in between."""
    at = torch.tensor([0, T // 2, 4129776 - 20, T - 40], device="cuda")
    return (at.unsqueeze(1) + torch.arange(40, device="cuda")).reshape(-1).clamp(max=T - 1).unique()


def test_results_and_gradients_past_32_bits():
    T, K, N = (1 << 22) + 5, 8, 520      # 2.2e9 elements
    x, w, b = whole((T, K), 1).requires_grad_(), whole((N, K), 2).requires_grad_(), whole((N,), 3).requires_grad_()
    r, dy = whole((T, N), 4).requires_grad_(), whole((T, N), 5, 1)
    y = fused.linear(x, w, bias=b, activation="relu", residual=r)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], dy)
    gemm.check()
    i = parts(T)
    z = x[i].detach().double() @ w.detach().double().t() + b.detach().double()
    assert torch.equal(y[i], (torch.relu(z) + r[i].detach().double()).to(BF))
    assert torch.equal(dx[i], ((dy[i].double() * (z > 0)) @ w.detach().double()).to(BF)) and dr.data_ptr() == dy.data_ptr()
    # every row has a part in these two; sums of 2^22 whole numbers up to 2, exact in fp32 where they stay below 2^24 (blocks of rows, added up in turn)
    want_w, want_b = torch.zeros(N, K, device="cuda", dtype=torch.float64), torch.zeros(N, device="cuda", dtype=torch.float64)
    for a in range(0, T, 1 << 19):
        rows = slice(a, min(a + (1 << 19), T))
        xd = x[rows].detach().double()
        dz = dy[rows].double() * (xd @ w.detach().double().t() + b.detach().double() > 0)
        want_w += dz.t() @ xd
        want_b += dz.sum(0)
    assert want_w.abs().max() < 1 << 24 and want_b.abs().max() < 1 << 24
    assert torch.equal(dw, want_w.to(BF)) and torch.equal(db, want_b.to(BF))


def test_swiglu_keeps_more_than_32_bits_count():
    T, K, I = 1 << 21, 8, 256            # gate and up, twice 16 bits each: 2.1e9 elements
    w = interleave_gate_up(whole((1, I, K), 2), whole((1, I, K), 3))[0].requires_grad_()
    x, dy = whole((T, K), 1).requires_grad_(), whole((T, I), 4, 1)
    y = fused.linear(x, w, activation="swiglu")
    (dx,) = torch.autograd.grad(y, x, dy)
    gemm.check()
    i = torch.cat([torch.arange(50, device="cuda"), torch.arange(T - 50, T, device="cuda")])
    small, leaf = fused.linear(x[i].detach(), w.detach(), activation="swiglu"), x[i].detach().requires_grad_()
    assert torch.equal(y[i], small)
    assert torch.equal(dx[i], torch.autograd.grad(fused.linear(leaf, w.detach(), activation="swiglu"), leaf, dy[i])[0])
