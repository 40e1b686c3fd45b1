"""gelu of a linear layer, value by value: z Phi(z) and its derivative rounded once, far negative values too.

The products are exact here (one weight of 1 a row), so z is the input. Tolerances: half a step of bf16 for the rounding; relative to the value, for the fit of the tail 2^-17.8, for
the exponential's argument, which is rounded twice, 2 * 128 * 2^-24 = 2^-16, a few fp32 roundings: 2^-15 together; and what no normal number of bf16 holds, 2^-126. The exponential itself ends there as well (fp32 without subnormals): what is lost of it, up to 2^-126, is multiplied
by z and q < 0.5 in the value, 13.5 * 0.5 / (1 + 0.3 * 13.5) < 2, and by |z| / sqrt(2 pi) + q < 13.5 * 0.399 + 0.5 < 6 in the derivative."""
import pytest
import torch

from fast_b200.ops import fused, gemm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF, REL, TINY = 2.0**-8, 2.0**-15, 2.0**-126


@pytest.mark.parametrize("N", [8, 2056])   # tiles of few tokens, and tiles of 256 features (thousands of rows)
def test_every_value_is_rounded_once(N):
    z = torch.cat([torch.linspace(-13.5, 13.5, 8000, device="cuda").to(BF), torch.logspace(-30, 0, 500, device="cuda").to(BF), -torch.logspace(-30, 0, 500, device="cuda").to(BF)])
    x, w = torch.zeros(z.numel(), 8, device="cuda", dtype=BF), torch.zeros(N, 8, device="cuda", dtype=BF)
    x[:, 0], w[:, 0] = z, 1
    leaf = x.requires_grad_()
    y = fused.linear(leaf, w, activation="gelu")
    d = z.double()
    phi, density = 0.5 * torch.special.erfc(-d / 2**0.5), torch.exp(-0.5 * d * d) / (2 * torch.pi) ** 0.5
    want = d * phi
    assert torch.equal(y, y[:, :1].expand_as(y))
    off = (y[:, 0].double() - want).abs()
    assert (off <= (HALF + REL) * want.abs() + 3 * TINY).all(), (off / want.abs()).max().item()
    dy = torch.zeros_like(y)
    dy[:, N - 1] = 1
    (g,) = torch.autograd.grad(y, leaf, dy)
    slope = phi + d * density
    assert ((g[:, 0].double() - slope).abs() <= HALF * slope.abs() + REL * (phi + d.abs() * density) + 7 * TINY).all()
    gemm.check()
