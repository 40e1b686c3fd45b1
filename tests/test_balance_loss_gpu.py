"""The router's balance loss, counts and gradient against a plain implementation in 64 bits.

Tolerances: an exponential of x in fp32 is off by 2^-21 and |x| 2^-23 relative (its argument is rounded, |x| <= 40 where it matters), a sum of n
positive terms by n 2^-24 of itself; scores and sums together are held to (2^-16 + n 2^-24)."""
import pytest
import torch

from fast_b200.ops import fused

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
REL = 2.0**-16


def make(T, E, K, seed, dtype=F32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = ((torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")) * std).to(dtype)
    idx = torch.rand(T, E, generator=g, device="cuda").add(torch.linspace(0, 0.5, E, device="cuda")).topk(K, dim=-1).indices.to(torch.int32) if E >= K else None
    return logits, idx, torch.rand(T, generator=g, device="cuda") < 0.7


def plain(logits, idx, mask, scores, dloss):
    """Loss, counts, gradient and what the gradient's terms add up to in magnitude, from the formulas."""
    l = logits.double().clone()
    l[l.isnan()] = float("-inf")
    T, E = l.shape
    K = idx.shape[1]
    live = torch.ones(T, device="cuda", dtype=torch.bool) if mask is None else mask
    counts = torch.zeros(E, dtype=torch.int64, device="cuda")
    chosen = idx[live].reshape(-1).long()
    counts += torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)[:E]
    if scores == "softmax":
        top = l.amax(-1, keepdim=True)
        e = torch.where(top == float("inf"), (l == float("inf")).double(), torch.exp(l - torch.where(top.isinf(), 0.0, top)))
        total = e.sum(-1, keepdim=True)
        s = torch.where(total > 0, e / total, 0.0)
        slope = s
    else:
        sig = torch.sigmoid(l)
        total = sig.sum(-1, keepdim=True)
        s = torch.where(total > 0, sig / total, 0.0)
        slope = torch.where(total > 0, sig * torch.sigmoid(-l) / total, 0.0)
    n = max(int(live.sum()), 1)
    s, slope = s * live.unsqueeze(1), slope * live.unsqueeze(1)
    loss = E / (K * n * n) * (counts.double() * s.sum(0)).sum()
    c = counts.double() - counts.double().mean()
    d = dloss * E / (K * n * n) * slope * (c - (s * c).sum(-1, keepdim=True))
    size = dloss * E / (K * n * n) * slope * (c.abs() + (s * c.abs()).sum(-1, keepdim=True))
    return loss, counts, d, size


def check(logits, idx, mask, scores, dloss=1.5):
    T = logits.shape[0]
    want, counts, d, size = plain(logits.detach(), idx, mask, scores, dloss)
    leaf = logits.detach().requires_grad_()
    loss, got = fused.balance_loss(leaf, idx, mask=mask, scores=scores)
    assert loss.shape == () and loss.dtype == F32 and got.dtype == torch.int32 and torch.equal(got.long(), counts)
    assert abs(loss.double() - want) <= (REL + T * 2.0**-24) * want, (loss.item(), want.item())
    with torch.no_grad():
        again, cnt = fused.balance_loss(logits, idx, mask=mask, scores=scores)
    assert torch.equal(again, loss) and torch.equal(cnt, got)
    (g,) = torch.autograd.grad(loss, leaf, torch.tensor(dloss, device="cuda"))
    half = torch.finfo(logits.dtype).eps / 2
    assert g.dtype == logits.dtype and g.shape == logits.shape
    # 2^-126 and 2^-133: what a type cannot hold
    assert ((g.double() - d).abs() <= half * d.abs() + REL * size + 2.0**-125).all(), ((g.double() - d).abs() - REL * size).max().item()
    return loss, got, g


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 2, 1), (3, 3, 2), (7, 5, 5), (61, 64, 6), (129, 8, 2), (513, 9, 3), (1000, 33, 4), (2049, 16, 2), (300, 256, 8), (5000, 256, 8), (700, 257, 8),
                                   (513, 1000, 8), (130, 1024, 32), (20011, 8, 2)])
def test_loss_counts_and_gradient(T, E, K, dtype, scores):
    logits, idx, mask = make(T, E, K, T + E, dtype)
    check(logits, idx, None, scores)
    check(logits, idx, mask, scores)


def test_even_routing_is_one_and_has_no_gradient():
    T, E, K = 4096, 8, 2
    idx = (torch.arange(T * K, device="cuda") % E).view(T, K).to(torch.int32)
    loss, counts, g = check(torch.randn(T, E, device="cuda"), idx, None, "softmax")
    assert (counts == T * K // E).all() and not g.any()
    assert abs(fused.balance_loss(torch.zeros(T, E, device="cuda"), idx)[0].item() - 1) <= REL


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [6, 64, 300])
def test_masked_experts_infinities_and_nan(E, scores):
    logits, idx, mask = make(200, E, 2, 5)
    logits[0] = float("-inf")
    logits[1, ::2] = float("-inf")
    logits[2] = torch.finfo(F32).min
    logits[3, 1::2] = torch.finfo(F32).min
    logits[4, 3] = float("inf")
    logits[5, 2:5] = float("inf")
    logits[6, 4] = float("nan")
    logits[7] = float("nan")
    logits[8] = 80.0
    logits[9] = -80.0
    idx[10, 0], idx[11, 1], idx[12] = -1, E, 3          # out of range, and the same expert twice
    _, _, g = check(logits, idx, None, scores)
    assert g.isfinite().all()
    logits[~mask] = float("nan")                          # padding may hold anything
    _, _, g = check(logits, idx, mask, scores)
    assert not g[~mask].any()
    none = torch.zeros_like(mask)
    loss, counts, g = check(logits, idx, none, scores)
    assert loss.item() == 0 and not counts.any() and not g.any()


def test_no_tokens():
    leaf = torch.empty(0, 8, device="cuda", requires_grad=True)
    loss, counts = fused.balance_loss(leaf, torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert loss.item() == 0 and not counts.any()
    assert torch.autograd.grad(loss, leaf)[0].shape == (0, 8)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides_and_shapes(dtype):
    logits, idx, mask = make(120, 24, 3, 9, dtype)
    loss, counts, g = check(logits, idx, mask, "softmax")
    wide = torch.full((120, 31), float("nan"), device="cuda", dtype=dtype)
    wide[:, 5:29] = logits
    for view in (wide[:, 5:29], logits.t().contiguous().t(), logits.view(5, 24, 24)):
        lead = view.shape[:-1]
        leaf = view.detach().requires_grad_()
        other_idx = torch.stack([idx, idx], -1)[..., 0].view(*lead, 3)
        other, cnt = fused.balance_loss(leaf, other_idx, mask=torch.stack([mask, mask], -1)[..., 0].view(*lead))
        assert torch.equal(other, loss) and torch.equal(cnt, counts)
        (d,) = torch.autograd.grad(other, leaf, torch.tensor(1.5, device="cuda"))
        assert torch.equal(d.reshape(120, 24), g)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_gradient_against_differences(scores):
    logits, idx, _ = make(40, 12, 2, 3)
    d, step = torch.randn(40, 12, device="cuda"), 2.0**-6
    leaf = logits.detach().requires_grad_()
    loss, _ = fused.balance_loss(leaf, idx, scores=scores)
    (g,) = torch.autograd.grad(loss, leaf)
    up, down = (fused.balance_loss(logits + s * step * d, idx, scores=scores)[0].double() for s in (1, -1))
    slope, want = (up - down) / (2 * step), (g.double() * d.double()).sum()
    # a loss of about one: its third derivative (a token's share, at most 1 / 40 of it, times d^3, added over the tokens) times step^2, and rounding by the step
    assert abs(slope - want) <= 8 * step**2 * d.abs().max().item() ** 3 + 2 * REL / step * 2.0**-4, (slope.item(), want.item())


def test_offsets_past_32_bits():
    T, E = 2200000, 1000
    logits = torch.zeros(T, E, device="cuda", dtype=BF)   # 2.2e9 elements
    logits[-1] = torch.arange(E, device="cuda").to(BF) / 100
    idx = torch.full((T, 1), 7, dtype=torch.int32, device="cuda")
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    mask[-1] = True
    leaf = logits.requires_grad_()
    loss, counts = fused.balance_loss(leaf, idx, mask=mask)
    want, cnt, d, size = plain(logits[-1:].detach(), idx[-1:], None, "softmax", 1.0)
    assert torch.equal(counts.long(), cnt) and abs(loss.double() - want) <= REL * want
    (g,) = torch.autograd.grad(loss, leaf)
    assert ((g[-1:].double() - d).abs() <= 2.0**-8 * d.abs() + REL * size + 2.0**-125).all() and not g[-1000000:-1].any()


def test_captured_and_replayed_and_on_another_stream():
    logits, idx, mask = make(3000, 64, 6, 2)

    def step(l):
        leaf = l.detach().requires_grad_()
        loss, counts = fused.balance_loss(leaf, idx, mask=mask)
        return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step(logits)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, step(logits)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(logits)
    for seed in (20, 21):
        logits.copy_(make(3000, 64, 6, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(logits)))


def test_its_backward_has_no_gradient():
    logits, idx, _ = make(10, 8, 2, 1)
    leaf = logits.requires_grad_()
    (g,) = torch.autograd.grad(fused.balance_loss(leaf, idx)[0], leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        g.sum().backward()


def test_counts_and_inputs_may_change_before_the_backward_pass():
    """The counts are the caller's (summed over ranks in place, say); so are the choices. Logits that change are noticed."""
    logits, idx, _ = make(500, 16, 2, 1)
    leaf = logits.detach().requires_grad_()
    (want,) = torch.autograd.grad(fused.balance_loss(leaf, idx)[0], leaf)
    loss, counts = fused.balance_loss(leaf, idx)
    counts.mul_(8)
    idx.zero_()
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
    moved = leaf * 1.0
    loss, _ = fused.balance_loss(moved, idx)
    moved.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
