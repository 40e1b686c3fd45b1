"""The dense operators read memory through pointers: what has no memory of its own is refused before anything runs, and gradients that are no memory yet are made it."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from fast_b200.ops import fused

BF = torch.bfloat16


def _calls(make):
    """Every tensor argument of every operator in turn: a call with `make` of that one."""
    shapes = {"x": (4, 64), "w": (256, 64), "b": (256,), "r": (4, 256), "nw": (64,), "nr": (4, 64)}

    def args(**other):
        t = {k: torch.ones(s, dtype=BF) for k, s in shapes.items()}
        t.update(logits=torch.ones(4, 8), idx=torch.zeros(4, 2, dtype=torch.int32), mask=torch.ones(4, dtype=torch.bool), q=torch.zeros(4, 128, dtype=torch.uint8), s=torch.ones(4, 1))
        for k in other:
            t[k] = make(t[k])
        return t

    runs = {
        "linear": (lambda t: fused.linear(t["x"], t["w"], bias=t["b"], residual=t["r"]), "xwbr"),
        "norm": (lambda t: fused.add_rms_norm(t["x"], t["nw"], residual=t["nr"]), ("x", "nw", "nr")),
        "balance": (lambda t: fused.balance_loss(t["logits"], t["idx"], mask=t["mask"]), ("logits", "idx", "mask")),
        "dequantise": (lambda t: fused.dequantise_rows(t["q"], t["s"]), "qs"),
    }
    for name, (run, keys) in runs.items():
        for key in keys:
            yield f"{name} {key}", lambda run=run, key=key: run(args(**{key: True}))


def _fake(t):
    with FakeTensorMode() as mode:
        return mode.from_tensor(t)


def test_fake_zero_and_negated_tensors_are_refused():
    # integers have no negated views, and truth values neither
    for make, skip in ((_fake, ()), (lambda t: torch._efficientzerotensor(t.shape, dtype=t.dtype), ()), (lambda t: torch._neg_view(t), ("mask",)), (lambda t: t.to_sparse(), ())):
        for name, call in _calls(make):
            if name.split()[1] in skip:
                continue
            with pytest.raises(RuntimeError, match="plain memory"):
                call()


def test_fake_tensors_of_the_device_are_refused():
    with FakeTensorMode():
        x, w = torch.empty(4, 64, device="cuda", dtype=BF), torch.empty(16, 64, device="cuda", dtype=BF)
        for call in (lambda: fused.linear(x, w), lambda: fused.linear(x[:0], w), lambda: fused.add_rms_norm(x, w[0]), lambda: fused.balance_loss(x, torch.empty(4, 1, device="cuda", dtype=torch.int32)),
                     lambda: fused.dequantise_rows(torch.empty(4, 128, device="cuda", dtype=torch.uint8), torch.empty(4, 1, device="cuda"))):
            with pytest.raises(RuntimeError, match="plain memory"):
                call()


def test_functional_transforms_are_refused():
    x, w = torch.ones(4, 64), torch.ones(16, 64)
    for transform in (lambda f: torch.func.grad(lambda v: f(v).sum())(x), lambda f: torch.func.vmap(f)(x.unsqueeze(0)), lambda f: torch.func.jvp(f, (x,), (x,))):
        with pytest.raises(RuntimeError, match="plain memory"):
            transform(lambda v: fused.linear(v, w))


def _t(*shape, seed=1, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _training(op):
    """(leaves, their results) of an operator that trains."""
    if op == "norm":
        leaves = [_t(5, 256, seed=s).requires_grad_() for s in (1, 2)] + [_t(256, seed=3).requires_grad_()]
        r = fused.add_rms_norm(leaves[0], leaves[2], residual=leaves[1])
        return leaves, [r.y, r.h]
    if op == "balance":
        leaf = _t(40, 8, dtype=torch.float32).requires_grad_()
        idx = torch.arange(40, device="cuda", dtype=torch.int32).remainder(5).view(40, 1)
        return [leaf], [fused.balance_loss(leaf, idx, mask=torch.arange(40, device="cuda") > 3)[0]]
    leaves = [_t(5, 64, seed=1).requires_grad_(), _t(256, 64, seed=2).requires_grad_()]
    if op == "swiglu":
        return leaves, [fused.linear(*leaves, activation="swiglu")]
    leaves += [_t(256, seed=3).requires_grad_(), _t(5, 256, seed=4).requires_grad_()]
    return leaves, [fused.linear(leaves[0], leaves[1], bias=leaves[2], activation=op, residual=leaves[3])]


OPS = ["norm", "balance", "swiglu", "silu", None]


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_zero_and_negated_gradients(op):
    leaves, outs = _training(op)
    real = [torch.full_like(o, 0.5) for o in outs]
    zeros = torch.autograd.grad(outs, leaves, [torch._efficientzerotensor(o.shape, dtype=o.dtype, device=o.device) for o in outs], retain_graph=True)
    assert all(not z.any() for z in zeros)
    negated = torch.autograd.grad(outs, leaves, [torch._neg_view(-g) for g in real], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(negated, torch.autograd.grad(outs, leaves, real)))


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("change", ["host", "type", "size"])
def test_saved_tensors_that_come_back_otherwise_are_refused(op, change):
    back = {"host": lambda t: t.cpu(), "type": lambda t: t.double(), "size": lambda t: t.reshape(-1)[:1].contiguous()}[change]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        leaves, outs = _training(op)
    with pytest.raises(RuntimeError, match="saved tensor|gradient of y"):
        torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):      # and those that come back as they were are not
        leaves, outs = _training(op)
    got = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
    leaves, outs = _training(op)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])))


@pytest.mark.gpu
def test_one_token_without_other_dimensions():
    logits, idx = _t(8, dtype=torch.float32), torch.tensor([1, 3], device="cuda", dtype=torch.int32)
    for live in (True, False):
        mask = torch.tensor(live, device="cuda")
        leaf, rows = logits.clone().requires_grad_(), logits.view(1, 8).clone().requires_grad_()
        (a, ca), (b, cb) = fused.balance_loss(leaf, idx, mask=mask), fused.balance_loss(rows, idx.view(1, 2), mask=mask.view(1))
        assert torch.equal(a, b) and torch.equal(ca, cb)
        assert torch.equal(torch.autograd.grad(a, leaf)[0], torch.autograd.grad(b, rows)[0].view(8))
    x, w = _t(256).requires_grad_(), _t(256, seed=2).requires_grad_()
    grads = torch.autograd.grad(fused.add_rms_norm(x, w).y, [x, w], torch.ones(256, device="cuda", dtype=BF))
    assert all(g.shape == (256,) and g.isfinite().all() for g in grads)
    lw = _t(264, 256, seed=3).requires_grad_()
    for act in (None, "gelu"):
        gx, gw = torch.autograd.grad(fused.linear(x, lw, activation=act), [x, lw], torch.ones(264, device="cuda", dtype=BF))
        assert gx.shape == (256,) and gw.shape == (264, 256) and gw.isfinite().all()
