"""The dense operators as the MoE layer and the block model use them, in a run together: residual sum and norm, routing, the balance loss, routed experts, the
shared expert on top, backward through all of it; forward-only layers with e4m3 rows, eager and captured."""
import pytest
import torch

from tests.test_moe_gpu import _ref_forward, _rel

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _layer(E, K, H, I, **kw):
    from fast_b200.models import MoELayer
    from fast_b200.parallel import Communicator

    comm = Communicator(heap_bytes=512 << 20, device=0)
    return comm, MoELayer(comm, H, I, E, K, max_tokens=1024, **kw)


def _randn(seed, *shape, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


def _shared(x, w13, w2):
    t = (x @ w13.t()).view(x.shape[0], -1, 2, 128)
    return (torch.nn.functional.silu(t[:, :, 0]) * t[:, :, 1]).reshape(x.shape[0], -1) @ w2.t()


def _balance(logits, idx, scores, mask):
    p = torch.softmax(logits, -1) if scores == "softmax" else torch.sigmoid(logits) / torch.sigmoid(logits).sum(-1, keepdim=True)
    keep = torch.ones(logits.shape[0], dtype=torch.bool, device="cuda") if mask is None else mask
    counts = torch.bincount(idx[keep].reshape(-1).long(), minlength=logits.shape[1]).float()
    n = keep.sum()
    return logits.shape[1] / (idx.shape[1] * n * n) * (counts * p[keep].sum(0)).sum(), counts


@pytest.mark.parametrize("E,K,T,scores,shared,add,masked", [(8, 2, 500, "softmax", 0, False, False), (8, 2, 500, "softmax", 256, True, True), (32, 6, 300, "sigmoid", 128, True, False),
                                                           (64, 4, 300, "softmax", 256, True, True), (64, 4, 300, "sigmoid", 0, False, True)])
def test_training_layer_with_balance_and_shared_expert(E, K, T, scores, shared, add, masked):
    """Up to 32 experts the router is fused with the norm, above it is not; gradients of everything against autograd in fp32."""
    H, I, eps, coef = 512, 256, 1e-5, 300.0   # the coefficient makes the balance loss's gradient as large as the others
    comm, layer = _layer(E, K, H, I, balance=scores, shared_inter=shared)
    h, more, nw = _randn(1, T, H), _randn(2, T, H), (1 + _randn(3, H, std=0.1).float()).to(BF)
    gout, gsum = _randn(4, T, H), _randn(5, T, H)
    mask = torch.arange(T, device="cuda") % 5 != 0 if masked else None
    leaves = [t.clone().requires_grad_() for t in ([h, nw, more] if add else [h, nw])]
    for _ in range(2):                        # the second step uses the buffers again
        layer.zero_grad()
        for t in leaves:
            t.grad = None
        out = layer.forward_from_residual(leaves[0], leaves[1], eps, add=leaves[2] if add else None, mask=mask)
        out, total = out if add else (out, None)
        loss = (out.float() * gout.float()).sum() + coef * layer.balance_loss
        if add:
            loss = loss + (total.float() * gsum.float()).sum()
        loss.backward()
    comm.check()
    idx = layer.last_route.topk_idx.long()
    ref = {k: v.detach().float().requires_grad_() for k, v in dict(layer.named_parameters()).items()}
    rl = [t.detach().float().requires_grad_() for t in leaves]
    s = rl[0] + rl[2] if add else rl[0]
    hn = s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + eps) * rl[1]
    want, _, _ = _ref_forward(hn, ref["gate"], ref["w13"], ref["w2"], K, idx=idx)
    if shared:
        want = want + _shared(hn, ref["shared_w13"], ref["shared_w2"])
    bal, counts = _balance(hn @ ref["gate"].t(), idx, scores, mask)
    assert _rel(out, want) < 2e-2
    assert abs(layer.balance_loss.item() - bal.item()) < 1e-2 * bal.item() and torch.equal(layer.expert_counts.float(), counts)
    if add:
        assert _rel(total, s) < 1e-2
    rloss = (want * gout.float()).sum() + coef * bal
    (rloss + (s * gsum.float()).sum() if add else rloss).backward()
    for name, p in layer.named_parameters():
        assert _rel(p.grad, ref[name].grad) < 3e-2, name
    for t, r in zip(leaves, rl):
        assert _rel(t.grad, r.grad) < 3e-2


def test_balance_gradient_alone_reaches_the_router():
    """Only the balance loss is differentiated: the experts get nothing, the router what the formula says."""
    comm, layer = _layer(8, 2, 512, 256, balance="softmax")
    h, nw = _randn(1, 400, 512).requires_grad_(), torch.ones(512, device="cuda", dtype=BF, requires_grad=True)
    layer.forward_from_residual(h, nw, 1e-5)
    (layer.balance_loss * 100).backward()
    comm.check()
    hr, gr = h.detach().float().requires_grad_(), layer.gate.detach().float().requires_grad_()
    hn = hr * torch.rsqrt(hr.pow(2).mean(-1, keepdim=True) + 1e-5)
    bal, _ = _balance(hn @ gr.t(), layer.last_route.topk_idx.long(), "softmax", None)
    (bal * 100).backward()
    assert _rel(layer.gate.grad, gr.grad) < 2e-2 and _rel(h.grad, hr.grad) < 2e-2
    assert not layer.w13.grad.any() and not layer.w2.grad.any()


def test_loss_in_the_layer_with_balance_is_the_separate_sum():
    comm, layer = _layer(8, 2, 512, 256, balance="softmax")
    plain_comm, plain = _layer(8, 2, 512, 256)
    h, nw = _randn(1, 300, 512), torch.ones(512, device="cuda", dtype=BF)
    a, b = h.clone().requires_grad_(), h.clone().requires_grad_()
    loss, base = layer.mean_square_from_residual(a, nw, 1e-5), plain.mean_square_from_residual(b, nw, 1e-5)
    assert torch.equal(loss, base) and 0.9 < layer.balance_loss.item() < 8
    (ga,), (gb,) = torch.autograd.grad(loss, a, retain_graph=True), torch.autograd.grad(base, b)
    assert _rel(ga, gb) < 1e-2          # the same sum with one logit after the other in another order


@pytest.mark.parametrize("overlap,fp8", [(False, False), (True, True), (False, True)])
@pytest.mark.parametrize("T", [1, 300])
def test_forward_layer_from_the_residual_stream(T, overlap, fp8):
    from fast_b200.ops import fused

    H = 512
    comm, layer = _layer(8, 2, H, 256, fp8_dispatch=fp8, training=False, overlap_dispatch=overlap, shared_inter=256)
    layer.eval()
    h, more, nw = _randn(1, T, H), _randn(2, T, H), (1 + _randn(3, H, std=0.1).float()).to(BF)
    with torch.no_grad():
        out, total = layer.forward_from_residual(h, nw, 1e-5, add=more)
        again, _ = layer.forward_from_residual(h, nw, 1e-5, add=more)
        rows = fused.add_rms_norm(h, nw, 1e-5, residual=more)
        apart = layer(rows.y)
    comm.check()
    assert torch.equal(total, rows.h) and torch.equal(out, again) and torch.equal(out, apart)   # the rows that the dispatch would make of y
    x = rows.y.float()
    want, _, _ = _ref_forward(x, layer.gate, layer.w13, layer.w2, 2, idx=layer.last_route.topk_idx.long())
    want = want + _shared(x, layer.shared_w13.float(), layer.shared_w2.float())
    assert _rel(out, want) < (6e-2 if fp8 else 2e-2)


def test_shared_expert_in_the_captured_layer():
    comm, layer = _layer(8, 2, 512, 256, training=False, graph_mode=True, shared_inter=128)
    layer.eval()
    x = _randn(1, 64, 512)
    layer.capture(64)
    for seed in (2, 3):
        x.copy_(_randn(seed, 64, 512))
        got = layer.forward_graphed(x).clone()
        ref, _, _ = _ref_forward(x, layer.gate, layer.w13, layer.w2, 2, idx=layer.last_route.topk_idx.long())
        want = ref + _shared(x.float(), layer.shared_w13.float(), layer.shared_w2.float())
        assert _rel(got, want) < 2e-2
    comm.check()


def test_block_model_trains_with_balance_and_shared_expert():
    from fast_b200.models import MixtralBlockModel
    from fast_b200.parallel import Communicator
    from fast_b200.utils import FusedAdamW

    comm = Communicator(heap_bytes=512 << 20, device=0)
    model = MixtralBlockModel(comm, vocab=1000, hidden=512, inter=256, num_experts=8, top_k=2, max_tokens=512, balance_coef=0.01, shared_inter=256)
    params = [*model.replicated_parameters(), *model.expert_parameters()]
    assert len(params) == len(list(model.parameters()))
    opt = FusedAdamW(params, lr=1e-3)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 1000, (512,), generator=g, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        loss = model(ids)
        loss.backward()
        assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() for p in params)
        opt.step()
    assert model.moe.expert_counts.sum().item() == 512 * 2
    comm.check()


def test_layer_options_that_are_refused():
    from fast_b200.models import MoELayer

    for kw in ({"balance": "l2"}, {"shared_inter": 100}, {"shared_inter": -128}):
        with pytest.raises(ValueError):
            MoELayer(None, 512, 256, 8, 2, 64, **kw)


@pytest.mark.parametrize("E,K,shared", [(8, 2, 0), (8, 2, 128), (64, 4, 0)])
def test_a_pass_that_nothing_was_made_of_is_let_go_before_the_next(E, K, shared):
    """What a pass keeps for its backward pass hangs on the layer's balance loss: no second one may live beside it."""
    H, T, eps = 512, 256, 1e-5
    comm, layer = _layer(E, K, H, 256, balance="softmax", shared_inter=shared)
    h, nw = _randn(1, T, H).requires_grad_(), torch.ones(H, device="cuda", dtype=BF)
    seen = []
    for name in ("route", "route_fused"):
        def wrapped(*a, _run=getattr(layer.engine, name), **kw):
            seen.append((layer.balance_loss, layer.expert_counts))
            return _run(*a, **kw)
        setattr(layer.engine, name, wrapped)
    for run in (lambda: layer.forward_from_residual(h, nw, eps), lambda: layer.mean_square_from_residual(h, nw, eps), lambda: layer(h)):
        for _ in range(2):
            run()
            assert layer.balance_loss.requires_grad and int(layer.expert_counts.sum()) == T * K
    comm.check()
    assert seen == [(None, None)] * 6
