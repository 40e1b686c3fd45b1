"""The block model and the layer outside training: a forward-only pass has no balance loss, and shows none of an earlier batch."""
import pytest
import torch

BF = torch.bfloat16


def _stubbed(monkeypatch, **layer_fields):
    """The block model around a layer whose engine is left out: its passes give zeros, and in training a balance loss of 7."""
    from fast_b200.models.moe import MixtralBlockModel, MoELayer
    from fast_b200.ops import fused

    layer = MoELayer.__new__(MoELayer)
    torch.nn.Module.__init__(layer)
    layer.balance, layer.shared_inter, layer.router_bias = "softmax", 0, None
    layer.balance_loss = layer.expert_counts = layer.gate = layer.w13 = layer.w2 = None
    rs = type("Route", (), {"topk_w": None, "topk_idx": None})()

    class Engine:
        def can_fuse_gate(self):
            return False

        def route_and_send(self, x, gate, bias, quantised):
            return rs

        def experts_forward(self, *a, **kw):
            pass

        def combine(self, rs, w):
            return torch.zeros(4, 8)

        def route(self, logits, bias):
            return rs

    layer.engine = Engine()
    model = MixtralBlockModel.__new__(MixtralBlockModel)
    torch.nn.Module.__init__(model)
    model.moe, model.eps, model.balance_coef = layer, 1e-5, 0.5
    model.norm_w, model.embed = torch.ones(8), torch.zeros(10, 8)
    monkeypatch.setattr(fused, "embedding", lambda ids, table: table[ids])
    monkeypatch.setattr(fused, "residual_mean_square", lambda a, b: (a + b).pow(2).mean())
    return model, layer


@pytest.mark.parametrize("how", ["no_grad", "eval", "both"])
def test_a_forward_only_pass_has_no_balance_loss(how, monkeypatch):
    model, layer = _stubbed(monkeypatch)
    ids = torch.arange(4)
    for left_over in (None, torch.tensor(7.0)):     # a fresh model, and one that has trained
        layer.balance_loss = layer.expert_counts = left_over
        model.train(how == "no_grad")
        with torch.set_grad_enabled(how == "eval"):
            assert model(ids).item() == 0
        assert layer.balance_loss is None and layer.expert_counts is None


def test_a_replayed_pass_drops_the_last_balance_loss(monkeypatch):
    _, layer = _stubbed(monkeypatch)
    layer._gx, layer._gout = torch.zeros(4, 8), torch.ones(4, 8)
    layer._graph = type("Graph", (), {"replay": lambda self: None})()
    layer.balance_loss = layer.expert_counts = torch.tensor(7.0)
    assert layer.forward_graphed(torch.zeros(4, 8)) is layer._gout
    assert layer.balance_loss is None and layer.expert_counts is None


@pytest.mark.parametrize("coef,want", [(0.5, 6.5), (0.0, 3.0)])
def test_a_training_pass_adds_the_balance_loss_only_with_a_coefficient(coef, want, monkeypatch):
    model, layer = _stubbed(monkeypatch)
    model.balance_coef = coef

    def trained(h, norm_w, eps):
        layer.balance_loss = torch.tensor(7.0 if coef else float("nan"))
        return torch.tensor(3.0)

    monkeypatch.setattr(layer, "mean_square_from_residual", trained)
    assert model(torch.arange(4)).item() == want


@pytest.mark.gpu
@pytest.mark.parametrize("E,shared", [(8, 0), (8, 128), (64, 0)])
def test_evaluation_between_training_steps(E, shared):
    from fast_b200.models import MixtralBlockModel
    from fast_b200.parallel import Communicator

    comm = Communicator(heap_bytes=512 << 20, device=0)
    kw = dict(vocab=1000, hidden=512, inter=256, num_experts=E, top_k=2, max_tokens=512, shared_inter=shared)
    model, plain = MixtralBlockModel(comm, balance_coef=0.25, **kw), MixtralBlockModel(comm, **kw)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids, other = (torch.randint(0, 1000, (n,), generator=g, device="cuda") for n in (512, 300))
    with torch.no_grad():
        fresh, want = model(ids), plain(ids)        # the same seed, the same weights
    assert torch.equal(fresh, want) and model.moe.balance_loss is None
    trained = model(other)
    assert trained.requires_grad and 0.9 < model.moe.balance_loss.item() < E
    with torch.no_grad():
        assert torch.equal(model(ids), want)
    model.eval()
    assert torch.equal(model(ids), want) and model.moe.balance_loss is None and model.moe.expert_counts is None
    model.train()
    again = model(other)
    assert torch.equal(again, trained) and model.moe.balance_loss is not None
    again.backward()
    comm.check()
