"""What the dense operators refuse, with the message that says why (no GPU: an argument is checked before anything runs)."""
import pytest
import torch

from fast_b200.ops import fused

BF = torch.bfloat16


def test_row_norm_refuses_tensors_of_the_host():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fused.add_rms_norm(torch.zeros(2, 128, dtype=BF), torch.ones(128, dtype=BF))
    with pytest.raises(RuntimeError, match="contiguous e4m3 bytes"):
        fused.dequantise_rows(torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(2, 1))


def test_balance_loss_refuses_what_it_does_not_know():
    logits, idx = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fused.balance_loss(logits, idx)
    with pytest.raises(ValueError, match="scores"):
        fused.balance_loss(logits, idx, scores="tanh")


def test_linear_refuses_what_it_does_not_know():
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(16, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fused.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        fused.linear(x, w, activation="tanh")


@pytest.mark.gpu
def test_linear_refusals():
    x, w, b, r = (torch.zeros(*s, device="cuda", dtype=BF) for s in ((4, 64), (256, 64), (256,), (4, 256)))
    for bad, match in [
        (lambda: fused.linear(x.float(), w), "x must be"),
        (lambda: fused.linear(x, w.float()), "weight"),
        (lambda: fused.linear(x, w[:, :32]), "weight"),
        (lambda: fused.linear(x, w.unsqueeze(0)), "weight"),
        (lambda: fused.linear(x, w.cpu()), "weight"),
        (lambda: fused.linear(x[:, :60], w[:, :60]), "multiples of 8"),
        (lambda: fused.linear(x, w[:250]), "multiples of 8"),
        (lambda: fused.linear(x[:, :0], w[:, :0]), "multiples of 8"),
        (lambda: fused.linear(x, w[:0]), "multiples of 8"),
        (lambda: fused.linear(x, w, bias=b.float()), "bias"),
        (lambda: fused.linear(x, w, bias=b[:128]), "bias"),
        (lambda: fused.linear(x, w, residual=r[:1]), "residual"),
        (lambda: fused.linear(x, w, residual=r.float()), "residual"),
        (lambda: fused.linear(x, w[:128], activation="swiglu"), "swiglu"),
        (lambda: fused.linear(x, w, bias=b, activation="swiglu"), "swiglu"),
        (lambda: fused.linear(x, w, residual=r[:, :128], activation="swiglu"), "swiglu"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()


@pytest.mark.gpu
def test_balance_loss_refusals():
    logits, idx = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    mask = torch.ones(4, dtype=torch.bool, device="cuda")
    for bad, match in [
        (lambda: fused.balance_loss(logits.half(), idx), "bf16 or fp32"),
        (lambda: fused.balance_loss(torch.zeros(4, 1025, device="cuda"), idx), "experts"),
        (lambda: fused.balance_loss(logits[:, :0], idx), "experts"),
        (lambda: fused.balance_loss(logits, idx.long()), "topk_idx"),
        (lambda: fused.balance_loss(logits, idx[:3]), "topk_idx"),
        (lambda: fused.balance_loss(logits, idx[:, :0]), "topk_idx"),
        (lambda: fused.balance_loss(logits, idx.cpu()), "topk_idx"),
        (lambda: fused.balance_loss(logits, idx, mask=mask[:3]), "mask"),
        (lambda: fused.balance_loss(logits, idx, mask=mask.float()), "mask"),
        (lambda: fused.balance_loss(logits, idx, mask=mask.unsqueeze(1)), "mask"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()


@pytest.mark.gpu
def test_row_norm_refusals():
    x, w = torch.zeros(4, 200, device="cuda", dtype=BF), torch.ones(200, device="cuda", dtype=BF)
    for bad, match in [
        (lambda: fused.add_rms_norm(x.half(), w), "bf16 or fp32"),
        (lambda: fused.add_rms_norm(x, w[:100].contiguous()), "weight"),
        (lambda: fused.add_rms_norm(x, torch.ones(400, device="cuda", dtype=BF)[::2]), "weight"),
        (lambda: fused.add_rms_norm(x, w.half()), "weight"),
        (lambda: fused.add_rms_norm(x, w.cpu()), "weight"),
        (lambda: fused.add_rms_norm(x, w, residual=x.float()), "residual"),
        (lambda: fused.add_rms_norm(x, w, residual=x[:2]), "residual"),
        (lambda: fused.add_rms_norm(x, w, residual=x[:1]), "residual"),
        (lambda: fused.add_rms_norm(x, w, quantise=True), "multiple of 128"),
        (lambda: fused.add_rms_norm(x, w, eps=-1.0), "eps"),
        (lambda: fused.add_rms_norm(x[:, :0], w[:0]), "hidden size"),
        (lambda: fused.add_rms_norm(torch.zeros(1, 49153, device="cuda"), torch.ones(49153, device="cuda")), "hidden size"),
        (lambda: fused.dequantise_rows(torch.zeros(2, 130, device="cuda", dtype=torch.uint8), torch.zeros(2, 1, device="cuda")), "multiple of 128"),
        (lambda: fused.dequantise_rows(torch.zeros(2, 256, device="cuda", dtype=torch.uint8), torch.zeros(2, 1, device="cuda")), "scales"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()


@pytest.mark.gpu
def test_more_rows_than_are_counted_are_refused_before_anything_is_allocated():
    def rows(n, cols, dtype=BF):   # one row's memory
        return torch.zeros(1, cols, device="cuda", dtype=dtype).expand(n, cols)

    n = 2**30 + 1
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    held = [rows(n, 8), torch.ones(8, device="cuda", dtype=BF), rows(n, 2), rows(n, 1, torch.int32), torch.zeros(8, 8, device="cuda", dtype=BF), rows(2**29, 2), rows(2**29, 4, torch.int32)]
    made = torch.cuda.memory_stats()["allocation.all.allocated"] - before
    for bad, match in [
        (lambda: fused.add_rms_norm(held[0], held[1]), "rows"),
        (lambda: fused.balance_loss(held[2], held[3]), "rows"),
        (lambda: fused.balance_loss(held[5], held[6]), "choices"),
        (lambda: fused.linear(held[0], held[4]), "rows"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == made


def test_memory_plan_counts_a_shared_expert():
    from fast_b200.models import DEEPSEEK_V3_MOE_LAYER, MIXTRAL_8X7B_BLOCK, flops_per_step, memory_plan, step_roofline

    for cfg in (MIXTRAL_8X7B_BLOCK, DEEPSEEK_V3_MOE_LAYER):
        a, b = memory_plan(cfg, 8), memory_plan(cfg.with_(shared_inter=2048), 8)
        assert b["weights"] - a["weights"] == 2 * 3 * cfg.hidden * 2048
        assert b["workspace"] - a["workspace"] == 2 * cfg.tokens_per_rank * 2048 * (8 if cfg.training else 1)
        f, g = flops_per_step(cfg, 8), flops_per_step(cfg.with_(shared_inter=2048), 8)
        assert f["shared_expert"] == 0 and g["total"] - f["total"] == g["shared_expert"] == 2.0 * cfg.tokens_per_rank * cfg.hidden * 2048 * 3 * (3 if cfg.training else 1)
        assert step_roofline(cfg.with_(shared_inter=2048), 8, 1500, 6500)["total_ms"] > step_roofline(cfg, 8, 1500, 6500)["total_ms"]
