"""Small fused autograd ops around the MoE block: embedding with a segmented-sum backward, the
mean-square loss of a residual sum computed without materialising fp32 copies, and the dense side of a block (residual
sum and RMS norm of rows, the router's balance loss, linear layers), whose derivatives are reverse mode, once: inputs with a forward-mode tangent are refused."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .. import runtime
from ..utils.config import CONFIG


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table):
        ctx.save_for_backward(ids)
        ctx.shape = table.shape
        return torch.nn.functional.embedding(ids, table)

    @staticmethod
    def backward(ctx, grad_out):
        (ids,) = ctx.saved_tensors
        # positions grouped by id by this library's counting sort (stable; its cost does not depend on duplicates), then one warp per
        # id adds up its rows in position order: an id that names many positions is a serial chain as long as they are
        grad_table = runtime.ext().embedding_grad(ids.reshape(-1).contiguous(), ctx.shape[0], grad_out.reshape(-1, ctx.shape[1]).contiguous())
        return None, grad_table


def embedding(ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """``table[ids]`` (bf16 table); backward sums duplicate ids in position order (deterministic)."""
    return _Embedding.apply(ids, table)


class _ResidualMeanSquare(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b):
        C = runtime.ext()
        a, b = a.contiguous(), b.contiguous()
        partial = torch.empty(148 * 8, dtype=torch.float32, device=a.device)
        out = torch.empty(1, dtype=torch.float32, device=a.device)
        C.sumsq_add(a, b, 1.0 / a.numel(), partial, out)
        ctx.save_for_backward(a, b)
        return out.reshape(())

    @staticmethod
    def backward(ctx, grad_loss):
        a, b = ctx.saved_tensors
        g = torch.empty_like(a)
        runtime.ext().scaled_sum(a, b, grad_loss.reshape(1).float().contiguous(), 2.0 / a.numel(), g)
        return g, g


def residual_mean_square(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """mean((a + b)^2) with the sum rounded to bf16, as a scalar fp32 tensor (bf16 inputs)."""
    return _ResidualMeanSquare.apply(a, b)


class NormRows(NamedTuple):
    """What ``add_rms_norm`` returns: the normalised rows ``y``, the sum ``h`` that was normalised (``x`` itself without a residual) and, if
    asked for, ``y`` in e4m3: bytes ``q`` (uint8) and fp32 ``scales``, one per 128 columns."""

    y: torch.Tensor
    h: torch.Tensor
    q: Optional[torch.Tensor]
    scales: Optional[torch.Tensor]


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, residual: Optional[torch.Tensor] = None, quantise: bool = False) -> NormRows:
    """RMS norm of rows, with the residual's addition in front of it and optionally an output in e4m3.

    ``h = x + residual`` rounded to x's type; ``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, rounded once. x: bf16 or
    fp32 [..., hidden], rows in any strides (16-byte aligned rows of whole 16-byte words are fastest); ``residual``: the same shape and type;
    ``weight``: bf16 or fp32 [hidden]; hidden up to 49152, up to 2^30 rows. ``quantise`` (hidden a multiple of 128): ``y`` also as the e4m3 rows that the
    fp8 dispatch would send for it (``dequantise_rows`` reads them back). Gradients flow through y and h, not through q and scales; the weight's
    gradient is summed in a fixed order."""
    return NormRows(*runtime.ext().add_rms_norm(x, weight, eps, residual, quantise))


def dequantise_rows(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """bf16 rows of e4m3 bytes (uint8 [..., hidden]) and fp32 scales [..., hidden / 128], as ``add_rms_norm`` makes them. Has no gradient: scales
    that require one are refused."""
    return runtime.ext().dequantise_rows(q, scales)


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, mask: Optional[torch.Tensor] = None, scores: str = "softmax") -> Tuple[torch.Tensor, torch.Tensor]:
    """Balance loss of a router and how often each expert was chosen: ``(loss, counts)``, an fp32 scalar and int32 [experts].

    ``loss = E / (K N^2) * sum_e counts[e] * sum_t s[t, e]`` over the N live tokens: 1 when choices and scores are spread evenly, more when the
    experts that are chosen often are also those with high scores. ``s``: the softmax of a token's logits, or with ``scores="sigmoid"`` their sigmoids
    divided by the sum of these. logits: bf16 or fp32 [..., experts] (up to 1024 experts, 2^30 tokens, 2^31 - 1 choices), without a bias that only the choice uses; ``topk_idx``: int32
    [..., k] as the routing returns it (entries outside the experts' range count for none); ``mask``: bool [...], False for padding, which has
    no part in anything. NaN logits count as -inf; a token whose scores are all zero adds no score; without live tokens the loss is 0. Gradients
    flow to the logits only. The result does not change from run to run."""
    if scores not in ("softmax", "sigmoid"):
        raise ValueError(f"balance_loss: scores must be 'softmax' or 'sigmoid', got {scores!r}")
    return runtime.ext().balance_loss(logits, topk_idx, mask, scores == "sigmoid")


_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "swiglu": 4}


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel (tcgen05, fp32 accumulation, the result rounded once), with its backward pass.

    x: bf16 [..., inputs]; ``weight``: bf16 [outputs, inputs], both sizes multiples of 8; ``bias``: bf16 [outputs]; ``residual``: bf16 with the
    result's shape. ``activation``: None, "relu", "silu", "gelu" (z Phi(z)), or "swiglu": the weight holds tiles of 128 gate rows and the 128 up rows of
    the same features, as an expert's does (``models.moe.interleave_gate_up``), outputs a multiple of 256, the result [..., outputs / 2] =
    silu(gate) * up, without bias and residual. From none to 2^30 rows; rows that are not contiguous, 16-byte aligned and a multiple of 16 bytes
    apart are copied first. Where a gradient needs it, what the activation was taken of is kept in bf16 (swiglu: in two bf16, 16 bits of each value). A device wait that gave up is
    reported by ``ops.gemm.check()`` and ``Communicator.check()``."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"linear: activation must be one of {', '.join(map(repr, _ACTIVATIONS))}, got {activation!r}")
    return runtime.ext().linear(x, weight, bias, residual, _ACTIVATIONS[activation], CONFIG.timeout_s)
