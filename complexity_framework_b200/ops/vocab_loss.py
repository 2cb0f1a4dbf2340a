"""Softmax cross-entropy over a large vocabulary without keeping its logits
(``csrc/vocab_loss.cu``).

With logits ``z = logit_scale * hidden @ weight.T`` and ``lse = logsumexp(z)``, a row whose
target is the word ``y`` has the loss

    lse - (1 - label_smoothing) z_y - label_smoothing * mean(z) + z_loss * lse^2

The logits exist a tile at a time: the forward pass leaves a row's log-sum-exp, the backward
pass computes the logits again, for as much of the vocabulary at a time as ``workspace_bytes``
holds gradients of (bf16), but 256 words at least.  Beside it are a copy of the counted rows and
one or more fp32 accumulators of ``hidden``'s gradient (few rows of few channels take more, so
that their products fill the GPU: 18 at 2048 x 50000 x 256), which ``workspace_bytes`` does not
count.  The logits are fp32 throughout, where ``ops.fused.linear_cross_entropy`` keeps them,
rounded to bf16, for the mean loss alone.

Rows whose target is ``ignore_index`` have the loss 0, add nothing to a gradient whatever they
hold, and cost nothing in the products.  A target that is neither a word nor ``ignore_index`` is
reported by ``ops.check_errors`` and its row's loss is NaN.

On CUDA ``hidden`` and ``weight`` are bfloat16 with a hidden size that is a multiple of 8 (any
number of rows and words); the gradients are bfloat16, and equal calls give equal bits.  The
gradients' own derivatives (``create_graph``) are computed in PyTorch from all logits in fp32.  On
the CPU the same formulas run in PyTorch, any floating-point type.
"""
from __future__ import annotations

import torch

from ._ext import require

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
WORKSPACE_BYTES = 512 << 20


def _rows_torch(h, w, y, ignore_index, smooth, z, scale):
    """Row losses in PyTorch, in fp32 (fp64 for fp64 tensors)."""
    valid = y != ignore_index
    if bool((valid & ((y < 0) | (y >= w.shape[0]))).any()):
        raise ValueError("a target is neither a word nor ignore_index")
    wide = torch.float64 if h.dtype == torch.float64 else torch.float32
    out = torch.zeros(h.shape[0], dtype=wide, device=h.device)
    hv, yv = h[valid].to(wide), y[valid]
    logits = (hv @ w.to(wide).t()) * scale
    lse = torch.logsumexp(logits, -1)
    loss = lse - (1 - smooth) * logits.gather(1, yv[:, None])[:, 0]
    if smooth > 0:
        loss = loss - smooth * logits.mean(-1)
    if z > 0:
        loss = loss + z * lse.square()
    return out.masked_scatter(valid, loss)


def vocab_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                        ignore_index: int = -100, label_smoothing: float = 0.0,
                        z_loss: float = 0.0, logit_scale: float = 1.0, reduction: str = "mean",
                        workspace_bytes: int = WORKSPACE_BYTES) -> torch.Tensor:
    """The loss of ``hidden`` ``[..., H]`` against ``targets`` ``[...]`` (int64) under the output
    matrix ``weight`` ``[V, H]``, fp32: the mean over the counted rows (0 without any), their
    sum, or, with ``reduction="none"``, every row's, shaped like ``targets``."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {list(_REDUCTIONS)}")
    return _loss(hidden, weight, targets, ignore_index, label_smoothing, z_loss, logit_scale,
                 reduction, 1.0, workspace_bytes)


def _loss(hidden, weight, targets, ignore_index, label_smoothing, z_loss, logit_scale, reduction,
          sign, workspace_bytes):
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing must be between 0 and 1")
    if not 0.0 <= z_loss < float("inf"):
        raise ValueError("z_loss must not be negative")
    if not 0.0 < logit_scale < float("inf"):
        raise ValueError("logit_scale must be positive and finite")
    if workspace_bytes < 0:
        raise ValueError("workspace_bytes must not be negative")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("hidden must be [..., H] and weight [V, H]")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must be {list(hidden.shape[:-1])}, got {list(targets.shape)}")
    if targets.dtype != torch.int64:
        raise TypeError("targets must be int64")
    h, y = hidden, targets
    if hidden.dim() != 2:
        h, y = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1)
    if h.is_cuda:
        grad = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
        loss = require().vocab_loss(h, weight, y, ignore_index, label_smoothing, z_loss, logit_scale,
                                    _REDUCTIONS[reduction], sign, workspace_bytes, grad)
        return loss.view(targets.shape) if loss.dim() and targets.dim() != 1 else loss
    rows = sign * _rows_torch(h, weight, y, ignore_index, label_smoothing, z_loss, logit_scale)
    if reduction == "none":
        return rows.view(targets.shape)
    if reduction == "sum":
        return rows.sum()
    return rows.sum() / (y != ignore_index).sum().clamp_min(1)


def token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                   ignore_index: int = -100, logit_scale: float = 1.0,
                   workspace_bytes: int = WORKSPACE_BYTES) -> torch.Tensor:
    """Log-probability of every target under ``softmax(logit_scale * hidden @ weight.T)``, fp32,
    shaped like ``targets``; 0 where the target is ``ignore_index``."""
    return _loss(hidden, weight, targets, ignore_index, 0.0, 0.0, logit_scale, "none", -1.0,
                 workspace_bytes)
