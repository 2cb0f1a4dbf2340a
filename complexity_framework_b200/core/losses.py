"""Causal-LM losses.

* ``causal_lm_loss``: cross-entropy from logits with optional label smoothing
  and z-loss (complexity/core/losses/causal_lm.py:1-104).
* ``causal_lm_loss_from_hidden`` / ``fused_linear_causal_lm_loss``: CE of
  ``hidden @ W^T`` without materialising all logits.  On CUDA bf16 it is the
  sm_100a fused linear-CE (ops.fused.linear_cross_entropy) for the plain mean, and
  ops.vocab_loss with label smoothing, z-loss, a positive logit scale or a vocabulary that is
  no multiple of 32; elsewhere, and under torch.func or forward-mode differentiation, a chunked
  PyTorch loop with per-chunk recomputation (complexity/core/losses/causal_lm.py:106-191,
  fused_ce.py:95-204).
* ``model_token_logprobs``: log-probabilities of given next tokens, without logits where
  ops.vocab_loss applies.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Tuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint as activation_checkpoint

from .layers import use_fused


@dataclass
class CausalLMLossMetrics:
    ce: float
    z_loss: float
    total: float

    def as_dict(self) -> dict:
        return {"ce": self.ce, "z_loss": self.z_loss, "total": self.total}


def causal_lm_loss(logits: torch.Tensor, labels: torch.Tensor, *, label_smoothing: float = 0.0,
                   z_loss_coef: float = 0.0, ignore_index: int = -100, shift: bool = False,
                   sync_metrics: bool = True) -> Tuple[torch.Tensor, CausalLMLossMetrics]:
    if shift:
        logits = logits[..., :-1, :]
        labels = labels[..., 1:]
    V = logits.shape[-1]
    lf = logits.reshape(-1, V).float()
    lb = labels.reshape(-1)
    ce = F.cross_entropy(lf, lb, ignore_index=ignore_index, label_smoothing=label_smoothing)
    total = ce
    z = torch.zeros((), device=lf.device)
    if z_loss_coef > 0:
        valid = lb != ignore_index
        lse = torch.logsumexp(lf, -1)
        z = z_loss_coef * (lse[valid] ** 2).mean() if bool(valid.any()) else z
        total = ce + z
    if sync_metrics:
        metrics = CausalLMLossMetrics(float(ce.detach()), float(z.detach()), float(total.detach()))
    else:
        metrics = CausalLMLossMetrics(float("nan"), float("nan"), float("nan"))
    return total, metrics


def _chunk_ce(h: torch.Tensor, w: torch.Tensor, y: torch.Tensor, ignore_index: int,
              scale: float, label_smoothing: float = 0.0, z_loss_coef: float = 0.0
              ) -> torch.Tensor:
    logits = F.linear(h, w).float() * scale
    ce = F.cross_entropy(logits, y, ignore_index=ignore_index, reduction="sum",
                         label_smoothing=label_smoothing)
    if z_loss_coef > 0:
        ce = ce + z_loss_coef * torch.logsumexp(logits[y != ignore_index], -1).square().sum()
    return ce


def _transformed(*tensors: torch.Tensor) -> bool:
    """Whether torch.func transforms or forward-mode differentiation are at work, which the
    kernels take no part in."""
    if torch._C._are_functorch_transforms_active():
        return True
    return forward_ad._current_level >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def causal_lm_loss_from_hidden(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                               *, ignore_index: int = -100, chunk_tokens: int = 8192,
                               logit_scale: float = 1.0, checkpoint_chunks: bool = True,
                               label_smoothing: float = 0.0, z_loss_coef: float = 0.0
                               ) -> torch.Tensor:
    """Mean CE over labels != ignore_index of ``(hidden @ weight.T) * logit_scale``, plus
    ``z_loss_coef`` times the mean square of their log-sum-exp.

    ``hidden [.., H]`` and ``labels [..]`` are aligned (shift beforehand).
    """
    H = hidden.shape[-1]
    h = hidden.reshape(-1, H)
    y = labels.reshape(-1)
    if use_fused(h) and weight.dtype == torch.bfloat16 and H % 8 == 0:
        # the plain mean keeps 16-bit logits: three products where ops.vocab_loss takes four, and
        # more memory (32768 x 32000 x 896: 6.4 ms and 2.2 GB against 7.1 ms and 0.5 GB)
        if (logit_scale == 1.0 and weight.shape[0] % 32 == 0 and label_smoothing == 0.0
                and z_loss_coef == 0.0):
            from ..ops.fused import linear_cross_entropy

            return linear_cross_entropy(h, weight, y, ignore_index=ignore_index)
        if 0.0 < logit_scale < float("inf") and not _transformed(h, weight):
            from ..ops.vocab_loss import vocab_cross_entropy

            return vocab_cross_entropy(h, weight, y.long(), ignore_index=ignore_index,
                                       label_smoothing=label_smoothing, z_loss=z_loss_coef,
                                       logit_scale=logit_scale)
    total = h.new_zeros((), dtype=torch.float32)
    for s in range(0, h.shape[0], chunk_tokens):
        hc, yc = h[s:s + chunk_tokens], y[s:s + chunk_tokens]
        if checkpoint_chunks and torch.is_grad_enabled():
            total = total + activation_checkpoint(_chunk_ce, hc, weight, yc, ignore_index,
                                                  logit_scale, label_smoothing, z_loss_coef,
                                                  use_reentrant=False)
        else:
            total = total + _chunk_ce(hc, weight, yc, ignore_index, logit_scale, label_smoothing,
                                      z_loss_coef)
    return total / (y != ignore_index).sum().clamp_min(1)


def fused_linear_causal_lm_loss(hidden: torch.Tensor, weight: torch.Tensor,
                                labels: torch.Tensor, *, ignore_index: int = -100,
                                shift: bool = True, label_smoothing: float = 0.0,
                                z_loss_coef: float = 0.0) -> torch.Tensor:
    """Reference-compatible entry: ``hidden[:, :-1]`` predicts ``labels[:, 1:]`` when shift."""
    if shift:
        hidden = hidden[..., :-1, :]
        labels = labels[..., 1:]
    return causal_lm_loss_from_hidden(hidden.contiguous(), weight, labels.contiguous(),
                                      ignore_index=ignore_index, label_smoothing=label_smoothing,
                                      z_loss_coef=z_loss_coef)


def model_token_logprobs(model, ids: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100) -> torch.Tensor:
    """Log-probability, fp32 ``[B, S]``, of each target under ``model`` after the tokens up to
    its position (``targets[b, s]`` follows ``ids[b, :s + 1]``); 0 where it is ``ignore_index``.

    A ``ComplexityModel`` in bf16 on CUDA computes them from its hidden states without logits;
    any other model from the logits it returns."""
    head = getattr(model, "lm_head", None)
    if (hasattr(model, "output_weight") and (head is None or type(head) is torch.nn.Linear)
            and isinstance(getattr(model, "logit_scale", None), float)):
        w = model.output_weight()
        if use_fused(w) and w.shape[1] % 8 == 0:
            from ..ops.vocab_loss import token_logprobs

            hidden = model(ids, return_logits=False)["last_hidden_state"]
            if use_fused(hidden):
                return token_logprobs(hidden, w, targets, ignore_index=ignore_index,
                                      logit_scale=model.logit_scale)
            return _logprobs(model.logits(hidden), targets, ignore_index)
    return _logprobs(model(ids)["logits"], targets, ignore_index)


def _logprobs(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int) -> torch.Tensor:
    counted = targets != ignore_index
    at = torch.where(counted, targets, torch.zeros_like(targets))
    lp = torch.log_softmax(logits.float(), -1).gather(-1, at[..., None])[..., 0]
    return torch.where(counted, lp, torch.zeros_like(lp))
