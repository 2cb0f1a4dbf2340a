"""Operators of the residual stream (``csrc/residual.cuh``): what joins a block's branch to the
stream, and dropout.

``residual_norm`` is one join of a decoder whose blocks have norms before and after them:

    n  = branch_weight * branch / rms(branch)          (n = branch without branch_weight)
    x' = x + scale * dropout(gate * n)
    y  = norm_weight * x' / rms(x')                    (the next block's input)

with ``rms(v) = sqrt(mean(v^2) + eps)`` over the last dimension, and ``gate`` a learned vector
of the channels.  ``dropout`` is the same dropout alone.

The dropout mask is never stored.  It comes from the counter-based generator Philox4x32-10
(Salmon, Moraes, Dror and Shaw, SC 2011), drawn again in the backward pass: the key is ``seed``,
the counter is (element // 8, ``stream``), an element takes 16 of the 128 bits, and is kept
where they are at least ``round(p * 65536)``; so ``p`` is rounded to a multiple of 2^-16, and
what is kept is divided by the kept share of the rounded one.  A dropped element is 0, also
where it was not finite.  The mask depends on the seed, the stream and the element's position
alone, not on the type, the device or the launch.  Calls that share a seed take different
``stream`` numbers.  ``seed`` is an int or an int64 tensor of one element, which a captured CUDA
graph reads anew at every replay (``new_seed`` draws one from PyTorch's generator, in a capture
too); an int is part of the capture.

On CUDA the operators run the sm_100a kernels on the current stream: bfloat16, float16 or
float32, weights and gate in the activations' type, rows of up to 16384 channels (16370 where
their number is no multiple of 8).  Sums and statistics are held in fp32 and each result is rounded once.
On the CPU the same formulas run in PyTorch.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from ._ext import require

Seed = Union[int, torch.Tensor]


def new_seed(device: Union[str, torch.device]) -> torch.Tensor:
    """A seed from PyTorch's generator of ``device``: int64 ``[1]`` on that device."""
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64, device=device)


def _threshold(p: float) -> int:
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be between 0 and 1")
    return int(p * 65536.0 + 0.5)


def _check_seed(seed: Optional[Seed], stream: int, x: torch.Tensor) -> Tuple[Optional[torch.Tensor], int]:
    """(seed tensor or None, seed value)."""
    if not 0 <= stream < 2 ** 32:
        raise ValueError("stream must fit 32 bits")
    if seed is None:
        raise ValueError("dropout needs a seed")
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64:
            raise TypeError("seed must be int64")
        if seed.numel() != 1:
            raise ValueError("seed must have one element")
        if seed.device != x.device:
            raise ValueError("seed must be on x's device")
        return seed, 0
    s = int(seed)
    if not -2 ** 63 <= s < 2 ** 64:
        raise ValueError("seed must fit 64 bits")
    return None, s - 2 ** 64 if s >= 2 ** 63 else s


def _mul32(a: int, b: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """High and low words of the 64-bit product of two 32-bit values (int64 tensors)."""
    lo, hi = (b & 0xFFFF) * a, (b >> 16) * a
    mid = (lo >> 16) + (hi & 0xFFFF)
    return (hi >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)


def _random16(n: int, seed: torch.Tensor, stream: int) -> torch.Tensor:
    """The 16 random bits of each of ``n`` elements, int64, on the seed's device."""
    s = seed.reshape(())
    k0, k1 = s & 0xFFFFFFFF, (s >> 32) & 0xFFFFFFFF
    i = torch.arange(-(-n // 8), device=seed.device, dtype=torch.int64)
    c0, c1, c2, c3 = i & 0xFFFFFFFF, i >> 32, torch.full_like(i, stream), torch.zeros_like(i)
    for _ in range(10):
        ah, al = _mul32(0xD2511F53, c0)
        bh, bl = _mul32(0xCD9E8D57, c2)
        c0, c1, c2, c3 = bh ^ c1 ^ k0, bl, ah ^ c3 ^ k1, al
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16,
                        c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16), -1).reshape(-1)[:n]


def dropout_factors(shape, p: float, seed: Seed, *, stream: int = 0,
                    device: Union[str, torch.device] = "cpu") -> torch.Tensor:
    """The factors (0, or one over the kept share) that ``dropout`` of this shape, seed and
    stream multiplies by, in fp32.  For tests and the CPU: the kernels never store them."""
    t = _threshold(p)
    n = 1
    for d in shape:
        n *= int(d)
    if n == 0 or t >= 65536:
        return torch.zeros(shape, device=device)
    if not torch.is_tensor(seed):
        s = int(seed)
        seed = torch.tensor([s - 2 ** 64 if s >= 2 ** 63 else s])
    u = _random16(n, seed.to(device), stream)
    return torch.where(u >= t, 65536.0 / (65536 - t), 0.0).view(shape)


# ------------------------------------------------------------------- dropout
def dropout(x: torch.Tensor, p: float, seed: Seed, *, stream: int = 0) -> torch.Tensor:
    """``x`` with a share ``p`` of its elements set to 0 and the others divided by the kept
    share, by the counter-based generator (see the module)."""
    _threshold(p)
    tensor, value = _check_seed(seed, stream, x)
    if not x.is_floating_point():
        raise TypeError("x must be a floating-point tensor")
    if not x.is_cuda:
        f = dropout_factors(x.shape, p, value if tensor is None else tensor, stream=stream,
                            device=x.device)
        wide = x if x.dtype == torch.float64 else x.float()
        return torch.where(f == 0, 0.0, wide * f).to(x.dtype)
    if torch.is_grad_enabled() and x.requires_grad:
        return require().dropout_grad(x, p, tensor, value, stream)
    return require().dropout(x, p, tensor, value, stream)


# -------------------------------------------------------------- residual join
def _residual_norm_torch(x, branch, w1, gate, w2, scale, factors, eps):
    """The formulas in PyTorch, in fp32 (fp64 for fp64 tensors), rounded at the ends."""
    dt = x.dtype
    wide = torch.float64 if dt == torch.float64 else torch.float32

    def rms(v):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)

    u = branch.to(wide)
    if w1 is not None:
        u = w1.to(wide) * rms(u)
    if gate is not None:
        u = gate.to(wide) * u
    if factors is not None:
        u = torch.where(factors == 0, 0.0, u * factors.to(wide))
    new = x.to(wide) + scale * u
    y = None if w2 is None else (w2.to(wide) * rms(new)).to(dt)
    return new.to(dt), y


def residual_norm(x: torch.Tensor, branch: torch.Tensor, *,
                  branch_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None,
                  norm_weight: Optional[torch.Tensor] = None, scale: float = 1.0, p: float = 0.0,
                  seed: Optional[Seed] = None, stream: int = 0, eps: float = 1e-6
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(x', y)`` of the module's formulas; ``y`` is None without ``norm_weight``.

    ``x`` and ``branch`` have one shape ``[..., H]`` and type, the weights and the gate are
    ``[H]`` of that type.  ``p`` > 0 drops elements of the branch and needs a ``seed``.
    """
    threshold = _threshold(p)
    tensor, value = (None, 0) if threshold == 0 else _check_seed(seed, stream, x)
    ts = (x, branch, branch_weight, gate, norm_weight)
    if x.is_cuda:  # shapes, types and devices are checked in the extension
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
            return require().residual_norm_grad(*ts, scale, p, tensor, value, stream, eps)
        return require().residual_norm_fwd(*ts, scale, p, tensor, value, stream, eps, False)[:2]
    if not x.is_floating_point():
        raise TypeError("x must be a floating-point tensor")
    for name, t in zip(("branch", "branch_weight", "gate", "norm_weight"), ts[1:]):
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError(f"{name} must have x's dtype {x.dtype}, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{name} must be on x's device")
        want = x.shape if name == "branch" else x.shape[-1:]
        if t.shape != want:
            raise ValueError(f"{name} must be {list(want)}, got {list(t.shape)}")
    f = None
    if threshold:
        f = dropout_factors(x.shape, p, value if tensor is None else tensor, stream=stream,
                            device=x.device)
    return _residual_norm_torch(*ts, scale, f, eps)
