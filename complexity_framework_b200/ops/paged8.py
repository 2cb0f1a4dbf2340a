"""Operators of a paged KV cache held in 8 bits (``csrc/paged8_*.cu``).

One layer of the cache is

* ``codes``  ``[pages, Hkv, 2, 16, D]`` int8 or float8_e4m3fn: K, then V, of each page and head;
* ``scales`` ``[pages, Hkv, 2]`` fp32: a block is one page of one head's K or V, and a code
  ``c`` stands for ``c * scale``;
* ``mass``   ``[pages, Hkv, 16]`` fp32, optional: attention weight each cached token has
  received, summed over steps, queries and the query heads of its KV head.

A batch of new tokens is ragged: sequence i owns the rows ``[cu_q[i], cu_q[i+1])``, which are
the last of its ``kv_lens[i]`` cached tokens (their own keys included), and token t of a
sequence is at ``page_table[i, t // 16]``, slot ``t % 16``.  Index tensors are int32.  A row
whose position would be negative (a padding row has ``kv_lens`` 0) stores nothing and attends
to nothing: its output is 0.  Sequences of one call must not share pages that are written
(append, mass, the new pages of an eviction).

On CUDA the operators run the sm_100a kernels (head_dim 64 or 128; bf16 or fp16 tensors) on
the current stream, and raise on what these cannot take.  Page ids outside the pool, lengths
past the page table and chunks longer than ``max_q_len`` are found on the device and raised
by ``ops.check_errors``.  On the CPU the same formulas run in PyTorch.  There are no gradients.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import require

PAGE = 16
#: largest magnitude of a code
LEVELS = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _no_grad(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("the 8-bit KV cache operators have no gradient; "
                           "call them under torch.no_grad()")


def _check_cpu(codes: torch.Tensor, scales: torch.Tensor) -> None:
    if codes.dtype not in LEVELS:
        raise ValueError("codes must be int8 or float8_e4m3fn")
    if codes.dim() not in (5, 6) or codes.shape[-3] != 2 or codes.shape[-2] != PAGE:
        raise ValueError("codes must be [(layers,) pages, kv_heads, 2, 16, head_dim]")
    if scales.shape != codes.shape[:-2] or scales.dtype != torch.float32:
        raise ValueError("scales must be fp32 and match codes")


def paged8_append(k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                  page_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                  max_q_len: int, mass: Optional[torch.Tensor] = None) -> None:
    """Quantise the new tokens' ``k``, ``v`` ``[N, Hkv, D]`` into one layer, in place.

    A block's scale is the largest magnitude among its new tokens over the largest code, or
    its present scale where that is larger and the block holds older tokens; the older codes
    are rounded anew when the scale grows.  ``kv_lens`` counts the new tokens; ``max_q_len``
    bounds the new tokens of a sequence; the new tokens' ``mass`` starts at 0.  A block with a
    value that is not finite reads as NaN or infinity throughout.
    """
    if codes.is_cuda:
        require().paged8_append(k, v, codes, scales, page_table, cu_q, kv_lens, max_q_len, mass)
        return
    _no_grad(k, v)
    _check_cpu(codes, scales)
    if k.shape != v.shape or k.shape[1] != codes.shape[1] or k.shape[2] != codes.shape[4]:
        raise ValueError("k and v must be [tokens, kv_heads, head_dim] of the cache")
    levels = LEVELS[codes.dtype]
    cu = cu_q.tolist()
    for i, n in enumerate(kv_lens.tolist()):
        start = n - (cu[i + 1] - cu[i])
        if cu[i + 1] - cu[i] > max_q_len:
            raise ValueError("a chunk is longer than max_q_len")
        for b in range(max(start, 0) // PAGE, -(-n // PAGE)):
            page = int(page_table[i, b])
            lo, hi = max(start, 0, b * PAGE), min(n, (b + 1) * PAGE)
            if lo >= hi:
                continue
            new = torch.stack((k[cu[i] + lo - start:cu[i] + hi - start],
                               v[cu[i] + lo - start:cu[i] + hi - start])).float()
            new = new.permute(2, 0, 1, 3)                            # [Hkv, 2, n, D]
            older = lo - b * PAGE
            s0 = scales[page] if older else torch.zeros_like(scales[page])
            s = torch.maximum(new.abs().amax((-1, -2)) / levels, s0)
            # the kernel's arithmetic, to the bit: a product with the reciprocal, or a quotient
            # where the scale is subnormal; codes of 0 where it is 0 or not finite
            fine = (s > 0) & torch.isfinite(s)
            div = torch.where(fine, s, torch.ones_like(s))[..., None, None]
            x = torch.where(torch.isinf(1 / div), new / div, new * (1 / div))
            fine = fine[..., None, None]
            block = codes[page].float()
            if older:
                ratio = torch.where(fine, s0[..., None, None] / div, 0.0)
                block[:, :, :older] *= torch.where(s[..., None, None] == s0[..., None, None], 1.0,
                                                   ratio)
            block[:, :, older:older + hi - lo] = torch.where(fine, x, 0.0)
            block = torch.nan_to_num(block)
            if codes.dtype == torch.int8:
                block = block.round().clamp(-levels, levels)
            codes[page] = block.to(codes.dtype)
            scales[page] = s
            if mass is not None:
                mass[page][:, older:older + hi - lo] = 0


def paged8_read(codes: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor,
                kv_lens: torch.Tensor, dtype: torch.dtype = torch.bfloat16
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached values ``(k, v)``, each ``[(layers,) S, Hkv, max_pages * 16, D]``, of one layer
    or (with a leading dimension of ``codes`` and ``scales``) of all; 0 past ``kv_lens``."""
    if codes.is_cuda:
        return require().paged8_read(codes, scales, page_table, kv_lens, dtype)
    _check_cpu(codes, scales)
    lead = codes.shape[:-5]
    S, P = page_table.shape
    H, D = codes.shape[-4], codes.shape[-1]
    t = page_table.long()
    if lead:
        x = codes[:, t].float() * scales[:, t][..., None, None]
    else:
        x = (codes[t].float() * scales[t][..., None, None])[None]
    x = x.permute(4, 0, 1, 3, 2, 5, 6).reshape(2, -1, S, H, P * PAGE, D)
    live = torch.arange(P * PAGE) < kv_lens[:, None]
    x = torch.where(live[:, None, :, None], x, torch.zeros_like(x)).to(dtype)
    return (x[0], x[1]) if lead else (x[0, 0], x[1, 0])


def paged8_attention(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                     page_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                     scale: float, max_q_len: int, mass: Optional[torch.Tensor] = None,
                     mass_out: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None,
                     workspace_bytes: int = 4 << 30) -> torch.Tensor:
    """Causal attention of ``q`` ``[N, Hq, D]`` over one layer of the cache -> ``[N, Hq, D]``.

    With ``mass`` the softmax weights every cached token receives from this call are added to
    it: in place, or into ``mass_out`` (which takes the tokens of this call's sequences only).
    Rows of ``out`` before ``cu_q[0]`` or from ``cu_q[-1]`` on, which are other calls', stay as
    they are.
    Long chunks expand keys and values to 16 bits first, and short ones with ``mass`` keep their
    scores, both as long as the page table is wide: in a workspace of about ``workspace_bytes``
    at most (or one sequence's, where that is more), with the sequences taken in parts.
    """
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    if mass is None and mass_out is not None:
        raise ValueError("mass_out needs mass")
    if mass is not None and mass_out is None:
        mass_out = mass
    if codes.is_cuda:
        return require().paged8_attention(q, codes, scales, page_table, cu_q, kv_lens, out, scale,
                                          max_q_len, mass, mass_out, workspace_bytes)
    _no_grad(q)
    _check_cpu(codes, scales)
    H, D = codes.shape[1], codes.shape[4]
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] % H:
        raise ValueError("q must be [tokens, heads, head_dim], heads a multiple of the KV heads")
    G = q.shape[1] // H
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype)
    cu = cu_q.tolist()
    for i, n in enumerate(kv_lens.tolist()):
        rows = cu[i + 1] - cu[i]
        if rows > max_q_len:
            raise ValueError("a chunk is longer than max_q_len")
        blocks = -(-n // PAGE)
        pages = page_table[i, :blocks].long()
        x = codes[pages].float() * scales[pages][..., None, None]
        x = x.permute(2, 1, 0, 3, 4).reshape(2, H, blocks * PAGE, D)[:, :, :n]
        qs = q[cu[i]:cu[i + 1]].float().view(rows, H, G, D).permute(1, 2, 0, 3)
        s = torch.matmul(qs, x[0][:, None].transpose(-1, -2)) * scale     # [H, G, rows, n]
        seen = torch.arange(n) <= (n - rows + torch.arange(rows))[:, None]
        s = s.masked_fill(~seen, float("-inf"))
        # 0 at hidden tokens also where the row is NaN, and for rows that see nothing
        p = torch.where(seen, torch.softmax(s, -1), torch.zeros_like(s))
        # what is not finite reaches the rows that see it only, not the others as 0 * NaN
        bad = ~torch.isfinite(x[1])
        o = torch.matmul(p, x[1].masked_fill(bad, 0.0)[:, None])
        if bad.any():
            hit = torch.matmul(seen.float(), bad.float()) > 0                 # [H, rows, D]
            o = o.masked_fill(hit[:, None], float("nan"))
        out[cu[i]:cu[i + 1]] = o.permute(2, 0, 1, 3).reshape(rows, H * G, D).to(out.dtype)
        if mass is not None:
            w = torch.zeros(H, blocks * PAGE)
            w[:, :n] = p.sum((1, 2))
            slots = torch.arange(blocks * PAGE).view(blocks, 1, PAGE) < n
            new = mass[pages] + w.view(H, blocks, PAGE).transpose(0, 1)
            mass_out[pages] = torch.where(slots, new, mass_out[pages])
    return out


def paged8_evict(codes: torch.Tensor, scales: torch.Tensor, mass: torch.Tensor,
                 page_table: torch.Tensor, kv_lens: torch.Tensor, dst_table: torch.Tensor, *,
                 budget: int, recent: int) -> torch.Tensor:
    """Cut each sequence to ``budget`` tokens and move those to the pages of ``dst_table``.

    Of one layer, or (with a leading dimension) of all layers at once, every KV head keeps the
    last ``recent`` tokens and, of the older ones, the ``budget - recent`` with the largest
    ``mass`` (ties: the lowest index), in their order.  Sequences of at most ``budget`` tokens
    are moved whole.  A new block takes the largest scale among its tokens' old blocks; codes
    from blocks of a smaller scale are rounded anew.  The old pages are left as they are and
    must not be among the new ones.  Returns the kept indices
    ``[(layers,) S, Hkv, budget]`` int32, -1 past a sequence's kept tokens.
    """
    if not 0 <= recent <= budget or budget < 1:
        raise ValueError("need 0 <= recent <= budget and budget >= 1")
    if codes.is_cuda:
        return require().paged8_evict(codes, scales, mass, page_table, kv_lens, dst_table, budget,
                                      recent)
    _check_cpu(codes, scales)
    lead = codes.shape[:-5]
    S, H, D = page_table.shape[0], codes.shape[-4], codes.shape[-1]
    keep = torch.empty(*lead, S, H, budget, dtype=torch.int32, device=codes.device)
    layers = codes.shape[0] if lead else 1
    cs, ss, ms, ks = [x if lead else x[None] for x in (codes, scales, mass, keep)]
    ks.fill_(-1)
    for lay in range(layers):
        for i, n in enumerate(kv_lens.tolist()):
            kept, blocks = min(n, budget), -(-n // PAGE)
            if kept == 0:
                continue
            room = -(-kept // PAGE) * PAGE
            if room > dst_table.shape[1] * PAGE:
                raise ValueError("dst_table has too few pages")
            pages = page_table[i, :blocks].long()
            m = ms[lay, pages].transpose(0, 1).reshape(H, -1)[:, :n]
            # the recent tokens apart: no older mass, infinite or NaN, may take their place
            older = n - recent if n > budget else 0
            idx = m[:, :older].sort(dim=-1, descending=True, stable=True).indices
            idx = torch.cat((idx[:, :kept - (n - older)].sort(-1).values,
                             torch.arange(older, n).expand(H, -1)), -1)
            ks[lay, i, :, :kept] = idx.int()
            page, slot, head = pages[idx // PAGE], idx % PAGE, torch.arange(H)[:, None]
            old = ss[lay, page, head]                                   # [H, kept, 2]
            x = cs[lay].float()[page, head, :, slot]                    # [H, kept, 2, D]
            pad = (0, 0, 0, room - kept)
            s = torch.nn.functional.pad(old, pad).view(H, -1, PAGE, 2).amax(2)   # [H, blocks, 2]
            wide = s.repeat_interleave(PAGE, 1)[:, :kept]
            x = torch.nan_to_num(x * (old / torch.where(wide == 0, torch.ones_like(wide),
                                                        wide))[..., None])
            if codes.dtype == torch.int8:
                x = x.round()
            full = torch.zeros(H, room, 2, D)
            full[:, :kept] = x
            to = dst_table[i, :room // PAGE].long()
            cs[lay, to] = full.view(H, -1, PAGE, 2, D).permute(1, 0, 3, 2, 4).to(codes.dtype)
            ss[lay, to] = s.transpose(0, 1)
            got = torch.nn.functional.pad(torch.gather(m, 1, idx), (0, room - kept))
            ms[lay, to] = got.view(H, -1, PAGE).transpose(0, 1)
    return keep
