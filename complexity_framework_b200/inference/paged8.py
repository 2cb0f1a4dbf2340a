"""Paged KV cache held in 8 bits, with eviction by accumulated attention weight.

``Paged8Pool`` / ``Paged8Batch`` / ``StaticDecode8Batch`` are ``PagePool`` / ``PagedBatch`` /
``StaticDecodeBatch`` over the operators of ``ops.paged8``: int8 or e4m3 codes with one fp32
scale for each 16-token page, KV head and K / V.  The cache takes half the bytes of a bf16 one,
and a decode step, which reads all of it once, half the time on it.

With ``track_mass`` every attention call adds the softmax weight each cached token receives to
its mass, and ``evict`` cuts sequences to a budget of tokens: each layer and KV head keeps its
most recent tokens and, of the older ones, those with the most mass.  A sequence then holds
fewer tokens than its positions count: ``lengths`` are cached tokens, ``dropped`` the evicted
ones, and a token's position is ``slot + dropped`` at the time it was appended (keys carry their
position in their rotation, so slots need not follow positions).
"""
from __future__ import annotations

import itertools
from typing import Dict, List, Sequence, Tuple

import torch

from ..ops import paged8 as ops
from .paged import OutOfPages, PagedBatch, PagePool, SeqChunk, StaticDecodeBatch

CODE_TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}

#: rows (new tokens x query heads of a KV head) up to which a sequence takes the decode kernel
#: (``kP8ShortRows`` of the kernels)
SHORT_ROWS = 64


class Paged8Pool(PagePool):
    """``num_pages`` pages for sequences, and ``evict_pages`` more that only ``evict`` takes: with
    a budget's worth of them one sequence at a time can be cut however full the pool is."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int = ops.PAGE, dtype=torch.bfloat16, device="cpu",
                 kv_dtype: str = "int8", track_mass: bool = False, evict_pages: int = 0):
        if kv_dtype not in CODE_TYPES:
            raise ValueError(f"kv_dtype must be one of {sorted(CODE_TYPES)}, got {kv_dtype!r}")
        if page_size != ops.PAGE:
            raise ValueError(f"the 8-bit cache has pages of {ops.PAGE} tokens, got {page_size}")
        self.device = torch.device(device)
        if self.device.type == "cuda":
            if head_dim not in (64, 128):
                raise ValueError(f"the 8-bit cache kernels take head_dim 64 or 128, got {head_dim}")
            if dtype not in (torch.bfloat16, torch.float16):
                raise ValueError(f"the 8-bit cache kernels take bf16 or fp16 models, got {dtype}")
        self.num_layers, self.num_kv_heads, self.head_dim = num_layers, num_kv_heads, head_dim
        num_pages += evict_pages
        self.num_pages, self.page_size, self.dtype, self.kv_dtype = num_pages, page_size, dtype, kv_dtype
        self.evict_pages = evict_pages
        shape = (num_layers, num_pages, num_kv_heads)
        self.codes = torch.zeros(*shape, 2, page_size, head_dim, dtype=CODE_TYPES[kv_dtype],
                                 device=self.device)
        self.scales = torch.zeros(*shape, 2, device=self.device)
        self.mass = torch.zeros(*shape, page_size, device=self.device) if track_mass else None
        self.free: List[int] = list(range(num_pages - 1, -1, -1))
        self.pages: Dict[int, List[int]] = {}
        self.lengths: Dict[int, int] = {}
        self.dropped: Dict[int, int] = {}
        # a number of its own for each time a sequence's pages were replaced
        self.moves: Dict[int, int] = {}
        self._move = itertools.count()

    def allocate_sequence(self, seq_id: int) -> None:
        super().allocate_sequence(seq_id)
        self.dropped[seq_id] = 0
        self.moves[seq_id] = next(self._move)

    def free_sequence(self, seq_id: int) -> None:
        super().free_sequence(seq_id)
        self.dropped.pop(seq_id, None)
        self.moves.pop(seq_id, None)

    def reserve(self, seq_id: int, new_tokens: int) -> None:
        if not self.can_reserve(seq_id, self.lengths[seq_id] + new_tokens):
            raise OutOfPages("KV page pool exhausted")
        super().reserve(seq_id, new_tokens)

    def can_reserve(self, seq_id, length_after: int, current: int = 0) -> bool:
        have = len(self.pages.get(seq_id, [])) if seq_id is not None else 0
        need = -(-length_after // self.page_size) - have
        return need <= max(0, len(self.free) - self.evict_pages)

    def truncate_sequence(self, seq_id: int, length: int) -> None:
        held = len(self.pages[seq_id])
        super().truncate_sequence(seq_id, length)
        if len(self.pages[seq_id]) < held:
            self.moves[seq_id] = next(self._move)

    def fork_sequence(self, src: int, dst: int) -> None:
        if dst in self.pages:
            self.free_sequence(dst)
        self.allocate_sequence(dst)
        n = self.lengths[src]
        self.reserve(dst, n)
        k = -(-n // self.page_size)
        if k:
            s_idx = torch.tensor(self.pages[src][:k], device=self.device)
            d_idx = torch.tensor(self.pages[dst][:k], device=self.device)
            for t in (self.codes.view(torch.uint8), self.scales, self.mass):
                if t is not None:
                    t[:, d_idx] = t[:, s_idx]
        self.lengths[dst] = n
        self.dropped[dst] = self.dropped[src]

    def memory_usage(self) -> Dict[str, float]:
        used = self.num_pages - len(self.free)
        per_page = sum(t[:, 0].numel() * t.element_size()
                       for t in (self.codes, self.scales, self.mass) if t is not None)
        return {"pages_used": used, "pages_total": self.num_pages,
                "gb_used": used * per_page / 1e9, "gb_total": self.num_pages * per_page / 1e9}

    def _table(self, seq_ids: Sequence[int]) -> torch.Tensor:
        width = max([1] + [len(self.pages[s]) for s in seq_ids])
        table = torch.zeros(len(seq_ids), width, dtype=torch.int32)
        for i, s in enumerate(seq_ids):
            table[i, :len(self.pages[s])] = torch.tensor(self.pages[s], dtype=torch.int32)
        return table.to(self.device)

    def read(self, seq_id: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The sequence's cached keys and values ``[L, Hkv, length, D]`` in the model's type."""
        n = self.lengths[seq_id]
        lens = torch.tensor([n], dtype=torch.int32, device=self.device)
        k, v = ops.paged8_read(self.codes, self.scales, self._table([seq_id]), lens, dtype=self.dtype)
        return k[:, 0, :, :n], v[:, 0, :, :n]

    def evict(self, seq_ids: Sequence[int], budget: int, recent: int) -> None:
        """Cut each sequence that holds more than ``budget`` tokens to ``budget``: its last
        ``recent`` tokens and the older ones of largest mass, by layer and KV head.  Takes the
        new pages from all that are free (``OutOfPages`` when they do not suffice) and returns
        the old ones, which are as many or more."""
        if self.mass is None:
            raise RuntimeError("eviction needs a pool with track_mass=True")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError("need 0 <= recent <= budget and budget >= 1")
        seqs = [s for s in seq_ids if self.lengths[s] > budget]
        if not seqs:
            return
        need = -(-budget // self.page_size)
        if need * len(seqs) > len(self.free):
            raise OutOfPages("no free pages to move the kept tokens to")
        new = [[self.free.pop() for _ in range(need)] for _ in seqs]
        dst = torch.tensor(new, dtype=torch.int32).to(self.device)
        lens = torch.tensor([self.lengths[s] for s in seqs], dtype=torch.int32).to(self.device)
        ops.paged8_evict(self.codes, self.scales, self.mass, self._table(seqs), lens, dst,
                         budget=budget, recent=recent)
        for s, pages in zip(seqs, new):
            self.free.extend(self.pages[s])
            self.pages[s] = pages
            self.dropped[s] += self.lengths[s] - budget
            self.lengths[s] = budget
            self.moves[s] = next(self._move)

    def batch(self, chunks: Sequence[SeqChunk]) -> "Paged8Batch":
        return Paged8Batch(self, chunks)

    def static_batch(self, size: int, max_pages: int, max_position: int) -> "StaticDecode8Batch":
        return StaticDecode8Batch(self, size, max_pages, max_position)


class _Attend8:
    """What the eager and the static batch share: the operators over ``page_table``, ``cu_q``
    and ``kv_lens``; ``new`` are the new tokens of each sequence."""

    def _groups(self, group: int) -> List[Tuple[int, int, int]]:
        """Runs of sequences (start, end, longest chunk) that take the same kernel: decode
        tokens and short chunks, or long ones."""
        got = self._runs.get(group)
        if got is None:
            got = []
            for i, n in enumerate(self.new):
                if got and (got[-1][2] * group <= SHORT_ROWS) == (n * group <= SHORT_ROWS):
                    got[-1] = (got[-1][0], i + 1, max(got[-1][2], n))
                else:
                    got.append((i, i + 1, n))
            self._runs[group] = got
        return got

    def _mass(self, layer: int):
        return None if self.pool.mass is None else self.pool.mass[layer]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        P = self.pool
        ops.paged8_append(k.to(P.dtype), v.to(P.dtype), P.codes[layer], P.scales[layer],
                          self.page_table, self.cu_q, self.kv_lens, max_q_len=max(self.new),
                          mass=self._mass(layer))

    def attend(self, layer: int, q: torch.Tensor, scale: float) -> torch.Tensor:
        P = self.pool
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        for a, e, longest in self._groups(q.shape[1] // P.num_kv_heads):
            ops.paged8_attention(q, P.codes[layer], P.scales[layer], self.page_table[a:e],
                                 self.cu_q[a:e + 1], self.kv_lens[a:e], scale=scale,
                                 max_q_len=longest, mass=self._mass(layer), out=out)
        return out

    def rope_target(self, layer: int):
        """Dense rows: the rotated keys and values are quantised from here."""
        P = self.pool
        k, v = torch.empty(2, 1, self.num_tokens, P.num_kv_heads, P.head_dim, dtype=P.dtype,
                           device=P.device)
        return self.rows, k, v

    def rope_done(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        self.write(layer, k[0], v[0])


class Paged8Batch(_Attend8, PagedBatch):
    """Per-step view of a ``Paged8Pool`` for a ragged batch (chunks start at positions; a
    sequence's cached tokens are its positions less the evicted ones)."""

    def __init__(self, pool: Paged8Pool, chunks: Sequence[SeqChunk]):
        self.pool, self.chunks = pool, list(chunks)
        dev = pool.device
        cu, pos, lens = [0], [], []
        for c in self.chunks:
            n = c.start + c.length - pool.dropped[c.seq_id]
            pool.reserve(c.seq_id, n - pool.lengths[c.seq_id])
            pos.extend(range(c.start, c.start + c.length))
            lens.append(n)
            cu.append(cu[-1] + c.length)
        self.num_tokens = cu[-1]
        self.max_position = max(pos) if pos else 0
        self._cu_host, self._lens = cu, lens
        self.positions = torch.tensor(pos, dtype=torch.long, device=dev)
        self.rows = torch.arange(self.num_tokens, device=dev)
        self.cu_q = torch.tensor(cu, dtype=torch.int32, device=dev)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.page_table = pool._table([c.seq_id for c in self.chunks])
        self.new = [c.length for c in self.chunks]
        self._runs: Dict[int, List[Tuple[int, int, int]]] = {}

    def commit(self) -> None:
        for c, n in zip(self.chunks, self._lens):
            self.pool.lengths[c.seq_id] = max(self.pool.lengths[c.seq_id], n)


class StaticDecode8Batch(_Attend8, StaticDecodeBatch):
    """``StaticDecodeBatch`` over a ``Paged8Pool``.  Padding rows have no cached tokens: they
    write nothing and attend to nothing, so no scratch page is held."""

    def __init__(self, pool: Paged8Pool, size: int, max_pages: int, max_position: int):
        self.pool, self.size, self.max_pages = pool, size, max_pages
        dev, B = pool.device, size
        n = B * (3 + max_pages)  # ids | positions | kv_lens | page table [size, max_pages]
        self.host = torch.zeros(n, dtype=torch.int32).pin_memory()
        self._h = self.host.numpy()
        self.dev = torch.zeros(n, dtype=torch.int32, device=dev)
        self.ids32, self._pos32 = self.dev[0:B], self.dev[B:2 * B]
        self.kv_lens = self.dev[2 * B:3 * B]
        self.page_table = self.dev[3 * B:].view(B, max_pages)
        self.max_position, self.num_tokens = max_position, B
        self.new = [1] * B
        self._runs: Dict[int, List[Tuple[int, int, int]]] = {}
        self.cu_q = torch.arange(B + 1, dtype=torch.int32, device=dev)
        self.rows = torch.arange(B, device=dev)
        self.positions = torch.zeros(B, dtype=torch.long, device=dev)
        self.ids = torch.zeros(B, dtype=torch.long, device=dev)
        self._row_seq = [None] * B   # (sequence, its last move) of each row
        self._row_pages = [0] * B    # pages of that sequence already in the table row
        self._live = []

    def _set_padding(self, i: int) -> None:
        B, mp, h = self.size, self.max_pages, self._h
        h[i] = h[B + i] = h[2 * B + i] = 0
        h[3 * B + i * mp:3 * B + (i + 1) * mp] = 0
        self._row_seq[i], self._row_pages[i] = None, 0

    def expand(self) -> None:
        self.positions.copy_(self._pos32)
        self.ids.copy_(self.ids32)

    def fill(self, entries) -> None:
        """``entries[i] = (seq_id, token, position)`` for row i, the rest padding."""
        P = self.pool
        B, mp, h = self.size, self.max_pages, self._h
        if len(entries) > B:
            raise ValueError(f"{len(entries)} requests for a decode batch of {B}")
        self._live = []
        for i in range(B):
            if i >= len(entries):
                if self._row_seq[i] is not None:
                    self._set_padding(i)
                continue
            sid, tok, t = entries[i]
            who = (sid, P.moves[sid])
            if self._row_seq[i] != who:
                self._set_padding(i)
                self._row_seq[i] = who
            n = t + 1 - P.dropped[sid]
            P.reserve(sid, n - P.lengths[sid])
            pages = P.pages[sid]
            if len(pages) > mp:
                raise ValueError(f"sequence {sid} needs {len(pages)} pages; the graph holds {mp}")
            for j in range(self._row_pages[i], len(pages)):
                h[3 * B + i * mp + j] = pages[j]
            self._row_pages[i] = len(pages)
            h[i], h[B + i], h[2 * B + i] = tok, t, n
            self._live.append((sid, n))
        self.dev.copy_(self.host, non_blocking=True)

    def commit(self) -> None:
        for sid, n in self._live:
            self.pool.lengths[sid] = max(self.pool.lengths[sid], n)
