"""Low-rank adapters of many requests beside a shared projection, on the in-tree kernel (``csrc/kernels/lora.cu``).

``lora_add(y, x, stack, plan)`` computes ``y[r] + scale[s] * (x[r] @ A[s].T) @ B[s].T`` for every row, ``s`` being the adapter
of row ``r``; rows without one keep ``y``. The adapters of one projection live in an :class:`AdapterStack`; which row uses which
is an :class:`AdapterPlan`, made once per batch and used by all layers and projections.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Sequence

import numpy as np
import torch

from .. import native
from .overlap import rows_meet

MAX_RANK = 128
MAX_PARTS = 4
_CALL, _PLAN = struct.Struct("3Q4i"), struct.Struct("3Q2i")      # XpLoraArgs: of a call, then of its plan, then of its stack
ITEM_ROWS = 16        # rows of one adapter that a cluster of CTAs takes at once; a plan's items hold at most so many


class AdapterStack:
    """The adapters of one projection, slot by slot in bf16, in the order in which the kernel's lanes read them
    (``XpLoraArgs``): ``a`` with room for ``[rank, in]`` of every part (``in`` padded to a multiple of 32), ``b`` for ``[out, rank]``, a
    scale and a rank per slot. ``out_features``: a number, or one per part of a fused projection (q, k and v: each part has an ``A``
    of its own). A slot's rank is its adapter's, padded with zeros to a multiple of 16 (``rank`` at most); its ``B`` lies without
    gaps, so that low ranks cost no more bytes than they have."""

    def __init__(self, slots: int, in_features: int, out_features: int | Sequence[int], max_rank: int, device: str | torch.device = "cuda"):
        self.parts = (int(out_features),) if isinstance(out_features, int) else tuple(int(n) for n in out_features)
        if slots < 1 or not 1 <= max_rank <= MAX_RANK or not 1 <= len(self.parts) <= MAX_PARTS:
            raise ValueError(f"{slots} slots, rank {max_rank}, {len(self.parts)} parts: at least one slot, ranks 1 to {MAX_RANK}, 1 to {MAX_PARTS} parts")
        if in_features < 1 or in_features % 8 or any(n < 1 or n % 8 for n in self.parts):
            raise ValueError(f"features {in_features} -> {self.parts}: multiples of 8 are supported")
        self.slots, self.in_features, self.out_features = slots, in_features, sum(self.parts)
        self.rank = (max_rank + 15) // 16 * 16
        self.a = torch.zeros(slots, len(self.parts), self.rank, (in_features + 31) // 32 * 32, dtype=torch.bfloat16, device=device)
        self.b = torch.zeros(slots, self.out_features * self.rank, dtype=torch.bfloat16, device=device)
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(slots, dtype=torch.int32, device=device)
        self.part_ranks = torch.zeros(slots, MAX_PARTS, dtype=torch.int32, device=device)
        self.device = self.a.device
        self._fresh = [True] * slots       # never loaded: still zero
        self.used = [0] * slots            # ranks in use, as in `ranks`
        end, ends = 0, []
        for n in self.parts:
            end += n
            ends.append(end)
        s = native.LoraArgs()
        s.a, s.b, s.scale, s.ranks = self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr(), self.ranks.data_ptr()
        s.part_ranks = self.part_ranks.data_ptr()
        s.k, s.n, s.rank, s.parts, s.slots = in_features, self.out_features, self.rank, len(self.parts), slots
        s.part_end = (C.c_int * 4)(*(ends + [end] * (4 - len(ends))))
        self._fields = bytes(s)[native.LoraArgs.a.offset:]
        if self.device.type == "cuda":          # a slot may be loaded on any stream from here on
            torch.cuda.current_stream(self.device).synchronize()

    @torch.no_grad()
    def load(self, slot: int, a: torch.Tensor | Sequence[torch.Tensor], b: torch.Tensor | Sequence[torch.Tensor], scale: float = 1.0) -> None:
        """Puts an adapter into ``slot``: ``a`` ``[r, in]`` and ``b`` ``[out, r]``, or one pair per part (``None`` for a part
        without one); ranks may differ between parts. Ordered with the work of the current stream."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        pa, pb = ([a], [b]) if isinstance(a, torch.Tensor) else (list(a), list(b))
        if len(pa) != len(self.parts) or len(pb) != len(self.parts):
            raise ValueError(f"{len(pa)} and {len(pb)} matrices for {len(self.parts)} parts")
        used = 0
        for n, x, y in zip(self.parts, pa, pb):
            if (x is None) != (y is None):
                raise ValueError("a part has both matrices or none")
            if x is None:
                continue
            r = x.shape[0]
            if x.dim() != 2 or y.dim() != 2 or not 1 <= r <= self.rank or tuple(x.shape) != (r, self.in_features) or tuple(y.shape) != (n, r):
                raise ValueError(f"matrices {tuple(x.shape)} and {tuple(y.shape)} for {self.in_features} -> {n} features, rank up to {self.rank}")
            used = max(used, r)
        if not self._fresh[slot]:
            self.a[slot].zero_()
            self.b[slot].zero_()
        self._fresh[slot] = False
        r16, at = (used + 15) // 16 * 16, 0
        for i, (n, x, y) in enumerate(zip(self.parts, pa, pb)):
            if x is not None:
                wide = torch.zeros(self.rank, self.a.shape[3], dtype=torch.bfloat16, device=self.device)
                wide[:x.shape[0], :self.in_features].copy_(x)
                self.a[slot, i].view(-1, self.rank, 32).copy_(wide.view(self.rank, -1, 32).transpose(0, 1))
                wide = torch.zeros(n, r16, dtype=torch.bfloat16, device=self.device)
                wide[:, :x.shape[0]].copy_(y)
                for f0, f1 in ((0, n // 32 * 32), (n // 32 * 32, n)):          # whole blocks, and a last one of fewer features
                    if f0 < f1:
                        e = min(f1 - f0, 32) // 8
                        block = wide[f0:f1].view(-1, e, 2, 2, 2, r16 // 16, 4, 4).permute(0, 5, 2, 1, 4, 6, 3, 7)
                        self.b[slot, (at + f0) * r16:(at + f1) * r16].view(block.shape).copy_(block)
            at += n
        self.scale[slot:slot + 1].fill_(float(scale))
        self.ranks[slot:slot + 1].fill_(r16)
        for i, x in enumerate(pa):
            self.part_ranks[slot, i].fill_(0 if x is None else x.shape[0])
        self.used[slot] = r16

    def clear(self, slot: int) -> None:
        """Empties ``slot``: rows that name it keep ``y``."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        self.ranks[slot:slot + 1].zero_()
        self.used[slot] = 0


def plan_words(rows: int) -> int:
    """32-bit words of a plan of up to ``rows`` rows."""
    return 4 + 5 * rows


def fill_plan(index: Sequence[int], words: np.ndarray, rows: int, bare: bool = True, ranks: Sequence[int] | None = None) -> int:
    """Writes the plan of ``index`` (adapter slot per row, negative: none) to ``words`` (``plan_words(rows)`` of them); returns its
    number of items. ``bare``: rows without an adapter get items too (they are copied when the result goes elsewhere). ``ranks``: of
    the slots; items of high ranks come first, so that the last ones to start are short."""
    idx = np.maximum(np.asarray(index, dtype=np.int64).reshape(-1), -1)
    order = np.argsort(idx, kind="stable")
    srt = idx[order]
    starts = np.flatnonzero(np.r_[True, srt[1:] != srt[:-1]]) if len(srt) else np.zeros(0, dtype=np.int64)
    counts = np.diff(np.r_[starts, len(srt)])
    pieces = -(-counts // ITEM_ROWS)
    run = np.repeat(np.arange(len(starts)), pieces)
    nth = np.arange(len(run)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
    first = starts[run] + nth * ITEM_ROWS
    n = np.minimum(ITEM_ROWS, counts[run] - nth * ITEM_ROWS)
    slot = srt[starts][run] if len(starts) else run
    if not bare:
        keep = slot >= 0
        first, n, slot = first[keep], n[keep], slot[keep]
    if ranks is not None and len(slot):
        cost = np.where(slot >= 0, np.asarray(ranks, dtype=np.int64)[np.maximum(slot, 0)], -1)
        by = np.argsort(-cost, kind="stable")
        first, n, slot = first[by], n[by], slot[by]
    items = words[4:4 + 4 * rows].reshape(rows, 4)
    items[:len(slot), 0], items[:len(slot), 1], items[:len(slot), 2] = slot, first, n
    words[4 + 4 * rows:4 + 4 * rows + len(order)] = order
    words[0] = len(slot)
    return len(slot)


class AdapterPlan:
    """Which adapter every row of a batch uses, in device memory (``words``), for up to ``rows`` rows. ``max_items`` bounds the
    items that the words may hold while the plan is in use (a captured graph replays with new words)."""

    def __init__(self, words: torch.Tensor, rows: int, max_items: int, slots: int):
        self.words, self.rows, self.max_items, self.slots = words, rows, max_items, slots
        base = words.data_ptr()
        self._fields = _PLAN.pack(base + 16, base, base + 16 + 16 * rows, max_items, 0)


def adapter_plan(index: Sequence[int], stack: "AdapterStack | int", device: str | torch.device | None = None) -> AdapterPlan:
    """The plan of a batch whose row ``r`` uses adapter slot ``index[r]`` (negative: none), for stacks of as many slots as ``stack``
    has (or is)."""
    slots = stack.slots if isinstance(stack, AdapterStack) else int(stack)
    if device is None:
        device = stack.device if isinstance(stack, AdapterStack) else "cuda"
    rows = len(index)
    if rows and max(index) >= slots:
        raise ValueError(f"adapter slot {max(index)} of {slots}")
    host = np.zeros(plan_words(rows), dtype=np.int32)
    n = fill_plan(index, host, rows, ranks=stack.used if isinstance(stack, AdapterStack) else None)
    return AdapterPlan(torch.from_numpy(host).to(device), rows, n, slots)


def lora_add(y: torch.Tensor, x: torch.Tensor, stack: AdapterStack, plan: AdapterPlan, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[rows, out] + scale * (x[rows, in] @ A.T) @ B.T`` with every row's own adapter, rounded once; sums in fp32. ``out`` may
    be ``y`` itself, or rows that no row of ``x`` or ``y`` lies over. bf16; rows may have a pitch (a multiple of 8 elements), so that a
    slice of a wider buffer can be read or written."""
    rows, fresh = x.shape[0], out is None
    if fresh:
        out = torch.empty_like(y)
    if x.shape != (rows, stack.in_features) or y.shape != (rows, stack.out_features) or out.shape != y.shape:
        raise ValueError(f"x {tuple(x.shape)}, y {tuple(y.shape)}, out {tuple(out.shape)} beside a {stack.in_features} -> {stack.out_features} stack")
    if rows != plan.rows or plan.slots > stack.slots:
        raise ValueError(f"a plan of {plan.rows} rows and {plan.slots} slots for {rows} rows and {stack.slots} slots")
    dev, bf16 = stack.device, torch.bfloat16
    for t in (x, y, out):
        if t.dtype is not bf16 or t.device != dev:
            raise ValueError(f"{t.dtype} on {t.device}: bf16 on the stack's device ({dev}) is supported")
    at_x, at_y, at_out = x.data_ptr(), y.data_ptr(), out.data_ptr()
    (ld_x, one_x), (ld_y, one_y), (ld_out, one_out) = x.stride(), y.stride(), out.stride()
    if not one_x == one_y == one_out == 1 or (at_x | at_y | at_out) & 15 or (rows > 1 and ((ld_x | ld_y | ld_out) & 7 or max(ld_x, ld_y, ld_out) >> 31)):
        raise ValueError("rows must be contiguous, 16-byte aligned, with pitches of whole 16 bytes")
    if rows > 1 and (ld_out < stack.out_features or (at_out == at_y and ld_out != ld_y)):
        raise ValueError("the rows of out must not overlap one another or other rows of y")
    if plan.words.device != dev:
        raise ValueError("the plan lives on another device")
    wide = 2 * stack.out_features
    if not fresh and ((at_out != at_y and rows_meet(rows, at_out, 2 * ld_out, wide, at_y, 2 * ld_y, wide))
                 or rows_meet(rows, at_out, 2 * ld_out, wide, at_x, 2 * ld_x, 2 * stack.in_features)):
        raise ValueError("out may be y, but not x, and lie over neither")
    if dev.type != "cuda":
        raise ValueError("the kernel runs on a GPU")
    if rows <= 1:
        ld_x = ld_y = ld_out = 0
    native.run_packed("xp_lora", _CALL.pack(at_x, at_y, at_out, rows, ld_x, ld_y, ld_out) + plan._fields + stack._fields, dev)
    return out
