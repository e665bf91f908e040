"""What requests of one batch share, or bring of their own, beside their prompts: shared prompt prefixes in decode attention,
low-rank adapters beside the attention projections, and controls on the logits.

Each class here owns the static device buffers of one of them and their pinned mirrors; the engine fills the mirrors before a pass,
copies them on its stream, and the captured decode graphs read them.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable

import numpy as np
import torch

from ..ops import attention as A
from ..ops import logits as L
from ..ops import lora


class RequestFailed(RuntimeError):
    """What one request brought along failed in the step of all (``__cause__``: its error). Nothing was launched: the step can be taken
    again, or without the request (``AttentionEngine.drop_request(sequence)``)."""

    def __init__(self, sequence, error: Exception):
        super().__init__(str(error))
        self.sequence, self.__cause__ = sequence, error


# ---------------------------------------------------------------------------------------------- shared prefixes

DEEPEST = 64      # groups within groups that are looked at


def shared_groups(tables: list[list[int]]) -> tuple[list[int], list[int], list[int]]:
    """Groups of sequences whose page tables begin alike: (order of the sequences, sizes of the groups, pages that each shares).
    Groups follow one another in the order; sequences that share nothing are groups of one with no pages. Where a group contains
    smaller ones that share more, the split that saves the most page reads is taken."""
    order = sorted(range(len(tables)), key=lambda i: tables[i])
    alike = []
    for a, b in zip(order, order[1:]):
        x, y, n = tables[a], tables[b], 0
        while n < len(x) and n < len(y) and x[n] == y[n]:
            n += 1
        alike.append(n)

    def split(lo: int, hi: int, depth: int = 0) -> tuple[int, list[tuple[int, int]]]:
        """(pages saved, [(size, pages)]) for the sequences [lo, hi) of the order."""
        if hi - lo == 1:
            return 0, [(1, 0)]
        common = min(alike[lo:hi - 1])
        one = ((hi - lo - 1) * common, [(hi - lo, common)])
        if common > 0 and (depth >= DEEPEST or len(set(alike[lo:hi - 1])) == 1):
            return one
        saved, parts, start = 0, [], lo
        for i in range(lo, hi):
            if i == hi - 1 or alike[i] == common:
                s, p = split(start, i + 1, depth + 1)
                saved, start = saved + s, i + 1
                parts += p
        return one if one[0] >= saved and common > 0 else (saved, parts)

    groups = split(0, len(tables))[1] if tables else []
    return order, [n for n, _ in groups], [p for _, p in groups]


class PrefixRows:
    """Plans of shared prefixes for the decode row buckets of an engine."""

    PARTS = 8        # pieces of a prefix, at most: a bound of the workspace

    def __init__(self, cfg, ecfg, buckets: list[int], max_len: int, device):
        self.cfg, self.page, self.max_len = cfg, ecfg.page_size, max_len
        self.heads = dict(q_heads=cfg.num_q_heads, kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim)
        most = max(A.shared_plan_words(b, self._pieces(b)) for b in buckets)
        self.words = torch.zeros(most, dtype=torch.int32, device=device)
        self.host = torch.zeros(most, dtype=torch.int32).pin_memory()
        self.plans = {b: A.SharedPrefixPlan(self.words[:A.shared_plan_words(b, self._pieces(b))], b, self._pieces(b), self.PARTS, max_len, **self.heads)
                      for b in buckets}
        self.ws = torch.zeros(max(p.workspace_floats(b) for b, p in self.plans.items()), dtype=torch.float32, device=device)
        self.dirty = False

    @staticmethod
    def _pieces(rows: int) -> int:
        return 148 + 2 * rows          # a piece per SM, and room for every group's last ones

    def order(self, batch: list, tables: list[list[int]], rows: int) -> list:
        """The batch with sequences that share pages side by side; fills the plan of the row bucket ``rows``."""
        order, sizes, pages = shared_groups(tables)
        prefixes = [p * self.page for p in pages]
        n = A.shared_plan_words(rows, self._pieces(rows))
        own = sum(batch[i].total_len for i in order) - sum(s * p for s, p in zip(sizes, prefixes))
        A.fill_shared_plan(sizes, prefixes, self.host.numpy()[:n], rows, self._pieces(rows), self.PARTS, own_tokens=max(own, 0), **self.heads)
        self.dirty = True
        return [batch[i] for i in order]

    def copy(self) -> None:
        """On the engine's stream, before the pass."""
        if self.dirty:
            self.words.copy_(self.host, non_blocking=True)
            self.dirty = False


# ---------------------------------------------------------------------------------------------- adapters

PROJECTIONS = ("q", "k", "v", "o")


class AdapterRows:
    """Adapters of the attention projections by name, and the plan of which row uses which. ``cfg``: the engine's model."""

    def __init__(self, cfg, slots: int, max_rank: int, decode_rows: int, prefill_rows: int, device):
        self.cfg, self.slots = cfg, slots
        self.qkv = [lora.AdapterStack(slots, cfg.hidden_size, (cfg.q_size, cfg.kv_size, cfg.kv_size), max_rank, device) for _ in range(cfg.num_layers)]
        self.o = [lora.AdapterStack(slots, cfg.q_size, cfg.hidden_size, max_rank, device) for _ in range(cfg.num_layers)]
        self.names: dict[str, int] = {}
        self.loads = 0
        self.generation: dict[str, int] = {}       # of the load a name stands for: cached prefixes of another one do not count
        words = lora.plan_words(max(decode_rows, prefill_rows))
        self.words = torch.zeros(words, dtype=torch.int32, device=device)
        self.host = torch.zeros(words, dtype=torch.int32).pin_memory()

    def load(self, name: str, layers: list[dict[str, tuple[torch.Tensor, torch.Tensor]]], scale: float = 1.0) -> None:
        """``layers[l]``: {projection: (A ``[rank, in]``, B ``[out, rank]``)} for any of ``q``, ``k``, ``v`` and ``o``."""
        if name in self.names:
            raise ValueError(f"adapter {name!r} is loaded")
        if len(layers) != self.cfg.num_layers:
            raise ValueError(f"{len(layers)} layers for a model of {self.cfg.num_layers}")
        for l in layers:
            if set(l) - set(PROJECTIONS):
                raise ValueError(f"projections {sorted(set(l) - set(PROJECTIONS))}: {', '.join(PROJECTIONS)} are supported")
        free = sorted(set(range(self.slots)) - set(self.names.values()))
        if not free:
            raise ValueError(f"all {self.slots} adapter slots are taken")
        none = (None, None)
        for l, qkv, o in zip(layers, self.qkv, self.o):
            a, b = zip(*(l.get(p, none) for p in ("q", "k", "v")))
            qkv.load(free[0], a, b, scale)
            o.load(free[0], *([x] for x in l.get("o", none)), scale)
        self.loads += 1
        self.names[name], self.generation[name] = free[0], self.loads

    def unload(self, name: str) -> None:
        slot = self.names.pop(name)
        for s in (*self.qkv, *self.o):
            s.clear(slot)

    def fill(self, index: list[int], rows: int) -> int:
        """Writes the plan of a pass over ``rows`` rows to the pinned mirror (``index``: slots of the first rows); number of items."""
        n = lora.plan_words(rows)
        return lora.fill_plan(index + [-1] * (rows - len(index)), self.host.numpy()[:n], rows, bare=False, ranks=self.qkv[0].used)

    def copy(self, rows: int) -> None:
        n = lora.plan_words(rows)
        self.words[:n].copy_(self.host[:n], non_blocking=True)

    def plan(self, rows: int, max_items: int) -> lora.AdapterPlan:
        return lora.AdapterPlan(self.words[:lora.plan_words(rows)], rows, max_items, self.slots)


# ---------------------------------------------------------------------------------------------- controls

@dataclass(frozen=True)
class TokenControls:
    """Controls on the tokens of one request. ``repetition`` (1: none), ``frequency``, ``presence`` and ``bias`` as in
    :class:`~crosspool_b200.ops.logits.LogitControls`. ``allowed``: called with the generated tokens before every token; gives the
    mask of the next one as ``ceil(vocab / 32)`` 32-bit words (bit i % 32 of word i / 32: token i), or None for no mask. Where it
    raises, or its mask has another shape or allows no token, the request fails (:class:`RequestFailed`), and no other does."""

    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: dict[int, float] = field(default_factory=dict)
    allowed: Callable[[list[int]], "np.ndarray | None"] | None = None

    @property
    def penalises(self) -> bool:
        return self.repetition != 1.0 or self.frequency != 0.0 or self.presence != 0.0

    def check(self, vocab: int, most_biases: int) -> None:
        # as the kernel gets them, in 32 bits
        try:
            with np.errstate(over="ignore", under="ignore"):
                values = np.array([self.repetition, self.frequency, self.presence, *self.bias.values()], dtype=np.float64).astype(np.float32)
        except (TypeError, ValueError, OverflowError) as e:
            raise ValueError(f"controls must be numbers: {e}") from None
        if not values[0] > 0:
            raise ValueError(f"repetition penalty {self.repetition} is not positive in 32 bits")
        if not np.isfinite(values).all():
            raise ValueError(f"a control of {values[~np.isfinite(values)][0]} in 32 bits")
        if len(self.bias) > most_biases:
            raise ValueError(f"{len(self.bias)} biases: up to {most_biases} are supported")
        if any(not 0 <= t < vocab for t in self.bias):
            raise ValueError(f"bias for a token outside [0, {vocab})")


class ControlRows:
    """Controls of the rows that a pass samples, histories of the sequences that have penalties."""

    MOST_BIASES = 300

    def __init__(self, rows: int, sequences: int, max_len: int, vocab: int, device):
        self.rows, self.vocab, self.max_len = rows, vocab, max_len
        self.words = (vocab + 31) // 32
        dev = dict(device=device)
        self.history = torch.zeros(sequences, max_len, dtype=torch.int32, **dev)
        self.history_host = torch.zeros(sequences, max_len, dtype=torch.int32).pin_memory()
        # slots | lens | prompt_lens | latest | mask_index | repetition | frequency | presence | bias_starts
        self.meta = torch.zeros(9 * rows + 1, dtype=torch.int32, **dev)
        self.meta_host = torch.zeros(9 * rows + 1, dtype=torch.int32).pin_memory()
        self.bias = torch.zeros(2, rows * self.MOST_BIASES, dtype=torch.int32, **dev)
        self.bias_host = torch.zeros(2, rows * self.MOST_BIASES, dtype=torch.int32).pin_memory()
        self.masks = torch.zeros(rows, self.words, dtype=torch.int32, **dev)
        self.masks_host = torch.zeros(rows, self.words, dtype=torch.int32).pin_memory()
        self.free = list(range(sequences - 1, -1, -1))
        self.slots: dict[int, int] = {}             # sequence -> history slot
        self.stored: dict[int, int] = {}            # sequence -> tokens of it that the device's history holds
        m = [self.meta[i * rows:(i + 1) * rows] for i in range(8)]
        f = [t.view(torch.float32) for t in m[5:]]
        self.controls = L.LogitControls(history=self.history, history_rows=m[0], lens=m[1], prompt_lens=m[2], latest=m[3], mask_index=m[4],
                                        repetition=f[0], frequency=f[1], presence=f[2], bias_ids=self.bias[0],
                                        bias_values=self.bias[1].view(torch.float32), bias_starts=self.meta[8 * rows:], masks=self.masks)
        self._neutral()
        self.meta.copy_(self.meta_host)

    def _neutral(self) -> None:
        h, n = self.meta_host.numpy(), self.rows
        h[:] = 0
        h[0:n] = h[3 * n:4 * n] = h[4 * n:5 * n] = -1
        h[5 * n:6 * n].view(np.float32)[:] = 1.0

    def release(self, seq_id: int) -> None:
        slot = self.slots.pop(seq_id, None)
        if slot is not None:
            self.free.append(slot)
            self.stored.pop(seq_id, None)

    def stage(self, seqs: list, samples: list[bool]) -> None:
        """Fills and copies the rows of a pass (on the engine's stream): ``seqs[i]`` samples its next token in row i unless
        ``samples[i]`` is False (a portion of a prompt that is not its last)."""
        # what may raise comes first: a step that failed here can be taken again
        words = [self.mask(s) if wanted and s.controls is not None and s.controls.allowed is not None else None for s, wanted in zip(seqs, samples)]
        self._neutral()
        n, h = self.rows, self.meta_host.numpy()
        f, ids, vals = h[5 * n:8 * n].view(np.float32).reshape(3, n), self.bias_host[0].numpy(), self.bias_host[1].numpy().view(np.float32)
        biases = masks = 0
        for i, (s, wanted) in enumerate(zip(seqs, samples)):
            h[8 * n + i] = biases
            c = s.controls
            if c is None or not wanted:
                continue
            if c.penalises:
                self._history(i, s, h)
                f[0, i], f[1, i], f[2, i] = c.repetition, c.frequency, c.presence
            for t, v in c.bias.items():
                ids[biases], vals[biases] = t, v
                biases += 1
            if words[i] is not None:
                self.masks_host[masks].numpy()[:] = words[i]
                h[4 * n + i] = masks
                masks += 1
        h[8 * n + len(seqs):] = biases
        self.meta.copy_(self.meta_host, non_blocking=True)
        if biases:
            self.bias[:, :biases].copy_(self.bias_host[:, :biases], non_blocking=True)
        if masks:
            self.masks[:masks].copy_(self.masks_host[:masks], non_blocking=True)

    def mask(self, s) -> "np.ndarray | None":
        """The mask of a sequence's next token; :class:`RequestFailed` where the request gives none that a token fits."""
        try:
            words = s.controls.allowed(list(s.generated))
            if words is None:
                return None
            words = np.asarray(words)
            if words.shape != (self.words,):
                raise ValueError(f"a mask of shape {words.shape} for {self.vocab} tokens ({self.words} words)")
            # (a copy: the callback may fill the same buffer for the next sequence)
            words = words.copy() if words.dtype == np.int32 else words.astype(np.uint32).view(np.int32)
            if not words[:-1].any() and not int(words[-1]) & ((1 << (self.vocab - 1) % 32 + 1) - 1):
                raise ValueError("the mask allows no token")
            return words
        except Exception as e:
            raise RequestFailed(s, e)

    def _history(self, i: int, s, h: np.ndarray) -> None:
        """Row i's history: its slot gets the whole sequence once, then every call the token that the sequence grew by."""
        n, total = self.rows, s.total_len
        slot = self.slots.get(s.seq_id)
        if slot is None:
            slot = self.slots[s.seq_id] = self.free.pop()
        have = self.stored.get(s.seq_id, 0)
        if have == total - 1 and s.generated:
            h[3 * n + i] = s.generated[-1]
        elif have != total:
            row = self.history_host[slot]
            row.numpy()[:total] = s.prompt + s.generated
            self.history[slot, :total].copy_(row[:total], non_blocking=True)
        self.stored[s.seq_id] = total
        h[i], h[n + i], h[2 * n + i] = slot, total, len(s.prompt)
