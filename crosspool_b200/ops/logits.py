"""Controls on logits, on the in-tree kernel (``csrc/kernels/logit_controls.cu``): penalties on the tokens that a row's prompt and
answer already hold, biases on listed tokens, and bit masks of the tokens that a grammar allows.

:func:`adjust_logits` stores the adjusted rows; :func:`select_tokens` reads the logits once and stores one token a row, greedily
or by temperature (the draw of :func:`crosspool_b200.ops.attention.sample`).
"""

from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from .. import native
from .overlap import rows_meet

_INT, _FLOAT = torch.int32, torch.float32
MAX_VOCAB = 1 << 20
_CALL = struct.Struct("6Q6i")      # what XpLogitArgs holds behind the controls


@dataclass(frozen=True)
class LogitControls:
    """What is done to the rows of a batch of logits; every tensor is optional and lives on the logits' device. Steps, in fp32 and
    in this order: ``v / repetition`` where ``v > 0`` and ``v * repetition`` elsewhere, for tokens of the history; minus ``frequency``
    times the occurrences behind the prompt; minus ``presence`` where there are any; plus the biases of the token; ``-inf`` where the
    mask does not allow it. Rows may name the same history, but then not bring a ``latest`` token for it.

    The tensors are read when a call runs: their contents may change between calls (and between replays of a captured graph)."""

    history: torch.Tensor | None = None        # int32 [slots, capacity] token ids; ids outside the vocabulary count for nothing
    lens: torch.Tensor | None = None           # int32 [rows] tokens of the history in use
    prompt_lens: torch.Tensor | None = None    # int32 [rows] how many of them are the prompt's (None: 0)
    history_rows: torch.Tensor | None = None   # int32 [rows] slot of each row (None: row r is slot r; negative: no history)
    latest: torch.Tensor | None = None         # int32 [rows] the last of the `lens` tokens, which the call stores into the history
    repetition: torch.Tensor | None = None     # fp32 [rows]
    frequency: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None       # int32 [entries], the rows' entries one after the other
    bias_values: torch.Tensor | None = None    # fp32 [entries]; entries of one token add up
    bias_starts: torch.Tensor | None = None    # int32 [rows + 1]
    masks: torch.Tensor | None = None          # int32 [masks, words] bit i % 32 of word i / 32: token i is allowed
    mask_index: torch.Tensor | None = None     # int32 [rows] mask of each row (outside the masks: none)

    def __post_init__(self) -> None:
        s = native.LogitArgs()
        for name, dtype, dims in (("history", _INT, 2), ("history_rows", _INT, 1), ("lens", _INT, 1), ("prompt_lens", _INT, 1), ("latest", _INT, 1),
                                  ("repetition", _FLOAT, 1), ("frequency", _FLOAT, 1), ("presence", _FLOAT, 1), ("bias_ids", _INT, 1),
                                  ("bias_values", _FLOAT, 1), ("bias_starts", _INT, 1), ("masks", _INT, 2), ("mask_index", _INT, 1)):
            t = getattr(self, name)
            if t is None:
                continue
            if t.dtype != dtype or t.dim() != dims or (t.numel() and t.stride(-1) != 1):
                raise ValueError(f"{name} must be {dtype} with {dims} dimensions and contiguous rows")
            setattr(s, name, t.data_ptr() or None)
        if (self.history is None) != (self.lens is None):
            raise ValueError("history and lens come together")
        for name in ("prompt_lens", "history_rows", "latest", "repetition", "frequency", "presence"):
            if getattr(self, name) is not None and self.history is None:
                raise ValueError(f"{name} needs a history")
        given = [getattr(self, n) is not None for n in ("bias_ids", "bias_values", "bias_starts")]
        if any(given) and not all(given):
            raise ValueError("bias_ids, bias_values and bias_starts come together")
        if (self.masks is None) != (self.mask_index is None):
            raise ValueError("masks and mask_index come together")
        rows, devices = set(), set()
        for name in ("history_rows", "lens", "prompt_lens", "latest", "repetition", "frequency", "presence", "mask_index"):
            if getattr(self, name) is not None:
                rows.add(getattr(self, name).shape[0])
        for name in self.__dataclass_fields__:
            if getattr(self, name) is not None:
                devices.add(getattr(self, name).device)
        if self.bias_ids is not None:
            if self.bias_ids.shape != self.bias_values.shape or not self.bias_starts.shape[0]:
                raise ValueError("bias_ids and bias_values have an entry each, bias_starts one more than there are rows")
            rows.add(self.bias_starts.shape[0] - 1)
            s.bias_total = self.bias_ids.shape[0]
        if len(rows) > 1 or len(devices) > 1:
            raise ValueError(f"controls of {sorted(rows)} rows on {len(devices)} devices")
        for t in (self.history, self.masks):
            if t is not None and t.shape[0] > 1 and not t.shape[1] <= t.stride(0) < 2 ** 31:
                raise ValueError(f"rows of {t.shape[1]} words {t.stride(0)} apart")
        if self.history is not None:
            s.history_slots, s.history_cap, s.ld_history = *self.history.shape, self.history.stride(0)
            if self.history_rows is None and rows and self.history.shape[0] < max(rows):
                raise ValueError(f"{self.history.shape[0]} histories for {max(rows)} rows")
        if self.masks is not None:
            s.mask_count, s.ld_mask = self.masks.shape[0], self.masks.stride(0)
        object.__setattr__(self, "_fields", bytes(s)[:native.LogitArgs.logits.offset])
        object.__setattr__(self, "_rows", rows.pop() if rows else None)
        object.__setattr__(self, "_device", devices.pop() if devices else None)

    @property
    def rows(self) -> int | None:
        """Rows of logits that the controls belong to (None: no tensor says so)."""
        return self._rows


def _check(logits: torch.Tensor, c: LogitControls) -> tuple[int, int, int, int]:
    """Refuses what the kernel does not take; (rows, vocab, pitch, whether fp32)."""
    f32 = logits.dtype is _FLOAT
    if logits.dim() != 2 or not (f32 or logits.dtype is torch.bfloat16) or logits.stride(1) != 1:
        raise ValueError("logits must be bf16 or fp32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    ld = logits.stride(0) if rows > 1 else vocab
    if not vocab <= ld < 2 ** 31:
        raise ValueError(f"rows of {vocab} logits {ld} elements apart")
    if vocab > MAX_VOCAB:
        raise ValueError(f"{vocab} tokens: up to {MAX_VOCAB} are supported")
    if c._rows is not None and c._rows < rows:
        raise ValueError(f"controls of {c._rows} rows for {rows} rows of logits")
    if c._device is not None and c._device != logits.device:
        raise ValueError(f"controls on {c._device} for logits on {logits.device}")
    if c.masks is not None and c.masks.shape[0] and c.masks.shape[1] * 32 < vocab:
        raise ValueError(f"masks of {c.masks.shape[1]} words for {vocab} tokens")
    return rows, vocab, ld, f32


def _check_rows(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple[int, ...], dev: torch.device) -> None:
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be contiguous {dtype} {shape} on the logits' device")


def _launch(controls: LogitControls, call: bytes, dev) -> None:
    if dev.type != "cuda":
        raise ValueError("the kernel runs on a GPU")
    native.run_packed("xp_logit_controls", controls._fields + call, dev)


def adjust_logits(logits: torch.Tensor, controls: LogitControls, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The logits after ``controls``, rounded once to ``out``'s type (bf16 or fp32; by default the logits' own). ``out`` may be
    ``logits`` itself, or rows that none of theirs lies over."""
    rows, vocab, ld, f32 = _check(logits, controls)
    fresh = out is None
    if fresh:
        out = torch.empty_like(logits)
    if out.shape != logits.shape or out.dtype not in (torch.bfloat16, _FLOAT) or out.stride(1) != 1 or out.device != logits.device:
        raise ValueError("out must be bf16 or fp32 of the logits' shape, with contiguous rows, on their device")
    ld_out = out.stride(0) if rows > 1 else vocab
    if not vocab <= ld_out < 2 ** 31:
        raise ValueError(f"rows of {vocab} results {ld_out} elements apart")
    if not rows or not vocab:
        return out
    at, to = logits.data_ptr(), out.data_ptr()
    if at == to and (out.dtype is not logits.dtype or ld_out != ld):
        raise ValueError("adjusting in place keeps type and pitch")
    size, size_out = logits.element_size(), out.element_size()
    if not fresh and at != to and rows_meet(rows, at, size * ld, size * vocab, to, size_out * ld_out, size_out * vocab):
        raise ValueError("out may be the logits themselves, but must not lie over other rows of them")
    _launch(controls, _CALL.pack(at, to, 0, 0, 0, 0, rows, vocab, ld, ld_out, f32, out.dtype is _FLOAT), logits.device)
    return out


def select_tokens(logits: torch.Tensor, controls: LogitControls, temps: torch.Tensor | None = None, seeds: torch.Tensor | None = None, *,
                  out: torch.Tensor | None = None, values: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row from the logits after ``controls``: the largest one (ties go to the lower id), or where ``temps[r] > 0`` a
    draw from ``softmax(adjusted / temperature)`` with ``seeds`` int32 ``[rows, 2]`` as in
    :func:`crosspool_b200.ops.attention.sample`. ``values`` (fp32 ``[rows]``) receives the adjusted logit of the token. A row without
    an allowed token gives token 0 and the value ``-inf``; NaN is never the largest."""
    rows, vocab, ld, f32 = _check(logits, controls)
    dev = logits.device
    if vocab == 0:
        raise ValueError("logits of no tokens")
    if out is None:
        out = torch.empty(rows, dtype=_INT, device=dev)
    else:
        _check_rows("out", out, _INT, (rows,), dev)
    if values is not None:
        _check_rows("values", values, _FLOAT, (rows,), dev)
    if (temps is None) != (seeds is None):
        raise ValueError("temps and seeds come together")
    if temps is not None:
        _check_rows("temps", temps, _FLOAT, (rows,), dev)
        _check_rows("seeds", seeds, _INT, (rows, 2), dev)
    if rows:
        at = [0 if t is None else t.data_ptr() for t in (temps, seeds, out, values)]
        _launch(controls, _CALL.pack(logits.data_ptr(), 0, *at, rows, vocab, ld, 0, f32, 0), dev)
    return out
