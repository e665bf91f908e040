"""Attention-side operators on the in-tree kernels: q/k-norm + RoPE + paged KV write, paged decode
attention (split-KV) and chunked causal prefill attention over the paged cache, embedding gather and
greedy sampling. The reference owns none of these (SGLang/FlashInfer do, pyproject.toml:17-35); the
oracles are plain fp32 PyTorch restatements in ``tests/``.
"""

from __future__ import annotations

import ctypes as C
import os
import math
import struct
from typing import Sequence

import numpy as np
import torch

from .. import native
from .gemm import status_words


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def rope_kv_write(qkv: torch.Tensor, q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  positions: torch.Tensor, slots: torch.Tensor, *, q_heads: int, kv_heads: int, head_dim: int,
                  theta: float, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                  eps: float = 1e-6) -> None:
    """qkv ``[rows, (q+2kv)*d]`` → RoPE'd q in ``q_out`` and k/v scattered to the paged cache."""
    a = rope_args(qkv, q_out, k_cache, v_cache, positions, slots, q_heads, kv_heads, head_dim, theta, q_norm, k_norm, eps)
    native.check(native.kernels().xp_rope_kv(C.byref(a), _stream(qkv.device)), "xp_rope_kv")


def rope_args(qkv, q_out, k_cache, v_cache, positions, slots, q_heads, kv_heads, head_dim, theta, q_norm, k_norm, eps) -> "native.RopeArgs":
    a = native.RopeArgs()
    a.qkv, a.q_out = qkv.data_ptr(), q_out.data_ptr()
    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    a.q_norm_weight = q_norm.data_ptr() if q_norm is not None else None
    a.k_norm_weight = k_norm.data_ptr() if k_norm is not None else None
    assert positions.dtype == torch.int32 and slots.dtype == torch.int32
    a.positions, a.slots = positions.data_ptr(), slots.data_ptr()
    a.rows, a.ld_qkv = qkv.shape[0], qkv.stride(0)
    a.q_heads, a.kv_heads, a.head_dim = q_heads, kv_heads, head_dim
    a.eps, a.log2_theta = eps, math.log2(theta)
    return a


def decode_splits(batch: int, kv_heads: int, max_len: int) -> int:
    return native.kernels().xp_decode_attn_splits(batch, kv_heads, max_len)


# Which prefill kernel runs when the caller does not say: "umma" (tcgen05 tensor cores, TMEM accumulators; shapes it
# does not cover fall back to "mma"), "mma" (TMA-fed mma.sync kernel) or "simple" (plain mma.sync kernel).
# "umma-alt" is the tcgen05 kernel with the other route for the probabilities (tensor memory <-> shared memory).
# XPOOL_PREFILL_KERNEL selects one, e.g. to bisect a numerical difference.
PREFILL_KERNELS = {"umma": 0, "simple": 1, "mma": 2, "umma-alt": 0x100}
PREFILL_KERNEL_DEFAULT = os.environ.get("XPOOL_PREFILL_KERNEL", "umma")


def decode_plan(batch: int, kv_heads: int, max_len: int) -> tuple[int, int]:
    """(num_splits, chunk_tokens) for a decode batch.

    A CTA covers one (sequence, KV head, slice); its fixed cost (first TMA round trip, cross-warp merge,
    partial write + merge kernel) is amortised best by long slices, so sequences are only cut when there
    are too few (sequence, head) pairs to fill the 148 SMs a few times over. Measured on B200 (16 q / 8 kv
    heads, d 128, lengths 128-2048): batch 256 reaches 0.92 of copy bandwidth unsplit, 0.87 with 512-token
    slices, 0.77 with 256-token slices."""
    pairs = batch * kv_heads
    if pairs >= 1024 or max_len <= 512:
        return 1, 0
    chunk = 1024 if pairs >= 256 else 512 if pairs >= 64 else 256
    if max_len <= chunk:
        return 1, 0
    return (max_len + chunk - 1) // chunk, chunk


def window_plan(batch: int, kv_heads: int, seen: int) -> tuple[int, int]:
    """(num_splits, chunk_tokens) for rows that see a window of ``seen`` tokens at most (first tokens and the edges of 16-token
    tiles included): slices of equal length, and only while (row, head) pairs leave SMs idle. Measured on B200 with 8 KV heads
    and 1104 tokens: one slice from 64 rows on, four for 1 and 8 rows."""
    splits = min(max(1, 256 // (batch * kv_heads)), (seen + 287) // 288)
    return (splits, (seen + splits * 16 - 1) // (splits * 16) * 16) if splits > 1 else (1, 0)


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, *, out: torch.Tensor | None = None, num_splits: int = 0,
                 ws: torch.Tensor | None = None, scale: float | None = None, max_len: int | None = None,
                 chunk_tokens: int = 0, force_simt: bool = False) -> torch.Tensor:
    """q ``[batch, q_heads, d]`` against caches ``[pages, page, kv_heads, d]``.

    Runs the tensor-core kernel (TMA-fed ``mma`` tiles) whenever pages hold a multiple of 16 tokens
    and at most 16 query heads share a KV head; ``force_simt`` selects the plain kernel."""
    batch, q_heads, d = q.shape
    page_size, kv_heads = k_cache.shape[1], k_cache.shape[2]
    if out is None:
        out = torch.empty_like(q)
    if num_splits <= 0:
        num_splits = decode_splits(batch, kv_heads, max_len or block_table.shape[1] * page_size)
    if num_splits > 1 and ws is None:
        ws = torch.empty(batch * q_heads * num_splits * (d + 2), dtype=torch.float32, device=q.device)
    a = native.DecodeAttnArgs()
    a.q, a.k_cache, a.v_cache, a.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    a.ws = ws.data_ptr() if ws is not None else None
    assert block_table.dtype == torch.int32 and seq_lens.dtype == torch.int32
    a.block_table, a.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
    a.batch, a.q_heads, a.kv_heads, a.head_dim = batch, q_heads, kv_heads, d
    a.page_size, a.max_blocks, a.num_splits = page_size, block_table.stride(0), num_splits
    a.scale = scale if scale is not None else d ** -0.5
    a.chunk_tokens = chunk_tokens
    a.num_pages = k_cache.shape[0] if k_cache.is_contiguous() and v_cache.is_contiguous() else 0
    a.force_simt = int(force_simt)
    from .gemm import status_words

    a.status = status_words(q.device).data_ptr()
    native.check(native.kernels().xp_decode_attn(C.byref(a), _stream(q.device)), "xp_decode_attn",
                 2 if num_splits > 1 else 1)
    return out


# ---------------------------------------------------------------------------------------------- shared prefixes

PREFIX_TOKENS = 16      # prefixes are shared in whole tiles of so many tokens; the rest of one is read by every row
PIECE_TOKENS = 128      # pieces of a prefix begin at multiples of this
MAX_PARTS = 32          # pieces of one prefix
MAX_SHARED_ROWS = 4096  # rows of a batch
_SHARED_CALL = struct.Struct("7Q7if2iQ2i")   # XpDecodeAttnArgs, which begins XpDecodeSharedArgs


def own_slots(rows: int, q_heads: int, kv_heads: int) -> int:
    """Shares that a row's own tokens may be cut into: the grid's workers (twelve warps on each of 148 SMs) take even shares of all
    own tokens, and a long row among short ones needs more of them than the rows of an even batch."""
    units = max(1, rows) * kv_heads * (2 if q_heads // kv_heads > 8 else 1)
    return min(64, max(8, -(-2 * 12 * 148 // units)))


def piece_rows(q_heads: int, kv_heads: int) -> int:
    """Rows that one piece of a prefix may hold: two tiles of 128 query heads of a KV head."""
    return 2 * (128 // (q_heads // kv_heads))


def prefix_piece_tokens(groups: Sequence[tuple[int, int]], kv_heads: int, rows_per_piece: int, own_tokens: int = 0, head_dim: int = 128,
                        q_heads: int = 0, num_sms: int = 148) -> int:
    """Tokens of a prefix that a CTA takes at once, for ``groups`` of (rows, prefix tokens) and about ``own_tokens`` behind them: the
    split with the least estimated time. The SMs that take pieces need the longest unit's time and stream own tokens afterwards,
    the others stream from the start; every part of a prefix is one more result to store and merge. Microseconds, as measured on
    B200 with heads of 128: a unit 3.5 and 1.9 per 128 tokens; 80 KB a us and SM streamed, 5.7 MB in all."""
    tiles = [(-(-n // rows_per_piece), p) for n, p in groups]
    own = own_tokens * kv_heads * head_dim * 4
    rows = sum(n for n, _ in groups)
    longest = max(p for _, p in tiles)
    best, best_cost, c = PIECE_TOKENS, None, PIECE_TOKENS
    while True:
        parts = -(-longest // c)
        if parts <= MAX_PARTS:
            units = kv_heads * sum(t * -(-p // c) for t, p in tiles)
            turns = -(-units // num_sms)
            busy, piece = -(-units // turns), turns * (3.5 + 1.9 * -(-min(c, longest) // PIECE_TOKENS))
            left = own - (num_sms - busy) * piece * 80e3                # streamed by all SMs behind the pieces
            cost = max(piece + (4.0 + left / 5.3e6 if left > 0 else 0.0), own / 5.7e6) + parts * (0.15 + rows * max(q_heads, kv_heads) * (head_dim + 2) * 8 / 5e6)
            if best_cost is None or cost < best_cost:
                best, best_cost = c, cost
        if c >= longest:
            return best
        c += max(PIECE_TOKENS, c // 8 // PIECE_TOKENS * PIECE_TOKENS)


def shared_plan_words(rows: int, max_pieces: int) -> int:
    """32-bit words of a plan for up to ``rows`` rows and ``max_pieces`` pieces."""
    return 4 + 8 * max_pieces + 2 * rows


def fill_shared_plan(sizes: Sequence[int], prefixes: Sequence[int], words: np.ndarray, rows: int, max_pieces: int, max_parts: int, *,
                     q_heads: int, kv_heads: int, head_dim: int = 128, own_tokens: int = 0) -> tuple[int, int]:
    """Writes the plan of consecutive groups of rows (``sizes``) with ``prefixes`` tokens shared in each to ``words``; returns its
    number of pieces and the most pieces of a row. Prefixes are cut so that neither exceeds its bound. ``own_tokens``: about how many
    tokens all rows have behind their prefixes."""
    per = piece_rows(q_heads, kv_heads)
    pieces = words[4:4 + 8 * max_pieces].reshape(max_pieces, 8)
    shared, parts = words[4 + 8 * max_pieces:][:rows], words[4 + 8 * max_pieces + rows:][:rows]
    shared[:], parts[:] = 0, 0
    groups, at = [], 0
    for n, p in zip(sizes, prefixes):
        p = p // PREFIX_TOKENS * PREFIX_TOKENS
        if n > 0 and p > 0:
            groups.append((at, n, p))
        at += n
    if not groups:
        words[0] = words[1] = 0
        return 0, 0
    longest = max(p for _, _, p in groups)
    c = prefix_piece_tokens([(n, p) for _, n, p in groups], kv_heads, per, own_tokens, head_dim, q_heads)
    while -(-longest // c) > max_parts or sum(-(-n // per) * -(-p // c) for _, n, p in groups) > max_pieces:
        if c >= longest:
            raise ValueError(f"{len(groups)} groups do not fit a plan of {max_pieces} pieces and {max_parts} parts")
        c += max(PIECE_TOKENS, c // 8 // PIECE_TOKENS * PIECE_TOKENS)
    count = most = tokens = 0
    for at, n, p in groups:
        k = -(-p // c)
        size = -(-p // (k * PIECE_TOKENS)) * PIECE_TOKENS          # even pieces
        k = -(-p // size)
        shared[at:at + n], parts[at:at + n] = p, k
        for r in range(at, at + n, per):
            m = min(per, at + n - r)
            for i in range(k):
                pieces[count] = (at, r, m, i * size, min(p, (i + 1) * size), i, 0, 0)
                count += 1
        most, tokens = max(most, k), max(tokens, size)
    words[0], words[1] = count, tokens
    return count, most


class SharedPrefixPlan:
    """Which rows of a decode batch share which prefix, in device memory (``words``), and the bounds that a call is launched with:
    a captured graph may be replayed with other words that keep to them. ``max_len`` bounds the sequences' lengths."""

    def __init__(self, words: torch.Tensor, rows: int, max_pieces: int, max_parts: int, max_len: int, q_heads: int, kv_heads: int, head_dim: int):
        _check_heads(q_heads, kv_heads, head_dim)
        _check_size(rows, max_len, kv_heads)
        self.words, self.rows, self.max_pieces, self.max_parts = words, rows, max_pieces, max_parts
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.slices = decode_plan(max(rows, 1), kv_heads, max(max_len, 1)) if max_pieces == 0 else (1, 0)   # without prefixes: paged_decode's
        base = words.data_ptr()
        s = native.DecodeSharedArgs()
        s.n_pieces, s.pieces = base, base + 16
        s.row_prefix = base + 16 + 32 * max_pieces
        s.row_parts = s.row_prefix + 4 * rows
        s.max_pieces, s.max_parts, s.plan_rows = max_pieces, max_parts, rows
        s.max_len = self.max_len = max_len
        s.own_slots = self.own = own_slots(rows, q_heads, kv_heads)
        self._fields = bytes(s)[native.DecodeSharedArgs.pieces.offset:]

    def workspace_floats(self, batch: int) -> int:
        """Elements of the fp32 workspace of a call over ``batch`` rows."""
        if self.max_pieces == 0:
            return batch * self.q_heads * self.slices[0] * (self.head_dim + 2) if self.slices[0] > 1 else 0
        return batch * self.q_heads * (self.max_parts + self.own) * (self.head_dim + 2) + batch + 4


def shared_prefix_plan(sizes: Sequence[int], prefixes: Sequence[int], *, rows: int, q_heads: int, kv_heads: int, head_dim: int, max_len: int,
                       device: str | torch.device = "cuda") -> SharedPrefixPlan:
    """The plan of a batch of ``rows`` rows whose first ``sizes[0]`` rows share their first ``prefixes[0]`` tokens (their block
    tables name the same pages for them; a group's prefix is read through its first row's table, whatever that row's length), the
    next ``sizes[1]`` rows ``prefixes[1]`` tokens and so on; rows behind the last group share nothing. ``max_len``: bound of the
    sequence lengths while the plan is in use; rows are read no further."""
    if len(sizes) != len(prefixes) or any(n < 0 for n in sizes) or any(p < 0 for p in prefixes):
        raise ValueError("a size and a prefix, neither negative, for every group")
    if sum(sizes) > rows or (prefixes and max(prefixes) > max_len):
        raise ValueError(f"groups of {sum(sizes)} rows and prefixes up to {max(prefixes, default=0)} for {rows} rows of {max_len} tokens")
    _check_heads(q_heads, kv_heads, head_dim)
    per = piece_rows(q_heads, kv_heads)
    most = sum(-(-n // per) * -(-p // PIECE_TOKENS) for n, p in zip(sizes, prefixes))
    host = np.zeros(shared_plan_words(rows, most), dtype=np.int32)
    # the longest tail behind a prefix is about what every row may have, and half of it what a row has
    own = rows * (max_len - max(prefixes, default=0)) // 2
    count, parts = fill_shared_plan(sizes, prefixes, host, rows, most, MAX_PARTS, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, own_tokens=own)
    words = np.concatenate([host[:4 + 8 * count], host[4 + 8 * most:]])
    return SharedPrefixPlan(torch.from_numpy(words).to(device), rows, count, parts, max_len, q_heads, kv_heads, head_dim)


def _check_size(rows: int, max_len: int, kv_heads: int) -> None:
    if rows > MAX_SHARED_ROWS or rows * -(-max_len // 16) * kv_heads * 2 >= 2 ** 31:
        raise ValueError(f"{rows} rows of up to {max_len} tokens: up to {MAX_SHARED_ROWS} rows and 2^31 tiles of 16 tokens are supported")


def _check_heads(q_heads: int, kv_heads: int, head_dim: int) -> None:
    if kv_heads < 1 or q_heads % kv_heads or not 1 <= q_heads // kv_heads <= 16 or head_dim not in (64, 128):
        raise ValueError(f"{q_heads} query and {kv_heads} KV heads of {head_dim}: up to 16 query heads per KV head of 64 or 128 are supported")


def paged_decode_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                        plan: SharedPrefixPlan, *, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                        scale: float | None = None) -> torch.Tensor:
    """:func:`paged_decode` for a batch whose rows share prefixes: every prefix of ``plan`` is read and multiplied once for all rows
    of its group (``csrc/kernels/shared_prefix.cu``), then each row adds its own tokens. ``seq_lens`` count prefix and own tokens; a
    row of fewer tokens than its group's prefix reads all of them on its own. Rows without tokens give zeros. ``out`` may be ``q``."""
    batch, q_heads, d = q.shape
    pages, page, kv_heads, kv_d = kv_shape = k_cache.shape
    if (q_heads, kv_heads, d, d) != (plan.q_heads, plan.kv_heads, plan.head_dim, kv_d) or v_cache.shape != kv_shape:
        raise ValueError(f"q {tuple(q.shape)}, caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} for a plan of {plan.q_heads} query and "
                         f"{plan.kv_heads} KV heads of {plan.head_dim}")
    if page < 16 or page & (page - 1):
        raise ValueError(f"pages of {page} tokens: powers of two from 16 on are supported")
    dev, bf16, i32 = q.device, torch.bfloat16, torch.int32
    at_q, at_k, at_v = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if (at_q | at_k | at_v) & 15 or not (q.dtype is k_cache.dtype is v_cache.dtype is bf16 and q.is_contiguous() and k_cache.is_contiguous()
                                         and v_cache.is_contiguous() and k_cache.device == dev and v_cache.device == dev):
        raise ValueError("queries and caches must be contiguous, 16-byte aligned bf16 on one device")
    if not (block_table.dtype is seq_lens.dtype is i32 and block_table.device == dev and seq_lens.device == dev):
        raise ValueError("block_table and seq_lens must be int32 on the queries' device")
    if block_table.dim() != 2 or seq_lens.shape != (batch,) or not seq_lens.is_contiguous():
        raise ValueError(f"block_table {tuple(block_table.shape)} and seq_lens {tuple(seq_lens.shape)} for {batch} rows")
    (rows, width), (pitch, one) = block_table.shape, block_table.stride()
    if rows < batch or (width and one != 1):
        raise ValueError(f"block_table {tuple(block_table.shape)} and seq_lens {tuple(seq_lens.shape)} for {batch} rows")
    if plan.rows > batch or plan.words.device != dev or width * page < plan.max_len:
        raise ValueError(f"a plan of {plan.rows} rows of up to {plan.max_len} tokens for {batch} rows of {width} pages")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not bf16 or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be like q")
    elif 0 < abs(out.data_ptr() - at_q) < 2 * batch * q_heads * d:
        raise ValueError("out may be q, but must not lie over other rows of it")
    if scale is None:
        scale = d ** -0.5
    elif not 0 < scale < math.inf:
        raise ValueError(f"scale {scale}: the kernel takes positive numbers")
    if batch > plan.rows:
        _check_size(batch, plan.max_len, kv_heads)
    need = plan.workspace_floats(batch)
    if ws is None:
        if need:
            ws = torch.empty(need, dtype=torch.float32, device=dev)
    elif ws.dtype != torch.float32 or ws.numel() < need or not ws.is_contiguous() or ws.device != dev:
        raise ValueError(f"the workspace must hold {need} contiguous fp32 elements on the queries' device")
    at_out, at_ws = out.data_ptr(), ws.data_ptr() if ws is not None else 0
    if (at_out | at_ws) & 15:
        raise ValueError("out and the workspace must be 16-byte aligned")
    if not batch:
        return out
    if dev.type != "cuda":
        raise ValueError("the kernel runs on a GPU")
    if not pages:
        raise ValueError("a cache of no pages")
    call = _SHARED_CALL.pack(at_q, at_k, at_v, at_out, at_ws, block_table.data_ptr(), seq_lens.data_ptr(), batch, q_heads, kv_heads, d, page, pitch,
                             plan.slices[0], scale, plan.slices[1], pages, status_words(dev).data_ptr(), 0, 0)
    native.run_packed("xp_decode_shared", call + plan._fields, dev, 1 + (plan.max_pieces > 0 or plan.slices[0] > 1))
    return out


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  q_starts: torch.Tensor, q_lens: torch.Tensor, ctx_lens: torch.Tensor, max_q_len: int, *,
                  out: torch.Tensor | None = None, scale: float | None = None,
                  force_simple: bool | str | None = None) -> torch.Tensor:
    """Causal attention of packed chunk queries ``[total_q, q_heads, d]`` over the paged cache.

    Runs the tcgen05 kernel (S and O in tensor memory, TMA-fed Q/K/V, the heads of a KV group packed into 128-row
    tiles) when pages hold a power-of-two number of at least 16 tokens and 1, 2, 4, 8 or 16 query heads share a KV
    head. ``force_simple``: True or ``"simple"`` selects the plain kernel, ``"mma"`` the TMA-fed mma.sync kernel."""
    if out is None:
        out = torch.empty_like(q)
    a = prefill_args(q, k_cache, v_cache, block_table, q_starts, q_lens, ctx_lens, max_q_len, out, scale, force_simple)
    native.check(native.kernels().xp_prefill_attn(C.byref(a), _stream(q.device)), "xp_prefill_attn")
    return out


def prefill_args(q, k_cache, v_cache, block_table, q_starts, q_lens, ctx_lens, max_q_len, out, scale=None, force_simple=None) -> "native.PrefillAttnArgs":
    _, q_heads, d = q.shape
    page_size, kv_heads = k_cache.shape[1], k_cache.shape[2]
    a = native.PrefillAttnArgs()
    a.q, a.k_cache, a.v_cache, a.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
    a.block_table = block_table.data_ptr()
    a.q_starts, a.q_lens, a.ctx_lens = q_starts.data_ptr(), q_lens.data_ptr(), ctx_lens.data_ptr()
    a.num_seqs, a.max_q_len = q_lens.shape[0], max_q_len
    a.q_heads, a.kv_heads, a.head_dim = q_heads, kv_heads, d
    a.page_size, a.max_blocks = page_size, block_table.stride(0)
    a.scale = scale if scale is not None else d ** -0.5
    a.num_pages = k_cache.shape[0] if k_cache.is_contiguous() and v_cache.is_contiguous() else 0
    which = PREFILL_KERNEL_DEFAULT if force_simple in (None, False) else ("simple" if force_simple is True else force_simple)
    a.force_simple = PREFILL_KERNELS[which]
    a.total_q = q.shape[0]
    from .gemm import status_words

    a.status = status_words(q.device).data_ptr()
    return a


def embedding(ids: torch.Tensor, table: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    rows, hidden = ids.shape[0], table.shape[1]
    if out is None:
        out = torch.empty(rows, hidden, dtype=table.dtype, device=table.device)
    hidden = hidden * table.element_size() // 2          # rows are copied as they are, counted in 16-bit elements
    native.check(native.kernels().xp_embedding(ids.data_ptr(), table.data_ptr(), out.data_ptr(), rows, hidden,
                                               table.shape[0], _stream(table.device)), "xp_embedding")
    return out


def argmax(logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    native.check(native.kernels().xp_argmax(logits.data_ptr(), int(logits.dtype == torch.float32), out.data_ptr(),
                                            rows, vocab, logits.stride(0), _stream(logits.device)), "xp_argmax")
    return out


def sample(logits: torch.Tensor, temps: torch.Tensor, seeds: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row from ``softmax(logits / temperature)`` (Gumbel-max); rows with temperature 0 are
    greedy. ``temps`` fp32 ``[rows]``; ``seeds`` int32 ``[rows, 2]`` = (request seed, step): the same pair
    always gives the same token."""
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    assert temps.dtype == torch.float32 and seeds.dtype == torch.int32 and seeds.shape[-1] == 2
    native.check(native.kernels().xp_sample(logits.data_ptr(), int(logits.dtype == torch.float32), temps.data_ptr(),
                                            seeds.data_ptr(), out.data_ptr(), rows, vocab, logits.stride(0),
                                            _stream(logits.device)), "xp_sample")
    return out
