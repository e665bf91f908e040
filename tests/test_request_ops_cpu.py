"""Plans and refusals of the operators of requests; no GPU is needed."""
import numpy as np
import pytest
import torch

from crosspool_b200.ops import attention as A
from crosspool_b200.ops import logits as L
from crosspool_b200.ops import lora


def plan(sizes, prefixes, rows, hq=8, hk=2, d=128, max_len=10000):
    return A.shared_prefix_plan(sizes, prefixes, rows=rows, q_heads=hq, kv_heads=hk, head_dim=d, max_len=max_len, device="cpu")


def read_plan(p):
    w = p.words.numpy()
    pieces = w[4:4 + 8 * p.max_pieces].reshape(-1, 8)[:w[0]]
    return pieces, w[4 + 8 * p.max_pieces:][:p.rows], w[4 + 8 * p.max_pieces + p.rows:][:p.rows]


@pytest.mark.parametrize("sizes,prefixes,rows", [([4], [512], 4), ([64], [2048], 64), ([300], [8192], 301), ([1, 70, 5, 0, 3], [16, 6000, 15, 90, 100], 90),
                                                 ([], [], 3), ([2] * 40, [64 * i for i in range(40)], 80)])
@pytest.mark.parametrize("hq,hk", [(8, 2), (14, 2), (16, 1), (64, 8), (3, 3)])
def test_pieces_cover_every_prefix_once(sizes, prefixes, rows, hq, hk):
    p = plan(sizes, prefixes, rows, hq, hk)
    pieces, shared, parts = read_plan(p)
    per, at = A.piece_rows(hq, hk), 0
    want = np.zeros(rows, dtype=int)
    seen = [set() for _ in range(rows)]
    for n, t in zip(sizes, prefixes):
        want[at:at + n] = t // 16 * 16
        at += n
    assert shared.tolist() == want.tolist()
    starts = np.cumsum([0] + list(sizes))
    for leader, row0, n, t0, t1, part, *_ in pieces.tolist():
        assert leader in starts and leader <= row0 and row0 + n <= starts[starts > leader][0]
        assert 0 < n <= per and t0 % A.PIECE_TOKENS == 0 and t1 % 16 == 0 and t0 < t1 <= want[row0]
        for r in range(row0, row0 + n):
            assert part not in [x[2] for x in seen[r]] and part < parts[r]
            seen[r].add((t0, t1, part))
    for r in range(rows):
        spans = sorted(seen[r])
        assert [s[2] for s in spans] == list(range(parts[r])) and (parts[r] > 0) == (want[r] > 0)
        assert not spans or (spans[0][0] == 0 and spans[-1][1] == want[r] and all(x[1] == y[0] for x, y in zip(spans, spans[1:])))


def test_plans_keep_to_their_bounds():
    words = np.zeros(A.shared_plan_words(64, 20), dtype=np.int32)
    n, parts = A.fill_shared_plan([32, 32], [8192, 4096], words, 64, 20, 6, q_heads=16, kv_heads=8)
    assert n <= 20 and parts <= 6 and words[0] == n
    with pytest.raises(ValueError, match="do not fit"):
        A.fill_shared_plan([2] * 30, [512] * 30, np.zeros(A.shared_plan_words(64, 20), dtype=np.int32), 64, 20, 6, q_heads=16, kv_heads=8)


@pytest.mark.parametrize("args", [([4], [64, 64], 4), ([-1], [64], 4), ([4], [-16], 4), ([5], [64], 4), ([4], [20000], 4)])
def test_plans_that_are_refused(args):
    with pytest.raises(ValueError):
        plan(*args)


@pytest.mark.parametrize("hq,hk,d", [(7, 2, 128), (34, 2, 128), (8, 2, 96), (8, 0, 64)])
def test_heads_that_are_refused(hq, hk, d):
    with pytest.raises(ValueError, match="heads"):
        plan([2], [64], 2, hq, hk, d)


def attention_args(**change):
    a = dict(q=torch.zeros(4, 8, 128, dtype=torch.bfloat16), k_cache=torch.zeros(9, 16, 2, 128, dtype=torch.bfloat16),
             v_cache=torch.zeros(9, 16, 2, 128, dtype=torch.bfloat16), block_table=torch.zeros(4, 8, dtype=torch.int32),
             seq_lens=torch.zeros(4, dtype=torch.int32), plan=plan([4], [64], 4, max_len=128))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(4, 8, 128)), dict(q=torch.zeros(4, 16, 128, dtype=torch.bfloat16)), dict(q=torch.zeros(4, 8, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(4, 16, 128, dtype=torch.bfloat16)[:, ::2]), dict(q=torch.zeros(3, 8, 128, dtype=torch.bfloat16), seq_lens=torch.zeros(3, dtype=torch.int32)),
    dict(k_cache=torch.zeros(9, 16, 4, 128, dtype=torch.bfloat16)), dict(v_cache=torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16)),
    dict(k_cache=torch.zeros(9, 24, 2, 128, dtype=torch.bfloat16), v_cache=torch.zeros(9, 24, 2, 128, dtype=torch.bfloat16)),
    dict(k_cache=torch.zeros(9, 8, 2, 128, dtype=torch.bfloat16), v_cache=torch.zeros(9, 8, 2, 128, dtype=torch.bfloat16)),
    dict(block_table=torch.zeros(4, 8, dtype=torch.int64)), dict(block_table=torch.zeros(3, 8, dtype=torch.int32)),
    dict(block_table=torch.zeros(4, 3, dtype=torch.int32)), dict(block_table=torch.zeros(8, 4, dtype=torch.int32).t()),
    dict(seq_lens=torch.zeros(5, dtype=torch.int32)), dict(seq_lens=torch.zeros(4, dtype=torch.int64)), dict(seq_lens=torch.zeros(8, dtype=torch.int32)[::2]),
    dict(out=torch.zeros(4, 8, 128)), dict(out=torch.zeros(3, 8, 128, dtype=torch.bfloat16)), dict(ws=torch.zeros(3)),
    dict(ws=torch.zeros(10 ** 6, dtype=torch.float64)),
    dict(k_cache=torch.zeros(0, 16, 2, 128, dtype=torch.bfloat16), v_cache=torch.zeros(0, 16, 2, 128, dtype=torch.bfloat16))])
def test_attention_calls_that_are_refused(change):
    a = attention_args(**change)
    with pytest.raises(ValueError):
        A.paged_decode_shared(**a)


def test_adapter_plans_hold_every_row_once():
    for index in ([], [0], [-1, -1], [3, 1, -1, 3, 1] * 20, [2] * 100, [-5, 0, 5]):
        p = lora.adapter_plan(index, 6, device="cpu")
        w, rows = p.words.numpy(), len(index)
        items, perm = w[4:4 + 4 * rows].reshape(-1, 4)[:w[0]], w[4 + 4 * rows:][:rows]
        assert sorted(perm.tolist()) == list(range(rows)) and p.max_items == w[0] <= rows
        got = {}
        for slot, first, n, _ in items.tolist():
            assert 0 < n <= lora.ITEM_ROWS
            for r in perm[first:first + n].tolist():
                assert r not in got
                got[r] = slot
        assert got == {r: max(s, -1) for r, s in enumerate(index)}
    words = np.zeros(lora.plan_words(5), dtype=np.int32)
    assert lora.fill_plan([1, -1, 0, -1, 1], words, 5, bare=False) == 2 and words[4:12].tolist() == [0, 2, 1, 0, 1, 3, 2, 0]


def test_stacks_and_adapters_that_are_refused():
    for args in ((0, 64, 64, 8), (1, 64, 64, 0), (1, 64, 64, 129), (1, 60, 64, 8), (1, 64, (64, 4), 8), (1, 64, (8,) * 5, 8), (1, 64, (), 8)):
        with pytest.raises(ValueError):
            lora.AdapterStack(*args, device="cpu")
    s = lora.AdapterStack(2, 64, (32, 16), 20, device="cpu")
    assert s.rank == 32 and s.a.shape == (2, 2, 32, 64) and s.b.shape == (2, 48 * 32)
    z = torch.zeros
    for slot, a, b in ((2, [z(4, 64), z(4, 64)], [z(32, 4), z(16, 4)]), (-1, [None, None], [None, None]), (0, z(4, 64), z(48, 4)),
                       (0, [z(4, 64), z(4, 64)], [z(32, 4), z(32, 4)]), (0, [z(4, 64), None], [z(32, 4), z(16, 4)]),
                       (0, [z(4, 60), None], [z(32, 4), None]), (0, [z(40, 64), None], [z(32, 40), None]), (0, [z(4, 64), None], [z(32, 5), None])):
        with pytest.raises(ValueError):
            s.load(slot, a, b)
    s.load(1, [z(4, 64) + 1, None], [z(32, 4) + 2, None], 0.5)
    assert s.ranks.tolist() == [0, 16] and s.a[1].sum() == 4 * 64 and s.b[1].sum() == 2 * 32 * 4 and s.scale.tolist() == [0, 0.5]
    s.load(1, [None, None], [None, None])
    assert s.ranks.tolist() == [0, 0] and not s.a.any() and not s.b.any()
    with pytest.raises(ValueError):
        lora.adapter_plan([0, 2], s)
    with pytest.raises(ValueError):
        s.clear(2)


def test_adapter_calls_that_are_refused():
    s, b = lora.AdapterStack(2, 64, 48, 16, device="cpu"), torch.bfloat16
    p = lora.adapter_plan([0, 1, -1], s)
    x, y = torch.zeros(3, 64, dtype=b), torch.zeros(3, 48, dtype=b)
    wide = torch.zeros(3, 80, dtype=b)
    for args, kw in (((y, x[:, :56], s, p), {}), ((y[:, :40], x, s, p), {}), ((y[:2], x[:2], s, p), {}), ((y.float(), x, s, p), {}), ((y, x.float(), s, p), {}),
                     ((y, x, s, lora.adapter_plan([0, 1, 2], 3, device="cpu")), {}), ((y, x, s, p), dict(out=y.float())), ((y, x, s, p), dict(out=y[:2])),
                     ((y, wide[:, 4:68], s, p), {}), ((y, torch.zeros(3, 68, dtype=b)[:, :64], s, p), {}), ((y, torch.zeros(64, 3, dtype=b).t(), s, p), {})):
        with pytest.raises(ValueError):
            lora.lora_add(*args, **kw)


def test_calls_on_the_cpu_are_refused():
    s, p = lora.AdapterStack(1, 64, 64, 8, device="cpu"), lora.adapter_plan([0, -1], 1, device="cpu")
    x, y = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: lora.lora_add(y, x, s, p), lambda: lora.lora_add(y, x, s, p, out=x), lambda: A.paged_decode_shared(**attention_args()),
                 lambda: L.adjust_logits(x, L.LogitControls()), lambda: L.select_tokens(x, L.LogitControls())):
        with pytest.raises(ValueError, match="GPU|not x"):
            call()


def test_controls_that_are_refused():
    i, f = (lambda *s: torch.zeros(*s, dtype=torch.int32)), (lambda *s: torch.zeros(*s))
    for kw in (dict(history=i(2, 5)), dict(lens=i(2)), dict(history=f(2, 5), lens=i(2)), dict(history=i(2, 5), lens=i(3)), dict(history=i(5), lens=i(2)),
               dict(repetition=f(2)), dict(history=i(2, 5), lens=i(2), repetition=f(3)), dict(history=i(2, 5), lens=i(2), presence=i(2)),
               dict(history=i(5, 2).t(), lens=i(2)), dict(bias_ids=i(3)), dict(bias_ids=i(3), bias_values=f(2), bias_starts=i(3)),
               dict(bias_ids=i(3), bias_values=f(3), bias_starts=i(0)), dict(masks=i(1, 4)), dict(masks=f(1, 4), mask_index=i(2)),
               dict(masks=i(1, 4), mask_index=i(2), history=i(3, 4), lens=i(3))):
        with pytest.raises(ValueError):
            L.LogitControls(**kw)
    c = L.LogitControls(masks=i(1, 4), mask_index=i(2))
    assert c.rows == 2 and L.LogitControls().rows is None
    x = f(2, 100)
    for call in (lambda: L.adjust_logits(x.half(), c), lambda: L.adjust_logits(f(3, 100), c), lambda: L.adjust_logits(f(2, 129), c),
                 lambda: L.adjust_logits(f(100, 2).t(), c), lambda: L.adjust_logits(x, c, out=f(2, 99)), lambda: L.adjust_logits(x, c, out=x.half()),
                 lambda: L.adjust_logits(x, c, out=x.view(torch.bfloat16)[:, ::2]), lambda: L.select_tokens(f(2, 0), c),
                 lambda: L.select_tokens(x, c, temps=f(2)), lambda: L.select_tokens(x, c, temps=f(3), seeds=i(3, 2)),
                 lambda: L.select_tokens(x, c, temps=f(2), seeds=i(2, 3)), lambda: L.select_tokens(x, c, out=i(3)), lambda: L.select_tokens(x, c, values=f(1)),
                 lambda: L.select_tokens(x, c, out=f(2))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("scale", [0.0, -0.1, float("inf"), float("nan")])
def test_scales_that_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        A.paged_decode_shared(**attention_args(), scale=scale)


def test_batches_that_are_too_large_for_a_small_plan():
    rows, max_len = 4096, 1 << 20
    a = attention_args(q=torch.zeros(rows, 8, 128, dtype=torch.bfloat16), k_cache=torch.zeros(9, 16, 4, 128, dtype=torch.bfloat16),
                       v_cache=torch.zeros(9, 16, 4, 128, dtype=torch.bfloat16), block_table=torch.zeros(1, max_len // 16, dtype=torch.int32).expand(rows, -1),
                       seq_lens=torch.zeros(rows, dtype=torch.int32), plan=plan([4], [64], 4, 8, 4, max_len=max_len))
    with pytest.raises(ValueError, match="tiles"):
        A.paged_decode_shared(**a)


def test_results_that_overlap_are_refused():
    b = torch.bfloat16
    s = lora.AdapterStack(2, 64, 48, 16, device="cpu")
    p, x = lora.adapter_plan([0, 1, -1], s), torch.zeros(3, 64, dtype=b)
    buf = torch.zeros(3 * 64, dtype=b)
    y = buf.view(3, 64)[:, :48]
    for out in (buf[:48].expand(3, 48), buf.as_strided((3, 48), (40, 1)), buf[:144].view(3, 48)):
        with pytest.raises(ValueError, match="overlap"):
            lora.lora_add(y, x, s, p, out=out)
    z = torch.zeros(100)
    with pytest.raises(ValueError, match="apart"):
        L.adjust_logits(z.expand(3, 100), L.LogitControls())
    with pytest.raises(ValueError, match="apart"):
        L.adjust_logits(torch.zeros(3, 100), L.LogitControls(), out=z.expand(3, 100))
    with pytest.raises(ValueError, match="apart"):
        L.LogitControls(masks=torch.zeros(4, dtype=torch.int32).expand(2, 4), mask_index=torch.zeros(2, dtype=torch.int32))


def test_adapters_that_are_trained_can_be_loaded():
    s = lora.AdapterStack(1, 64, (32, 16), 20, device="cpu")
    a, b = torch.ones(3, 64, requires_grad=True), torch.ones(16, 3, requires_grad=True)
    s.load(0, [None, a], [None, b])
    s.load(0, [None, a], [None, b], 2.0)
    assert not s.a.requires_grad and not s.b.requires_grad and s.part_ranks.tolist() == [[0, 3, 0, 0]] and s.a.sum() == 3 * 64
