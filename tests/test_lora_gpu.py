"""Adapters of many requests beside a projection, against 64 bits."""
import pytest
import torch

from request_oracle import adapters

pytestmark = pytest.mark.gpu


def make(rows, k, parts, ranks, max_rank, index, seed=0, missing=()):
    from crosspool_b200.ops import lora

    g = torch.Generator().manual_seed(seed)
    n = sum(parts)
    x, y = torch.randn(rows, k, generator=g).bfloat16(), torch.randn(rows, n, generator=g).bfloat16()
    stack = lora.AdapterStack(len(ranks), k, parts, max_rank)
    pairs, scales = [], []
    for s, r in enumerate(ranks):
        scales.append(0.5 + 0.25 * s)
        if r == 0:
            pairs.append(None)
            continue
        mine = [(((torch.randn(r, k, generator=g) / k ** 0.5).bfloat16(), (torch.randn(f, r, generator=g) / r ** 0.5).bfloat16())
                 if (s, i) not in missing else None, f) for i, f in enumerate(parts)]
        pairs.append(mine)
        stack.load(s, [p[0] if p else None for p, _ in mine], [p[1] if p else None for p, _ in mine], scales[s])
    return x.cuda(), y.cuda(), stack, [None if p is None else [(None if m is None else (m[0].cuda(), m[1].cuda()), f) for m, f in p] for p in pairs], scales


def check(got, x, y, pairs, scales, index, rank):
    """The result is rounded to bf16 once (half a step: 2^-8). The products' sums are fp32 (k + rank steps of 2^-24), the low-rank
    values enter the second product with 16 bits (2^-16)."""
    want, mass = adapters(y, x, pairs, scales, index)
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * (2.0 ** -16 + (x.shape[1] + rank + 4) * 2.0 ** -24) * mass + 1e-30
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("rank", [1, 8, 16, 24, 64, 128])
@pytest.mark.parametrize("k,parts", [(1024, (2048, 1024, 1024)), (896, (896, 128, 128)), (8, (8,)), (72, (200, 8)), (5120, (5120,)), (520, (64, 72, 8, 16))])
def test_ranks_and_widths(rank, k, parts):
    from crosspool_b200.ops import lora

    index = [0, 2, -1, 1, 0, 0, 2]
    x, y, stack, pairs, scales = make(7, k, parts, [rank, 0, max(1, rank - 3)], rank, index)
    got = lora.lora_add(y, x, stack, lora.adapter_plan(index, stack))
    check(got, x, y, pairs, scales, index, stack.rank)
    assert torch.equal(got[2], y[2]) and torch.equal(got[3], y[3])      # no adapter, an empty slot


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 100, 300])
@pytest.mark.parametrize("order", ["one", "runs", "shuffled", "none"])
def test_rows_and_orders(rows, order):
    from crosspool_b200.ops import lora

    slots = [16, 8, 32, 4]
    g = torch.Generator().manual_seed(rows)
    index = {"one": [2] * rows, "runs": [i * 5 // rows - 1 for i in range(rows)], "none": [-1] * rows,
             "shuffled": (torch.randint(-1, 4, (rows,), generator=g)).tolist()}[order]
    x, y, stack, pairs, scales = make(rows, 512, (384, 128), slots, 32, index, seed=rows)
    plan = lora.adapter_plan(index, stack)
    got = lora.lora_add(y, x, stack, plan)
    check(got, x, y, pairs, scales, index, 32)
    again = lora.lora_add(y, x, stack, plan)
    assert torch.equal(got, again)
    assert lora.lora_add(y, x, stack, plan, out=y) is y and torch.equal(y, got)


def test_rows_with_pitches_and_nothing_else_written():
    from crosspool_b200.ops import lora

    index = [1, 0, 1, -1, 0]
    x, y, stack, pairs, scales = make(5, 256, (128, 64), [16, 40], 48, index)
    wide_x, wide_y = torch.full((5, 264), float("nan"), device="cuda").bfloat16(), torch.full((5, 208), float("nan"), device="cuda").bfloat16()
    wide_o = torch.full((7, 200), 3.0, device="cuda").bfloat16()
    wide_x[:, :256], wide_y[:, 8:200] = x, y
    got = lora.lora_add(wide_y[:, 8:200], wide_x[:, :256], stack, lora.adapter_plan(index, stack), out=wide_o[1:6, :192])
    check(got, x, y, pairs, scales, index, 48)
    wide_o[1:6, :192] = 3.0
    assert (wide_o == 3.0).all()


def test_parts_without_an_adapter():
    from crosspool_b200.ops import lora

    index = [0, 1, 1]
    x, y, stack, pairs, scales = make(3, 128, (64, 32, 64), [8, 16], 16, index, missing={(0, 1), (1, 0), (1, 2)})
    got = lora.lora_add(y, x, stack, lora.adapter_plan(index, stack))
    check(got, x, y, pairs, scales, index, 16)
    assert torch.equal(got[0, 64:96], y[0, 64:96]) and torch.equal(got[1, :64], y[1, :64])


def test_slots_are_reloaded_and_cleared():
    from crosspool_b200.ops import lora

    index = [0, 1]
    x, y, stack, pairs, scales = make(2, 128, (64,), [64, 8], 64, index)
    plan = lora.adapter_plan(index, stack)
    a, b = torch.randn(5, 128).bfloat16().cuda(), torch.randn(64, 5).bfloat16().cuda()
    stack.load(0, a, b, -2.0)
    pairs[0], scales[0] = [((a, b), 64)], -2.0
    check(lora.lora_add(y, x, stack, plan), x, y, pairs, scales, index, 64)
    stack.clear(1)
    pairs[1] = None
    check(lora.lora_add(y, x, stack, plan), x, y, pairs, scales, index, 64)


def test_infinities_stay_in_their_row():
    from crosspool_b200.ops import lora

    index = [0, 0, -1, 0]
    x, y, stack, pairs, scales = make(4, 256, (128,), [16], 16, index)
    x[1] = float("inf")
    x[2] = float("nan")
    got = lora.lora_add(y, x, stack, lora.adapter_plan(index, stack))
    keep = [0, 2, 3]
    x[2] = 0
    assert torch.equal(got[2], y[2])
    check(got[keep], x[keep], y[keep], pairs, scales, [index[i] for i in keep], 16)


def test_graph_replays_with_other_plans():
    from crosspool_b200.ops import lora

    rows = 40
    x, y, stack, pairs, scales = make(rows, 256, (128, 128), [16, 32, 8], 32, None)
    words = torch.zeros(lora.plan_words(rows), dtype=torch.int32, device="cuda")
    plan = lora.AdapterPlan(words, rows, rows, 3)
    out = torch.empty_like(y)

    def fill(index):
        import numpy as np

        host = np.zeros(lora.plan_words(rows), dtype=np.int32)
        lora.fill_plan(index, host, rows)
        words.copy_(torch.from_numpy(host))

    cases = [[-1] * rows, [i % 3 for i in range(rows)], [i % 4 - 1 for i in range(rows)], [2] * rows]
    fill(cases[1])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        lora.lora_add(y, x, stack, plan, out=out)
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        lora.lora_add(y, x, stack, plan, out=out)
    for index in cases:
        fill(index)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, y, pairs, scales, index, 32)


def test_infinities_go_through_the_ranks_that_there_are():
    """Ranks that only fill up a tile, and parts without an adapter, add nothing to a row of infinities. Every A and B is positive:
    the formula gives infinities, no NaN."""
    from crosspool_b200.ops import lora

    index = [0, 1, 0, 1]
    x, y, stack, pairs, scales = make(4, 256, (64, 32, 64), [8, 21], 32, index, missing={(0, 1), (1, 0)})
    pairs = [[(None if m is None else tuple(t.abs() + 0.125 for t in m), f) for m, f in p] for p in pairs]
    for s, p in enumerate(pairs):
        stack.load(s, [m[0] if m else None for m, _ in p], [m[1] if m else None for m, _ in p], scales[s])
    x[0, 3], x[1, 200] = float("inf"), float("-inf")
    got, inf = lora.lora_add(y, x, stack, lora.adapter_plan(index, stack)), float("inf")
    assert (got[0, :64] == inf).all() and torch.equal(got[0, 64:96], y[0, 64:96]) and (got[0, 96:] == inf).all()
    assert torch.equal(got[1, :64], y[1, :64]) and (got[1, 64:] == -inf).all()
    check(got[2:], x[2:], y[2:], pairs, scales, index[2:], 32)
