"""Decode attention of rows that share prefixes, against the same rows attended one by one in 64 bits."""
import pytest
import torch

from request_oracle import paged_attention

pytestmark = pytest.mark.gpu


def make(sizes, prefixes, alone, own, hq, hk, d, page, seed=0, poison=True):
    """A paged cache in which the rows of a group name the same pages for their whole shared pages. ``own``: tokens behind the
    prefix per row, in turn. What no row may see is NaN."""
    g = torch.Generator().manual_seed(seed)
    pre, owner, at = [], [], 0
    for n, p in zip(sizes, prefixes):
        pre += [p] * n
        owner += [at] * n
        at += n
    pre += [0] * alone
    owner += list(range(at, at + alone))
    lens = [p + own[i % len(own)] for i, p in enumerate(pre)]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 5
    perm, used = torch.randperm(total, generator=g).int(), 0
    table = torch.full((len(lens), max(need + [1]) + 2), total - 1, dtype=torch.int32)
    for r, n in enumerate(need):
        # a page is shared when the whole of it belongs to the prefix
        s = min(pre[r] // page, n) if owner[r] != r else 0
        table[r, :s] = table[owner[r], :s]
        table[r, s:n] = perm[used:used + n - s]
        used += n - s
    k = torch.randn(total, page, hk, d, generator=g).bfloat16()
    v = torch.randn(total, page, hk, d, generator=g).bfloat16()
    if poison:
        seen = torch.zeros(total, page, dtype=torch.bool)
        for r, n in enumerate(lens):
            t = torch.arange(n)
            seen[table[r, (t // page).long()].long(), t % page] = True
        k[~seen] = float("nan")
        v[~seen] = float("nan")
    q = (1.5 * torch.randn(len(lens), hq, d, generator=g)).bfloat16()
    return q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def close(got, q, k, v, table, lens, scale=None):
    """The weights are rounded to bf16 (half a step: 2^-8 of each), the result once more; what fp32 sums and 2 ** x add is below
    2^-14 of the weighted values: scores below 64 carry d 2^-24 64 of error."""
    want, mass = paged_attention(q, k, v, table, lens, scale)
    tol = (2.0 ** -8 + 2.0 ** -14) * mass + 2.0 ** -8 * want.abs() + 1e-30
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), (off / tol).max()


def run(sizes, prefixes, q, k, v, table, lens, **kw):
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    plan = A.shared_prefix_plan(sizes, prefixes, rows=q.shape[0], q_heads=q.shape[1], kv_heads=k.shape[2], head_dim=q.shape[2],
                                max_len=max(max(prefixes, default=0), int(lens.max())) if len(lens) else 1)
    out = A.paged_decode_shared(q, k, v, table, lens, plan, **kw)
    gemm.check_status(q.device)
    return out


HEADS = [(16, 8, 128), (32, 8, 128), (14, 2, 64), (16, 1, 128), (3, 3, 64)]


@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("page", [16, 64, 128])
def test_groups_and_rows_alone(hq, hk, d, page):
    sizes, prefixes, own = [5, 1, 2, 19], [208, 64, 513, 1000], [1, 17, 64, 130]
    data = make(sizes, prefixes, 3, own, hq, hk, d, page)
    close(run(sizes, [p // page * page for p in prefixes], *data), *data)


@pytest.mark.parametrize("prefix", [16, 48, 64, 80, 128, 144, 1008])
@pytest.mark.parametrize("rows", [1, 2, 64, 65, 129])
def test_prefix_lengths_and_row_counts(prefix, rows):
    # 65 and 129 rows of two heads: a tile of 128 query heads and one more row; the second tile and one more
    data = make([rows], [prefix], 0, [1, 2, 40], 4, 2, 128, 16, seed=prefix)
    close(run([rows], [prefix], *data), *data)


@pytest.mark.parametrize("prefix", [0, 5, 15, 17, 100])
def test_prefixes_that_are_no_whole_tiles(prefix):
    data = make([6], [prefix // 16 * 16], 0, [33, 90], 8, 4, 64, 16, poison=False)
    close(run([6], [prefix], *data), *data)


def test_rows_without_own_tokens_and_rows_shorter_than_the_prefix():
    data = list(make([7], [256], 2, [0, 3], 8, 2, 128, 64, poison=False))
    lens = data[4].clone()
    lens[1], lens[2], lens[3], lens[7] = 0, 1, 255, 0
    data[4] = lens
    got = run([7], [256], *data)
    close(got, *data)
    assert not got[1].any() and not got[7].any()


def test_every_row_shorter_than_a_prefix_whose_pages_hold_nothing():
    q, k, v, table, lens = make([4], [128], 0, [0], 8, 2, 128, 16, poison=False)
    lens.fill_(20)
    k.view(-1, 2, 128)[:] = float("nan")
    v.view(-1, 2, 128)[:] = float("nan")
    for r in range(4):
        for t in range(20):
            for c in (k, v):
                c[table[r, t // 16].long(), t % 16] = torch.randn(2, 128, device="cuda").bfloat16()
    data = (q, k, v, table, lens)
    close(run([4], [128], *data), *data)


def test_long_own_tails_in_slices():
    data = make([3], [320], 1, [700, 1, 2500], 4, 2, 128, 64)
    close(run([3], [320], *data), *data)


def test_a_short_row_has_more_tokens_than_the_slices_of_the_tails_cover():
    data = list(make([3], [4096], 0, [600], 4, 2, 128, 64, poison=False))
    data[4][1] = 4000
    close(run([3], [4096], *data), *data)


def test_large_scores_and_equal_scores():
    q, k, v, table, lens = make([9], [192], 0, [10], 8, 2, 128, 64, poison=False)
    data = (q * 8, k, v, table, lens)
    close(run([9], [192], *data, scale=0.05), *data, scale=0.05)
    data = (q * 0, k, v, table, lens)
    close(run([9], [192], *data), *data)


def test_scores_grow_along_the_prefix():
    """The running maximum moves in every tile."""
    q, k, v, table, lens = make([9], [512], 0, [40], 4, 2, 64, 64, poison=False)
    pos = torch.zeros(k.shape[0], 64, device="cuda")
    for r in range(9):
        for b in range(int(lens[r] + 63) // 64):
            pos[table[r, b].long()] = torch.arange(64, device="cuda").float() + 64 * b
    k = (q[0, 0][None, None, None] * (pos / 200)[:, :, None, None]).expand_as(k).bfloat16().contiguous()
    q = q[:1, :1].expand_as(q).contiguous()
    data = (q, k, v, table, lens)
    close(run([9], [512], *data), *data)


def test_same_bits_every_time_and_where_the_result_goes():
    data = make([40, 3], [512, 64], 2, [1, 30], 16, 8, 128, 64)
    first = run([40, 3], [512, 64], *data)
    out = torch.full_like(first, 7.0)
    assert run([40, 3], [512, 64], *data, out=out) is out and torch.equal(out, first)
    for _ in range(3):
        assert torch.equal(run([40, 3], [512, 64], *data), first)


def test_no_rows_and_no_groups():
    data = make([], [], 4, [9, 70], 8, 2, 128, 64)
    close(run([], [], *data), *data)
    q, k, v, table, lens = data
    assert run([], [], q[:0], k, v, table, lens[:0]).shape == (0, 8, 128)


def test_graph_replays_with_other_plans():
    from crosspool_b200.ops import attention as A

    rows, hq, hk, d, page = 12, 8, 2, 128, 16
    cases = [([12], [512]), ([4, 8], [256, 64]), ([], []), ([3, 3, 3], [16, 512, 128])]
    words = torch.zeros(A.shared_plan_words(rows, 64), dtype=torch.int32, device="cuda")
    plan = A.SharedPrefixPlan(words, rows, 64, 8, 700, hq, hk, d)
    ws = torch.empty(plan.workspace_floats(rows), device="cuda")

    def load(i):
        sizes, prefixes = cases[i]
        data = make(sizes, prefixes, rows - sum(sizes), [1, 20, 100], hq, hk, d, page, seed=i)
        host = words.cpu().numpy()
        A.fill_shared_plan(sizes, prefixes, host, rows, 64, 8, q_heads=hq, kv_heads=hk)
        return data, torch.from_numpy(host)

    sets = [load(i) for i in range(len(cases))]
    pages = max(s[0][1].shape[0] for s in sets)
    wide = max(s[0][3].shape[1] for s in sets)
    k, v = (torch.zeros(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, out = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, hq, d, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(rows, max(wide, 44), dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")

    def fill(i):
        (q1, k1, v1, t1, n1), w = sets[i]
        q.copy_(q1), k[:k1.shape[0]].copy_(k1), v[:v1.shape[0]].copy_(v1), table[:, :t1.shape[1]].copy_(t1), lens.copy_(n1), words.copy_(w)

    fill(0)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        A.paged_decode_shared(q, k, v, table, lens, plan, out=out, ws=ws)
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        A.paged_decode_shared(q, k, v, table, lens, plan, out=out, ws=ws)
    for i in (1, 2, 3, 0):
        fill(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        close(out, q, k, v, table, lens)


def test_two_streams_at_once():
    sets = [make([20], [640], 0, [5, 50], 8, 2, 128, 64, seed=i) for i in range(2)]
    want = [run([20], [640], *s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run_quietly([20], [640], *sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def run_quietly(sizes, prefixes, q, k, v, table, lens):
    from crosspool_b200.ops import attention as A

    plan = A.shared_prefix_plan(sizes, prefixes, rows=q.shape[0], q_heads=q.shape[1], kv_heads=k.shape[2], head_dim=q.shape[2], max_len=700)
    return A.paged_decode_shared(q, k, v, table, lens, plan)


def test_a_cache_of_more_than_two_billion_elements():
    """Pages at both ends of caches whose offsets do not fit 32 bits."""
    q, k, v, table, lens = make([6], [640], 1, [1, 70, 300], 8, 8, 128, 64, poison=False)
    pages = 2 ** 31 // (64 * 8 * 128) + 4096                         # 2.4 G elements each
    used = torch.unique(torch.cat([table[r, :(int(n) + 63) // 64] for r, n in enumerate(lens)])).long()
    to = torch.cat([torch.arange(len(used) // 2), pages - 1 - torch.arange(len(used) - len(used) // 2)]).cuda()[torch.randperm(len(used), generator=torch.Generator().manual_seed(2)).cuda()]
    new = torch.zeros(k.shape[0], dtype=torch.int64, device="cuda")
    new[used] = to
    big = [torch.empty(pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b, c in zip(big, (k, v)):
        b[to] = c[used]
    moved = new[table.long()].int()
    got = run([6], [640], q, *big, moved, lens)
    close(got, q, k, v, table, lens)
    assert torch.equal(got, run([6], [640], q, k, v, table, lens))


def test_most_rows():
    """As many rows as a batch may have, in groups and alone."""
    sizes, prefixes = [3000, 500], [96, 32]
    data = make(sizes, prefixes, 596, [1, 3, 18], 2, 1, 64, 16)
    close(run(sizes, prefixes, *data), *data)


def test_workspaces_of_two_captured_graphs():
    """Two graphs captured on one stream, each with memory of its own, replayed on two streams at once."""
    from crosspool_b200.ops import attention as A

    sets = [make([24], [512], 0, [5, 80], 8, 2, 128, 64, seed=i) for i in range(2)]
    want = [run([24], [512], *s) for s in sets]
    plans = [A.shared_prefix_plan([24], [512], rows=24, q_heads=8, kv_heads=2, head_dim=128, max_len=int(s[4].max())) for s in sets]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    stream.wait_stream(torch.cuda.current_stream())
    for s, p in zip(sets, plans):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(A.paged_decode_shared(*s, p))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [0, 512])
def test_keys_of_minus_infinity_weigh_nothing(prefix, d):
    """The first 40 own tokens of every row, and (but for one) the first 160 of the prefix, have scores of -inf. Without a prefix the
    plan has one piece all the same, of rows that are empty."""
    hk, page, rows = 2, 16, 5
    q, k, v, table, lens = make([rows - 2, 2], [prefix, 64], 0, [90, 41, 300], 8, hk, d, page)
    lens[rows - 2:] = 0
    q = q.abs()
    low = torch.tensor(float("-inf"), device="cuda").bfloat16()
    for r in range(rows - 2):
        for t in [*range(prefix, prefix + 40), *range(min(160, max(prefix - 1, 0)))]:
            k[table[r, t // page].long(), t % page, :, 5] = low
    k[table[rows - 2, :4].long()] = 0
    v[table[rows - 2, :4].long()] = 0
    got = run([rows - 2, 2], [prefix, 64], q, k, v, table, lens)
    close(got, q, k, v, table, lens)
    assert (got[rows - 2:] == 0).all()
