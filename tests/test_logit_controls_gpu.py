"""Controls on logits: every step equal to the same step in 32 bits, and near 64 bits."""
import pytest
import torch

from request_oracle import controls

pytestmark = pytest.mark.gpu


def batch(rows, vocab, dtype, seed=0, history=40, biases=6, masks=2, wide=0):
    """Rows with different amounts of everything; returns (logits, LogitControls, list of the oracle's arguments per row)."""
    from crosspool_b200.ops import logits as L

    g = torch.Generator().manual_seed(seed)
    ints = lambda n, hi: torch.randint(0, max(hi, 1), (n,), generator=g).tolist()
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    words = -(-vocab // 32) + wide
    mask = torch.randint(-2 ** 31, 2 ** 31, (max(masks, 1), words), generator=g).to(torch.int32)
    hist = torch.zeros(rows + 2, history + 3, dtype=torch.int32)
    lens, prompts, slots, starts, ids, vals, which, args = [], [], [], [0], [], [], [], []
    rep, freq, pres = (1 + torch.rand(rows, generator=g)), torch.rand(rows, generator=g) - 0.3, torch.rand(rows, generator=g) - 0.3
    order = torch.randperm(rows + 2, generator=g)[:rows].tolist()
    for r in range(rows):
        n = [0, 1, history // 2, history][r % 4]
        p = [0, n, n // 3][r % 3]
        toks = ints(n, vocab)
        if n > 4:
            toks[1], toks[2], toks[n - 1] = vocab - 1, -7, vocab + 5          # the last token; two that are none
            toks[3] = toks[0] = int(x[r].argmax())
        e = [0, biases, 1][r % 3] if biases else 0
        bi = ints(e, vocab)
        if e > 3:
            bi[0], bi[1], bi[2], bi[3] = vocab - 1, toks[0] if toks else 0, -3, vocab     # the last token, one of the history, none
            bi[e - 1] = bi[1]                                                             # twice
        bv = (6 * torch.rand(e, generator=g) - 3).tolist()
        hist[order[r], :n] = torch.tensor(toks, dtype=torch.int32)
        lens.append(n), prompts.append(p), slots.append(order[r])
        ids += bi
        vals += bv
        starts.append(len(ids))
        m = r % (masks + 1) - 1 if masks else -1
        which.append(m)
        args.append(dict(history=toks, prompt=p, repetition=float(rep[r]), frequency=float(freq[r]), presence=float(pres[r]),
                         biases=list(zip(bi, bv)), mask=mask[m].tolist() if m >= 0 else None))
    t = lambda v, d=torch.int32: torch.tensor(v, dtype=d).cuda()
    c = L.LogitControls(history=hist.cuda(), lens=t(lens), prompt_lens=t(prompts), history_rows=t(slots), repetition=rep.cuda(), frequency=freq.cuda(),
                        presence=pres.cuda(), bias_ids=t(ids), bias_values=t(vals, torch.float32), bias_starts=t(starts), masks=mask.cuda(),
                        mask_index=t(which))
    return x.cuda(), c, args


def oracle(x, args, dtype=torch.float64):
    return torch.stack([controls(row.cpu(), dtype=dtype, **a) for row, a in zip(x, args)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 8191, 8192, 8200, 20011])
def test_adjusted_rows(vocab, dtype):
    from crosspool_b200.ops import logits as L

    x, c, args = batch(9, vocab, dtype, seed=vocab)
    same = oracle(x, args, torch.float32)
    got = L.adjust_logits(x, c, out=torch.empty(x.shape, device="cuda"))
    assert torch.equal(got.cpu(), same)
    assert torch.equal(L.adjust_logits(x, c).cpu(), same.to(dtype))
    # five steps, each off by at most half a step of the largest number on the way (at most twice the logits, plus biases and penalties)
    want = oracle(x, args)
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got).cpu(), inf)
    assert ((got.cpu().double() - want).abs()[~inf] <= 5 * 2.0 ** -24 * (2 * x.float().abs().max().item() + 60)).all()
    y = x.clone()
    assert L.adjust_logits(y, c, out=y) is y and torch.equal(y.cpu(), same.to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 151936), (5, 32), (7, 8193), (70, 4100), (33, 50021)])
def test_selected_tokens(rows, vocab, dtype):
    from crosspool_b200.ops import logits as L

    x, c, args = batch(rows, vocab, dtype, seed=rows + vocab, history=30 if rows * vocab < 10 ** 6 else 200)
    adjusted = L.adjust_logits(x, c, out=torch.empty(x.shape, device="cuda"))
    values = torch.empty(rows, device="cuda")
    got = L.select_tokens(x, c, values=values)
    want = torch.stack([(r == r.max()).nonzero()[0, 0] for r in adjusted]).int()       # ties go to the lower id
    assert torch.equal(got, want)
    assert torch.equal(values, adjusted.gather(1, want.long()[:, None])[:, 0])
    if rows * vocab < 400000:
        assert torch.equal(adjusted.cpu(), oracle(x, args, torch.float32))


def test_nothing_to_do_is_the_plain_sampler():
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import logits as L

    x = torch.randn(6, 5003, device="cuda").bfloat16()
    temps = torch.tensor([0.0, 0.7, 1.0, 0.0, 2.0, 0.1], device="cuda")
    seeds = torch.arange(12, dtype=torch.int32, device="cuda").view(6, 2)
    none = L.LogitControls()
    assert torch.equal(L.select_tokens(x, none), A.argmax(x))
    assert torch.equal(L.select_tokens(x, none, temps, seeds), A.sample(x, temps, seeds))
    assert torch.equal(L.adjust_logits(x, none), x)


def test_draws_are_those_of_the_sampler_on_the_adjusted_row():
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import logits as L

    x, c, _ = batch(12, 3001, torch.float32, seed=5)
    temps = torch.linspace(0, 1.5, 12).cuda()
    adjusted, values = L.adjust_logits(x, c), torch.empty(12, device="cuda")
    for step in range(20):
        seeds = torch.tensor([[r, step] for r in range(12)], dtype=torch.int32, device="cuda")
        got = L.select_tokens(x, c, temps, seeds, values=values)
        assert torch.equal(got, A.sample(adjusted, temps, seeds))
        assert torch.equal(values, adjusted.gather(1, got.long()[:, None])[:, 0])
        assert torch.isfinite(values).all()


def test_rows_without_an_allowed_token_infinities_and_the_lowest_value():
    from crosspool_b200.ops import logits as L

    low = torch.finfo(torch.float32).min
    x = torch.randn(5, 100, device="cuda")
    x[1] = low
    x[2, 40:] = -float("inf")
    x[3, 7] = float("inf")
    x[4, 50] = float("nan")
    masks = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    masks[1, 2] = 1 << 6                                  # token 70 alone
    masks[2] = -1
    masks[2, 1] = ~(1 << 18)                              # all but token 50
    index = torch.tensor([0, 1, 1, -1, 2], dtype=torch.int32, device="cuda")
    c = L.LogitControls(masks=masks, mask_index=index)
    values = torch.empty(5, device="cuda")
    got = L.select_tokens(x, c, values=values).tolist()
    assert got[:2] == [0, 70] and got[3] == 7
    assert values.tolist()[:4] == [-float("inf"), low, -float("inf"), float("inf")]
    assert got[4] != 50 and torch.isfinite(values[4])     # what the mask hides may be anything
    adjusted = L.adjust_logits(x, c)
    assert torch.isneginf(adjusted[0]).all() and torch.isneginf(adjusted[4, 50]) and torch.equal(adjusted[3], x[3])


def test_histories_longer_than_their_room_and_slots_that_are_none():
    from crosspool_b200.ops import logits as L

    x = torch.ones(4, 64, device="cuda")
    history = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    c = L.LogitControls(history=history, history_rows=t(0, 1, -1, 2), lens=t(9, -3, 4, 4), repetition=torch.full((4,), 2.0, device="cuda"))
    want = x.clone()
    want[0, :4] = 0.5
    assert torch.equal(L.adjust_logits(x, c), want)


def test_the_latest_token_joins_the_history():
    from crosspool_b200.ops import logits as L

    x = torch.full((3, 50), 4.0, device="cuda")
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    history = torch.full((3, 6), 49, dtype=torch.int32, device="cuda")
    c = L.LogitControls(history=history, lens=t(1, 3, 0), prompt_lens=t(0, 0, 0), latest=t(7, 8, 9), presence=torch.ones(3, device="cuda"),
                        frequency=torch.full((3,), 0.5, device="cuda"))
    got = L.adjust_logits(x, c)
    want = x.clone()
    want[0, 7], want[1, 8], want[1, 49] = 2.5, 2.5, 2.0
    assert torch.equal(got, want)
    assert history.tolist() == [[7, 49, 49, 49, 49, 49], [49, 49, 8, 49, 49, 49], [49] * 6]


def test_rows_with_a_pitch_and_nothing_else_written():
    from crosspool_b200.ops import logits as L

    x, c, args = batch(5, 1003, torch.bfloat16, seed=3, wide=2)
    wide = torch.full((5, 1011), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:1006] = x
    out = torch.full((6, 1010), 9.0, device="cuda")
    got = L.adjust_logits(wide[:, 3:1006], c, out=out[:5, 1:1004])
    assert torch.equal(got.cpu(), oracle(x, args, torch.float32))
    out[:5, 1:1004] = 9.0
    assert (out == 9.0).all()
    assert torch.equal(L.select_tokens(wide[:, 3:1006], c), L.select_tokens(x, c))


@pytest.mark.parametrize("select", [False, True])
def test_histories_of_more_different_tokens_than_are_counted_at_once(select):
    from crosspool_b200.ops import logits as L

    g = torch.Generator().manual_seed(4)
    x = (2 * torch.randn(3, 30000, generator=g)).cuda()
    toks = torch.cat([torch.randperm(30000, generator=g)[:9000], torch.randint(0, 400, (3000,), generator=g)]).int()
    history = torch.stack([toks, toks.flip(0), toks]).cuda()
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    ids = toks[::40].contiguous()
    vals = torch.randn(len(ids), generator=g)
    c = L.LogitControls(history=history, lens=t(12000, 12000, 5), prompt_lens=t(4000, 0, 0), repetition=torch.full((3,), 1.3, device="cuda"),
                        frequency=torch.full((3,), 0.2, device="cuda"), presence=torch.full((3,), 0.4, device="cuda"), bias_ids=ids.cuda(),
                        bias_values=vals.cuda(), bias_starts=t(0, len(ids), len(ids), len(ids)))
    want = torch.stack([controls(x[r].cpu(), history[r, :n].tolist(), p, 1.3, 0.2, 0.4, list(zip(ids.tolist(), vals.tolist())) if r == 0 else (),
                                 dtype=torch.float32) for r, (n, p) in enumerate(((12000, 4000), (12000, 0), (5, 0)))])
    if select:
        assert L.select_tokens(x, c).tolist() == want.argmax(1).tolist()
    else:
        y = x.clone()
        assert torch.equal(L.adjust_logits(x, c).cpu(), want) and torch.equal(L.adjust_logits(y, c, out=y).cpu(), want)


@pytest.mark.parametrize("dtype,to", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("vocab", [3, 1021, 12291])
def test_rows_that_begin_anywhere(vocab, dtype, to):
    """A contiguous batch of an odd vocabulary, and results of the same pitch and of another one."""
    from crosspool_b200.ops import logits as L

    x, c, args = batch(17, vocab, dtype, seed=vocab + 1)
    same = oracle(x, args, torch.float32).to(to)
    assert torch.equal(L.adjust_logits(x, c, out=torch.empty(x.shape, dtype=to, device="cuda")).cpu(), same)
    wide = torch.full((17, vocab + 5), 7.0, dtype=to, device="cuda")
    assert torch.equal(L.adjust_logits(x, c, out=wide[:, :vocab]).cpu(), same) and (wide[:, vocab:] == 7.0).all()
    full = L.adjust_logits(x, c, out=torch.empty(x.shape, device="cuda"))
    want = torch.stack([(r == r.max()).nonzero()[0, 0] for r in full]).int()
    assert torch.equal(L.select_tokens(x, c), want)


def test_many_biases_of_few_tokens():
    from crosspool_b200.ops import logits as L

    x = torch.zeros(1, 40, device="cuda")
    g = torch.Generator().manual_seed(1)
    ids, vals = torch.randint(0, 5, (700,), generator=g).int(), torch.randn(700, generator=g)
    c = L.LogitControls(bias_ids=ids.cuda(), bias_values=vals.cuda(), bias_starts=torch.tensor([0, 700], dtype=torch.int32, device="cuda"))
    want = controls(x[0].cpu(), biases=list(zip(ids.tolist(), vals.tolist())), dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(L.adjust_logits(x, c)[0].cpu(), want)


def test_graph_replays_with_other_contents():
    from crosspool_b200.ops import logits as L

    x, c, _ = batch(6, 2000, torch.bfloat16, seed=8)
    out = torch.empty(6, dtype=torch.int32, device="cuda")
    L.select_tokens(x, c, out=out)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        L.select_tokens(x, c, out=out)
    for seed in (9, 10):
        y, d, _ = batch(6, 2000, torch.bfloat16, seed=seed)
        x.copy_(y)
        for name in ("history", "lens", "prompt_lens", "history_rows", "repetition", "frequency", "presence", "masks", "mask_index"):
            getattr(c, name).copy_(getattr(d, name))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, L.select_tokens(x, c))
