"""Calls of the operators of requests at the edges of what their documentation allows."""
import pytest
import torch

from request_oracle import paged_attention

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ shared prefixes

def cache(rows, tokens, hq, hk, d, page, seed=0):
    """Rows of ``tokens`` tokens each, in pages of their own."""
    g = torch.Generator().manual_seed(seed)
    wide = -(-tokens // page)
    table = torch.randperm(rows * wide, generator=g).int().view(rows, wide)
    k, v = (torch.randn(rows * wide, page, hk, d, generator=g).bfloat16() for _ in range(2))
    q = (1.5 * torch.randn(rows, hq, d, generator=g)).bfloat16()
    return [t.cuda() for t in (q, k, v, table)]


def close(got, q, k, v, table, lens, scale=None):
    """The weights are rounded to bf16 (half a step: 2^-8 of each), the result once more; what fp32 sums and 2 ** x add is below
    2^-14 of the weighted values: scores below 64 carry d 2^-24 64 of error."""
    want, mass = paged_attention(q, k, v, table, lens, scale)
    off, tol = (got.double() - want).abs(), (2.0 ** -8 + 2.0 ** -14) * mass + 2.0 ** -8 * want.abs() + 1e-30
    assert torch.isfinite(got).all() and (off <= tol).all(), (off / tol).max()


@pytest.mark.parametrize("sizes,prefixes,max_len", [([], [], n) for n in (0, 1, 100, 640, 2000)] + [(s, p, n) for s, p in (([5], [7]), ([3], [64])) for n in (100, 640, 2000)])
@pytest.mark.parametrize("rows,d", [(5, 128), (5, 64), (300, 64)])
def test_rows_are_read_no_further_than_the_plans_bound(sizes, prefixes, max_len, rows, d):
    """Whether the plan holds a prefix or not, and whether rows are read in one slice or in several. The tables hold all tokens
    that the lengths name, so that reading on would stay in the cache."""
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    q, k, v, table = cache(rows, max(max_len, 16) + 200, 8, 4, d, 16, seed=max_len)
    for r in range(1, sum(sizes)):
        table[r, :prefixes[0] // 16] = table[0, :prefixes[0] // 16]
    lens = torch.full((rows,), max_len, dtype=torch.int32, device="cuda")
    lens[0], lens[1], lens[2], lens[3] = max_len + 1, max_len + 200, max_len // 2, -3
    plan = A.shared_prefix_plan(sizes, prefixes, rows=rows, q_heads=8, kv_heads=4, head_dim=d, max_len=max_len)
    got = A.paged_decode_shared(q, k, v, table, lens, plan)
    gemm.check_status(q.device)
    close(got, q, k, v, table, lens.clamp(0, max_len))
    assert not got[3].any()


# ------------------------------------------------------------------------------------------------ adapters

def behind(stream, ms=60):
    """Keeps ``stream`` busy for about so long."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 1.9e6))


def test_adapters_computed_on_the_callers_stream_are_loaded_when_they_are_there():
    from test_request_options_gpu import build

    from crosspool_b200.ops import lora

    cfg, eng, _ = build(adapters=1, adapter_rank=16)
    g = torch.Generator().manual_seed(3)
    a, b = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((8, cfg.hidden_size), (cfg.kv_size, 8)))
    want = lora.AdapterStack(1, cfg.hidden_size, (cfg.q_size, cfg.kv_size, cfg.kv_size), 16)
    want.load(0, [None, 2 * a, None], [None, 4 * b, None])
    torch.cuda.synchronize()
    late, side = [(torch.zeros_like(a), torch.zeros_like(b)) for _ in range(cfg.num_layers)], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    behind(side)
    with torch.cuda.stream(side):
        for x, y in late:
            x.copy_(a).mul_(2)
            y.copy_(b).mul_(4)
        eng.load_adapter("x", [{"k": pair} for pair in late])
    for stack in eng.adapter_rows.qkv:
        assert torch.equal(stack.a, want.a) and torch.equal(stack.b, want.b)


def test_slots_of_a_stack_made_behind_other_work_are_loaded_on_any_stream():
    from crosspool_b200.ops import lora

    a, b = torch.ones(8, 256, device="cuda").bfloat16(), torch.ones(128, 8, device="cuda").bfloat16()
    torch.cuda.synchronize()
    maker, loader = torch.cuda.Stream(), torch.cuda.Stream()
    behind(maker)
    with torch.cuda.stream(maker):
        stack = lora.AdapterStack(2, 256, 128, 8)
    with torch.cuda.stream(loader):
        stack.load(1, a, b, 0.5)
    torch.cuda.synchronize()
    assert stack.ranks.tolist() == [0, 16] and stack.scale.tolist() == [0.0, 0.5] and stack.part_ranks.tolist() == [[0] * 4, [8, 0, 0, 0]]
    assert stack.a[1].float().sum() == 8 * 256 and stack.b[1].float().sum() == 128 * 8


# ------------------------------------------------------------------------------------------------ masks

@pytest.mark.parametrize("mixed", [False, True])
def test_requests_whose_mask_fails_leave_the_engine_with_all_they_held(mixed):
    import queue

    import numpy as np
    from test_request_options_gpu import adapter, build, prompts

    from crosspool_b200.deployment import Deployment, InstanceHandle
    from crosspool_b200.engine.request_options import TokenControls
    from crosspool_b200.runtime.serving import EngineLoop

    cfg, eng, _ = build(controls=True, shared_prefix=True, prefix_cache=True, adapters=1, max_batch=8, mixed_batches=mixed)
    eng.load_adapter("a", adapter(cfg, 5))
    eng.warmup()
    full = eng.kv.allocator.free_pages
    words = (cfg.vocab_size + 31) // 32

    def until(n):
        def allowed(g):
            if len(g) == n:
                raise KeyError(n)
            return None
        return TokenControls(repetition=1.2, presence=0.5, allowed=allowed)

    cs = [None, until(0), until(1), until(6), TokenControls(allowed=lambda g: np.zeros(words, dtype=np.uint32) if len(g) == 4 else None),
          TokenControls(allowed=lambda g: [1]), TokenControls(repetition=1.3)]
    loop = EngineLoop(Deployment([InstanceHandle("m", cfg, eng)]))
    ps = [loop.submit("m", p, 12, options={**({} if c is None else {"controls": c}), **({"adapter": "a"} if i % 2 else {})})
          for i, (p, c) in enumerate(zip(prompts(cfg, [30, 41, 5, 18, 60, 7, 22], shared=40, seed=3), cs))]
    loop.start()
    try:
        got = []
        for p in ps:
            toks = []
            while True:
                item = p.out.get(timeout=60)
                if isinstance(item, Exception):
                    got.append((len(toks), type(item).__name__))
                    break
                toks.append(item[0])
                if item[1]:
                    got.append((len(toks), None))
                    break
        assert got == [(12, None), (0, "KeyError"), (1, "KeyError"), (6, "KeyError"), (4, "ValueError"), (0, "ValueError"), (12, None)]
        with pytest.raises(queue.Empty):
            ps[0].out.get_nowait()
    finally:
        loop.stop()
    assert loop.error is None and not eng.has_work and not eng.control_rows.slots and len(eng.control_rows.free) == 8
    eng.kv.allocator.free(eng.prefix.evict(10 ** 6))
    assert eng.kv.allocator.free_pages == full and not eng.kv.tables


# ------------------------------------------------------------------------------------------------ shared prefixes, infinities

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,lens", [(3, [90, 41, 300]), (200, [90, 41, 300, 57]), (3, [700, 1500, 900])])
def test_keys_of_minus_infinity_weigh_nothing_where_no_rows_share(rows, lens, d):
    """The first 40 tokens of every row have scores of -inf; with long rows the first of several slices begins with them."""
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    q, k, v, table = cache(rows, 1500, 8, 2, d, 16, seed=d)
    n = torch.tensor([lens[r % len(lens)] for r in range(rows)], dtype=torch.int32, device="cuda")
    q = q.abs()
    for r in range(rows):
        k[table[r, 0:2].long(), :, :, 5] = float("-inf")
        k[table[r, 2].long(), :8, :, 5] = float("-inf")
    plan = A.shared_prefix_plan([], [], rows=rows, q_heads=8, kv_heads=2, head_dim=d, max_len=int(n.max()))
    for got in (A.paged_decode_shared(q, k, v, table, n, plan), A.paged_decode(q, k, v, table, n, max_len=1500)):
        gemm.check_status(q.device)
        close(got, q, k, v, table, n)


@pytest.mark.parametrize("sizes,prefixes", [([], []), ([5], [320])])
@pytest.mark.parametrize("tokens", [400, 2000])
def test_results_may_lie_over_their_queries(sizes, prefixes, tokens):
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    q, k, v, table = cache(9, tokens, 8, 2, 128, 16)
    table[1:sum(sizes), :20] = table[:1, :20]
    n = torch.tensor([tokens - 7 * r for r in range(9)], dtype=torch.int32, device="cuda")
    plan = A.shared_prefix_plan(sizes, prefixes, rows=9, q_heads=8, kv_heads=2, head_dim=128, max_len=tokens)
    want = A.paged_decode_shared(q, k, v, table, n, plan)
    assert A.paged_decode_shared(q, k, v, table, n, plan, out=q) is q and torch.equal(q, want)
    gemm.check_status(q.device)


# ------------------------------------------------------------------------------------------------ draws

def highest_hashes(rows, vocab, steps):
    """(row, step, token) of the draws whose noise comes from the last of 2^24 steps (``csrc/include/xpool/gumbel.cuh``)."""
    import numpy as np

    out = []
    with np.errstate(over="ignore"):
        for step in range(steps):
            a, c = np.arange(rows, dtype=np.uint64)[:, None] << np.uint64(32), np.arange(vocab, dtype=np.uint64)[None]
            x = a ^ (np.uint64(step) * np.uint64(0x9E3779B97F4A7C15)) ^ c
            x ^= x >> np.uint64(30)
            x *= np.uint64(0xBF58476D1CE4E5B9)
            x ^= x >> np.uint64(27)
            x *= np.uint64(0x94D049BB133111EB)
            x ^= x >> np.uint64(31)
            r, t = np.nonzero(((x >> np.uint64(16)) & np.uint64(0xFFFFFFFF)) >> np.uint64(8) == np.uint64(0xFFFFFF))
            out += [(int(i), step, int(j)) for i, j in zip(r, t)]
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_noise_draws_a_token_that_has_no_weight(dtype):
    """Every draw's highest noise is finite: a token 100 below another one at temperature 1 has a chance of e^-100."""
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import logits as L

    rows, vocab = 64, 4096
    hits = highest_hashes(rows, vocab, 400)                          # 6 are expected of 10^8 draws
    assert len(hits) >= 2
    temps = torch.ones(rows, device="cuda")
    for row, step, token in hits:
        x = torch.full((rows, vocab), -50.0, device="cuda", dtype=dtype)
        best = (token + 7) % vocab
        x[:, best] = 50.0
        seeds = torch.stack([torch.arange(rows), torch.full((rows,), step)], 1).int().cuda()
        for got in (A.sample(x, temps, seeds), L.select_tokens(x, L.LogitControls(), temps, seeds)):
            assert (got == best).all(), (row, step, token)


# ------------------------------------------------------------------------------------------------ host threads

FIRST_CALLS = """
import sys, threading
import torch
from crosspool_b200.ops import attention as A, logits as L, lora

torch.manual_seed(0)
rows = 6
q = torch.randn(rows, 8, 128, device="cuda").bfloat16()
k, v = (torch.randn(rows * 8, 16, 2, 128, device="cuda").bfloat16() for _ in range(2))
table = torch.arange(rows * 8, dtype=torch.int32, device="cuda").view(rows, 8)
table[:, :4] = table[0, :4]
lens = torch.full((rows,), 100, dtype=torch.int32, device="cuda")
plan = A.shared_prefix_plan([rows], [64], rows=rows, q_heads=8, kv_heads=2, head_dim=128, max_len=128)
stack = lora.AdapterStack(1, 256, 512, 16)
stack.load(0, torch.randn(16, 256, device="cuda"), torch.randn(512, 16, device="cuda"))
adapters = lora.adapter_plan([0] * rows, stack)
x, y, z = torch.randn(rows, 256, device="cuda").bfloat16(), torch.randn(rows, 512, device="cuda").bfloat16(), torch.randn(rows, 9000, device="cuda")
none = L.LogitControls()
torch.cuda.synchronize()
got, start = [None] * 4, threading.Barrier(4)


def work(i):
    out = []
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        for _ in range(50):
            out = [A.paged_decode_shared(q, k, v, table, lens, plan), lora.lora_add(y, x, stack, adapters), L.select_tokens(z, none), L.adjust_logits(z, none)]
        torch.cuda.current_stream().synchronize()
    got[i] = out


threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[t.start() for t in threads]
[t.join() for t in threads]
want = [A.paged_decode_shared(q, k, v, table, lens, plan), lora.lora_add(y, x, stack, adapters), L.select_tokens(z, none), L.adjust_logits(z, none)]
sys.exit(0 if all(g is not None and all(torch.equal(a, b) for a, b in zip(g, want)) for g in got) else 1)
"""


def test_first_calls_of_four_threads_at_once():
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ calls that the documentation allows

@pytest.mark.parametrize("hq,hk,d", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("parts", [1, 8, 32])
def test_long_prefixes_in_few_pieces(hq, hk, d, parts):
    """Plans of few pieces, as an engine's captured steps bound them, and more rows in the call than in the plan."""
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    rows, prefix, extra = 4, 20000, 2
    q, k, v, table = cache(rows + extra, prefix + 96, hq, hk, d, 32, seed=parts)
    table[1:rows, :prefix // 32] = table[0, :prefix // 32]
    words = torch.zeros(A.shared_plan_words(rows, 40), dtype=torch.int32)
    count, most = A.fill_shared_plan([rows], [prefix], words.numpy(), rows, 40, parts, q_heads=hq, kv_heads=hk, head_dim=d, own_tokens=200)
    assert 1 <= most <= parts and count == most
    plan = A.SharedPrefixPlan(words.cuda(), rows, 40, parts, prefix + 96, hq, hk, d)
    lens = torch.tensor([prefix + 1, prefix + 96, prefix, prefix - 1, 33, 19000], dtype=torch.int32, device="cuda")
    got = A.paged_decode_shared(q, k, v, table, lens, plan)
    gemm.check_status(q.device)
    close(got, q, k, v, table, lens)


def test_rows_of_one_table():
    """Every row reads the same sequence, through a table that is there once."""
    from crosspool_b200.ops import attention as A
    from crosspool_b200.ops import gemm

    q, k, v, table = cache(70, 400, 8, 2, 128, 16)
    one = table[:1].expand(70, -1)
    lens = torch.full((70,), 400, dtype=torch.int32, device="cuda")
    plan = A.shared_prefix_plan([70], [400], rows=70, q_heads=8, kv_heads=2, head_dim=128, max_len=400)
    got = A.paged_decode_shared(q, k, v, one, lens, plan)
    gemm.check_status(q.device)
    close(got, q, k, v, one, lens)


@pytest.mark.parametrize("rows", [3, 200])
def test_selected_tokens_go_where_the_latest_ones_came_from(rows):
    """A decode loop whose tokens of a step are the latest ones of the next."""
    from crosspool_b200.ops import logits as L

    vocab, steps = 9000, 5
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    history = torch.full((rows, steps + 2), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    c = L.LogitControls(history=history, lens=lens, latest=tokens, presence=torch.full((rows,), 100.0, device="cuda"))
    x = torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    want = x.topk(steps, dim=1).indices.int()                         # the penalty keeps every token from coming twice
    for step in range(steps):
        L.select_tokens(x, c, out=tokens)
        assert torch.equal(tokens, want[:, step])
        lens += 1
    assert torch.equal(history[:, :steps - 1], want[:, :steps - 1])
