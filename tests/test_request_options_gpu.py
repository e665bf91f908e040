"""Engines whose requests share prompt pages, use adapters and put controls on their tokens, against the plain engine and the
monolithic PyTorch forward, alone and all together."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LAYERS = 3


def build(seed=1, **ecfg):
    from crosspool_b200.engine.atn_engine import AttentionEngine, EngineConfig
    from crosspool_b200.engine.ffn_local import LocalFfnPort
    from crosspool_b200.models import config as mc
    from crosspool_b200.models.reference import ReferenceModel
    from crosspool_b200.models.weights import random_attention_weights, random_ffn_weights

    cfg = mc.preset("Qwen/Qwen3-0.6B").with_layers(LAYERS)
    aw, fw = random_attention_weights(cfg, seed, "cuda", torch.bfloat16), random_ffn_weights(cfg, seed, "cuda", torch.bfloat16)
    eng = AttentionEngine(cfg, aw, LocalFfnPort(cfg, fw), EngineConfig(**{**dict(max_batch=16, prefill_chunk=512, max_seq_len=512, page_size=16), **ecfg}))
    return cfg, eng, ReferenceModel(cfg, aw, fw)


def adapter(cfg, seed, rank=8, only=("q", "k", "v", "o")):
    g = torch.Generator().manual_seed(seed)
    dims = {"q": (cfg.hidden_size, cfg.q_size), "k": (cfg.hidden_size, cfg.kv_size), "v": (cfg.hidden_size, cfg.kv_size), "o": (cfg.q_size, cfg.hidden_size)}
    out = []
    for _ in range(cfg.num_layers):
        out.append({p: ((torch.randn(rank, dims[p][0], generator=g) / dims[p][0] ** 0.5).bfloat16().cuda(),
                        (0.5 * torch.randn(dims[p][1], rank, generator=g) / rank ** 0.5).bfloat16().cuda()) for p in only})
    return out


def merged(cfg, aw, layers, scale):
    """Attention weights with an adapter added to them."""
    import copy

    out = copy.copy(aw)
    out.layers = []
    for lw, ad in zip(aw.layers, layers):
        n = copy.copy(lw)
        qkv, at = lw.qkv.float().clone(), 0
        for p, f in (("q", cfg.q_size), ("k", cfg.kv_size), ("v", cfg.kv_size)):
            if p in ad:
                qkv[at:at + f] += scale * ad[p][1].float() @ ad[p][0].float()
            at += f
        n.qkv = qkv.bfloat16()
        n.o = (lw.o.float() + (scale * ad["o"][1].float() @ ad["o"][0].float() if "o" in ad else 0)).bfloat16()
        out.layers.append(n)
    return out


def run(eng, requests):
    """Steps the requests to their ends."""
    for a, kw in requests:
        eng.add_request(*a, **kw)
    while eng.has_work:
        eng.step()


def logits_of(eng, requests):
    """As :func:`run`: (sequences, the logits that each of their tokens was chosen from). Row i of a step belongs to its i-th
    sequence."""
    seqs, got = [eng.add_request(*a, **kw) for a, kw in requests], {}
    while eng.has_work:
        eng.launch_step()
        rows = [s for s, _ in eng._pre_inflight] if eng._pre_inflight is not None else list(eng._inflight[0]) if eng._inflight else []
        done = dict((s.seq_id, t) for s, t in eng.collect_step())
        torch.cuda.synchronize()
        for i, s in enumerate(rows):
            if s.seq_id in done:
                got.setdefault(s.seq_id, []).append(eng.logits[i].float().clone())
    from crosspool_b200.ops import gemm

    gemm.check_status(eng.device)
    return seqs, [torch.stack(got[s.seq_id]) for s in seqs]


def kl(p, q):
    p, q = p.float().log_softmax(-1), q.float().log_softmax(-1)
    return (p.exp() * (p - q)).sum(-1)


def prompts(cfg, lens, shared=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    first = torch.randint(0, cfg.vocab_size, (shared,), generator=g).tolist()
    return [first + torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in lens]


def compare(a, b, limit=1e-3):
    """Two engines' logits while their tokens agree: bf16 residual streams of another order of sums (the limits of the plain
    engine's own test: 0.001 nats a decoded token)."""
    (sa, la), (sb, lb) = a, b
    for x, y, u, v in zip(sa, sb, la, lb):
        n = 1
        while n < len(x.generated) and x.generated[:n] == y.generated[:n]:
            n += 1
        assert kl(u[:n], v[:n]).max().item() <= limit, (x.seq_id, n)


@pytest.mark.parametrize("graph", [False, True])
def test_shared_prefix_decode_is_the_plain_engines(graph):
    ecfg = dict(prefix_cache=True, use_cuda_graph=graph)
    cfg, eng, _ = build(shared_prefix=True, **ecfg)
    _, plain, _ = build(**ecfg)
    results = []
    for e in (eng, plain):
        e.warmup()
        first = prompts(cfg, [5], 130, seed=1)[0]
        run(e, [((first, 1), {})])                                  # the prompt's pages are cached
        reqs = [((p, n), {}) for p, n in zip(prompts(cfg, [3, 20, 1, 40], 130, seed=1) + prompts(cfg, [17, 50], 0, seed=2), (9, 5, 12, 7, 9, 3))]
        results.append(logits_of(e, reqs))
        more = prompts(cfg, [9, 2, 33], 64, seed=5)                  # a second batch shares another prompt, in pages as they come
        results.append(logits_of(e, [((p, 6), {}) for p in more]))
    compare(results[0], results[2])
    compare(results[1], results[3])


def test_shared_prefix_reads_pages_once():
    """Sequences that share pages are side by side in the batch, and the plan says so."""
    cfg, eng, _ = build(shared_prefix=True, prefix_cache=True)
    eng.warmup()
    p = prompts(cfg, [4, 4, 4, 4, 4], 96, seed=3)
    run(eng, [((p[0], 1), {})])
    other = prompts(cfg, [60], seed=9)[0]
    for q in (p[1], other, p[2], p[3]):
        eng.add_request(q, 20)
    seen = []
    while eng.has_work:
        eng.step()
        if len(eng.running) == 4:
            seen.append(eng.prefix_rows.host.numpy().copy())
    w = seen[-1]
    b = eng._bucket(4)
    n = eng.prefix_rows._pieces(b)
    shared = w[4 + 8 * n:][:4].tolist()
    assert w[0] >= 1 and sorted(shared) == [0, 96, 96, 96]


def test_adapters_are_merged_weights():
    from crosspool_b200.models.reference import ReferenceModel

    cfg, eng, ref = build(adapters=4, adapter_rank=24)
    eng.warmup()
    ads = {"a": (adapter(cfg, 1), 2.0), "b": (adapter(cfg, 2, rank=24, only=("q", "v")), 1.0), "c": (adapter(cfg, 3, only=("o",)), -1.5)}
    for name, (layers, scale) in ads.items():
        eng.load_adapter(name, layers, scale)
    ps = prompts(cfg, [5, 33, 70, 12, 64, 7], seed=4)
    names = ["a", None, "b", "c", "a", "b"]
    seqs, got = logits_of(eng, [((p, 5), dict(adapter=n)) for p, n in zip(ps, names)])
    for s, p, n, l in zip(seqs, ps, names, got):
        model = ref if n is None else ReferenceModel(cfg, merged(cfg, eng.w, *ads[n]), ref.ffn)
        toks, want = model.generate(torch.tensor(p, device="cuda"), 5)
        agree = 1
        while agree < 5 and s.generated[:agree] == list(toks[:agree]):
            agree += 1
        # 0.05 nats: the engine's limit for prompts; merging rounds the weights once more
        d = kl(want[:agree], l[:agree])
        assert d.max() <= 0.05, (n, d)
        if n is not None:                                            # far nearer to the merged model than the plain one is
            assert 10 * d[0] < kl(want[:1], ref.generate(torch.tensor(p, device="cuda"), 1)[1])[0]


def test_adapters_come_and_go_and_do_not_share_cached_prompts():
    cfg, eng, _ = build(adapters=1, prefix_cache=True, shared_prefix=True)
    eng.warmup()
    p = prompts(cfg, [40], 64, seed=6)[0]
    plain = logits_of(eng, [((p, 3), {})])[1][0]
    eng.load_adapter("x", adapter(cfg, 7), 2.0)
    with pytest.raises(ValueError, match="is loaded"):
        eng.load_adapter("x", adapter(cfg, 7))
    with pytest.raises(ValueError, match="slots"):
        eng.load_adapter("y", adapter(cfg, 7))
    seqs, both = logits_of(eng, [((p, 3), dict(adapter="x")), ((p, 3), {})])
    hits = eng.prefix.hit_tokens
    assert torch.equal(both[1][0], plain[0]) or kl(plain[:1], both[1][:1]).max() <= 1e-3
    assert kl(plain[:1], both[0][:1]).max() > 0.01
    again = logits_of(eng, [((p, 3), dict(adapter="x"))])[1][0]
    assert eng.prefix.hit_tokens > hits and kl(both[0][:1], again[:1]).max() <= 1e-3     # its own cached pages count
    eng.add_request(p, 3, adapter="x")
    with pytest.raises(ValueError, match="in use"):
        eng.unload_adapter("x")
    while eng.has_work:
        eng.step()
    eng.unload_adapter("x")
    with pytest.raises(ValueError, match="no adapter"):
        eng.add_request(p, 3, adapter="x")
    eng.load_adapter("x", adapter(cfg, 8), 2.0)                      # another one under the name: old pages do not count
    hits = eng.prefix.hit_tokens
    other = logits_of(eng, [((p, 3), dict(adapter="x"))])[1][0]
    assert eng.prefix.hit_tokens == hits and kl(again[:1], other[:1]).max() > 0.01


def oracle_tokens(seq, logits, c, vocab):
    """The tokens that the controls choose greedily from the recorded logits."""
    from request_oracle import controls

    out = []
    for i, row in enumerate(logits):
        mask = c.allowed(seq.generated[:i]) if c.allowed is not None else None
        history = (seq.prompt + seq.generated[:i]) if c.penalises else []
        v = controls(row.cpu(), history, len(seq.prompt) if c.penalises else 0, c.repetition, c.frequency, c.presence, list(c.bias.items()),
                     None if mask is None else [int(w) for w in mask], dtype=torch.float32)
        out.append(int((v == v.max()).nonzero()[0, 0]))
    return out


def only(vocab, tokens):
    w = np.zeros((vocab + 31) // 32, dtype=np.uint32)
    for t in tokens:
        w[t // 32] |= np.uint32(1) << np.uint32(t % 32)
    return w


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("sampling", [False, True])
def test_controls_choose_the_tokens(graph, sampling):
    from crosspool_b200.engine.request_options import TokenControls

    cfg, eng, _ = build(controls=True, use_cuda_graph=graph, sampling=sampling, max_batch=8)
    eng.warmup()
    v = cfg.vocab_size
    cs = [None, TokenControls(repetition=1.5, frequency=0.7, presence=0.4), TokenControls(bias={11: 50.0}), TokenControls(presence=30.0, bias={12: 45.0, 13: 35.0}),
          TokenControls(allowed=lambda g: only(v, [5, 700, v - 1]) if len(g) % 2 else None), TokenControls(repetition=0.5)]
    reqs = [((p, n), dict(controls=c)) for p, n, c in zip(prompts(cfg, [5, 40, 17, 3, 100, 9], seed=8), (6, 12, 5, 6, 7, 9), cs)]
    seqs, got = logits_of(eng, reqs)
    for s, l, c in zip(seqs, got, cs):
        assert s.generated == oracle_tokens(s, l, c or TokenControls(), v), s.seq_id
    assert seqs[2].generated == [11] * 5 and seqs[3].generated[:2] == [12, 13]
    assert all(t in (5, 700, v - 1) for t in seqs[4].generated[1::2])
    assert not eng.control_rows.slots and sorted(eng.control_rows.free) == list(range(8))
    # the slots' next sequences begin with histories of their own
    seqs, got = logits_of(eng, reqs)
    for s, l, c in zip(seqs, got, cs):
        assert s.generated == oracle_tokens(s, l, c or TokenControls(), v), s.seq_id


def test_controls_after_a_retraction_and_in_chunks():
    from crosspool_b200.engine.request_options import TokenControls

    cfg, eng, _ = build(controls=True, max_batch=4, prefill_chunk=64, max_seq_len=256, num_pages=24)
    eng.warmup()
    c = TokenControls(repetition=1.4, frequency=0.6, presence=0.3)
    seqs, got = logits_of(eng, [((p, 60), dict(controls=c)) for p in prompts(cfg, [90, 80, 70], seed=11)])
    assert any(s.refill_len for s in seqs)                           # the cache has no room for all three at their ends
    for s, l in zip(seqs, got):
        assert s.generated == oracle_tokens(s, l, c, cfg.vocab_size)


@pytest.mark.parametrize("mixed", [False, True])
def test_everything_at_once(mixed):
    """Requests that share a prompt, with adapters and controls of their own, in one batch: the logits are those of an engine
    without shared-prefix attention, the tokens those that the controls choose from them."""
    from crosspool_b200.engine.request_options import TokenControls

    results = []
    for shared in (True, False):
        cfg, eng, _ = build(controls=True, adapters=3, adapter_rank=16, prefix_cache=True, shared_prefix=shared, max_batch=12, mixed_batches=mixed)
        eng.warmup()
        for i, name in enumerate(("a", "b", "c")):
            eng.load_adapter(name, adapter(cfg, 20 + i, rank=4 + 6 * i), 1.0)
        v = cfg.vocab_size
        ps = prompts(cfg, [4, 9, 30, 5, 18, 2, 11, 6], 100, seed=13)
        names = [None, "a", "a", "b", None, "c", "b", None]
        cs = [None, TokenControls(repetition=1.3), TokenControls(bias={3: 40.0}, presence=50.0), None, TokenControls(frequency=1.0),
              TokenControls(allowed=lambda g: only(v, range(64))), None, TokenControls(0.7, -0.2, 0.5)]
        run(eng, [((ps[0], 1), {}), ((ps[1], 1), dict(adapter="a")), ((ps[3], 1), dict(adapter="b"))])
        seqs, got = logits_of(eng, [((p, 10), dict(adapter=n, controls=c)) for p, n, c in zip(ps, names, cs)])
        for s, l, c in zip(seqs, got, cs):
            assert s.generated == oracle_tokens(s, l, c or TokenControls(), v), s.seq_id
        results.append((seqs, got))
    compare(*results)


def test_engines_that_are_refused():
    with pytest.raises(ValueError, match="pages"):
        build(shared_prefix=True, page_size=8)
    cfg, eng, _ = build(adapters=1)
    with pytest.raises(ValueError, match="layers"):
        eng.load_adapter("a", [])
    with pytest.raises(ValueError, match="projections"):
        eng.load_adapter("a", [{"gate": None}] * LAYERS)
    with pytest.raises(ValueError, match="rank"):
        eng.load_adapter("a", adapter(cfg, 1, rank=17))
    assert not eng.adapter_rows.names


@pytest.mark.parametrize("graph", [False, True])
def test_a_step_whose_mask_failed_can_be_taken_again(graph):
    from crosspool_b200.engine.request_options import TokenControls

    results = []
    for fail in (False, True):
        cfg, eng, _ = build(controls=True, shared_prefix=True, prefix_cache=True, use_cuda_graph=graph, max_batch=8)
        eng.warmup()
        failed = []

        def allowed(g):
            if fail and len(g) in (0, 3, 4) and len(g) not in failed:
                failed.append(len(g))
                raise RuntimeError("no mask yet")
            return only(cfg.vocab_size, range(len(g), 3000))

        a, b = prompts(cfg, [30, 41], shared=20, seed=3)
        seqs = [eng.add_request(a, 8, controls=TokenControls(repetition=1.3, frequency=0.5)), eng.add_request(b, 8, controls=TokenControls(allowed=allowed))]
        while eng.has_work:
            try:
                eng.step()
            except RuntimeError as e:
                assert str(e) == "no mask yet"
        assert failed == ([0, 3, 4] if fail else [])
        results.append([s.generated for s in seqs])
    assert results[0] == results[1]


def test_an_engine_is_warmed_up_again():
    """The plans' words of the last batch lie as its row bucket's; the other buckets' graphs find none."""
    cfg, eng, ref = build(shared_prefix=True, prefix_cache=True, adapters=2, max_batch=16)
    eng.load_adapter("a", adapter(cfg, 5))
    reqs = [((p, 6), dict(adapter=n)) for p, n in zip(prompts(cfg, [50, 60, 70, 40, 33], shared=32, seed=4), ["a", None, "a", None, "a"])]
    eng.warmup()
    first, got = logits_of(eng, reqs)
    eng.warmup()
    assert not eng.prefix_rows.words.any() and not eng.adapter_rows.words.any()
    second, again = logits_of(eng, reqs)
    assert [s.generated for s in first] == [s.generated for s in second]
