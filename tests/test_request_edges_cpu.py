"""Operators of requests, their engine and their serving loop at the edges of what their documentation allows; no GPU is needed."""
import contextlib
import random

import numpy as np
import pytest
import torch

from test_engine_bookkeeping import bare_engine


# ------------------------------------------------------------------------------------------------ adapters

@pytest.mark.parametrize("fails", [False, True])
def test_adapters_are_read_behind_the_callers_stream_and_before_the_call_returns(monkeypatch, fails):
    done = []

    class Stream:
        def wait_stream(self, other):
            done.append(("wait", other))

        def synchronize(self):
            done.append("synchronize")

    class Rows:
        def load(self, name, layers, scale):
            done.append((on[-1], name, layers, scale))
            if fails:
                raise ValueError("rank")

    @contextlib.contextmanager
    def stream(s):
        on.append(s)
        yield
        on.pop()

    eng, on = bare_engine(), ["caller"]
    eng.stream, eng.adapter_rows, eng.device = Stream(), Rows(), torch.device("cpu")
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: on[-1])
    with pytest.raises(ValueError, match="rank") if fails else contextlib.nullcontext():
        eng.load_adapter("x", [1], 2.0)
    assert done == [("wait", "caller"), (eng.stream, "x", [1], 2.0), "synchronize"]


# ------------------------------------------------------------------------------------------------ masks

def control_rows(vocab):
    from crosspool_b200.engine.request_options import ControlRows

    rows = ControlRows.__new__(ControlRows)
    rows.vocab, rows.words = vocab, (vocab + 31) // 32
    return rows


def with_mask(allowed, generated=()):
    from crosspool_b200.engine.atn_engine import Sequence
    from crosspool_b200.engine.request_options import TokenControls

    return Sequence(3, [1], 4, generated=list(generated), controls=TokenControls(allowed=allowed))


@pytest.mark.parametrize("vocab,words", [(40, [0, 1]), (40, [0, 0x80]), (64, [0, 0x80000000]), (32, [1]), (1, [1]), (40, [0x80000000, 0])])
@pytest.mark.parametrize("dtype", ["uint32", "int32", "int64"])
def test_masks_that_a_token_fits(vocab, words, dtype):
    want = np.array(words, dtype=np.uint32).view(np.int32)
    given = want if dtype == "int32" else np.array(words, dtype=dtype)
    assert control_rows(vocab).mask(with_mask(lambda g: given)).tolist() == want.tolist()
    assert control_rows(vocab).mask(with_mask(lambda g: None)) is None


@pytest.mark.parametrize("vocab,mask,match", [(40, [0, 0], "no token"), (40, [0, 0xffffff00], "no token"), (1, [0xfffffffe], "no token"), (64, [0, 0], "no token"),
                                              (40, [1], "shape"), (40, [[1, 1]], "shape"), (40, "x", "shape")])
def test_masks_that_fail_their_request(vocab, mask, match):
    from crosspool_b200.engine.request_options import RequestFailed

    s = with_mask(lambda g: mask if isinstance(mask, str) else np.array(mask, dtype=np.uint32))
    with pytest.raises(RequestFailed, match=match) as e:
        control_rows(vocab).mask(s)
    assert e.value.sequence is s and isinstance(e.value.__cause__, ValueError)


def test_a_request_is_dropped_with_its_pages():
    eng = bare_engine()
    eng._pending = eng._pre_inflight = eng._inflight = eng.capacity = None
    a, b, c, d = (eng.add_request([i + 1], 4) for i in range(4))
    eng.waiting.remove(b)
    eng.waiting.remove(c)
    eng.prefilling.append(b)
    eng.running.append(c)
    eng._b_key = (c.seq_id,)
    why = ValueError("why")
    for s in (a, b, c):
        eng.drop_request(s, why)
    assert list(eng.waiting) == [d] and not eng.prefilling and not eng.running and eng._b_key is None
    assert eng.kv.released == [a.seq_id, b.seq_id, c.seq_id] and a.error is why and d.error is None
    with pytest.raises(ValueError, match="not in"):
        eng.drop_request(a)
    eng._inflight = ([d], 1)
    with pytest.raises(RuntimeError, match="in flight"):
        eng.drop_request(d)


class MaskedEngine:
    """Stands for an engine: every request gets a token a step, the next one's number; one with a mask asks it first."""

    def __init__(self):
        self.live, self._out, self._next = [], None, 0

    def add_request(self, prompt, max_new_tokens, arrival=None, controls=None):
        from crosspool_b200.engine.atn_engine import Sequence

        s = Sequence(self._next, list(prompt), max_new_tokens, controls=controls)
        self._next += 1
        self.live.append(s)
        return s

    has_work = property(lambda self: bool(self.live))
    step_in_flight = property(lambda self: self._out is not None)

    def step_ready(self):
        return True

    def drop_request(self, s, error=None):
        assert self._out is None
        self.live.remove(s)
        s.error = error

    def launch_step(self):
        assert self._out is None, "launched twice"
        for s in self.live:
            if s.controls is not None:
                control_rows(40).mask(s)
        self._out = list(self.live)

    def collect_step(self):
        seqs, self._out = self._out or [], None
        for s in seqs:
            s.generated.append(len(s.generated))
            if s.finished:
                self.live.remove(s)
        return [(s, s.generated[-1]) for s in seqs]


def drain(p, timeout=20):
    got = []
    while True:
        item = p.out.get(timeout=timeout)
        if isinstance(item, Exception):
            return got, item
        got.append(item[0])
        if item[1]:
            return got, None


@pytest.mark.parametrize("stepping", ["step", "step_async"])
def test_a_mask_that_fails_ends_its_request_alone(stepping):
    from crosspool_b200.deployment import Deployment, InstanceHandle
    from crosspool_b200.engine.request_options import TokenControls
    from crosspool_b200.runtime.serving import EngineLoop

    dep = Deployment([InstanceHandle(m, None, MaskedEngine()) for m in ("a", "b")])
    if stepping == "step":
        dep.step_async = dep.step
    loop = EngineLoop(dep)

    def raises(g):
        if len(g) == 2:
            raise KeyError("grammar")
        return None

    masks = [raises, lambda g: np.zeros(2, dtype=np.uint32) if len(g) == 3 else None, lambda g: np.zeros(9, dtype=np.uint32)]
    plain = [loop.submit(m, [1], 9) for m in ("a", "b")]
    bad = [loop.submit("b", [1], 9, options={"controls": TokenControls(allowed=f)}) for f in masks]
    alone = loop.submit("a", [1], 9, options={"controls": TokenControls(allowed=raises)})
    loop.start()
    try:
        assert all(drain(p) == (list(range(9)), None) for p in plain)
        got = [drain(p) for p in (*bad, alone)]
        assert [(g, type(e)) for g, e in got] == [([0, 1], KeyError), ([0, 1, 2], ValueError), ([], ValueError), ([0, 1], KeyError)]
        later = loop.submit("b", [1], 3)                        # the loop goes on, also after an Instance that was left without work
        assert drain(later) == ([0, 1, 2], None) and loop.error is None and not loop._by_seq
    finally:
        loop.stop()


def test_the_only_request_of_a_deployment_may_fail():
    from crosspool_b200.deployment import Deployment, InstanceHandle
    from crosspool_b200.engine.request_options import TokenControls

    dep = Deployment([InstanceHandle("a", None, MaskedEngine())])
    s = dep.add_request("a", [1], 4, controls=TokenControls(allowed=lambda g: np.zeros(2, dtype=np.int32)))
    res = dep.step()
    assert [(m, x) for m, x, _ in res.failed] == [("a", s)] and res.num_tokens == 0 and not dep.has_work and isinstance(s.error, ValueError)


def test_masks_of_one_buffer_are_read_when_they_are_given():
    """A grammar library may fill the same words for every call."""
    words = np.zeros(2, dtype=np.int32)

    def allowed(token):
        def f(g):
            words[:] = [1 << token, 0]
            return words
        return f

    rows = control_rows(40)
    got = [rows.mask(with_mask(allowed(t))) for t in (3, 9)]
    assert [m.tolist() for m in got] == [[8, 0], [512, 0]]


# ------------------------------------------------------------------------------------------------ replicated requests

def _tp_rank(rank, port, q):
    import os
    import threading
    import time

    import torch.distributed as dist
    from test_tp_replication import FakeDeployment

    from crosspool_b200.engine.request_options import TokenControls
    from crosspool_b200.runtime.tp_replication import TpEngineLoop

    class Deployment(FakeDeployment):
        def add_request(self, model, prompt, max_new_tokens, **kw):
            s = super().add_request(model, prompt, max_new_tokens, **kw)
            self.log[-1] += (kw,)
            return s

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    dep = Deployment()
    loop = TpEngineLoop(dep, None, leader=rank == 0, idle_sleep=0.001)
    loop.start()
    out = None
    if rank == 0:
        options = [{"controls": TokenControls(1.2, allowed=lambda g: None)}, {"controls": TokenControls(allowed=print)}, {"adapter": threading.Lock()},
                   {"controls": TokenControls(1.5)}, {}]
        asked = [loop.submit("m", [i + 1], 2, options=o) for i, o in enumerate(options)]
        try:
            out = [(g, type(e).__name__) for g, e in (drain(p) for p in asked)]
        except Exception as e:
            out = repr(e)
        later = loop.submit("m", [9], 1)
        time.sleep(0.05)
        out = (out, drain(later)[0])
        loop.stop()
    else:
        loop._thread.join(30)
    q.put((rank, out, [e[2:] for e in dep.log if e[0] == "add"], repr(loop.error)))
    dist.destroy_process_group()


def test_options_that_cannot_be_replicated_fail_their_request_alone():
    import multiprocessing as mp
    import os

    from crosspool_b200.engine.request_options import TokenControls

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    ps = [ctx.Process(target=_tp_rank, args=(r, 29900 + os.getpid() % 90, q), daemon=True) for r in (0, 1)]
    for p in ps:
        p.start()
    try:
        res = {r[0]: r[1:] for r in (q.get(timeout=60) for _ in ps)}
    finally:
        for p in ps:
            p.join(10)
            if p.is_alive():
                p.terminate()
    refused, done = res[0][0]
    assert refused == [([], "ValueError")] * 3 + [([0, 1], "NoneType"), ([100, 101], "NoneType")] and done == [200]
    added = [((4,), 2, {"controls": TokenControls(1.5)}), ((5,), 2, {}), ((9,), 1, {})]
    assert res[0][1] == res[1][1] == added and res[0][2] == res[1][2] == "None"


# ------------------------------------------------------------------------------------------------ results over inputs

def test_rows_that_meet():
    from crosspool_b200.ops.overlap import rows_meet

    rng = random.Random(7)
    for _ in range(3000):
        rows = rng.randrange(0, 5)
        pitch = rng.randrange(1, 12)
        a, b = ((rng.randrange(0, 40), p, rng.randrange(1, 8)) for p in (pitch, pitch if rng.random() < 0.7 else rng.randrange(0, 12)))
        sa, sb = ({at + r * p + i for r in range(rows) for i in range(w)} for at, p, w in (a, b))
        got = rows_meet(rows, *a, *b)
        assert got or not sa & sb                                   # never missed
        wide = min(a[1], b[1]) >= max(a[2], b[2])
        apart = not sa or not sb or max(sa) < min(sb) or max(sb) < min(sa)
        assert not (got and apart)
        if got and not sa & sb:                                     # what is refused all the same: pitches that differ, rows that wrap
            assert a[1] != b[1] or not wide or (b[0] - a[0]) % a[1] + b[2] > a[1] or (b[0] - a[0]) % a[1] < a[2]


def lora_case(rows=4):
    from crosspool_b200.ops import lora

    stack = lora.AdapterStack(2, 64, 48, 16, device="cpu")
    return stack, lora.adapter_plan([0, 1, -1, 0][:rows], stack)


def test_adapters_refuse_results_that_lie_over_other_rows():
    from crosspool_b200.ops import lora

    s, p = lora_case()
    b = torch.bfloat16
    buf, flat, x, y = torch.zeros(5, 128, dtype=b), torch.zeros(1024, dtype=b), torch.zeros(4, 64, dtype=b), torch.zeros(4, 48, dtype=b)
    side = flat.as_strided((4, 64), (80, 1))                        # 64 of every 80 columns
    for yy, xx, out in ((buf[:4, :48], x, buf[:4, 16:64]), (buf[:4, :48], x, buf[1:, :48]), (buf[1:, :48], x, buf[:4, :48]), (y, buf[:4, :64], buf[:4, 56:104]),
                        (y, buf[:4, :64], buf[1:, :48]), (y, buf[:4, 64:], buf[:4, 64:112]), (y, side, flat.as_strided((4, 48), (64, 1), 64)),
                        (y, side, flat.as_strided((4, 48), (80, 1), 72))):
        with pytest.raises(ValueError, match="over"):
            lora.lora_add(yy, xx, s, p, out=out)
    for yy, xx, out in ((y, x, y), (buf[:4, :48], x, buf[:4, :48]), (buf[:4, :48], buf[:4, 64:], buf[:4, :48]), (y, buf[:4, :64], buf[:4, 64:112]),
                        (buf[:4, :48], x, buf[:4, 48:96]), (y, side, flat.as_strided((4, 48), (64, 1), 512))):
        with pytest.raises(ValueError, match="GPU"):
            lora.lora_add(yy, xx, s, p, out=out)
    one, plan = lora_case(1)
    with pytest.raises(ValueError, match="over"):
        lora.lora_add(buf[:1, :48], x[:1], one, plan, out=buf[:1, 40:88])
    with pytest.raises(ValueError, match="GPU"):
        lora.lora_add(buf[:1, :48], x[:1], one, plan, out=buf[:1, 48:96])


def test_adjusted_logits_refuse_results_that_lie_over_other_rows():
    from crosspool_b200.ops import logits as L

    none, z, b = L.LogitControls(), torch.zeros(5, 100), torch.zeros(5, 200, dtype=torch.bfloat16)
    for x, out in ((z[:4], z[1:]), (z[1:], z[:4]), (z[:, :60], z[:, 40:]), (b[:4, :100], b.view(torch.float32)[1:]), (z[:1, :60], z[:1, 40:]),
                   (z.view(torch.bfloat16)[:, 100:], z)):
        with pytest.raises(ValueError, match="over|in place"):
            L.adjust_logits(x, none, out=out)
    for x, out in ((z, z), (z[:2], z[2:4]), (z[:, :50], z[:, 50:]), (b[:4, :100], torch.zeros(4, 100)), (b[:, :100], b[:, 100:]), (z[:, 1:50], z[:, 51:])):
        with pytest.raises(ValueError, match="GPU"):
            L.adjust_logits(x, none, out=out)


@pytest.mark.parametrize("prefixes", [[64], []])
def test_shared_prefix_attention_refuses_results_that_lie_over_other_queries(prefixes):
    from crosspool_b200.ops import attention as A

    bf, i32 = torch.bfloat16, torch.int32
    buf = torch.zeros(5 * 8 * 128, dtype=bf)
    rest = dict(k_cache=torch.zeros(9, 16, 2, 128, dtype=bf), v_cache=torch.zeros(9, 16, 2, 128, dtype=bf), block_table=torch.zeros(4, 8, dtype=i32),
                seq_lens=torch.zeros(4, dtype=i32))
    rest["plan"] = A.shared_prefix_plan([4] if prefixes else [], prefixes, rows=4, q_heads=8, kv_heads=2, head_dim=128, max_len=128, device="cpu")
    q = buf[:4096].view(4, 8, 128)
    for out in (buf[1024:].view(4, 8, 128), buf[8:4104].view(4, 8, 128)):
        for a, b in ((q, out), (out, q)):
            with pytest.raises(ValueError, match="over"):
                A.paged_decode_shared(a, out=b, **rest)
    for out in (q, torch.zeros_like(q)):
        with pytest.raises(ValueError, match="GPU"):
            A.paged_decode_shared(q, out=out, **rest)


# ------------------------------------------------------------------------------------------------ controls of a request

@pytest.mark.parametrize("kw", [dict(repetition=1e-60), dict(repetition=1e39), dict(frequency=1e39), dict(presence=-1e39), dict(bias={1: 1e300}),
                                dict(repetition=10 ** 400), dict(bias={1: -10 ** 400}), dict(repetition="x"), dict(frequency=None)])
@pytest.mark.filterwarnings("error")
def test_controls_that_32_bits_do_not_hold_are_refused(kw):
    from crosspool_b200.engine.atn_engine import EngineConfig
    from crosspool_b200.engine.request_options import TokenControls

    eng = bare_engine()
    eng.ecfg = EngineConfig(controls=True)
    with pytest.raises(ValueError):
        eng.add_request([1, 2], 4, controls=TokenControls(**kw))
    assert not eng.waiting


def test_controls_that_32_bits_hold_are_taken():
    from crosspool_b200.engine.request_options import TokenControls

    TokenControls(1e-30, 3e38, -3e38, {5: 3.4e38, 6: 1e-45}).check(40, 300)
    TokenControls(np.float64(1.5), np.float32(0.1), 1, {5: np.float16(2)}).check(40, 300)


# ------------------------------------------------------------------------------------------------ HTTP

def ask(loop, models, bodies):
    """Status codes and answers of ``POST /generate`` with ``bodies``."""
    import asyncio

    import httpx

    from crosspool_b200.runtime.serving import create_serving_app

    app = create_serving_app(loop, models)

    async def go():
        async with httpx.AsyncClient(transport=httpx.ASGITransport(app=app), base_url="http://t") as c:
            return [await c.post("/generate", json={"input_ids": [1, 2], "max_new_tokens": 2, **b}) for b in bodies]

    return [(r.status_code, r.json()) for r in asyncio.run(go())]


def served(loop, bodies):
    loop.start()
    try:
        return ask(loop, ["m"], bodies)
    finally:
        loop.stop()


def test_the_cpu_engine_answers_requests_with_options():
    """Options that it does not have are the request's fault, not the server's."""
    from crosspool_b200.models import config as mc
    from crosspool_b200.models.weights import random_attention_weights, random_ffn_weights
    from crosspool_b200.models import reference
    from crosspool_b200.runtime.cpu_backends import CpuDeployment, CpuOracleEngine
    from crosspool_b200.runtime.serving import EngineLoop

    cfg = mc.preset("Qwen/Qwen3-0.6B").with_layers(1)
    aw, fw = random_attention_weights(cfg, 1, "cpu", torch.float32), random_ffn_weights(cfg, 1, "cpu", torch.float32)
    loop = EngineLoop(CpuDeployment({"m": CpuOracleEngine(cfg, aw, None, model=reference.ReferenceModel(cfg, aw, fw))}))
    got = served(loop, [{"repetition_penalty": 1.3}, {"frequency_penalty": 0.2}, {"logit_bias": {"5": 1.0}}, {"adapter": "x"}])
    assert [c for c, _ in got] == [422] * 4 and all("CPU engine" in b["detail"] for _, b in got)
    assert loop.error is None


def test_http_fields_that_are_null_are_neutral():
    """Clients of other servers send null for fields that they leave alone."""
    from crosspool_b200.runtime.serving import EngineLoop, GenerateRequest
    from test_serving import FakeDeployment

    nulls = {f: None for f in ("repetition_penalty", "frequency_penalty", "presence_penalty", "logit_bias", "adapter")}
    assert GenerateRequest.model_validate({"input_ids": [1], **nulls}).options() == {}
    r = GenerateRequest.model_validate({"input_ids": [1], **nulls, "presence_penalty": 0.5})
    assert r.options()["controls"].presence == 0.5 and r.options()["controls"].repetition == 1.0
    got = served(EngineLoop(FakeDeployment()), [nulls, {"logit_bias": None}])
    assert [(c, b["output_ids"]) for c, b in got] == [(200, [3, 4])] * 2


# ------------------------------------------------------------------------------------------------ plans

@pytest.mark.parametrize("hq,hk,d", [(34, 2, 128), (8, 2, 96), (7, 2, 64), (8, 0, 64)])
def test_plans_of_heads_that_no_kernel_takes_are_refused_when_they_are_made(hq, hk, d):
    from crosspool_b200.ops import attention as A

    with pytest.raises(ValueError, match="heads"):
        A.SharedPrefixPlan(torch.zeros(A.shared_plan_words(4, 8), dtype=torch.int32), 4, 8, 4, 100, hq, hk, d)


def test_an_in_process_consumer_hears_of_requests_that_fail():
    import threading

    from crosspool_b200.deployment import Deployment, InstanceHandle
    from crosspool_b200.engine.request_options import TokenControls
    from crosspool_b200.runtime.serving import EngineLoop

    heard, over = [], threading.Event()

    def sink(batch, stamp):
        heard.extend((p.tag, item) for p, item in batch)
        if any(isinstance(item, Exception) for _, item in batch):
            over.set()

    def allowed(g):
        if len(g) == 2:
            raise KeyError("grammar")
        return None

    loop = EngineLoop(Deployment([InstanceHandle("a", None, MaskedEngine())]), sink=sink)
    loop.submit("a", [1], 5, queued=False, tag="x", options={"controls": TokenControls(allowed=allowed)})
    loop.start()
    try:
        assert over.wait(20)
    finally:
        loop.stop()
    assert [t for t, _ in heard] == ["x"] * 3 and [i for _, i in heard[:2]] == [(0, False), (1, False)] and isinstance(heard[2][1], KeyError)
