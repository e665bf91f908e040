"""Groups of shared pages, request options of the HTTP endpoint and refusals of the engine; no GPU is needed."""
import asyncio
import random

import httpx
import pytest

from crosspool_b200.engine.atn_engine import EngineConfig
from crosspool_b200.engine.prefix_cache import PrefixCache
from crosspool_b200.engine.request_options import TokenControls, shared_groups
from crosspool_b200.runtime.serving import EngineLoop, GenerateRequest, create_serving_app
from test_engine_bookkeeping import bare_engine
from test_serving import FakeDeployment


def saved(order, sizes, pages):
    return sum((n - 1) * p for n, p in zip(sizes, pages))


def test_groups_of_pages():
    assert shared_groups([]) == ([], [], [])
    assert shared_groups([[5, 6]])[1:] == ([1], [0])
    order, sizes, pages = shared_groups([[1, 2, 9], [7], [1, 2, 8], [3, 4]])
    assert sorted(zip(sizes, pages)) == [(1, 0), (1, 0), (2, 2)] and set(order[:2]) == {0, 2}
    # all share a system prompt of four pages; two long documents below it save more than the prompt does
    tables = [[1, 2, 3, 4] + [10 + d] * 1 + list(range(100 * d, 100 * d + 30)) + [1000 + i] for d in (1, 2) for i in range(3)]
    order, sizes, pages = shared_groups(tables)
    assert sizes == [3, 3] and pages == [35, 35]
    # ... but not where the prompt is long and the documents are short
    tables = [list(range(50)) + [100 + d, 200 + i] for d in (1, 2) for i in (10 * d, 10 * d + 1)]
    assert shared_groups(tables)[1:] == ([4], [50])


def test_groups_are_valid_and_never_save_less_than_one_of_all():
    rng = random.Random(3)
    for _ in range(200):
        stems = [[rng.randrange(1000, 1100) * 50 + i for i in range(rng.randrange(0, 6))] for _ in range(3)]
        fresh = iter(range(10 ** 6, 2 * 10 ** 6))
        tables = [list(rng.choice(stems))[:rng.randrange(0, 7)] + [next(fresh) for _ in range(rng.randrange(1, 4))] for _ in range(rng.randrange(1, 20))]
        order, sizes, pages = shared_groups(tables)
        assert sorted(order) == list(range(len(tables))) and sum(sizes) == len(tables)
        at = 0
        for n, p in zip(sizes, pages):
            rows = [tables[i] for i in order[at:at + n]]
            assert all(r[:p] == rows[0][:p] and len(r) >= p for r in rows) and (n > 1 or p == 0)
            at += n
        common = 0
        while all(len(t) > common and t[common] == tables[0][common] for t in tables):
            common += 1
        assert saved(order, sizes, pages) >= (len(tables) - 1) * common


def test_cached_prefixes_of_another_space_do_not_count():
    c = PrefixCache(2)
    assert c.insert([1, 2, 3, 4], [7, 8], ("a", 1)) == [7, 8]
    assert c.match([1, 2, 3, 4, 5]) == [] and c.match([1, 2, 3, 4, 5], ("a", 2)) == []
    assert c.match([1, 2, 3, 4, 5], ("a", 1)) == [7, 8]
    assert c.insert([1, 2, 3, 4], [3, 4]) == [3, 4] and c.match([1, 2, 3], ("a", 1)) == [7]
    for p in ([7, 8], [7, 8], [7], [3, 4]):
        c.release(p)
    assert sorted(c.evict(10)) == [3, 4, 7, 8] and c.match([1, 2, 3], ("a", 1)) == []


@pytest.mark.parametrize("kw,match", [(dict(controls=TokenControls(repetition=1.1)), "EngineConfig"), (dict(adapter="x"), "adapter")])
def test_options_need_an_engine_that_has_them(kw, match):
    eng = bare_engine()
    with pytest.raises(ValueError, match=match):
        eng.add_request([1, 2], 4, **kw)
    with pytest.raises(ValueError, match="adapters"):
        eng.load_adapter("x", [])
    with pytest.raises(ValueError, match="no adapter"):
        eng.unload_adapter("x")
    assert not eng.waiting


@pytest.mark.parametrize("c", [TokenControls(repetition=0.0), TokenControls(repetition=-1.0), TokenControls(frequency=float("nan")),
                               TokenControls(presence=float("inf")), TokenControls(bias={-1: 1.0}), TokenControls(bias={10 ** 7: 1.0}),
                               TokenControls(bias={1: float("nan")}), TokenControls(bias={t: 1.0 for t in range(301)})])
def test_controls_that_are_refused(c):
    eng = bare_engine()
    eng.ecfg = EngineConfig(controls=True)
    with pytest.raises(ValueError):
        eng.add_request([1, 2], 4, controls=c)
    eng.add_request([1, 2], 4, controls=TokenControls(1.2, 0.1, -0.1, {5: -2.0}))


def test_http_options():
    assert GenerateRequest(input_ids=[1]).options() == {}
    r = GenerateRequest.model_validate({"input_ids": [1], "presence_penalty": 0.5, "logit_bias": {"7": -3}, "adapter": "a"})
    assert r.options() == {"controls": TokenControls(presence=0.5, bias={7: -3.0}), "adapter": "a"}
    seen = []

    class Recording(FakeDeployment):
        def add_request(self, model_id, prompt, max_new_tokens, arrival=None, **kw):
            seen.append(kw)
            return super().add_request(model_id, prompt, max_new_tokens, arrival)

    loop = EngineLoop(Recording())
    loop.start()
    app = create_serving_app(loop, ["a"])

    async def go():
        async with httpx.AsyncClient(transport=httpx.ASGITransport(app=app), base_url="http://t") as c:
            for body in ({}, {"repetition_penalty": 1.3}, {"adapter": "z"}):
                assert (await c.post("/generate", json={"input_ids": [1], "max_new_tokens": 1, **body})).status_code == 200

    asyncio.run(go())
    loop.stop()
    assert seen == [{}, {"controls": TokenControls(repetition=1.3)}, {"adapter": "z"}]


def test_groups_nested_deeper_than_is_looked_at():
    """Every sequence shares one page more than the one before it: the groups cover all of them, and share no more than they have."""
    from crosspool_b200.engine.request_options import shared_groups

    n = 3000
    tables = [list(range(i + 1)) + [10 ** 6 + i] for i in range(n)]
    order, sizes, pages = shared_groups(tables)
    assert sorted(order) == list(range(n)) and sum(sizes) == n
    at = 0
    for size, shared in zip(sizes, pages):
        first = tables[order[at]][:shared]
        assert len(first) == shared and all(tables[order[i]][:shared] == first for i in range(at, at + size))
        at += size
