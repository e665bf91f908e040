"""Operators of requests, their engine and their serving loop at the edges of what their documentation allows; no GPU is needed."""
import contextlib

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
