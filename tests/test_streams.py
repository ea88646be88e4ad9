"""Memory that a call allocates for a stream beside the current one, on the CPU: whose
blocks it is taken from, and where it is marked as used."""
import contextlib
from types import SimpleNamespace

import pytest

import llmoxide_amd as lmx
from llmoxide_amd import paged, spec


class Tensor:
    def __init__(self, torch):
        self.torch, self.made_on, self.used_on = torch, torch.now, []

    def record_stream(self, stream):
        self.used_on.append(stream)

    def new_empty(self, shape):
        return Tensor(self.torch)

    def data_ptr(self):
        return 4096


class Torch:
    """What the calls take of torch: streams, and an allocator that notes its stream."""
    uint8 = None

    def __init__(self):
        self.now = "main"
        self.cuda = SimpleNamespace(current_stream=lambda *a: self.now, stream=self.on)

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def device(self, name):
        return name

    def empty(self, *shape, **kw):
        return Tensor(self)


@pytest.fixture
def torch(monkeypatch):
    t = Torch()
    for m in (lmx, paged, spec):
        monkeypatch.setattr(m, "_torch", lambda: t)
    monkeypatch.setattr(lmx, "_stream", lambda s: 0)
    monkeypatch.setattr(lmx, "_check", lambda *a: None)
    monkeypatch.setattr(lmx, "lib", lambda: SimpleNamespace(lmx_workspace_init=lambda *a: 0))
    return t


def grown(t, stream):
    return lmx.Workspace(device="cuda").ensure(100, stream).buf


MAKES = [lambda t, s: paged._new_out((4,), None, "cuda", s), lambda t, s: spec._fresh(Tensor(t), 4, s),
         lambda t, s: spec._space(64, None, "cuda", s)[0], grown]


@pytest.mark.parametrize("make", MAKES)
def test_a_stream_fills_memory_of_its_own(torch, make):
    """The current stream's work may still use what it freed: another stream's work, which
    nothing holds back, must not get those blocks.  Nor may its own go back to it while the
    current stream uses the result."""
    x = make(torch, "side")
    assert x.made_on == "side" and x.used_on in (["main"], ["main", "side"])
    for stream in (None, "main"):
        x = make(torch, stream)
        assert x.made_on == "main" and x.used_on in ([], ["main"])


def test_a_workspace_that_grows_waits_for_the_stream_that_used_it(torch):
    ws = lmx.Workspace(device="cuda").ensure(100, "side")
    first = ws.buf
    ws.ensure(10000)  # ordered behind the side stream's work by the caller
    assert ws.buf is not first and ws.buf.made_on == "main" and "main" in first.used_on
    second = ws.buf
    ws.ensure(100000, "side")
    assert ws.buf.made_on == "side" and "side" in second.used_on
