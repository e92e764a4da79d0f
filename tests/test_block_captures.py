"""Block products' captures keep Python's cyclic collector off, whichever thread's
capture ends first.  The captures are stand-ins: no GPU is needed."""
import contextlib
import gc
import threading

import pytest
import torch

from jlust_b200 import block


class Graph:
    def replay(self):
        pass


class Product(block._Graphed):
    def __init__(self, inside):
        self.graphs, self.inside = {}, inside

    def spmv(self, x, y):
        self.inside()


@pytest.fixture
def stand_ins(monkeypatch):
    capturing = threading.local()

    @contextlib.contextmanager
    def graph(g):
        capturing.now = True
        yield
        capturing.now = False

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"synchronize": lambda s: None})())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    yield lambda: getattr(capturing, "now", False)
    gc.enable()


@pytest.mark.parametrize("enabled", [True, False])
def test_overlapping_captures(stand_ins, enabled):
    (gc.enable if enabled else gc.disable)()
    first_in, second_in, first_out = (threading.Event() for _ in range(3))
    seen = []

    def first():
        if stand_ins():
            first_in.set()
            assert second_in.wait(10)

    def second():
        if stand_ins():
            second_in.set()
            assert first_out.wait(10)
            seen.append(gc.isenabled())

    def run(inside, after=None, before=None):
        if before:
            assert before.wait(10)
        x = torch.zeros(4)
        Product(inside).run(x, torch.zeros(4))
        if after:
            after.set()

    threads = [threading.Thread(target=run, args=(first, first_out)),
               threading.Thread(target=run, args=(second, None, first_in))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert seen == [False]                 # still off when the first capture has ended
    assert gc.isenabled() == enabled


def test_a_capture_that_raises_puts_the_collector_back(stand_ins):
    def inside():
        if stand_ins():
            raise RuntimeError("no")

    gc.enable()
    with pytest.raises(RuntimeError):
        Product(inside).run(torch.zeros(4), torch.zeros(4))
    assert gc.isenabled()
