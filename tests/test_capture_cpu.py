"""Captures of several threads and the garbage collector of their process; no GPU: the capture itself is a stand-in."""
import contextlib
import gc
import threading

import pytest
import torch

from neuratensor_b200.inference.decode import capturing


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())
    assert gc.isenabled()
    yield
    gc.enable()


def test_a_capture_that_ends_does_not_start_the_collector_in_another(fake):
    first_in, second_in, first_out, seen = threading.Event(), threading.Event(), threading.Event(), {}

    def first():
        with capturing(None):
            first_in.set()
            seen["together"] = second_in.wait(0.5)
            seen["first"] = gc.isenabled()
        first_out.set()

    def second():
        first_in.wait(5)
        with capturing(None):
            second_in.set()
            first_out.wait(5)
            seen["second"] = gc.isenabled()

    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(10)
        assert not t.is_alive()
    assert seen == {"together": False, "first": False, "second": False}
    assert gc.isenabled()


def test_the_collector_is_as_it_was(fake):
    with capturing(None):
        assert not gc.isenabled()
    assert gc.isenabled()
    with pytest.raises(KeyError):
        with capturing(None):
            raise KeyError
    assert gc.isenabled()
    gc.disable()
    with capturing(None):
        pass
    assert not gc.isenabled()
