"""CPU: how a prepared projection weight orders its users after the preparation, with stand-ins for torch's events."""
import types

import pytest
import torch

from weftmoe_b200.fp8 import PreparedFP8Linear


class Event:
    def __init__(self, done):
        self.done, self.waited = done, []

    def query(self):
        return self.done


@pytest.fixture
def prepared(monkeypatch):
    made = object.__new__(PreparedFP8Linear)
    made.weight = types.SimpleNamespace(data=types.SimpleNamespace(device=torch.device("cuda", 0)))
    stream = types.SimpleNamespace(wait_event=lambda event: event.waited.append(True))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def test_waits_until_the_preparation_is_known_to_be_done(prepared):
    event = prepared._ready = Event(False)
    prepared.wait()
    assert event.waited == [True] and prepared._ready is event
    event.done = True
    prepared.wait()
    prepared.wait()
    assert event.waited == [True] and prepared._ready is None


@pytest.mark.parametrize("done", (False, True))
@pytest.mark.parametrize("when", ("is_current_stream_capturing", "query"))
def test_another_thread_may_find_it_done_meanwhile(prepared, monkeypatch, when, done):
    event = prepared._ready = Event(done)

    def meanwhile(result):
        def call(*_):
            prepared._ready = None
            return result
        return call

    if when == "query":
        monkeypatch.setattr(Event, "query", meanwhile(done))
    else:
        monkeypatch.setattr(torch.cuda, when, meanwhile(False))
    prepared.wait()
    assert prepared._ready is None and event.waited == ([] if done else [True])
