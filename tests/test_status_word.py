"""The device's status word: made once, whoever asks first (no GPU: torch's device
calls are stood in for)."""
import threading

import torch


class _Stream:
    """A stream whose synchronisation lets other threads run, as the real one does."""

    def __init__(self, others):
        self.others = others

    def synchronize(self):
        try:
            self.others.wait(timeout=0.5)  # both threads here at once: the word is made twice
        except threading.BrokenBarrierError:
            pass


def test_two_first_calls_get_one_word(monkeypatch):
    from eraserdit_b200 import _native
    monkeypatch.setattr(_native, "_status", {})
    monkeypatch.setattr(_native, "_capturing", lambda index: False, raising=False)
    make = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: make(1, dtype=torch.int32))
    others = threading.Barrier(2)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: _Stream(others))
    words = []
    threads = [threading.Thread(target=lambda: words.append(_native.status_word(torch.device("cuda", 0))))
               for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(words) == 2 and words[0] is words[1] is _native._status[0]
