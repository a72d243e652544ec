"""The ragged-batch operators' status word on the host: one per device, whichever thread comes first."""
import threading
import time
import types

import torch

from halftone_quantizedkvcache_b200 import kernels


def test_first_calls_from_many_threads_share_one_word(monkeypatch):
    """A word that another thread's replaces would take its errors with it."""
    zeros = torch.zeros
    stream = types.SimpleNamespace(synchronize=lambda: time.sleep(0.05))
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(kernels, "_ragged_status", {})
    start, got = threading.Barrier(8), []

    def first_call():
        start.wait()
        got.append(kernels._status_word(torch.device("cuda", 0)))

    threads = [threading.Thread(target=first_call) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 8 and all(t is got[0] for t in got)
    assert kernels._ragged_status == {0: got[0]}
