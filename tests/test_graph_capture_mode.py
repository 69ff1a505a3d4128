"""
Captures beside another host thread that queries events, as the watchdog thread of an RCCL process group does.
"""
import threading
import time

import pytest
import torch


def test_capture_mode_follows_the_process_group(monkeypatch):
    import torch.distributed as dist
    from pygho_amd import graphs
    assert graphs._capture_mode() == "global"
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    for backend, mode in (("nccl", "thread_local"), ("cpu:gloo,cuda:nccl", "thread_local"), ("gloo", "global")):
        monkeypatch.setattr(dist, "get_backend", lambda *a, b=backend: b)
        assert graphs._capture_mode() == mode


@pytest.mark.gpu
def test_events_are_queried_while_a_step_is_captured(monkeypatch):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from pygho_amd import graphs
    monkeypatch.setattr(graphs, "_capture_mode", lambda: "thread_local")
    x = torch.zeros(1024, device="cuda:0")
    event = torch.cuda.Event()
    event.record()
    torch.cuda.synchronize()
    stop, errors, polls = threading.Event(), [], [0]

    def poll():
        try:
            while not stop.is_set():
                event.query()
                polls[0] += 1
                time.sleep(0.001)
        except Exception as e:                                   # noqa: BLE001  (what the other thread sees is the test)
            errors.append(e)
    thread = threading.Thread(target=poll)

    def step():
        x.add_(1.0)
        if torch.cuda.is_current_stream_capturing():
            if not thread.is_alive():
                thread.start()
            n = polls[0]
            until = time.monotonic() + 5.0
            while polls[0] < n + 10 and not errors and time.monotonic() < until:      # the capture stays open over ten queries
                time.sleep(0.002)
        return x
    try:
        g = graphs.GraphedStep(step, warmup=2)
    finally:
        stop.set()
        if thread.is_alive():
            thread.join()
    assert not errors and polls[0] >= 10
    before = float(x[0])
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert bool((x == before + 3).all())
