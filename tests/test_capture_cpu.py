"""What TrainStep does before it captures a step into a graph, on stand-ins for the device (no GPU)."""
import contextlib
import types

import pytest
import torch
import torch.distributed as dist


class _Group:
    """RCCL's process group as far as a capture goes: a collective stays with the watchdog thread, which keeps querying the
    event recorded behind it, until the device has run it and the thread has seen that."""

    def __init__(self):
        self.running, self.polled, self.waits = 0, 0, 0

    def collective(self):
        self.running += 1
        self.polled += 1

    def _wait_for_pending_works(self):
        assert self.running == 0, "the host would wait for collectives that nothing has waited for on the device"
        self.polled, self.waits = 0, self.waits + 1


@pytest.fixture
def device(monkeypatch):
    log = types.SimpleNamespace(world=_Group(), own=_Group(), captures=0)

    @contextlib.contextmanager
    def graph(g, stream=None, capture_error_mode="global"):
        assert capture_error_mode == "thread_local"
        assert log.world.polled == 0 and log.own.polled == 0, "the watchdog still queries events of a stream that is captured"
        log.captures += 1
        yield

    def synchronize(*_):
        log.world.running = log.own.running = 0

    stream = types.SimpleNamespace(wait_stream=lambda s: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: types.SimpleNamespace(replay=lambda: None))
    monkeypatch.setattr(torch.cuda, "graph", graph)
    monkeypatch.setattr(torch.cuda, "synchronize", synchronize)
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "nccl")
    monkeypatch.setattr(dist.distributed_c10d, "_get_default_group", lambda: log.world)
    return log


class _Flat:
    grad = torch.zeros(4)


@pytest.mark.parametrize("which", ["own", "world", "no reducer"])
def test_no_collective_is_polled_while_a_step_is_captured(device, which):
    from mobilefinetuner_amd.train.engine import TrainStep
    dp = None
    if which != "no reducer":
        dp = types.SimpleNamespace(group=device.own if which == "own" else None, begin_step=lambda: None, finish=lambda: None,
                                   wants_graph_comm=lambda: True)
    st = TrainStep(None, _Flat(), types.SimpleNamespace(step=lambda: None), dp=dp, use_graph=True)
    st._fwd_bwd = lambda batches: None
    for g in (device.world, device.own if which == "own" else device.world):
        g.collective()  # an eager step's, still under way
    st._capture([(torch.zeros(1, 2), torch.zeros(1, 2))])
    assert device.captures == 1 and device.world.waits == 1 and device.own.waits == (which == "own")


def test_capture_without_a_process_group(device, monkeypatch):
    from mobilefinetuner_amd.train.engine import TrainStep
    monkeypatch.setattr(dist, "is_initialized", lambda: False)
    st = TrainStep(None, _Flat(), types.SimpleNamespace(step=lambda: None), use_graph=True)
    st._fwd_bwd = lambda batches: None
    st._capture([(torch.zeros(1, 2), torch.zeros(1, 2))])
    assert device.captures == 1 and device.world.waits == 0
