"""The capture error path, on the CPU.

`ldsgnn.engine.capture_into` wraps every HIP-graph capture of the engine.
An error raised by a launch inside the capture (here a NativeError, as
`lds_engine_fill_x_linear` raised on the GPU box in round 5) must propagate
ALONE: no hipErrorStreamCaptureUnjoined chained on top of it, the side
stream the capture forked joined back, the capture ended and the partial
graph reset, so the stream is usable afterwards.

The graph and the streams are stand-ins with torch.cuda.CUDAGraph's and
torch.cuda.Stream's capture semantics (capture_end fails while a forked
stream has unjoined work); the GPU form of the same check is
tests/test_engine_gpu.py::test_capture_error_is_raised_alone_and_the_engine_recovers.
"""
import contextlib

import pytest
import torch

from ldsgnn import _native as nat
from ldsgnn import engine as E


class _Stream:
    def __init__(self, name):
        self.name = name
        self.capturing = False   # part of an open capture (the main stream, or forked into it)
        self.unjoined = False    # forked work not yet joined back into the main stream

    def wait_stream(self, other):  # joining a forked stream back clears its unjoined work
        if other.capturing and other.unjoined:
            other.unjoined = False


class _Graph:
    def __init__(self, main, side, end_error=None):
        self.main, self.side, self.end_error = main, side, end_error
        self.calls = []

    def capture_begin(self, pool=None, capture_error_mode="global"):
        self.calls.append(("begin", capture_error_mode))
        self.main.capturing = True

    def capture_end(self):
        self.calls.append("end")
        was = self.main.capturing
        self.main.capturing = False
        self.side.capturing = False
        if not was:
            raise RuntimeError("HIP error: operation not permitted when stream is not capturing")
        if self.side.unjoined:
            self.side.unjoined = False
            raise RuntimeError("HIP error: capturing stream has unjoined work")
        if self.end_error:
            raise RuntimeError(self.end_error)

    def reset(self):
        self.calls.append("reset")


@pytest.fixture
def fake_cuda(monkeypatch):
    cur = {"s": None}

    @contextlib.contextmanager
    def stream(s):
        prev, cur["s"] = cur["s"], s
        try:
            yield
        finally:
            cur["s"] = prev

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: bool(cur["s"] is not None and cur["s"].capturing))
    return cur


def _fork(main, side):
    """side.wait_stream(main) inside a capture: the side stream joins the
    capture; a launch on it is then unjoined work."""
    side.capturing = True
    side.unjoined = True


def test_error_inside_capture_is_raised_alone(fake_cuda):
    main, side = _Stream("capture"), _Stream("side")
    g = _Graph(main, side)

    def body():
        _fork(main, side)
        raise nat.NativeError("lds_engine_fill_x_linear failed: hip error 1 (invalid argument)")

    with pytest.raises(nat.NativeError) as ei:
        E.capture_into(g, main, body, error_mode="thread_local", joins=(side,))
    assert ei.value.__context__ is None and ei.value.__cause__ is None
    assert g.calls == [("begin", "thread_local"), "end", "reset"]
    assert not main.capturing and not side.capturing and not side.unjoined


def test_error_of_capture_end_after_a_body_error_is_dropped(fake_cuda):
    main, side = _Stream("capture"), _Stream("side")
    g = _Graph(main, side, end_error="HIP error: operation failed due to a previous error during capture")

    def body():
        raise nat.NativeError("lds_engine_fwd_layer1 failed: hip error 1 (invalid argument)")

    with pytest.raises(nat.NativeError) as ei:
        E.capture_into(g, main, body, joins=(side,))
    assert ei.value.__context__ is None
    assert g.calls[-2:] == ["end", "reset"]
    assert not main.capturing


def test_successful_capture_ends_once(fake_cuda):
    main, side = _Stream("capture"), _Stream("side")
    g = _Graph(main, side)
    E.capture_into(g, main, lambda: None, joins=(side,))
    assert g.calls == [("begin", "global"), "end"]


@pytest.mark.parametrize("fails", [False, True])
def test_no_garbage_collection_inside_a_capture(fake_cuda, fails):
    import gc
    main, side = _Stream("capture"), _Stream("side")
    seen = []

    def body():
        seen.append(gc.isenabled())
        if fails:
            raise RuntimeError("launch")

    assert gc.isenabled()
    with pytest.raises(RuntimeError) if fails else contextlib.nullcontext():
        E.capture_into(_Graph(main, side), main, body, joins=(side,))
    assert seen == [False] and gc.isenabled()
    gc.disable()  # a caller's own choice stays
    try:
        E.capture_into(_Graph(_Stream("a"), side), _Stream("a"), lambda: None)
        assert not gc.isenabled()
    finally:
        gc.enable()


def test_overlapping_captures_keep_collection_off():
    """Two threads capture at once: the first to finish does not turn collection
    back on under the other."""
    import gc
    import threading
    a_in, b_in, a_out = (threading.Event() for _ in range(3))
    seen = []

    def first():
        with nat.no_collection():
            a_in.set()
            assert b_in.wait(30)
        a_out.set()

    def second():
        assert a_in.wait(30)
        with nat.no_collection():
            b_in.set()
            assert a_out.wait(30)
            seen.append(gc.isenabled())

    assert gc.isenabled()
    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert seen == [False] and gc.isenabled()
    with nat.no_collection():  # one inside another
        with nat.no_collection():
            pass
        assert not gc.isenabled()
    assert gc.isenabled()


@pytest.mark.parametrize("fails", [False, True])
def test_no_garbage_collection_inside_the_captured_collective(monkeypatch, fails):
    """The probe that captures an all-reduce holds collection off for the capture."""
    import gc

    from ldsgnn import replicas
    seen = []

    class Graph:
        def replay(self):
            pass

    class Stream:
        def wait_stream(self, other):
            pass

    @contextlib.contextmanager
    def capture(graph, stream=None, capture_error_mode=None):
        seen.append(("begin", gc.isenabled()))
        yield
        seen.append(("end", gc.isenabled()))

    def all_reduce(t, op=None):
        if t.dtype == torch.float32:
            seen.append(("collective", gc.isenabled()))
            if fails:
                raise RuntimeError("cannot be captured")

    monkeypatch.setattr(replicas, "_group_up", lambda: True)
    monkeypatch.setattr(replicas, "exchange_capturable", lambda: True)
    monkeypatch.setattr(replicas.dist, "get_world_size", lambda: 1)
    monkeypatch.setattr(replicas.dist, "all_reduce", all_reduce)
    for name, fake in (("CUDAGraph", Graph), ("Stream", lambda d: Stream()), ("current_stream", lambda d: Stream()),
                       ("stream", lambda s: contextlib.nullcontext()), ("graph", capture),
                       ("synchronize", lambda d: None)):
        monkeypatch.setattr(torch.cuda, name, fake)
    assert replicas.collective_capture_probe(torch.device("cpu")) is (not fails)
    assert [on for _, on in seen] == [False] * len(seen) and len(seen) == (2 if fails else 3)
    assert gc.isenabled()


def test_capture_status_classes():
    assert E._capture_status(None) == E._CAPTURE_OK
    assert E._capture_status(nat.NativeError("x")) == E._CAPTURE_FATAL
    assert E._capture_status(ValueError("x")) == E._CAPTURE_FATAL
    assert E._capture_status(RuntimeError("collective cannot be captured")) == E._CAPTURE_RETRY_SPLIT
    assert E._CAPTURE_FATAL < E._CAPTURE_RETRY_SPLIT < E._CAPTURE_OK  # agreed over ranks as the MIN


def test_collective_reducer_needs_a_group_of_more_than_one_rank():
    def red(grad):
        return None
    assert not E._collective_reducer(None)
    assert not E._collective_reducer(red)          # no `capturable`: not the replicas' collective
    red.capturable = lambda: True
    assert not E._collective_reducer(red)          # no process group in this process


def _agree_worker(rank, world, port, statuses, out):
    import os

    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)

    def red(grad):
        return None
    red.capturable = lambda: False
    out[rank] = (E._collective_reducer(red), E._ranks_agree(statuses[rank], "cpu"))
    dist.destroy_process_group()


@pytest.mark.parametrize("statuses,want", [((2, 2), 2), ((2, 1), 1), ((0, 2), 0), ((1, 0), 0)])
def test_ranks_agree_on_the_worst_capture_outcome(statuses, want):
    """with a collective exchange every rank learns the worst
    capture outcome of any rank (an eager MIN all-reduce, before any replay),
    so one rank's failed capture moves every rank to the split graphs
    (RETRY_SPLIT) or makes every rank raise (FATAL) instead of leaving the
    others replaying a graph that waits inside the collective."""
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mgr = mp.Manager()
    out = mgr.dict()
    mp.spawn(_agree_worker, args=(2, port, statuses, out), nprocs=2, join=True)
    for r in range(2):
        collective, agreed = out[r]
        assert collective  # the replicas' reducer over a 2-rank group: the agreement runs
        assert agreed == want
