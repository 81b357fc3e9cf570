"""Replays of graphs that share a stream's library scratch or arrival tickets never overlap, whichever streams they run on: read off the queue of records,
waits and launches that the host runtime gives the fake device (tests/test_runtime_cpu.py says how that is built)."""
import ctypes as C
import itertools

import pytest

from cubecl_amd import _native as N
from test_runtime_cpu import ctx, lib  # noqa: F401  (fixtures)


class Queue:
    """The launches so far, each with the launches that have to be over before it starts."""
    def __init__(self, lib):
        self.lib, self.before, self.streams, self.events = lib, [], {}, {}
        lib.faketest_queue_order.argtypes, lib.faketest_queue_order.restype = [C.POINTER(C.c_uint64), C.c_uint64], C.c_uint64
        lib.faketest_ticket_slot.argtypes, lib.faketest_ticket_slot.restype = [C.c_void_p, C.c_void_p, C.POINTER(C.c_int64)], C.c_int32
        lib.faketest_queue_order((C.c_uint64 * 3)(), 0)

    def read(self):
        raw = (C.c_uint64 * 1500)()
        self.touched = set()                                   # streams of the entries read last
        for i in range(self.lib.faketest_queue_order(raw, 500)):
            kind, stream, what = chr(raw[3 * i]), raw[3 * i + 1], raw[3 * i + 2]
            self.touched.add(stream)
            done = self.streams.setdefault(stream, set())
            if kind == "r":
                self.events[what] = set(done)
            elif kind == "w":
                done |= self.events.get(what, set())
            else:
                self.before.append(set(done))
                done.add(len(self.before) - 1)
        return self.before

    def in_turn(self, launches):
        before = self.read()
        return len(before) == launches and all(i in before[j] for i, j in itertools.combinations(range(launches), 2))


def stream(lib, ctx):
    s = C.c_void_p()
    assert lib.mi355_stream_create(ctx, C.byref(s)) == N.OK
    return s


def use(lib, ctx, s, what):
    if what == "scratch":
        assert lib.faketest_scratch_get(ctx, s, 0, 1 << 16, C.byref(C.c_void_p())) == N.OK
    elif what == "tickets":
        assert lib.faketest_ticket_slot(ctx, s, C.byref(C.c_int64())) == N.OK


def captured(lib, ctx, s, what):
    use(lib, ctx, s, what)                                     # warm-up
    graph = C.c_void_p()
    assert lib.mi355_graph_begin_capture(ctx, s) == N.OK
    use(lib, ctx, s, what)
    assert lib.mi355_graph_end_capture(ctx, s, C.byref(graph)) == N.OK
    return graph


@pytest.mark.parametrize("what", ["scratch", "tickets"])
@pytest.mark.parametrize("own", [True, False], ids=["stream", "default"])
def test_replays_of_one_streams_graphs_take_turns_on_any_streams(lib, ctx, what, own):  # noqa: F811
    home = stream(lib, ctx) if own else C.c_void_p()
    away = [stream(lib, ctx) for _ in range(2)]
    graphs = [captured(lib, ctx, home, what) for _ in range(2)]
    q = Queue(lib)
    order = [(0, home), (0, away[0]), (1, away[1]), (1, home), (0, home), (1, away[0]), (1, away[0]), (0, away[1]), (0, home)]
    for g, s in order:
        assert lib.mi355_graph_replay(ctx, s, graphs[g]) == N.OK
    assert q.in_turn(len(order))
    for g in graphs:
        assert lib.mi355_graph_destroy(ctx, g) == N.OK


@pytest.mark.parametrize("what", ["scratch", "tickets"])
def test_replays_take_turns_while_their_stream_is_under_capture(lib, ctx, what):  # noqa: F811
    """Inside the window nothing of the stream is recorded or made to wait (that would be part of the new graph); its work after the window waits."""
    home, away = stream(lib, ctx), [stream(lib, ctx) for _ in range(2)]
    graph = captured(lib, ctx, home, what)
    q = Queue(lib)
    assert lib.mi355_graph_replay(ctx, home, graph) == N.OK
    assert lib.mi355_graph_begin_capture(ctx, home) == N.OK
    q.read()
    for s in away:
        assert lib.mi355_graph_replay(ctx, s, graph) == N.OK
    q.read()
    assert q.touched == {s.value for s in away}
    second = C.c_void_p()
    assert lib.mi355_graph_end_capture(ctx, home, C.byref(second)) == N.OK
    assert lib.mi355_graph_replay(ctx, home, graph) == N.OK
    assert lib.mi355_graph_replay(ctx, away[0], graph) == N.OK
    assert q.in_turn(5)
    assert lib.mi355_graph_destroy(ctx, graph) == N.OK and lib.mi355_graph_destroy(ctx, second) == N.OK


def test_replays_take_turns_after_their_stream_is_gone(lib, ctx):  # noqa: F811
    home, away = stream(lib, ctx), [stream(lib, ctx) for _ in range(2)]
    graphs = [captured(lib, ctx, home, "scratch") for _ in range(2)]
    assert lib.mi355_stream_destroy(ctx, home) == N.OK
    q = Queue(lib)
    for g, s in ((0, away[0]), (1, away[1]), (0, away[1]), (1, away[0])):
        assert lib.mi355_graph_replay(ctx, s, graphs[g]) == N.OK
    assert q.in_turn(4)
    for g in graphs:
        assert lib.mi355_graph_destroy(ctx, g) == N.OK


def test_replays_that_share_nothing_stay_independent(lib, ctx):  # noqa: F811
    """No scratch and no tickets, the capture stream itself, or graphs of two streams: no wait is queued."""
    home, other = stream(lib, ctx), stream(lib, ctx)
    plain, one, two = captured(lib, ctx, home, None), captured(lib, ctx, home, "scratch"), captured(lib, ctx, other, "scratch")
    q = Queue(lib)
    for g, s in ((plain, home), (plain, other), (one, home), (two, other)):
        assert lib.mi355_graph_replay(ctx, s, g) == N.OK
    before = q.read()
    assert before == [set(), set(), {0}, {1}]
    for g in (plain, one, two):
        assert lib.mi355_graph_destroy(ctx, g) == N.OK
