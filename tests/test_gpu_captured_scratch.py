"""Scratch of calls captured into graphs: it stays with the graph and its
executables while any of them lives, and returns to the library's cache after
the last one, so a program that captures again does not grow."""
import ctypes

import numpy as np
import pytest

import chelis_amd as C
from chelis_amd import hiprt

pytestmark = pytest.mark.gpu
ROWS, N = 64, 60000  # column sums of 7.7 MB partial rows, a size no other test asks for


class Graph:
    def __init__(self, enqueue, executables=1):
        self.hip, self.stream = hiprt.hip(), ctypes.c_void_p(C.lib().chelis_hip_stream())
        self.graph, self.execs = ctypes.c_void_p(), [ctypes.c_void_p() for _ in range(executables)]
        assert self.hip.hipStreamBeginCapture(self.stream, 0) == 0
        try:
            enqueue()
        finally:
            end = self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph))
        assert end == 0
        for e in self.execs:
            assert self.hip.hipGraphInstantiate(ctypes.byref(e), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def launch(self, which=0):
        assert self.hip.hipGraphLaunch(self.execs[which], self.stream) == 0

    def drop_graph(self):
        assert self.hip.hipGraphDestroy(self.graph) == 0

    def drop(self, which=0):
        C.synchronize()
        assert self.hip.hipGraphExecDestroy(self.execs[which]) == 0


def operands(seed):
    rng = np.random.default_rng(seed)
    x, g = (C.to_device(rng.standard_normal((ROWS, N)).astype(np.float32)) for _ in range(2))
    gamma, mean, rstd = (C.to_device(v.astype(np.float32)) for v in (np.ones(N), np.zeros(ROWS), np.ones(ROWS)))
    return x, gamma, mean, rstd, g


def outputs():
    return C.empty((N,), np.float32), C.empty((N,), np.float32)


def gradients(t, out):
    C.layer_norm_adjoint(*t, want_dx=False, dgamma=out[0], dbeta=out[1])


def same(out, want):
    return all(np.array_equal(a.numpy().view(np.uint32), b) for a, b in zip(out, want))


def test_capturing_again_and_again_does_not_grow():
    t, out = operands(1), outputs()
    gradients(t, out)
    want = [o.numpy().view(np.uint32) for o in out]
    C.synchronize()
    start = C.allocation_counts()[1]
    for _ in range(24):
        graph = Graph(lambda: gradients(t, out))
        graph.drop_graph()
        graph.launch()
        graph.drop()
        assert same(out, want)
    # the runtime may hand a block back a little after the call that dropped it
    assert C.allocation_counts()[1] - start <= 8


def test_a_block_stays_with_the_last_executable():
    """The graph and one executable go, the other replays between eager calls
    of the same size on other data, and captures that are dropped unused."""
    t, other, out = operands(2), operands(3), outputs()
    gradients(t, out)
    want = [o.numpy().view(np.uint32) for o in out]
    graph = Graph(lambda: gradients(t, out), executables=2)
    graph.drop_graph()
    graph.launch(0)
    graph.drop(0)
    aside = outputs()
    for _ in range(3):
        graph.launch(1)
        gradients(other, aside)
        unused = Graph(lambda: gradients(other, aside))
        unused.drop_graph()
        unused.drop()
        gradients(other, aside)
        C.synchronize()
        assert same(out, want)
    graph.drop(1)


def test_two_calls_of_one_graph_take_scratch_of_their_own():
    t, other = operands(4), operands(5)
    a, b = outputs(), outputs()
    want = []
    for x, o in ((t, a), (other, b)):
        gradients(x, o)
        want.append([v.numpy().view(np.uint32) for v in o])

    def both():
        gradients(t, a)
        gradients(other, b)

    graph = Graph(both)
    for _ in range(3):
        graph.launch()
        gradients(t, outputs())
        C.synchronize()
        assert same(a, want[0]) and same(b, want[1])
    graph.drop_graph()
    graph.drop()
