"""Feed-forward calls in HIP graphs and across handles: a captured backward pass, two graphs of one handle, a chain over two
streams.  Whole numbers and ReLU make every result exact, so replays are compared bit by bit."""
import ctypes as C

import numpy as np
import pytest

import sycl_blas_amd as sb
from sycl_blas_amd import _lib, helper

import ffn_ref as ref
from common import seeded
from test_ffn_gpu import Mat, int8_operands

pytestmark = pytest.mark.gpu
DTYPE = "bfloat16"


class Graph:
    """What `calls` puts on the handle's stream, as an executable graph."""

    def __init__(self, h, calls):
        self.hip, self.stream = C.CDLL("libamdhip64.so"), C.c_void_p(h.get_stream())
        self.graph, self.exe = C.c_void_p(), C.c_void_p()
        h.wait()
        assert self.hip.hipStreamBeginCapture(self.stream, 0) == 0
        calls()
        assert self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0 and self.graph.value
        assert self.hip.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, 0) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exe, self.stream) == 0

    def close(self):
        self.hip.hipGraphExecDestroy(self.exe)
        self.hip.hipGraphDestroy(self.graph)


class Layer:
    """The operands of one backward pass."""

    def __init__(self, h, n, m, k):
        self.h, self.n, self.m, self.k = h, n, m, k
        shapes = dict(w=(2 * m, k), x=(n, k), p=(n, 2 * m), dc=(n, m), dp=(n, 2 * m), da=(2 * m, k), db=(n, k))
        self.mats = {name: Mat(h, DTYPE, *s) for name, s in shapes.items()}

    def load(self, rng):
        self.v = {}
        for name in ("w", "x", "p", "dc"):
            g = self.mats[name]
            self.v[name] = rng.integers(-2, 3, (g.rows, g.cols)).astype(np.float32)
            g.window(g.host)[...] = ref.to_bits(self.v[name], DTYPE)[0]
            self.h.wait(helper.copy_to_device(self.h, g.host, g.alloc))

    def call(self):
        b = {name: g.buf.ptr for name, g in self.mats.items()}
        n, m, k = self.n, self.m, self.k
        assert _lib.load().sbamd_bgated_gemm_grad(self.h._h, _lib.ACT_RELU, b"t", b"n", m, n, k, b["w"], k, b["x"], k, b["p"], 2 * m, b["dc"], m,
                                                  b["dp"], 2 * m, 0.0, b["da"], k, 0.0, b["db"], k) == _lib.OK

    def clear(self):
        for name in ("dp", "da", "db"):
            g = self.mats[name]
            self.h.wait(helper.copy_to_device(self.h, g.host, g.alloc))

    def check(self, what):
        v, m = self.v, self.m
        dp = np.concatenate([v["dc"] * v["p"][:, m:] * (v["p"][:, :m] > 0), v["dc"] * np.maximum(v["p"][:, :m], 0)], 1)
        for name, want in (("dp", dp), ("da", dp.T @ v["x"]), ("db", dp @ v["w"])):
            got = ref.from_bits(self.mats[name].get(), DTYPE)
            assert (got == ref.to_bits(want, DTYPE)[1]).all(), (what, name)

    def free(self):
        for g in self.mats.values():
            helper.deallocate(g.alloc)


# 1104 x 302: the products read a padded copy of dP, sums cut along k; 2048 x 128: one cut product; 40 x 24: neither
@pytest.mark.parametrize("n,m,k", [(1104, 302, 136), (2048, 128, 128), (40, 24, 32)])
def test_captured_gradient_replays(n, m, k):
    rng = seeded("captured gradient", n, m, k)
    h = sb.SB_Handle(0)
    layer, other = Layer(h, n, m, k), Layer(h, n + 8, m + 10, k + 8)
    graph = None
    try:
        layer.load(rng)
        layer.call()  # the scratch has to exist before the capture
        layer.check("eager")
        graph = Graph(h, layer.call)
        for i in range(4):
            layer.load(rng)
            layer.clear()
            graph.replay()
            h.wait()
            layer.check(f"replay {i}")
            other.load(rng)  # eager work between the replays that uses, and the first time outgrows, the same areas
            other.call()
            h.wait()
            other.check(f"eager {i}")
    finally:
        if graph:
            graph.close()
        h.wait()
        layer.free()
        other.free()
        h.close()


def test_two_graphs_of_one_handle_in_turn():
    """Both use the handle's areas; on its stream one runs after the other."""
    rng = seeded("two graphs")
    h = sb.SB_Handle(0)
    layers = [Layer(h, 1104, 302, 136), Layer(h, 2048, 130, 128)]
    graphs = []
    try:
        for layer in layers:
            layer.load(rng)
            layer.call()
        for layer in layers:
            graphs.append(Graph(h, layer.call))
        for i in range(4):
            for layer in layers:
                layer.load(rng)
                layer.clear()
            for graph in graphs if i % 2 else graphs[::-1]:
                graph.replay()
            h.wait()
            for layer in layers:
                layer.check(f"replay {i}")
    finally:
        for graph in graphs:
            graph.close()
        h.wait()
        for layer in layers:
            layer.free()
        h.close()


def test_chain_over_two_handles():
    """quantise on one handle's stream, the product on another's, ordered by the call's dependencies alone."""
    n, m, k = 300, 260, 512
    rng = seeded("chain")
    first, second = sb.SB_Handle(0), sb.SB_Handle(0)
    try:
        _, w = int8_operands(rng, 1, m, k)
        wg, c = Mat(second, "int8", m, k, values=w), Mat(second, "float32", n, m)
        x, q, s = Mat(first, "float32", n, k), Mat(first, "int8", n, k), Mat(first, "float32", 1, n)
        for i in range(8):
            values = (rng.integers(-127, 128, (n, k)) * 0.5).astype(np.float32)
            values[:, 0] = 63.5  # scale 1/2 exactly
            loaded = helper.copy_to_device(first, np.concatenate([x.host[:x.start], values.ravel(), x.host[x.start + n * k:]]), x.alloc)
            done = sb._quantize(first, k, n, x.buf, k, q.buf, k, s.buf, [loaded])
            # and the next quantisation must not overtake this product
            product = sb._gemm_scaled(second, "t", "n", m, n, k, 1.0, wg.buf, k, None, q.buf, k, s.buf, 0.0, c.buf, m, done)
            first.depends_on(product)
            second.wait()
            want = (values @ w.T.astype(np.float32))
            assert (c.get() == want).all(), i
        first.wait()
    finally:
        for g in (wg, c, x, q, s):
            helper.deallocate(g.alloc)
        first.close()
        second.close()
