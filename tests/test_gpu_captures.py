"""Graphs for every batch size of attention with a wide table, on the GPU: each is captured in the form with scratch, gives the
bits of the call outside a capture, and leaves the linears theirs."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from _attn import Scene
from _lib import check, Dev
from _ops import ops, Stream, Graph, hip

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


class Dim3(ctypes.Structure):
    _fields_ = [("x", ctypes.c_uint), ("y", ctypes.c_uint), ("z", ctypes.c_uint)]


class KernelNode(ctypes.Structure):
    _fields_ = [("block", Dim3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p), ("grid", Dim3),
                ("params", ctypes.c_void_p), ("shared", ctypes.c_uint)]


def kernels_of(graph):
    """(workgroup, grid) of a graph's kernels."""
    n = ctypes.c_size_t()
    assert hip().hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip().hipGraphGetNodes(graph, nodes, ctypes.byref(n)) == 0
    out = []
    for node in nodes:
        p = KernelNode()
        assert hip().hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(p)) == 0
        out.append((p.block.x, (p.grid.x, p.grid.y)))
    return out


def a_graph_for_every_batch_size():
    """In a process of its own, whose library has no scratch at first."""
    heads, kv, dim, page, room = 40, 8, 128, 16, 131072
    s, w = Stream(), heads * dim
    kept = []
    lens = [(700 * i) % 2500 + 1 for i in range(64)]
    lens[3] = 9000
    a = Scene(1, 8, page, heads, kv, dim, lens, [1] * 64, 0.5, ldt=room // page).device()
    Q = Dev.of(a.q)

    def call(b, Y, E, stream):
        return ops().ak_paged_attn(8, Q.p, b, w, a.P.p, a.npages, page, heads, kv, dim, b, None, a.L.p, a.T.p, a.ldt, a.scale,
                                   Y.p, w, E.p, stream)
    for twice in range(2):
        for b in (1, 2, 4, 8, 16, 32, 64):
            Y, E = Dev(b * w * 2), Dev(b * heads * 4)
            check(call(b, Y, E, None))
            check(ops().ak_synchronize())
            want = Y.get(np.uint16, b * w), E.get(np.float32, b * heads)
            g = Graph(s, lambda stream: call(b, Y, E, stream))
            forms = kernels_of(g.graph)
            # parts or blocks, and the kernel that adds them up; a wave for a head has workgroups of 128
            assert len(forms) == 2 and all(t == 256 for t, _ in forms), (b, forms)
            kept.append((g, Y, E, want, b))
    for rep in range(2):
        for g, Y, E, want, b in kept:
            check(ops().ak_memcpy_h2d(Y.p, ctypes.c_void_p(np.full(b * w, 0x7FC1, dtype=np.uint16).ctypes.data), b * w * 2))
        for g, *_ in kept:
            g.launch()
        s.sync()
        for g, Y, E, want, b in kept:
            assert np.array_equal(Y.get(np.uint16, b * w), want[0]) and np.array_equal(E.get(np.float32, b * heads), want[1])
    # captured linears find all of theirs: the two kernels of a split prefill GEMM, in as many pieces as 256 MB hold of it
    from test_gpu_scratch import Call
    K = ops()
    K.ak_w4_set_mma(1)
    c = Call(K, 5, 128, 2, 200, 640, 9344, True)
    for i in range(16):
        g = Graph(s, c.enqueue)
        assert len(kernels_of(g.graph)) == 2, i
        c.clear()
        g.launch()
        s.sync()
        assert np.array_equal(c.out(), c.want)
    print("all captured with scratch")


def test_a_graph_for_every_batch_size():
    r = subprocess.run([sys.executable, "-u", "-c", "import test_gpu_captures as t; t.a_graph_for_every_batch_size()"], cwd=HERE,
                       capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "all captured with scratch" in r.stdout, r.stdout + r.stderr
