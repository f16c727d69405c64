"""The adapter, top-logit and distillation calls captured into a graph, on streams of the caller and on two streams at once: none
of them keeps scratch memory, so a captured or concurrent call has to give the bits of an eager one."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32 = np.float32
P = ctypes.c_void_p


class Step:
    """A teacher's table, a student's loss towards it and the adapters around a layer, on buffers of their own."""

    def __init__(self, h, seed, N=300, I=96, O=520, num=7, rank=20, K=24):
        rs = np.random.RandomState(seed)
        self.h, self.N, self.I, self.O, self.num, self.K = h, N, I, O, num, K
        D = h.DevMatrix.from_numpy
        self.x = D(rs.rand(N, I).astype(f32))
        self.W, self.bias = D((rs.randn(O, I) / 8).astype(f32)), D(rs.randn(O).astype(f32), False)
        ranks = rs.randint(1, rank + 1, num)
        begin = np.concatenate([[0], np.cumsum(ranks)]).astype(np.int32)
        total = int(begin[-1])
        self.begin, self.scale = D(begin, False), D(rs.rand(num).astype(f32), False)
        self.down, self.up = D((rs.randn(total, I) / 8).astype(f32)), D(rs.randn(total, O).astype(f32))
        self.ids = D(rs.randint(-1, num, N).astype(np.int32), False)
        self.teacher = D((3 * rs.randn(N, O)).astype(f32))
        self.label = D(rs.randint(0, O, N).astype(np.int32), False)
        M = h.DevMatrix
        self.order, self.row_begin = M(1, N, np.int32, False), M(1, num + 1, np.int32, False)
        self.t, self.z = M(N, rank), M(N, O)
        self.idx, self.val, self.lse = M(N, K, np.int32), M(N, K), M(1, N, pitched=False)
        self.diff, self.row_loss, self.loss = M(N, O), M(1, N, pitched=False), M(1, 1, np.float64, False)
        self.u, self.eout, self.gdown, self.gup = M(N, rank), M(N, I), M(total, I), M(total, O)
        self.ad = h.Adapters(num, rank, total, self.begin.ptr.value, self.scale.ptr.value, self.down.ptr.value, self.down.stride,
                             self.up.ptr.value, self.up.stride)

    def run(self, s):
        h, ad = self.h, ctypes.byref(self.ad)
        h.call("hipI32_adapter_plan", s, self.ids.ptr, self.N, self.num, self.order.ptr, self.row_begin.ptr)
        h.call("hipF_adapter_forward", s, 0, self.N, self.O, self.I, self.x.ptr, self.x.stride, self.W.ptr, self.W.stride,
               self.bias.ptr, ad, self.ids.ptr, self.order.ptr, self.t.ptr, self.t.stride, self.z.ptr, self.z.stride)
        h.call("hipF_row_top", s, self.teacher.ptr, self.teacher.dim, self.K, self.idx.ptr, self.idx.stride, self.val.ptr,
               self.val.stride, self.lse.ptr)
        h.call("hipF_distill_eval", s, self.z.ptr, self.z.dim, self.idx.ptr, self.idx.stride, self.val.ptr, self.val.stride, self.K,
               self.label.ptr, None, 2.0, 0.5, self.diff.ptr, self.diff.stride, self.row_loss.ptr, self.loss.ptr)
        h.call("hipF_adapter_backward", s, self.N, self.O, self.I, self.diff.ptr, self.diff.stride, self.x.ptr, self.x.stride,
               self.W.ptr, self.W.stride, ad, self.ids.ptr, self.order.ptr, self.row_begin.ptr, self.t.ptr, self.t.stride,
               self.u.ptr, self.u.stride, self.x.ptr, self.x.stride, self.eout.ptr, self.eout.stride, self.gdown.ptr,
               self.gdown.stride, self.gup.ptr, self.gup.stride)

    def change(self, k):
        """Other inputs at the same places."""
        rs = np.random.RandomState(1000 + k)
        self.x.set(rs.rand(self.N, self.I).astype(f32))
        self.ids.set(rs.randint(-1, self.num, (1, self.N)).astype(np.int32))
        self.teacher.set((3 * rs.randn(self.N, self.O)).astype(f32))
        self.loss.set(np.zeros((1, 1)))

    def results(self):
        self.h.synchronize()
        return [m.numpy() for m in (self.order, self.row_begin, self.t, self.z, self.idx, self.val, self.lse, self.diff,
                                    self.row_loss, self.loss, self.u, self.eout, self.gdown, self.gup)]


def same(a, b):
    assert all(np.array_equal(p, q) for p, q in zip(a, b))


def test_captured_and_replayed(hip):
    h = hip
    rt = ctypes.CDLL("libamdhip64.so.7")  # (the runtime that the library uses)

    def ok(rc):
        assert rc == 0, "HIP error %d" % rc

    eager, captured = Step(h, 1), Step(h, 1)
    stream = P()
    h.call("hipK_stream_create", ctypes.byref(stream))
    eager.run(None)  # (kernels are loaded)
    h.synchronize()
    graph, instance = P(), P()
    ok(rt.hipStreamBeginCapture(stream, 0))
    captured.run(stream)
    ok(rt.hipStreamEndCapture(stream, ctypes.byref(graph)))
    ok(rt.hipGraphInstantiate(ctypes.byref(instance), graph, None, None, ctypes.c_size_t(0)))
    for k in range(4):
        eager.change(k)
        captured.change(k)
        h.synchronize()
        eager.run(None)
        ok(rt.hipGraphLaunch(instance, stream))
        h.call("hipK_stream_synchronize", stream)
        same(eager.results(), captured.results())
    ok(rt.hipGraphExecDestroy(instance))
    ok(rt.hipGraphDestroy(graph))
    h.call("hipK_stream_destroy", stream)


def test_two_streams_at_once(hip):
    h = hip
    a, b = Step(h, 2), Step(h, 3, N=1100, I=130, O=700, num=3, rank=33, K=40)
    a.run(None)
    b.run(None)
    want = a.results(), b.results()
    s, t = P(), P()
    h.call("hipK_stream_create", ctypes.byref(s))
    h.call("hipK_stream_create", ctypes.byref(t))
    for m in (a.loss, b.loss):
        m.set(np.zeros((1, 1)))
    h.synchronize()
    for k in range(3):
        if k:
            for m in (a.loss, b.loss):
                m.set(np.zeros((1, 1)))
            h.synchronize()
        a.run(s)
        b.run(t)
        same(a.results(), want[0])
        same(b.results(), want[1])
    h.call("hipK_stream_destroy", s)
    h.call("hipK_stream_destroy", t)


def test_results_do_not_depend_on_the_bunch(hip):
    """A row's narrow product is the same whoever shares its bunch; the layer's product, whose tiles depend on the number of
    rows, to rounding, and to the bit where hipK_gemm_row_invariant asks for it."""
    h = hip
    rs = np.random.RandomState(5)
    N, I, O, rank = 1500, 200, 300, 12
    x = rs.rand(N, I).astype(f32)
    W, down, up = (rs.randn(O, I) / 14).astype(f32), (rs.randn(3 * rank, I) / 14).astype(f32), rs.randn(3 * rank, O).astype(f32)
    ids = rs.randint(-1, 3, N).astype(np.int32)
    D = h.DevMatrix.from_numpy
    dW, dd, du, db = D(W), D(down), D(up), D(np.arange(4, dtype=np.int32) * rank, False)
    ad = h.Adapters(3, rank, 3 * rank, db.ptr.value, None, dd.ptr.value, dd.stride, du.ptr.value, du.stride)

    def forward(rows):
        dx, di = D(x[rows]), D(ids[rows], False)
        t, out = h.DevMatrix(len(rows), rank), h.DevMatrix(len(rows), O)
        h.call("hipF_adapter_forward", None, 1, len(rows), O, I, dx.ptr, dx.stride, dW.ptr, dW.stride, None, ctypes.byref(ad), di.ptr,
               None, t.ptr, t.stride, out.ptr, out.stride)
        return t.numpy(), out.numpy()

    t, out = forward(np.arange(N))
    for rows in (np.arange(1), np.arange(40, 57), np.arange(100, 500), rs.permutation(N)):
        t2, out2 = forward(rows)
        assert np.array_equal(t2, t[rows])
        # two sums of 200 + 12 products, each good to 2^-24 (24 * 7 + 24 + 16) of their magnitudes (below 8), a slope of 1/4
        np.testing.assert_allclose(out2, out[rows], rtol=0, atol=2 * 2.0 ** -24 * 208 * 8 / 4)
    h.call("hipK_gemm_row_invariant", 1)
    try:
        t, out = forward(np.arange(N))
        for rows in (np.arange(1), np.arange(40, 57), np.arange(100, 500), rs.permutation(N), np.tile(np.arange(N), 4)):
            t2, out2 = forward(rows)
            assert np.array_equal(t2, t[rows]) and np.array_equal(out2, out[rows])
    finally:
        h.call("hipK_gemm_row_invariant", 0)
