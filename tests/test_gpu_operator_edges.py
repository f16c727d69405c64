"""The adapter, top-logit and distillation entry points at the ends of what their interface allows, against the same oracles and
tolerances as test_gpu_adapters.py and test_gpu_distill.py."""
import ctypes

import numpy as np
import pytest

from test_gpu_adapters import Case, bound, check_backward, within
from test_gpu_distill import check_distill

pytestmark = pytest.mark.gpu
f32, f64 = np.float32, np.float64


def wave_columns(C, threads, vec):
    """Which wave of a row's workgroup holds a column: neighbouring threads hold neighbouring 16 bytes, or single floats where
    rows are not aligned."""
    return (np.arange(C) // (4 if vec else 1)) % threads // 64


@pytest.mark.parametrize("C,threads", [(1483, 256), (9000, 512), (20000, 1024)])
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("T,level", [(1.0, -100.0), (0.1, -20.0), (2.0, -400.0)])
@pytest.mark.parametrize("hard", [0.0, 0.4, 1.0])
def test_distill_mask_over_all_columns_of_a_wave(hip, C, threads, pad, T, level, hard):
    """Every column that one wave (or all but one) holds is masked out, the others are far below zero: what is masked has a
    gradient of zero, whatever the other logits' level."""
    rs = np.random.RandomState(C + pad)
    of = wave_columns(C, threads, pad == 0)
    gone = [of == 0, of == 2, of == threads // 64 - 1, of % 2 == 1, of != 1]
    R, K = len(gone), 6
    x = (level + rs.randn(R, C)).astype(f32)
    idx, val = np.zeros((R, K), int), rs.randn(R, K).astype(f32)
    label = np.zeros(R, int)
    for r in range(R):
        x[r, gone[r]] = -np.inf
        there = np.flatnonzero(~gone[r])
        idx[r], label[r] = rs.permutation(there)[:K], rs.choice(there)
    check_distill(hip, x, idx, val, label if hard else None, None, T, hard, pad=pad)


@pytest.mark.parametrize("N", [3, 50, 600])
def test_begins_far_below_zero_stay_inside(hip, N):
    """An adapter that ends before it begins has no rows, however far before: the stacks' neighbours are not touched, and rows of
    such adapters come out as rows without one.  (One that begins below zero begins at zero.)"""
    c = Case(hip, N, 33, 40, 4, 8, "shuffled", seed=4, ragged=False, none=0.0, pad=1)
    t = c.forward(0)[1].astype(f32)
    plain = Case(hip, N, 33, 40, 4, 8, "shuffled", seed=4, ragged=False, none=0.0)
    plain.ids[:] = -1
    alone, _ = plain.run_forward(0)
    for begin in ([1, -2 ** 31, 34, -2 ** 31, -2 ** 31 + 5], [34, -2 ** 31 + 1, 34, -5, -2 ** 31], [-2 ** 31, -2 ** 31, -2 ** 31, -1, -1]):
        c.begin = np.array(begin, np.int32)
        out, got_t = c.run_forward(0, True)
        u, eo, gd, gu = c.run_backward(t)  # (the windows' surroundings are checked as they come back)
        untouched = np.ones(len(c.down), bool)
        for g in range(4):
            m, lo, hi = c.ids == g, max(begin[g], 0), begin[g + 1]
            if hi <= lo:
                assert not got_t[m].any() and not u[m].any()
                np.testing.assert_allclose(out[m], alone[m], rtol=0, atol=1e-4)
                continue
            r = slice(lo, lo + min(hi - lo, 8))  # (a range longer than the largest rank is cut there)
            untouched[r] = False
            x, down, up, e = c.x[m].astype(f64), c.down[r].astype(f64), c.up[r].astype(f64), c.e[m].astype(f64)
            within(got_t[m], c.scale[g] * (x @ down.T), bound(40) * c.scale[g] * (x @ np.abs(down.T)) + 1e-37)
            within(u[m], c.scale[g] * (e @ up.T), bound(33) * c.scale[g] * (np.abs(e) @ np.abs(up.T)) + 1e-37)
        assert np.isnan(gd[untouched]).all() and np.isnan(gu[untouched]).all()
        assert np.isfinite(gd[~untouched]).all() and np.isfinite(gu[~untouched]).all()


def test_distill_loss_over_almost_2_to_31_rows(hip):
    """Rows are counted past where 32 bits with a sign end: two equal logits everywhere, so every row's loss is the float next to
    log 2.  Sums in double of fewer than 2^24 addends per thread are good to 2^24 * 2^-53 = 2^-29 of themselves."""
    R = 2 ** 31 - 1
    x = hip.DevMatrix(R, 2, f32, False)
    label, row_loss = hip.DevMatrix(1, R, np.int32, False), hip.DevMatrix(1, R, f32, False)
    loss = hip.DevMatrix(1, 1, f64, False)
    # (the teacher's table is not looked at where only hard labels count)
    hip.call("hipF_distill_eval", None, x.ptr, hip.MatrixDim(R, 2, 2), label.ptr, 1, x.ptr, 1, 1, label.ptr, None, 1.0, 1.0, None, 0,
             row_loss.ptr, loss.ptr)
    want = R * float(f32(np.log(2.0)))
    assert abs(loss.numpy()[0, 0] - want) <= 2.0 ** -29 * want
    for m in (x, label, row_loss):
        m.free()


def side_by_side(h, rows, *cols):
    """A buffer of NaN, and where matrices of these columns begin that lie next to each other in its rows."""
    m = h.DevMatrix.from_numpy(np.full((rows, sum(cols) + 3), np.nan, f32), False)
    at = np.concatenate([[1], 1 + np.cumsum(cols)])[:-1]
    return m, [ctypes.c_void_p(m.ptr.value + 4 * int(a)) for a in at], [slice(a, a + c) for a, c in zip(at, cols)]


@pytest.mark.parametrize("N", [1, 40, 700])
def test_outputs_side_by_side_in_one_matrix(hip, N):
    """Matrices that share rows of a larger one, and no element, are apart: the same bits as with each on its own."""
    h = hip
    c = Case(h, N, 50, 70, 5, 9, "shuffled", seed=N, pad=1)
    out, t = c.run_forward(1, True)
    grads = c.run_backward(t)
    ad = c.adapters()
    x, W, e = c.put("x", c.x), c.put("W", c.W), c.put("e", c.e)
    ids, order, begin = c.vec(c.ids), c.vec(c.order), c.vec(c.row_begin)
    m, (pt, pout, pu, peout), (st, sout, su, seout) = side_by_side(h, N, 9, 50, 9, 70)
    h.call("hipF_adapter_forward", None, 1, N, 50, 70, *x, *W, c.vec(c.bias), ctypes.byref(ad), ids, order, pt, m.stride, pout, m.stride)
    g, (pgd, pgu), (sgd, sgu) = side_by_side(h, len(c.down), 70, 50)
    h.call("hipF_adapter_backward", None, N, 50, 70, *e, *x, *W, ctypes.byref(ad), ids, order, begin, pt, m.stride, pu, m.stride, *x,
           peout, m.stride, pgd, g.stride, pgu, g.stride)
    got, gg = m.numpy(), g.numpy()
    for a, b in ((got[:, sout], out), (got[:, st], t), (got[:, su], grads[0]), (got[:, seout], grads[1]), (gg[:, sgd], grads[2]),
                 (gg[:, sgu], grads[3])):
        assert np.array_equal(a, b, equal_nan=True)
    assert np.isnan(got[:, [0, -2, -1]]).all() and np.isnan(gg[:, [0, -2, -1]]).all()


@pytest.mark.parametrize("T", [2.0 ** -126, 1e-30, 1e30, 3.4e38])
@pytest.mark.parametrize("C", [37, 1483, 30000])
def test_distill_ends_of_the_temperature(hip, C, T):
    """The softmax at the smallest temperature names the largest logit, at the largest all columns alike; nothing in between is
    not a number.  Logits of -1, 0 and a single 1, weights that bring T (p - q) back to about 1."""
    rs = np.random.RandomState(C)
    R, K = 4, 3
    x = -rs.randint(0, 2, (R, C)).astype(f32)
    idx = np.stack([rs.permutation(C)[:K] for _ in range(R)])
    val = np.tile(np.array([2, 1, 0], f32), (R, 1))
    best = np.array([rs.randint(C) for _ in range(R)])
    best[0], best[1] = idx[0, 0], idx[1, 2]
    x[np.arange(R), best] = 1
    weight = np.full(R, f32(2.0 ** -63) if T > 1 else f32(2.0 ** 63), f32)
    m, di, dv = hip.DevMatrix.from_numpy(x), hip.DevMatrix.from_numpy(idx.astype(np.int32)), hip.DevMatrix.from_numpy(val)
    dw = hip.DevMatrix.from_numpy(weight, False)
    diff = hip.DevMatrix(R, C)
    hip.call("hipF_distill_eval", None, m.ptr, m.dim, di.ptr, di.stride, dv.ptr, dv.stride, K, None, dw.ptr, T, 0.0, diff.ptr, diff.stride,
             None, None)
    p, q = np.zeros((R, C)), np.zeros((R, C))
    if T < 1:
        p[np.arange(R), best] = 1
        q[np.arange(R), idx[:, 0]] = 1
    else:
        p[:] = 1.0 / C
        np.put_along_axis(q, idx, 1.0 / K, 1)
    ws = f64(weight[:, None]) * float(f32(T))
    # p and q to 2^-17 of themselves (see test_gpu_distill.py), their product with w T and the difference to three roundings
    tol = ws * (2.0 ** -17 + 3 * 2.0 ** -24) * (p + q) + 2.0 ** -126
    assert (np.abs(diff.numpy() - ws * (p - q)) <= tol).all()


@pytest.mark.parametrize("O", [2, 3])
def test_softmax_layer_of_more_rows_than_one_launch_takes(hip, O):
    """2^24 rows and more of a softmax output layer: rows of the softmax go in launches whose threads 32 bits count.  One input x
    with weights 0, 1, ... and no bias: posteriors of exp(0), exp(x), ..., products of one and so exact up to the softmax (2^-20)."""
    R = 2 ** 24 + 5
    x = np.random.RandomState(O).randint(-64, 65, (R, 1)).astype(f32) / f32(32)
    dx, dW = hip.DevMatrix.from_numpy(x, False), hip.DevMatrix.from_numpy(np.arange(O, dtype=f32)[:, None], False)
    out = hip.DevMatrix(R, O, f32, False)
    ad = hip.Adapters(0, 1, 0, None, None, None, 1, None, O)
    hip.call("hipF_adapter_forward", None, hip.ACT_SOFTMAX, R, O, 1, dx.ptr, 1, dW.ptr, 1, None, ctypes.byref(ad), None, None, None, 0,
             out.ptr, O)
    z = x.astype(f64) * np.arange(O)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    assert (np.abs(out.numpy() - p) <= 2.0 ** -20 * p).all()


@pytest.mark.parametrize("backward", [False, True])
def test_a_row_of_almost_a_thousand_million_columns(hip, backward):
    """Tiles by the million: as many threads as a grid counts.  One row of one input 1: out is the weights' column, bit by bit."""
    h, C = hip, 2 ** 29
    w = np.arange(C, dtype=np.int32).astype(f32)
    dw, out, one = h.DevMatrix.from_numpy(w, False), h.DevMatrix(1, C, f32, False), h.DevMatrix.from_numpy(np.ones(1, f32), False)
    ad = h.Adapters(0, 1, 0, None, None, None, 1, None, 1)
    if backward:  # W is 1 x C: eout = e * W
        h.call("hipF_adapter_backward", None, 1, 1, C, one.ptr, 1, None, 0, dw.ptr, C, ctypes.byref(ad), None, None, None, None, 0, None,
               0, None, 0, out.ptr, C, None, 0, None, 0)
    else:  # W is C x 1
        h.call("hipF_adapter_forward", None, 0, 1, C, 1, one.ptr, 1, dw.ptr, 1, None, ctypes.byref(ad), None, None, None, 0, out.ptr, C)
    assert np.array_equal(out.numpy()[0], w)
    for m in (dw, out):
        m.free()


LARGEST = np.array([np.finfo(f32).max, np.finfo(f32).min, float.fromhex("0x1.ffp127"), float.fromhex("-0x1.ffp127"),
                    float.fromhex("0x1.fefffep127"), float.fromhex("0x1.fep127")], f32)  # around where bfloat16 ends
# which operand holds the largest floats, and what is scaled down so that the sums stay finite
SCALED = {"x": "W down e", "W": "x e", "down": "x e", "up": "x e", "e": "W up x", "t": "x e"}


@pytest.mark.parametrize("where", sorted(SCALED))
@pytest.mark.parametrize("shape", [
    (1, 33, 70, 2, 5, "each"), (17, 130, 100, 7, 33, "each"), (64, 259, 440, 80, 32, "each"), (300, 512, 511, 3, 128, "segments"),
    (1000, 320, 256, 500, 7, "shuffled"), (2000, 2048, 40, 12, 33, "segments"), (2000, 40, 2048, 12, 33, "segments"),
    (4000, 2048, 36, 12, 128, "shuffled"), (4000, 36, 2048, 12, 128, "shuffled")])
def test_the_largest_floats(hip, shape, where):
    """Finite floats that round to an infinite bfloat16 are floats like any other: the tolerances of test_gpu_adapters.py."""
    c = Case(hip, *shape, seed=sum(shape[:5]), none=0.0)
    rs = np.random.RandomState(sum(shape[:5]))
    for name in SCALED[where].split():
        getattr(c, name)[:] *= f32(2.0 ** -60)
    t = c.forward(0)[1].astype(f32)
    a = t if where == "t" else getattr(c, where)
    hit = rs.rand(*a.shape) < 0.03
    hit.flat[rs.randint(a.size)] = True
    if where == "t":  # (what lies behind an adapter's rank is not read)
        t *= f32(2.0 ** -60)
    a[hit] = rs.choice(LARGEST, hit.sum())
    if where != "t":
        t = c.forward(0)[1].astype(f32)
        out, got_t = c.run_forward(0, True)
        want, t64, mag, tmag = c.forward(0)
        within(got_t, t64, bound(c.I) * tmag + 1e-37)
        within(out, want, (bound(c.I, c.rank) + bound(c.I)) * mag + 1e-37)
    check_backward(c, t, with_y=False)


def test_infinities_beside_the_largest_floats(hip):
    """... stay what they were: NaN in their rows, the others as they are."""
    for N, O, I in ((40, 70, 64), (300, 70, 64), (4000, 300, 64)):
        c = Case(hip, N, O, I, 6, 8, "shuffled", seed=9, ragged=False, none=0.2)
        c.W *= f32(2.0 ** -60)
        c.down *= f32(2.0 ** -60)
        c.x[::3, 5] = np.finfo(f32).max
        good_out, good_t = c.run_forward(0, True)
        assert np.isfinite(good_out).all() and np.isfinite(good_t).all()
        c.x[17, 3] = np.inf
        c.x[33, 3] = np.nan
        out, t = c.run_forward(0, True)
        rest = np.setdiff1d(np.arange(N), [17, 33])
        assert np.array_equal(out[rest], good_out[rest]) and np.array_equal(t[rest], good_t[rest])
        assert np.isnan(out[[17, 33]]).all()


class Strided:
    """A matrix whose rows are far apart; its last rows begin behind 2^31 elements."""

    def __init__(self, h, a, stride):
        self.h, self.shape, self.stride, self.dtype = h, a.shape, stride, a.dtype
        self.m = h.DevMatrix((a.shape[0] - 1) * stride + a.shape[1], 1, a.dtype, False, False)
        self.ptr = self.m.ptr
        self.copy(np.ascontiguousarray(a), 0)

    def copy(self, a, kind):
        es = self.dtype.itemsize
        host, dev = (a.ctypes.data_as(ctypes.c_void_p), a.shape[1] * es), (self.ptr, self.stride * es)
        self.h.synchronize()
        self.h.call("hipK_memcpy_2d", None, *(dev + host if kind == 0 else host + dev), a.shape[1] * es, a.shape[0], kind)
        return a

    def numpy(self):
        return self.copy(np.empty(self.shape, self.dtype), 1)


@pytest.mark.parametrize("invariant", [0, 1])
@pytest.mark.parametrize("stride", [700000000, 700000001])
def test_adapters_strides_that_pass_32_bits(hip, stride, invariant):
    """Small tiles and (rows independent of the bunch) large ones, aligned rows and others, every matrix with rows 2.8 GB apart: the
    same as with rows close together, to the tolerances of test_gpu_adapters.py."""
    h = hip
    c = Case(h, 5, 5, 5, 2, 3, "each", ragged=False, seed=8, none=0.0)
    want_out, _, mag, _ = c.forward(0)
    h.call("hipK_gemm_row_invariant", invariant)
    try:
        put = lambda a: Strided(h, a, stride)  # noqa: E731
        x, W, e, down, up = put(c.x), put(c.W), put(c.e), put(c.down[:6]), put(c.up[:6])
        blank = lambda r, n: put(np.full((r, n), np.nan, f32))  # noqa: E731
        t, out, u, eout, gd, gu = blank(5, 3), blank(5, 5), blank(5, 3), blank(5, 5), blank(6, 5), blank(6, 5)
        ad = h.Adapters(2, 3, 6, c.vec(c.begin).value, c.vec(c.scale).value, down.ptr.value, stride, up.ptr.value, stride)
        ids, order, begin = c.vec(c.ids), c.vec(c.order), c.vec(c.row_begin)
        h.call("hipF_adapter_forward", None, 0, 5, 5, 5, x.ptr, stride, W.ptr, stride, c.vec(c.bias), ctypes.byref(ad), ids, order, t.ptr,
               stride, out.ptr, stride)
        within(out.numpy(), want_out, (bound(5, 3) + bound(5)) * mag)
        h.call("hipF_adapter_backward", None, 5, 5, 5, e.ptr, stride, x.ptr, stride, W.ptr, stride, ctypes.byref(ad), ids, order, begin,
               t.ptr, stride, u.ptr, stride, None, 0, eout.ptr, stride, gd.ptr, stride, gu.ptr, stride)
        got = [m.numpy() for m in (u, eout, gd, gu)]
        c.run_backward = lambda *a: [got[0], got[1]] + [np.vstack([g, np.full((2, 5), np.nan, f32)]) for g in got[2:]]
        check_backward(c, t.numpy(), with_y=False)
    finally:
        h.call("hipK_gemm_row_invariant", 0)


@pytest.mark.parametrize("stride", [700000000, 700000001])
@pytest.mark.parametrize("C", [50, 25000])
def test_top_and_distill_strides_that_pass_32_bits(hip, stride, C):
    h, rs = hip, np.random.RandomState(C)
    R, K = 5, 4
    x = rs.randn(R, C).astype(f32)
    m = Strided(h, x, stride)
    idx, val = Strided(h, np.zeros((R, K), np.int32), stride), Strided(h, np.zeros((R, K), f32), stride)
    h.call("hipF_row_top", None, m.ptr, h.MatrixDim(R, C, stride), K, idx.ptr, stride, val.ptr, stride, None)
    at = np.argsort(-x, 1, kind="stable")[:, :K]
    assert np.array_equal(idx.numpy(), at) and np.array_equal(val.numpy(), np.take_along_axis(x, at, 1))
    z = rs.randn(R, C).astype(f32)
    near = h.DevMatrix.from_numpy(z), h.DevMatrix.from_numpy(at.astype(np.int32)), h.DevMatrix.from_numpy(val.numpy()), h.DevMatrix(R, C)
    far = Strided(h, z, stride), idx, val, Strided(h, np.zeros((R, C), f32), stride)
    loss = [h.DevMatrix(1, R, f32, False) for _ in range(2)]
    for (a, i, v, d), r in zip((near, far), loss):
        h.call("hipF_distill_eval", None, a.ptr, h.MatrixDim(R, C, a.stride), i.ptr, i.stride, v.ptr, v.stride, K, None, None, 2.0, 0.0, d.ptr,
               d.stride, r.ptr, None)
    if stride % 4 == 0:  # (other rows are summed in another order)
        assert np.array_equal(near[3].numpy(), far[3].numpy()) and np.array_equal(loss[0].numpy(), loss[1].numpy())
    else:  # two results, each good to 2^-17 + 2^-24 * 10 of the probabilities times T
        assert np.abs(near[3].numpy() - far[3].numpy()).max() <= 2 * 2 * 2.0 ** -16
        assert np.abs(loss[0].numpy() - loss[1].numpy()).max() <= 2 * 9 * 2.0 ** -18 + 2.0 ** -20
