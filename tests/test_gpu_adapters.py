"""Low-rank adapters beside a shared affine layer (hipI32_adapter_plan, hipF_adapter_forward, hipF_adapter_backward) against
their formulas in 64 bits.

Tolerances.  A product of two floats is computed to 2^-26 of itself, so errors come from the float sums.  An output of inner
dimension K is summed by eight waves, each over K / 256 (rounded up) steps of six matrix instructions, then over the waves,
the bias and the adapters' part of (rank / 32) steps more.  An instruction adds 32 products; it is allowed four roundings.  Each
rounding is at most 2^-24 of a partial sum, and no partial sum exceeds the sum of the products' magnitudes, M:

    |error| <= 2^-24 * M * (24 * ceil(K / 256) + 24 * ceil(rank / 32) + 16)

Variants that sum K in one piece take K / 32 steps in a row: 24 * ceil(K / 32) in its place; the tests use that, the larger.
With few rows the adapters' part is a chain of `rank` fused multiply-adds, one rounding each: up to 32 * ceil(rank / 32) in the
place of 24 * ceil(rank / 32); the tests use that, the larger.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32, f64 = np.float32, np.float64
EPS = 2.0 ** -24


def bound(K, rank=0):
    return EPS * (24 * -(-K // 32) + 32 * -(-rank // 32) + 16)


class Case:
    """One layer with its adapters, a bunch of rows, and everything the formulas give for them in 64 bits."""

    def __init__(self, h, N, O, I, num, rank, mix, ragged=True, seed=0, pad=0, scale=True, none=0.1):
        rs = np.random.RandomState(seed)
        self.h, self.N, self.O, self.I, self.num, self.rank = h, N, O, I, num, rank
        self.x = rs.rand(N, I).astype(f32)
        self.e = (0.1 * rs.randn(N, O)).astype(f32)
        self.W = (rs.randn(O, I) / np.sqrt(max(I, 1))).astype(f32)
        self.bias = rs.randn(O).astype(f32)
        ranks = rs.randint(0, rank + 1, num) if ragged else np.full(num, rank)
        if num:
            ranks[rs.randint(num)] = rank
        self.begin = np.concatenate([[0], np.cumsum(ranks)]).astype(np.int32)
        total = int(self.begin[-1]) + 2  # two rows behind the last adapter
        self.down = (rs.randn(total, I) / np.sqrt(max(I, 1))).astype(f32)
        self.up = (0.5 * rs.randn(total, O)).astype(f32)
        self.scale = (0.5 + rs.rand(num)).astype(f32) if scale else np.ones(num, f32)
        if mix == "segments":
            ids = rs.randint(0, max(num, 1), N + 1)[np.cumsum(rs.rand(N) < 0.05)]
        elif mix == "each":
            ids = np.arange(N) % max(num, 1)
        else:
            ids = rs.randint(0, max(num, 1), N)
        ids = np.where(rs.rand(N) < none, rs.choice([-1, num, 2 ** 30, -2 ** 31], N), ids)
        self.ids = ids.astype(np.int32) if num else np.zeros(N, np.int32)
        valid = (self.ids >= 0) & (self.ids < num)
        key = np.where(valid, self.ids.astype(np.int64), num)
        self.order = np.argsort(key, kind="stable").astype(np.int32)
        self.row_begin = np.searchsorted(np.sort(key), np.arange(num + 1)).astype(np.int32)
        self.member = [np.flatnonzero(self.ids == g) for g in range(num)]
        self.scale_ptr = scale
        self.pad = pad
        self.dev = {}

    def rows(self, g):
        return slice(int(self.begin[g]), int(self.begin[g + 1]))

    def forward(self, act):
        x, W = self.x.astype(f64), self.W.astype(f64)
        t = np.zeros((self.N, max(self.rank, 1)))
        out = x @ W.T + self.bias
        mag = np.abs(x) @ np.abs(W).T + np.abs(self.bias)
        tmag = np.zeros_like(t)
        for g, m in enumerate(self.member):
            r = self.rows(g)
            k = r.stop - r.start
            t[m, :k] = self.scale[g] * (x[m] @ self.down[r].T.astype(f64))
            tmag[m, :k] = self.scale[g] * (np.abs(x[m]) @ np.abs(self.down[r].T.astype(f64)))
            out[m] += t[m, :k] @ self.up[r]
            mag[m] += tmag[m, :k] @ np.abs(self.up[r]).astype(f64)
        if act:
            out = 1.0 / (1.0 + np.exp(-out))
        return out, t, mag, tmag

    def put(self, name, a, pitched=True):
        """The array on the device; with `pad`, as an unaligned window of a larger buffer."""
        h = self.h
        a = np.atleast_2d(a)
        if not self.pad:
            m = h.DevMatrix.from_numpy(a, pitched)
            self.dev[name] = (m, a.shape)
            return m.ptr, m.stride
        big = np.full((a.shape[0] + 2, a.shape[1] + 5 + self.pad), np.nan if a.dtype == f32 else -7, a.dtype)
        big[1:-1, self.pad:self.pad + a.shape[1]] = a
        m = h.DevMatrix.from_numpy(big, False)
        self.dev[name] = (m, a.shape)
        return ctypes.c_void_p(m._p.value + 4 * (m.stride + self.pad)), m.stride

    def get(self, name, fill=np.nan):
        """What came back; the buffer around it has to be as it was."""
        m, shape = self.dev[name]
        a = m.numpy()
        if self.pad:
            inner = a[1:-1, self.pad:self.pad + shape[1]].copy()
            a[1:-1, self.pad:self.pad + shape[1]] = np.nan
            assert np.isnan(a).all(), "%s: written outside its window" % name
            return inner
        return a[:shape[0], :shape[1]]

    def vec(self, a):
        m = self.h.DevMatrix.from_numpy(np.asarray(a), False)
        self.dev[id(m)] = (m, None)
        return m.ptr

    def adapters(self):
        down, ldd = self.put("down", self.down)
        up, ldu = self.put("up", self.up)
        return self.h.Adapters(self.num, max(self.rank, 1), len(self.down), self.vec(self.begin).value,
                               self.vec(self.scale).value if self.scale_ptr else None, down.value, ldd, up.value, ldu)

    def run_forward(self, act, order=False, stream=None):
        ad = self.adapters()
        x, W = self.put("x", self.x), self.put("W", self.W)
        t = self.put("t", np.full((self.N, max(self.rank, 1)), np.nan, f32))
        out = self.put("out", np.full((self.N, self.O), np.nan, f32))
        self.h.call("hipF_adapter_forward", stream, act, self.N, self.O, self.I, *x, *W, self.vec(self.bias), ctypes.byref(ad),
                    self.vec(self.ids), self.vec(self.order) if order else None, *t, *out)
        return self.get("out"), self.get("t")

    def run_backward(self, t, with_y=True, eout=True, grads=True):
        ad = self.adapters()
        x, W, e, tt = self.put("x", self.x), self.put("W", self.W), self.put("e", self.e), self.put("t", t)
        u = self.put("u", np.full((self.N, max(self.rank, 1)), np.nan, f32))
        eo = self.put("eout", np.full((self.N, self.I), np.nan, f32)) if eout else (None, 0)
        gd = self.put("gdown", np.full(self.down.shape, np.nan, f32)) if grads else (None, 0)
        gu = self.put("gup", np.full(self.up.shape, np.nan, f32)) if grads else (None, 0)
        self.h.call("hipF_adapter_backward", None, self.N, self.O, self.I, *e, *x, *W, ctypes.byref(ad), self.vec(self.ids),
                    self.vec(self.order), self.vec(self.row_begin), *tt, *u, *(x if with_y else (None, 0)), *eo, *gd, *gu)
        return [self.get("u"), self.get("eout") if eout else None] + ([self.get("gdown"), self.get("gup")] if grads else [None, None])


def within(got, want, tol):
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%d of %d off, worst %g of its tolerance" % (bad.sum(), bad.size, np.nanmax(np.abs(got - want) / tol))


SHAPES = [
    # N, O, I, num, rank, mix
    (1, 64, 64, 3, 16, "each"), (1, 1, 1, 1, 1, "each"), (3, 17, 33, 2, 5, "each"), (16, 16, 32, 1, 16, "segments"),
    (17, 130, 100, 7, 33, "each"), (64, 259, 440, 80, 32, "each"), (100, 2048, 1320, 5, 16, "shuffled"),
    (256, 1483, 1024, 40, 16, "shuffled"), (300, 512, 511, 3, 128, "segments"), (1000, 320, 256, 500, 7, "shuffled"),
    (2100, 192, 130, 12, 64, "segments"), (4097, 257, 96, 9, 24, "shuffled"),
    # the other tiles, forward and backward
    (60, 1483, 70, 9, 40, "each"), (50, 70, 1483, 9, 40, "shuffled"), (1000, 2048, 70, 12, 20, "shuffled"),
    (1000, 50, 2048, 12, 20, "shuffled"), (2000, 2048, 40, 12, 33, "segments"), (2000, 40, 2048, 12, 33, "segments"),
    (4000, 2048, 36, 12, 128, "shuffled"), (4000, 36, 2048, 12, 128, "shuffled")]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("order", [False, True])
def test_forward(hip, shape, act, order):
    c = Case(hip, *shape, seed=sum(shape[:5]))
    out, t = c.run_forward(act, order)
    want, t64, mag, tmag = c.forward(act)
    within(t, t64, bound(c.I) * tmag + 1e-37)
    # t is rounded before it is multiplied: its own bound counts once more; the sigmoid's slope is at most 1/4, its own
    # rounding two units of at most 1
    tol = (bound(c.I, c.rank) + bound(c.I)) * mag
    within(out, want, tol / 4 + 4 * EPS if act else tol)


@pytest.mark.parametrize("shape", [(5, 7, 9, 2, 3, "each"), (33, 70, 37, 4, 18, "shuffled"), (260, 301, 129, 6, 40, "segments")])
@pytest.mark.parametrize("pad", [1, 3])
def test_forward_and_backward_on_windows(hip, shape, pad):
    c = Case(hip, *shape, seed=pad, pad=pad, scale=False)
    out, t = c.run_forward(1, True)
    want, t64, mag, tmag = c.forward(1)
    within(out, want, (bound(c.I, c.rank) + bound(c.I)) * mag / 4 + 4 * EPS)
    check_backward(c, t)


def check_backward(c, t, with_y=True, eout=True):
    u, eo, gd, gu = c.run_backward(t, with_y, eout)
    e, x, t = c.e.astype(f64), c.x.astype(f64), t.astype(f64)
    u64 = np.zeros_like(t)
    umag = np.zeros_like(t)
    want = e @ c.W.astype(f64)
    mag = np.abs(e) @ np.abs(c.W).astype(f64)
    for g, m in enumerate(c.member):
        r = c.rows(g)
        k = r.stop - r.start
        up, down = c.up[r].astype(f64), c.down[r].astype(f64)
        u64[m, :k] = c.scale[g] * (e[m] @ up.T)
        umag[m, :k] = c.scale[g] * (np.abs(e[m]) @ np.abs(up.T))
        want[m] += u64[m, :k] @ down
        mag[m] += umag[m, :k] @ np.abs(down)
        # the gradient's sums run over the adapter's rows
        b = bound(len(m))
        within(gu[r], t[m, :k].T @ e[m], b * (np.abs(t[m, :k]).T @ np.abs(e[m])) + 1e-37)
        within(gd[r], u64[m, :k].T @ x[m], (b + bound(c.O)) * (umag[m, :k].T @ np.abs(x[m])) + 1e-37)
    within(u, u64, bound(c.O) * umag + 1e-37)
    if eout:
        if with_y:
            want, mag = want * x * (1 - x), mag * x * (1 - x)
        within(eo, want, (bound(c.O, c.rank) + bound(c.O) + 4 * EPS) * mag + 1e-37)
    else:
        assert eo is None
    last = int(c.begin[-1])
    assert np.isnan(gd[last:]).all() and np.isnan(gu[last:]).all(), "rows outside every adapter were written"


@pytest.mark.parametrize("shape", SHAPES)
def test_backward(hip, shape):
    c = Case(hip, *shape, seed=sum(shape[:5]) + 1)
    t = c.forward(0)[1].astype(f32)
    check_backward(c, t, with_y=shape[0] % 2 == 0)


def test_more_rows_than_the_small_tiles_take(hip):
    c = Case(hip, 2 ** 20 + 3, 6, 5, 3, 4, "segments", seed=14)
    out, t = c.run_forward(0)
    want, t64, mag, tmag = c.forward(0)
    within(t, t64, bound(c.I) * tmag + 1e-37)
    within(out, want, (bound(c.I, c.rank) + bound(c.I)) * mag)
    check_backward(c, t)


def test_backward_of_the_lowest_layer_and_of_frozen_adapters(hip):
    c = Case(hip, 70, 96, 64, 5, 8, "shuffled", seed=3)
    t = c.forward(0)[1].astype(f32)
    check_backward(c, t, eout=False)
    u, eo, gd, gu = c.run_backward(t, grads=False)
    u2, eo2, _, _ = c.run_backward(t)
    assert gd is None and gu is None and np.array_equal(u, u2) and np.array_equal(eo, eo2)


def test_gradients_against_differences(hip):
    """With act none the layer is linear in `up` and in `down` each, so a difference quotient of any width is the gradient."""
    c = Case(hip, 48, 40, 56, 3, 6, "shuffled", seed=5, ragged=False)
    out, t = c.run_forward(0, True)
    _, _, gd, gu = c.run_backward(t, with_y=False)
    L = lambda: float((c.run_forward(0, True)[0].astype(f64) * c.e).sum())  # noqa: E731
    _, _, mag, _ = c.forward(0)
    # one value of L is off by the sum of its outputs' bounds (a rank-64 layer: bound() of 2 + 2 steps)
    off = 2 * (bound(c.I, c.rank) + bound(c.I)) * (mag * np.abs(c.e)).sum()
    rs = np.random.RandomState(1)
    for name, grad in (("up", gu), ("down", gd)):
        w = getattr(c, name)
        for _ in range(6):
            i, j = rs.randint(c.begin[-1]), rs.randint(w.shape[1])
            old = w[i, j]
            w[i, j] = old + 8
            hi = L()
            w[i, j] = old - 8
            lo = L()
            w[i, j] = old
            # (the perturbed layer's magnitudes: 8 more on one weight)
            wide = off * 4
            assert abs((hi - lo) / 16 - grad[i, j]) <= wide / 8 + 1e-4 * abs(grad[i, j])


def test_grouping(hip):
    h = hip
    for N, num, seed in ((0, 3, 0), (1, 1, 1), (255, 4, 2), (256, 1000, 3), (5000, 37, 4), (1025, 0, 5), (3000, 1, 6)):
        rs = np.random.RandomState(seed)
        ids = rs.choice([-1, num, 2 ** 31 - 1, -2 ** 31] + list(range(num)) * 3, N).astype(np.int32)
        valid = (ids >= 0) & (ids < num)
        key = np.where(valid, ids.astype(np.int64), num)
        order, begin = h.DevMatrix(1, max(N, 1), np.int32, False), h.DevMatrix(1, num + 1, np.int32, False)
        dids = h.DevMatrix.from_numpy(ids if N else np.zeros(1, np.int32), False)
        h.call("hipI32_adapter_plan", None, dids.ptr, N, num, order.ptr, begin.ptr)
        assert np.array_equal(order.numpy()[0, :N], np.argsort(key, kind="stable"))
        assert np.array_equal(begin.numpy()[0], np.searchsorted(np.sort(key), np.arange(num + 1)))


def test_products_of_one_are_exact(hip):
    """A layer of unit rows gives back its input bit by bit, whatever the 24 bits of its floats: nothing is lost by the split."""
    h = hip
    rs = np.random.RandomState(0)
    for N, n in ((3, 40), (200, 512), (2048, 512)):
        x = (rs.randn(N, n) * 10.0 ** rs.randint(-20, 20, (N, n))).astype(f32)
        c = Case(h, N, n, n, 0, 1, "each")
        c.x, c.W, c.bias = x, np.eye(n, dtype=f32), np.zeros(n, f32)
        out, _ = c.run_forward(0)
        assert np.array_equal(out, x)
        c.e = x
        assert np.array_equal(c.run_backward(np.zeros((N, 1), f32), with_y=False, grads=False)[1], x)


def test_no_adapters_no_rows_no_inputs(hip):
    h = hip
    c = Case(h, 9, 20, 30, 0, 1, "each", seed=1)
    out, _ = c.run_forward(1)
    want, _, mag, _ = c.forward(1)
    within(out, want, bound(30) * mag / 4 + 4 * EPS)
    c = Case(h, 4, 6, 5, 2, 3, "each", seed=2)
    ad = c.adapters()
    one = h.DevMatrix(4, 8)
    h.call("hipF_adapter_forward", None, 0, 0, 6, 5, None, 5, one.ptr, 8, None, ctypes.byref(ad), one.ptr, None, None, 3, None, 6)
    h.call("hipF_adapter_forward", None, 0, 0, 6, 5, None, 0, one.ptr, 8, None, ctypes.byref(ad), one.ptr, None, None, 0, None, 0)
    # no inputs: the bias alone
    out = h.DevMatrix(4, 6)
    t = h.DevMatrix.from_numpy(np.full((4, 3), 7, f32))
    h.call("hipF_adapter_forward", None, 0, 4, 6, 0, None, 0, None, 0, c.vec(c.bias), ctypes.byref(ad), c.vec(c.ids), None, t.ptr,
           t.stride, out.ptr, out.stride)
    assert np.array_equal(out.numpy(), np.tile(c.bias, (4, 1))) and not t.numpy().any()
    # a bunch without rows: the gradients are zeros
    gd, gu = h.DevMatrix.from_numpy(np.ones(c.down.shape, f32)), h.DevMatrix.from_numpy(np.ones(c.up.shape, f32))
    h.call("hipF_adapter_backward", None, 0, 6, 5, None, 0, None, 0, None, 0, ctypes.byref(ad), c.vec(c.ids), None,
           c.vec(np.zeros(3, np.int32)), None, 0, None, 0, None, 0, None, 0, gd.ptr, gd.stride, gu.ptr, gu.stride)
    n = int(c.begin[-1])
    assert not gd.numpy()[:n].any() and not gu.numpy()[:n].any() and gd.numpy()[n:].all() and gu.numpy()[n:].all()


def test_softmax_output_layer(hip):
    c = Case(hip, 33, 100, 64, 4, 8, "shuffled", seed=8)
    out, _ = c.run_forward(2)
    z, _, mag, _ = c.forward(0)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    # an error d of a logit changes a posterior by at most a factor exp(2 d); the row kernel's own: 2^-20
    d = ((bound(64, 8) + bound(64)) * mag).max(1, keepdims=True)
    within(out, p, p * (np.expm1(2 * d) + 2.0 ** -20))


@pytest.mark.parametrize("what", ["row", "adapter"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_bad_values_stay_in_their_rows(hip, what, bad):
    for N in (40, 300):
        c = Case(hip, N, 70, 64, 6, 8, "shuffled", seed=9, ragged=False, none=0.2)
        good_out, good_t = c.run_forward(0, True)
        gu, geo, gg, _ = c.run_backward(good_t)
        if what == "row":
            hit = np.arange(N) == 17
            c.x[17, 3] = bad
            c.e[17, 5] = bad
        else:
            hit = c.ids == 2
            assert hit.any() and not hit.all()
            c.down[c.rows(2)][1, 3] = bad
            c.up[c.rows(2)][2, 4] = bad
        out, t = c.run_forward(0, True)
        u, eo, gd, _ = c.run_backward(good_t)
        assert np.array_equal(out[~hit], good_out[~hit]) and np.array_equal(t[~hit], good_t[~hit])
        assert np.array_equal(u[~hit], gu[~hit]) and np.array_equal(eo[~hit], geo[~hit])
        if what == "adapter":
            others = np.ones(len(c.down), bool)
            others[c.rows(2)] = False
            others[c.begin[-1]:] = False
            assert np.array_equal(gd[others], gg[others])
            assert not np.isfinite(out[hit]).all(1).any()
        else:
            assert np.isnan(out[17]).all() and np.isnan(eo[17]).all()


def test_broken_tables_stay_inside(hip):
    """begin[] and order[] come from the device: whatever they hold, nothing outside the matrices is touched."""
    c = Case(hip, 50, 33, 40, 4, 8, "shuffled", seed=4, ragged=False, none=0.0)
    good, t = c.run_forward(0, True)
    keep = c.order.copy()
    c.order = keep.copy()
    c.order[[3, 20, 49]] = [-5, 2 ** 30, 50]
    out, _ = c.run_forward(0, True)
    lost = keep[[3, 20, 49]]
    rest = np.setdiff1d(np.arange(50), lost)
    assert np.allclose(out[rest], good[rest], rtol=0, atol=1e-4)
    # (a row that the order does not list is left as it was, or computed where rows are not put together)
    assert all(np.isnan(out[r]).all() or np.allclose(out[r], good[r], rtol=0, atol=1e-4) for r in lost)
    c.order = keep
    begin = c.begin.copy()
    for b in ([-100, 8, 16, 24, 32], [0, 8, 4, 2 ** 31 - 1, 32], [10 ** 9, 10 ** 9 + 5, 0, 0, 0], [0, 30, 31, 32, 33]):
        c.begin = np.array(b, np.int32)
        out, _ = c.run_forward(0, True)
        assert np.isfinite(out).all()
        c.row_begin = np.array([-7, 60, 3, 2 ** 31 - 1, 10], np.int32)
        c.run_backward(t)
    c.begin = begin


def test_a_row_of_t_whoever_shares_the_call(hip):
    """Other row counts take other tiles and other windows: a row's narrow product is summed in the same order in all."""
    whole = Case(hip, 600, 1483, 1024, 9, 32, "shuffled", seed=21)
    want = whole.run_forward(0)[1]
    for rows in (1, 40, 64, 300):
        c = Case(hip, 600, 1483, 1024, 9, 32, "shuffled", seed=21)
        c.N, c.ids = rows, whole.ids[:rows]
        c.x = whole.x[:rows]
        assert np.array_equal(c.run_forward(0)[1], want[:rows])


def test_same_bits_again(hip):
    c = Case(hip, 700, 300, 260, 11, 40, "shuffled", seed=12)
    a = c.run_forward(1, True)
    g = c.run_backward(a[1])
    for _ in range(3):
        b = c.run_forward(1, True)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
        for p, q in zip(g, c.run_backward(a[1])):
            assert np.array_equal(p, q, equal_nan=True)
