"""The largest logits of a row (hipF_row_top) and the distillation loss towards them (hipF_distill_eval) against their
definitions in 64 bits.

Tolerances of the loss.  A term exp((x - m) / T) is good to 2^-22 of itself (two units in the last place, and the subtraction
x - m, whose rounding 2^-24 |x - m| is multiplied by 1 / T: counted with the row's spread D = max |x - m| / T, but a term that
far down weighs exp(-D): D exp(-D) <= 1/2.72, so 2^-24 covers it in a sum).  A sum over at most 20 terms per thread and 1024
threads in a tree has at most 20 + 6 + 16 roundings, all terms positive: 42 * 2^-24 of itself.  So sums are good to 2^-18, their
logarithms to 2^-18 absolute, and probabilities to 2^-17 plus the term's own 2^-24 D.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f32, f64 = np.float32, np.float64


def dev(h, a, pitched=True):
    return h.DevMatrix.from_numpy(np.asarray(a), pitched)


class Window:
    """A matrix at an odd place of a larger buffer of `fill`; got() checks that the rest is as it was."""

    def __init__(self, h, a, pad, fill):
        self.a, self.pad, self.fill = a, pad, fill
        big = np.full((a.shape[0] + 2, a.shape[1] + 2 * pad + 1), fill, a.dtype)
        big[1:-1, pad:pad + a.shape[1]] = a
        self.m = dev(h, big, False)
        self.ptr = ctypes.c_void_p(self.m._p.value + 4 * (self.m.stride + pad))
        self.stride = self.m.stride
        self.dim = h.MatrixDim(a.shape[0], a.shape[1], self.stride)

    def numpy(self):
        big = self.m.numpy()
        inner = big[1:-1, self.pad:self.pad + self.a.shape[1]].copy()
        big[1:-1, self.pad:self.pad + self.a.shape[1]] = self.fill
        assert (big == self.fill).all(), "written outside the window"
        return inner


def put(h, a, pad=0, fill=-77):
    return Window(h, np.asarray(a), pad, fill) if pad else dev(h, a)


# ---- row top -------------------------------------------------------------------------------------------------------------
def top64(x, K):
    """Columns of the K largest by (value, NaN above all, -0 = +0), equal ones by column."""
    key = np.where(np.isnan(x), np.inf, x) + 0.0
    nan = np.isnan(x)
    idx = np.full((x.shape[0], K), -1, np.int64)
    for r in range(x.shape[0]):
        o = np.lexsort((np.arange(x.shape[1]), -key[r], ~nan[r]))[:K]
        idx[r, :len(o)] = o
    return idx


def check_top(h, x, K, pad=0):
    R, C = x.shape
    m = put(h, x, pad)
    idx, val = put(h, np.full((R, K), 9, np.int32), pad), put(h, np.full((R, K), 9, f32), pad)
    lse = dev(h, np.zeros(max(R, 1), f32), False)
    h.call("hipF_row_top", None, m.ptr, m.dim, K, idx.ptr, idx.stride, val.ptr, val.stride, lse.ptr)
    want = top64(x, K)
    got = idx.numpy()
    assert np.array_equal(got, want)
    v = np.where(want >= 0, np.take_along_axis(x, np.maximum(want, 0), 1), -np.inf) if C else np.full((R, K), -np.inf)
    assert np.array_equal(val.numpy(), v.astype(f32), equal_nan=True)
    with np.errstate(all="ignore"):
        x64 = x.astype(f64)
        peak = np.max(x64, 1, initial=-np.inf, keepdims=True)
        base = np.where(np.isfinite(peak), peak, 0)
        ref = (base[:, 0] + np.log(np.exp(x64 - base).sum(1))) if C else np.full(R, -np.inf)
    ref[np.isposinf(x).any(1)] = np.nan
    l = lse.numpy()[0][:R]
    assert np.array_equal(np.isnan(l), np.isnan(ref)) and np.array_equal(np.isneginf(l), np.isneginf(ref))
    ok = np.isfinite(ref)
    assert (np.abs(l - ref)[ok] <= 2.0 ** -18 + 2.0 ** -24 * np.abs(ref[ok])).all()
    # the same without the sum
    h.call("hipF_row_top", None, m.ptr, m.dim, K, idx.ptr, idx.stride, val.ptr, val.stride, None)
    assert np.array_equal(idx.numpy(), want)


@pytest.mark.parametrize("C", [1, 2, 63, 64, 65, 255, 1280, 1281, 1483, 5121, 9000, 10241, 20480, 20481, 70001])
@pytest.mark.parametrize("K", [1, 8, 64, 65, 128])
def test_row_top(hip, C, K):
    rs = np.random.RandomState(C + K)
    check_top(hip, (3 * rs.randn(5, C)).astype(f32), K)


@pytest.mark.parametrize("pad", [1, 2])
def test_row_top_on_windows(hip, pad):
    rs = np.random.RandomState(pad)
    for R, C, K in ((3, 7, 9), (4, 1500, 32), (2, 9001, 20)):
        check_top(hip, rs.randn(R, C).astype(f32), K, pad)


def test_row_top_many_rows_and_none(hip):
    rs = np.random.RandomState(0)
    check_top(hip, rs.randn(3000, 90).astype(f32), 5)
    h = hip
    h.call("hipF_row_top", None, None, h.MatrixDim(0, 5, 5), 3, None, 3, None, 3, None)
    idx, val, lse = dev(h, np.zeros((2, 3), np.int32)), dev(h, np.zeros((2, 3), f32)), dev(h, np.zeros(2, f32), False)
    h.call("hipF_row_top", None, None, h.MatrixDim(2, 0, 0), 3, idx.ptr, idx.stride, val.ptr, val.stride, lse.ptr)
    assert (idx.numpy() == -1).all() and np.isneginf(val.numpy()).all() and np.isneginf(lse.numpy()).all()


@pytest.mark.parametrize("C", [50, 1283, 9000, 25000])
def test_row_top_rows_that_make_it_hard(hip, C):
    """Equal values, rows in order, large values crowded together, what a mask leaves, and what is not a number."""
    rs = np.random.RandomState(C)
    a = np.arange(C, dtype=f32)
    crowd = rs.randn(C).astype(f32)
    crowd[C // 3:C // 3 + C // 4] += 100  # more than any candidate list holds, in few threads
    stride = rs.randn(C).astype(f32)
    stride[::4 * 64] += 50
    mask = rs.randn(C).astype(f32)
    mask[rs.rand(C) < 0.98] = -np.inf
    low = np.full(C, np.finfo(f32).min, f32)
    low[C // 2] = 1
    odd = rs.randn(C).astype(f32)
    odd[[0, C // 2, C - 1]] = np.nan, np.inf, -np.nan
    zero = np.where(rs.rand(C) < 0.5, f32(0.0), f32(-0.0))
    tiny = (rs.randn(C) * 1e-42).astype(f32)
    coarse = rs.randint(-3, 4, C).astype(f32)
    rows = np.stack([a, -a, a % 7, np.zeros(C, f32), zero, crowd, stride, mask, np.full(C, -np.inf, f32), low, odd, tiny, coarse,
                     np.full(C, np.nan, f32), np.full(C, np.inf, f32)]).astype(f32)
    for K in (1, 5, 32, 64, 128):
        check_top(hip, rows, K)


# ---- distillation ----------------------------------------------------------------------------------------------------------
def distill64(x, idx, val, label, weight, T, hard):
    """-> row_loss, diff from the definition, entry by entry."""
    R, C = x.shape
    x = x.astype(f64)
    loss, diff = np.zeros(R), np.zeros((R, C))
    hard = float(f32(hard))
    with np.errstate(all="ignore"):
        for r in range(R):
            w = 1.0 if weight is None else float(weight[r])
            if w == 0 or np.isneginf(x[r]).all():
                continue
            def soft(v, t):
                e = np.exp((v - v.max()) / t)
                return e / e.sum(), (v - v.max()) / t - np.log(e.sum())
            p, logp = soft(x[r], T)
            p1, logp1 = soft(x[r], 1.0)
            if hard < 1:
                k = np.flatnonzero((idx[r] >= 0) & (idx[r] < C) & ~np.isneginf(val[r]))
                if len(k):
                    q, logq = soft(val[r, k].astype(f64), T)
                    on = q > 0
                    loss[r] += (1 - hard) * T * T * (q[on] * (logq[on] - logp[idx[r, k][on]])).sum()
                    diff[r] += (1 - hard) * T * p
                    np.subtract.at(diff[r], idx[r, k], (1 - hard) * T * q)
            if hard > 0 and 0 <= label[r] < C:
                loss[r] -= hard * logp1[label[r]]
                diff[r] += hard * p1
                diff[r, label[r]] -= hard
            loss[r] *= w
            diff[r] *= w
    return loss, diff


def run_distill(h, x, idx, val, label, weight, T, hard, pad=0, alias=False, diff=True):
    R, C = x.shape
    K = idx.shape[1]
    m = put(h, x, pad)
    out = m if alias else put(h, np.full((R, C), 9, f32), pad)
    di, dv = put(h, idx.astype(np.int32), pad), put(h, val.astype(f32), pad)
    row_loss, loss = dev(h, np.full(R, 9, f32), False), dev(h, np.array([1000.0]), False)
    dl = dev(h, label.astype(np.int32), False) if label is not None else None
    dw = dev(h, weight.astype(f32), False) if weight is not None else None
    h.call("hipF_distill_eval", None, m.ptr, m.dim, di.ptr, di.stride, dv.ptr, dv.stride, K, dl.ptr if dl else None,
           dw.ptr if dw else None, T, hard, out.ptr if diff else None, out.stride, row_loss.ptr, loss.ptr)
    rl, total = row_loss.numpy()[0], loss.numpy()[0, 0]
    with np.errstate(all="ignore"):
        if np.isfinite(rl).all():
            assert abs(total - 1000.0 - rl.astype(f64).sum()) <= 1e-12 * (1000 + np.abs(rl).sum())
    return rl, out.numpy() if diff else None


def check_distill(h, x, idx, val, label, weight, T, hard, **kw):
    rl, diff = run_distill(h, x, idx, val, label, weight, T, hard, **kw)
    want_l, want_d = distill64(x, idx, val, label, weight, T, hard)
    w = np.ones(len(x)) if weight is None else np.abs(weight)
    # logarithms to 2^-18 (of p, q and p1), each multiplied by at most T^2 and 1; rounding of the result
    tol_l = w * (2 * T * T + 1) * 2.0 ** -18 + 2.0 ** -23 * np.abs(want_l)
    # (a loss beyond the floats, of a teacher's choice that has the lowest logit, is a float's infinity)
    over = want_l > np.finfo(f32).max
    assert np.isposinf(rl[over]).all()
    rl, want_l, tol_l = rl[~over], want_l[~over], tol_l[~over]
    assert (np.abs(rl - want_l) <= tol_l).all(), np.max(np.abs(rl - want_l) / tol_l)
    if diff is not None:
        with np.errstate(all="ignore"):
            spread = np.where(np.isfinite(x), x.max(1, keepdims=True) - x, 0).max(1, keepdims=True) / min(T, 1.0)
        # p, q and p1 each to 2^-17 + 2^-24 D of themselves, times T or 1
        tol_d = w[:, None] * (2.0 ** -17 + 2.0 ** -24 * np.minimum(spread, 110)) * (np.abs(want_d) / np.maximum(w, 1e-30)[:, None] + T * 2.0 ** -6) + 1e-37
        exactp = np.abs(diff - want_d) <= tol_d
        assert exactp.all(), np.max(np.abs(diff - want_d) / tol_d)


def table(rs, R, C, K, dup=False):
    idx = np.stack([rs.permutation(C)[:K] if K <= C else rs.randint(0, C, K) for _ in range(R)])
    if dup and K > 2:
        idx[:, K // 2] = idx[:, 0]
    return idx, (3 * rs.randn(R, K)).astype(f32)


@pytest.mark.parametrize("C", [1, 2, 65, 1483, 5120, 5121, 9000, 10241, 20480, 20481, 70001])
@pytest.mark.parametrize("T,hard", [(1.0, 0.0), (2.0, 0.0), (2.0, 0.5), (1.0, 0.3), (3.5, 1.0), (0.5, 0.25)])
def test_distill(hip, C, T, hard):
    rs = np.random.RandomState(C)
    R, K = 6, min(C, 20)
    x = (3 * rs.randn(R, C)).astype(f32)
    idx, val = table(rs, R, C, K, dup=True)
    label = rs.randint(0, C, R)
    label[1] = idx[1, 0]
    check_distill(hip, x, idx, val, label, 0.5 + rs.rand(R), T, hard)


@pytest.mark.parametrize("K", [1, 2, 33, 127, 128])
@pytest.mark.parametrize("diff", [True, False])
def test_distill_table_sizes(hip, K, diff):
    rs = np.random.RandomState(K)
    x = rs.randn(40, 700).astype(f32)
    idx, val = table(rs, 40, 700, K, dup=True)
    check_distill(hip, x, idx, val, rs.randint(0, 700, 40), None, 2.0, 0.4, diff=diff)


@pytest.mark.parametrize("pad", [1, 3])
def test_distill_on_windows(hip, pad):
    rs = np.random.RandomState(pad)
    for C in (5, 1283, 9001):
        x = rs.randn(4, C).astype(f32)
        idx, val = table(rs, 4, C, 4)
        check_distill(hip, x, idx, val, rs.randint(0, C, 4), None, 2.0, 0.5, pad=pad)


@pytest.mark.parametrize("C", [300, 9000, 50000])
def test_distill_in_place(hip, C):
    rs = np.random.RandomState(C)
    x = rs.randn(7, C).astype(f32)
    idx, val = table(rs, 7, C, 16, dup=True)
    label = rs.randint(0, C, 7)
    a = run_distill(hip, x, idx, val, label, None, 2.0, 0.5)
    b = run_distill(hip, x, idx, val, label, None, 2.0, 0.5, alias=True)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("C", [70, 9000, 30000])
@pytest.mark.parametrize("hard", [0.0, 0.5])
def test_distill_rows_with_little_in_them(hip, C, hard):
    """Entries that are not there, rows without any, masked logits and entries, weight 0 over NaN, labels that are none."""
    rs = np.random.RandomState(C)
    R, K = 12, 8
    x = rs.randn(R, C).astype(f32)
    idx, val = table(rs, R, C, K)
    label = rs.randint(0, C, R)
    idx[0] = -1                                   # nothing from the teacher
    idx[1, 3:] = [-1, C, 2 ** 31 - 1, -2 ** 31, -7]
    val[1, 3:] = np.nan                           # (of entries that are not there)
    idx[2], label[2] = -1, -1                     # nothing at all
    val[3] = -np.inf                              # entries without mass
    val[4, 1:] = -np.inf                          # one entry with all the mass
    keep = np.unique(np.concatenate([idx[5], [label[5]]]))
    x[5][np.setdiff1d(np.arange(C), keep)] = -np.inf  # a mask that leaves the named columns
    x[6] = -np.inf                                # a mask that leaves nothing
    x[7] = np.nan
    x[8, 5] = np.inf
    weight = np.ones(R, f32)
    weight[[7, 8]] = 0                            # rows that do not count, whatever they hold
    label[9] = C
    val[10] = 5.0                                 # equal entries
    x[11] = np.finfo(f32).min                     # a flat row of the lowest value
    x[11, idx[11, 0]] = 0
    if hard == 0.0:
        check_distill(hip, x, idx, val, None, weight, 2.0, hard)
    else:
        x[11, label[11]] = -1  # (a finite loss)
        x[11, idx[11]] = 0
        check_distill(hip, x, idx, val, label, weight, 2.0, hard)


def test_distill_infinite_and_not_numbers(hip):
    rs = np.random.RandomState(1)
    C = 100
    x = rs.randn(4, C).astype(f32)
    idx, val = table(rs, 4, C, 4)
    x[0, idx[0, 0]] = -np.inf   # the teacher wants what the network excludes
    x[1, 7] = np.nan
    val[2, 1] = np.nan
    rl, diff = run_distill(hip, x, idx, val, None, None, 2.0, 0.0)
    _, want = distill64(x, idx, val, None, None, 2.0, 0.0)
    assert rl[0] == np.inf and np.allclose(diff[0], want[0], rtol=1e-4, atol=1e-6)
    assert np.isnan(rl[1]) and np.isnan(diff[1]).all()
    assert np.isnan(rl[2]) and np.isnan(diff[2][idx[2]]).all()
    assert np.isfinite(rl[3]) and np.isfinite(diff[3]).all()


def test_distill_gradient_against_differences(hip):
    rs = np.random.RandomState(2)
    C, K = 37, 6
    x = rs.randn(3, C).astype(f32)
    idx, val = table(rs, 3, C, K, dup=True)
    label, weight = rs.randint(0, C, 3), (0.5 + rs.rand(3)).astype(f32)
    _, diff = run_distill(hip, x, idx, val, label, weight, 2.0, 0.5)
    step = f32(2.0 ** -4)
    for c in rs.permutation(C)[:12]:
        hi, lo = x.copy(), x.copy()
        hi[:, c] += step
        lo[:, c] -= step
        a = run_distill(hip, hi, idx, val, label, weight, 2.0, 0.5, diff=False)[0].astype(f64)
        b = run_distill(hip, lo, idx, val, label, weight, 2.0, 0.5, diff=False)[0].astype(f64)
        width = hi[:, c].astype(f64) - lo[:, c]
        # the central difference is off by h^2 / 6 of the third derivative: at most w (1 - h) / T + w h <= 1.5 of it, and by
        # two losses' errors (at most 2^-17 each at this size) over the width
        assert (np.abs((a - b) / width - diff[:, c]) <= 1.5 / 6 * (width / 2) ** 2 + 2 * 9 * 2.0 ** -18 / width).all()


def test_distill_adds_up_and_repeats(hip):
    h = hip
    rs = np.random.RandomState(3)
    x = rs.randn(5000, 130).astype(f32)
    idx, val = table(rs, 5000, 130, 5)
    a = run_distill(h, x, idx, val, None, None, 1.0, 0.0)
    b = run_distill(h, x, idx, val, None, None, 1.0, 0.0)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_teacher_to_student(hip):
    """The two together, as they are used: the teacher's table from one call, the student's gradient from the other; with all
    columns in the table it is softmax(x) - softmax(teacher)."""
    h = hip
    rs = np.random.RandomState(4)
    R, C = 300, 100
    teacher, x = (2 * rs.randn(R, C)).astype(f32), rs.randn(R, C).astype(f32)
    dt, dx = dev(h, teacher), dev(h, x)
    idx, val, lse = dev(h, np.zeros((R, C), np.int32)), dev(h, np.zeros((R, C), f32)), dev(h, np.zeros(R, f32), False)
    h.call("hipF_row_top", None, dt.ptr, dt.dim, C, idx.ptr, idx.stride, val.ptr, val.stride, lse.ptr)
    row_loss = dev(h, np.zeros(R, f32), False)
    h.call("hipF_distill_eval", None, dx.ptr, dx.dim, idx.ptr, idx.stride, val.ptr, val.stride, C, None, None, 1.0, 0.0, dx.ptr,
           dx.stride, row_loss.ptr, None)
    p, q = h.DevMatrix.from_numpy(x), h.DevMatrix.from_numpy(teacher)
    h.call("hipF_softmax", None, p.ptr, p.ptr, p.dim)
    h.call("hipF_softmax", None, q.ptr, q.ptr, q.dim)
    np.testing.assert_allclose(dx.numpy(), p.numpy() - q.numpy(), rtol=0, atol=2.0 ** -16)
    assert (row_loss.numpy() > 0).all()


def test_more_rows_than_one_launch_takes(hip):
    """Rows go in launches of 2^21: what the second one reads and writes lies behind the first one's.  Of the last rows, with
    |x| <= 1, K = 2, T = 1: a probability is good to 2^-16 (above), the gradient, two of them, to 2^-15; a loss is at most five
    logarithms of size <= 4, each weighed by a probability, so good to 5 * 4 * 2^-17 < 2^-12."""
    R, C, K, n = 2 ** 21 + 3, 5, 2, 9
    rs = np.random.RandomState(5)
    x = rs.uniform(-1, 1, (R, C)).astype(f32)
    dx, di, dv, dl = dev(hip, x, False), hip.DevMatrix(R, K, np.int32, False), hip.DevMatrix(R, K, f32, False), dev(hip, np.zeros((1, R), f32), False)
    hip.call("hipF_row_top", None, dx.ptr, hip.MatrixDim(R, C, C), K, di.ptr, K, dv.ptr, K, dl.ptr)
    idx, val = di.numpy(), dv.numpy()
    assert np.array_equal(idx, np.argsort(-x, axis=1, kind="stable")[:, :K])
    assert np.array_equal(val, np.take_along_axis(x, idx, 1))
    lse = np.log(np.exp(x.astype(f64)).sum(1))
    assert np.abs(dl.numpy()[0] - lse).max() <= 2.0 ** -17
    label = rs.randint(0, C, R).astype(np.int32)
    diff, row_loss = hip.DevMatrix(R, C, f32, False), dev(hip, np.zeros((1, R), f32), False)
    loss = dev(hip, np.zeros((1, 2), f32), False)  # a double
    dlabel = dev(hip, label[None], False)
    student = np.roll(x, 1, 1)
    ds = dev(hip, student, False)
    hip.call("hipF_distill_eval", None, ds.ptr, hip.MatrixDim(R, C, C), di.ptr, K, dv.ptr, K, K, dlabel.ptr, None, 1.0, 0.5, diff.ptr, C,
             row_loss.ptr, loss.ptr)
    z = student[-n:].astype(f64)
    lp = z - np.log(np.exp(z).sum(1, keepdims=True))
    q = np.zeros_like(z)
    v = val[-n:].astype(f64)
    np.put_along_axis(q, idx[-n:], np.exp(v) / np.exp(v).sum(1, keepdims=True), 1)
    hot = np.eye(C)[label[-n:]]
    want = 0.5 * (q * (np.log(np.where(q > 0, q, 1)) - lp)).sum(1) - 0.5 * (hot * lp).sum(1)
    got = row_loss.numpy()[0]
    assert np.abs(got[-n:] - want).max() <= 2.0 ** -12
    assert np.abs(diff.numpy()[-n:] - (np.exp(lp) - 0.5 * q - 0.5 * hot)).max() <= 2.0 ** -15
    assert np.isclose(loss.numpy().view(f64)[0, 0], got.astype(f64).sum(), rtol=1e-9, atol=0)
