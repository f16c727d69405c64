"""Products of the adapter kernels one at a time: every one of the part products that the interface promises is there.

With a 1 on one side a product is the other side, bit by bit.  With full mantissas on both sides and one product per sum: what is
left out is below 2^-26 of the product; hi * hi is exact; the five small ones, at most 2^-7 of it together, are rounded by at most 20
times 2^-23 of that (an instruction may cut off instead of rounding), below 2^-25; adding the two sums rounds once, 2^-24.  Together
below 2^-23.  Where one sum takes all six (the adapters' part in the tiles) the last instruction may cut off 2^-23 more: 2^-22.  Any of
the six lost would be at least ten times that somewhere, which each test checks on its own numbers."""

import numpy as np
import pytest

from test_gpu_adapters import Case

pytestmark = pytest.mark.gpu
f32, f64 = np.float32, np.float64
# rows x columns for which the six tiles are taken, with few inner indices
TILES = [(1, 130), (60, 1483), (256, 1100), (1000, 2048), (2000, 2048), (4000, 2048)]


def full(rs, *shape):
    """Floats of 24 random bits, magnitudes from 2^-3 to 2^3, either sign."""
    return (np.ldexp(1 + rs.rand(*shape), rs.randint(-3, 3, shape)) * rs.choice([-1, 1], shape)).astype(f32)


def parts(x):
    """The three bfloat16 numbers that add up to a float."""
    out = []
    rest = x.astype(f32)
    for _ in range(3):
        b = rest.view(np.uint32).astype(np.uint64)
        b = ((b + 0x7fff + ((b >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(f32)
        out.append(b.astype(f64))
        rest = (rest - b).astype(f32)
    assert not rest.any()
    return out


def worst(got, a, b, tol):
    """got = a * b to `tol` of each product; without any one of the small part products it would not be (one factor alone, as a
    single row has, may be short of bits: that is looked at where there are some dozens)."""
    want = a.astype(f64) * b.astype(f64)
    assert (np.abs(got - want) <= tol * np.abs(want)).all(), np.max(np.abs(got - want) / np.abs(want))
    if min(np.unique(a).size, np.unique(b).size) < 50:
        return
    pa, pb = parts(a), parts(b)
    for i, j in ((0, 1), (1, 0), (1, 1), (0, 2), (2, 0)):
        assert np.max(np.abs(pa[i] * pb[j] / want)) > 3 * tol


def layer(h, N, O, I, num, rank):
    c = Case(h, N, O, I, num, rank, "each", ragged=False, scale=False, none=0.0)
    c.bias[:] = 0
    c.up[:], c.down[:], c.W[:], c.x[:], c.e[:] = 0, 0, 0, 0, 0
    return c


@pytest.mark.parametrize("N,O", TILES)
def test_ones_on_the_rows_side(hip, N, O):
    """x and e of unit rows give back the weights: the other half of test_products_of_one_are_exact."""
    rs = np.random.RandomState(N)
    I = max(N, 7)
    c = layer(hip, N, O, I, 0, 1)
    c.x = np.eye(N, I, dtype=f32)
    c.W = full(rs, O, I)
    assert np.array_equal(c.run_forward(0)[0], c.W.T[:N])
    c = layer(hip, N, I, O, 0, 1)  # I outputs, O inputs
    c.e = np.eye(N, I, dtype=f32)
    c.W = full(rs, I, O)
    assert np.array_equal(c.run_backward(np.zeros((N, 1), f32), with_y=False, grads=False)[1], c.W[:N])


@pytest.mark.parametrize("N,O", TILES)
def test_one_product_per_sum(hip, N, O):
    rs = np.random.RandomState(N + 1)
    c = layer(hip, N, O, 1, 0, 1)
    c.x, c.W = full(rs, N, 1), full(rs, O, 1)
    worst(c.run_forward(0)[0], *np.broadcast_arrays(c.x, c.W.T), 2.0 ** -23)
    c = layer(hip, N, 1, O, 0, 1)
    c.e, c.W = full(rs, N, 1), full(rs, 1, O)
    worst(c.run_backward(np.zeros((N, 1), f32), with_y=False, grads=False)[1], *np.broadcast_arrays(c.e, c.W), 2.0 ** -23)


@pytest.mark.parametrize("N,O", TILES)
@pytest.mark.parametrize("rank", [16, 40])
def test_adapters_one_product_per_sum(hip, N, O, rank):
    """t = x * down with one input, then out = t * up with one rank row that is not zero, beside a layer of zeros; u and eout likewise."""
    rs = np.random.RandomState(N + rank)
    c = layer(hip, N, O, 1, 3, rank)
    c.x, c.down[:] = full(rs, N, 1), full(rs, len(c.down), 1)
    k = 11
    rows = c.begin[c.ids] + k
    c.up[c.begin[:-1] + k] = full(rs, 3, O)
    out, t = c.run_forward(0, True)
    worst(t, *np.broadcast_arrays(c.x, c.down[c.begin[c.ids][:, None] + np.arange(rank), 0]), 2.0 ** -23)
    worst(out, *np.broadcast_arrays(t[:, k:k + 1], c.up[rows]), 2.0 ** -22)
    c = layer(hip, N, 1, O, 3, rank)
    c.e, c.up[:] = full(rs, N, 1), full(rs, len(c.up), 1)
    c.down[c.begin[:-1] + k] = full(rs, 3, O)
    u, eout, _, _ = c.run_backward(np.zeros((N, rank), f32), with_y=False, grads=False)
    worst(u, *np.broadcast_arrays(c.e, c.up[c.begin[c.ids][:, None] + np.arange(rank), 0]), 2.0 ** -23)
    worst(eout, *np.broadcast_arrays(u[:, k:k + 1], c.down[rows]), 2.0 ** -22)


@pytest.mark.parametrize("num,N", [(300, 300), (4, 1500)])
@pytest.mark.parametrize("rank", [16, 40])
def test_gradients_one_product_per_sum(hip, num, N, rank):
    """An adapter's rows are zeros but for one: by one wave where adapters have few rows, by eight where they have many."""
    rs = np.random.RandomState(num)
    O, I = 90, 33
    c = layer(hip, N, O, I, num, rank)
    first = np.array([m[len(m) // 2] for m in c.member])
    c.e[first], c.x[first] = full(rs, num, O), full(rs, num, I)
    t = np.zeros((N, rank), f32)
    t[first] = full(rs, num, rank)
    # u = e * up: up takes output k for rank row k, so that u is e's first columns, bit by bit
    for g in range(num):
        c.up[c.rows(g)] = np.eye(rank, O, dtype=f32)
    u, _, gdown, gup = c.run_backward(t, with_y=False, eout=False)
    assert np.array_equal(u[first], c.e[first, :rank])
    n = int(c.begin[-1])
    worst(gup[:n].reshape(num, rank, O), *np.broadcast_arrays(t[first][:, :, None], c.e[first][:, None, :]), 2.0 ** -23)
    worst(gdown[:n].reshape(num, rank, I), *np.broadcast_arrays(u[first][:, :, None], c.x[first][:, None, :]), 2.0 ** -23)
    # ones on either side
    ones = np.zeros((N, rank), f32)
    ones[first, np.arange(num) % rank] = 1
    _, _, _, gup = c.run_backward(ones, with_y=False, eout=False)
    for g in range(num):
        assert np.array_equal(gup[c.rows(g)][g % rank], c.e[first[g]])
    c.e[:] = 0
    c.e[first, np.arange(num) % O] = 1
    _, _, _, gup = c.run_backward(t, with_y=False, eout=False)
    for g in range(num):
        assert np.array_equal(gup[c.rows(g)][:, g % O], t[first[g]])


@pytest.mark.parametrize("N", [3, 256, 2048])
def test_small_floats(hip, N):
    """Products of one are exact down to 2^-110; below, an operand is taken to half of bfloat16's last place, 2^-134."""
    rs = np.random.RandomState(N)
    for e, off in ((-90, 0.0), (-110, 0.0), (-118, 2.0 ** -134), (-126, 2.0 ** -134), (-140, 2.0 ** -134)):
        c = layer(hip, N, 512, 512, 0, 1)
        c.x = (np.ldexp(1 + rs.rand(N, 512), e) * rs.choice([-1, 1], (N, 512))).astype(f32)
        for up in (0, 60):
            c.W = np.eye(512, dtype=f32) * f32(2.0 ** up)
            out, _ = c.run_forward(0)
            # (an answer below the normal floats is one of its own last places off, 2^-149)
            assert (np.abs(out.astype(f64) * 2.0 ** -up - c.x) <= off + (2.0 ** -149 if off else 0)).all()
