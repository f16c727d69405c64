"""Speaker adaptation by distillation through the C++ classes (tests/fuzz/adapt_walk.cc: cu::RowTop, AdapterRows, Adapters,
Distill), every step's results against the same formulas in 64 bits on the step's own inputs.

Tolerances: inner dimensions stay below 130, so a sum of products is good to 2^-24 (24 * 5 + 24 + 16) <= 2^-16 of the products'
magnitudes (see test_gpu_adapters.py), a softmax to 2^-17 and a row's loss to (2 T^2 + 1) 2^-18 (see test_gpu_distill.py); chains
of these add up.  The bound of a chain here: 2^-14 of the magnitudes that went through it, taken as the largest value of the
result's matrix times its inner dimension."""
import os
import subprocess

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WALK = os.path.join(ROOT, "kaldi_amd", "bin", "adapt_walk")


def read(path):
    out = {}
    for line in open(path):
        f = line.split()
        a = np.array([float(v) for v in f[3:]])
        out.setdefault(f[0], []).append(a.reshape(int(f[1]), int(f[2])) if len(a) else np.zeros((int(f[1]), int(f[2]))))
    return out


def sigmoid(x):
    return 1 / (1 + np.exp(-x))


def softmax(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def near(got, want, inner):
    np.testing.assert_allclose(got, want, rtol=0, atol=2.0 ** -14 * max(1.0, np.abs(want).max(initial=0)) + 2.0 ** -22 * inner)


@pytest.mark.parametrize("seed", [1, 2, 3, 4, 5, 6])
def test_adaptation_by_distillation(tmp_path, seed):
    assert os.path.exists(WALK), "kaldi_amd/bin/adapt_walk missing: make -C kaldi_amd/csrc host"
    dump = str(tmp_path / "dump")
    r = subprocess.run([WALK, str(seed), "3", dump, str(tmp_path / "adapters")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    d = read(dump)
    one = lambda k: d[k][0]  # noqa: E731
    x, w1, w2, b1, b2 = one("x"), one("w1"), one("w2"), one("b1")[0], one("b2")[0]
    ranks, ids, labels, weight = one("ranks")[0].astype(int), one("ids")[0].astype(int), one("labels")[0].astype(int), one("weight")[0]
    begin = np.concatenate([[0], np.cumsum(ranks)])
    down, up, scale = one("down"), one("up"), one("scale")[0]
    teacher, k = one("teacher"), one("val").shape[1]
    idx = np.argsort(-teacher, 1, kind="stable")[:, :k]
    assert np.array_equal(one("id").reshape(-1, k), idx) and np.array_equal(one("val"), np.take_along_axis(teacher, idx, 1))
    T, hard, total = 2.0, 0.25, 0.0
    rows = np.arange(len(x))
    for s in range(3):
        add = np.zeros((len(x), w1.shape[0]))
        narrow = [None] * len(ranks)
        for g in range(len(ranks)):
            m, a = ids == g, slice(begin[g], begin[g + 1])
            narrow[g] = scale[g] * x[m] @ down[a].T
            add[m] = narrow[g] @ up[a]
        h = sigmoid(x @ w1.T + b1 + add)
        near(d["h"][s], h, 1)
        z = h @ w2.T + b2
        q = np.zeros_like(z)
        np.put_along_axis(q, idx, softmax(np.take_along_axis(teacher, idx, 1) / T), 1)
        p, p1 = softmax(z / T), softmax(z)
        onehot = np.eye(z.shape[1])[labels]
        diff = weight[:, None] * ((1 - hard) * T * (p - q) + hard * (p1 - onehot))
        near(d["diff"][s], diff, 1)
        with np.errstate(divide="ignore", invalid="ignore"):
            kl = np.where(q > 0, q * (np.log(q) - np.log(p)), 0).sum(1)
        total += (weight * ((1 - hard) * T * T * kl - hard * np.log(p1[rows, labels]))).sum()
        err = (diff @ w2) * h * (1 - h)
        ex = err @ w1
        gd, gu = np.zeros_like(down), np.zeros_like(up)
        for g in range(len(ranks)):
            m, a = ids == g, slice(begin[g], begin[g + 1])
            u = scale[g] * err[m] @ up[a].T
            ex[m] += u @ down[a]
            gd[a], gu[a] = u.T @ x[m], narrow[g].T @ err[m]
        near(d["err_x"][s], ex, w1.shape[0])
        if len(down):
            near(d["down_grad"][s], gd, len(x))
            near(d["up_grad"][s], gu, len(x))
            # the next step starts from what the device has
            down = down - 0.01 * d["down_grad"][s]
            up = up - 0.01 * d["up_grad"][s]
    near(one("down_end"), down, 1)
    near(one("up_end"), up, 1)
    loss, frames = one("loss")[0]
    assert frames == 3 * len(x) and abs(loss - total) <= 3 * weight.sum() * 9 * 2.0 ** -16
    assert r.stdout.startswith("Distill:") and "frames:%d " % frames in r.stdout
    for way in ("text", "binary"):
        tol = 1e-5 if way == "text" else 0  # (six digits of a text model)
        np.testing.assert_allclose(one("down_" + way), one("down_end"), rtol=tol)
        np.testing.assert_allclose(one("up_" + way), one("up_end"), rtol=tol)
    assert np.array_equal(one("h_binary"), d["h_end"][1])
    np.testing.assert_allclose(one("h_text"), d["h_end"][0], atol=1e-4)
