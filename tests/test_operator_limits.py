"""More of what the adapter, top-logit and distillation entry points refuse (see test_operator_refusals.py): no GPU is needed, a
refused call never reaches a kernel."""
import os
import subprocess

import pytest

import kaldi_amd.hip as h
from test_operator_refusals import BACKWARD, DISTILL, FORWARD, INVALID, PLAN, TOO_LARGE, TOP, adapters, status

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("change", [dict(N=2 ** 26 + 1), dict(N=2 ** 31 - 1, num=0), dict(N=2 ** 31 - 1024, num=3),
                                    dict(N=2 ** 26, num=2 ** 14), dict(N=2 ** 20, num=2 ** 20 + 1)])
def test_adapter_plan_too_many(change):
    """Rows are counted in 32 bits, and every adapter's workgroup reads all ids."""
    assert status("hipI32_adapter_plan", PLAN, **change) == TOO_LARGE
    assert str(change["N"]).encode() in h.lib.hipK_error_string(TOO_LARGE)


def test_no_rows_need_no_ids():
    """An empty vector of ids has no address.  (Neither call has anything to launch.)"""
    assert status("hipF_adapter_forward", FORWARD, N=0, row_adapter=None, in_=None, out=None, t=None) != INVALID
    nothing = dict(N=0, row_adapter=None, e=None, in_=None, order=None, t=None, u=None, y=None, eout=None, gdown=None, gup=None)
    assert status("hipF_adapter_backward", BACKWARD, **nothing) != INVALID


def test_overlap_against_sets_of_bytes(tmp_path):
    exe = str(tmp_path / "overlap_check")
    subprocess.run(["g++", "-O2", "-o", exe, os.path.join(ROOT, "tests", "fuzz", "overlap_check.cc")], check=True, timeout=120)
    r = subprocess.run([exe, "300000"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


M = 2 ** 20  # matrices that are apart
AD = adapters(begin=10 * M, scale=11 * M, down=12 * M, up=13 * M)
APART = {
    "hipI32_adapter_plan": dict(PLAN, row_adapter=M, order=2 * M, row_begin=3 * M),
    "hipF_adapter_forward": dict(FORWARD, in_=M, W=2 * M, bias=3 * M, ad=AD, row_adapter=4 * M, order=5 * M, t=6 * M, out=7 * M),
    "hipF_adapter_backward": dict(BACKWARD, e=M, in_=2 * M, W=3 * M, ad=AD, row_adapter=4 * M, order=5 * M, row_begin=6 * M, t=7 * M,
                                  u=8 * M, y=9 * M, ldy=32, eout=14 * M, gdown=15 * M, gup=16 * M),
    "hipF_row_top": dict(TOP, mat=M, idx=2 * M, val=3 * M, lse=4 * M),
    "hipF_distill_eval": dict(DISTILL, x=M, idx=2 * M, val=3 * M, label=4 * M, weight=5 * M, diff=6 * M, row_loss=7 * M, loss=8 * M),
}
OVER = [("hipI32_adapter_plan", o, i) for o in ("order", "row_begin") for i in ("row_adapter", "order", "row_begin") if o != i] + \
    [("hipF_adapter_forward", o, i) for o in ("t", "out") for i in ("in", "W", "bias", "row_adapter", "order", "begin", "scale", "down",
                                                                    "up", "t", "out") if o != i] + \
    [("hipF_adapter_backward", o, i) for o in ("u", "eout", "gdown", "gup")
     for i in ("e", "in", "W", "row_adapter", "order", "row_begin", "begin", "scale", "down", "up", "t", "y", "u", "eout", "gdown", "gup")
     if o != i] + \
    [("hipF_row_top", o, i) for o in ("idx", "val", "lse") for i in ("mat", "idx", "val", "lse") if o != i] + \
    [("hipF_distill_eval", o, i) for o in ("diff", "row_loss", "loss")
     for i in ("x", "idx", "val", "label", "weight", "diff", "row_loss", "loss") if o != i and (o, i) != ("diff", "x")]


@pytest.mark.parametrize("name,out,other", OVER)
def test_outputs_over_anything(name, out, other):
    """The output begins at the other's first element, and where both have four, at its second."""
    a = APART[name]
    at = getattr(AD, other) if other in ("begin", "scale", "down", "up") else a["in_" if other == "in" else other]
    for off in (0,) if other == "loss" else (0, 4):
        assert status(name, a, **{out: at + off}) == INVALID
        message = h.lib.hipK_error_string(INVALID).decode()
        assert "overlap" in message and name in message and out in message and other in message


def test_distill_in_place_but_not_quite():
    a = APART["hipF_distill_eval"]
    assert status("hipF_distill_eval", a, diff=a["x"] + 512) == INVALID
    assert b"diff and x" in h.lib.hipK_error_string(INVALID)
    # with the gradient in the logits' place, what lies over them lies over it
    assert status("hipF_distill_eval", a, diff=a["x"], row_loss=a["x"] + 4) == INVALID
    assert status("hipF_distill_eval", a, diff=a["x"], weight=a["x"] + 128 * 4 * 2) == INVALID


@pytest.mark.parametrize("T", [2.0 ** -149, 1e-40, 2.0 ** -127])
def test_distill_temperatures_whose_inverse_is_no_float(T):
    assert status("hipF_distill_eval", APART["hipF_distill_eval"], temperature=T) == INVALID
    assert b"temperature" in h.lib.hipK_error_string(INVALID)
