"""What the adapter, top-logit and distillation entry points refuse.  Arguments are checked before the device is looked for,
so these run without a GPU: a refused call never reaches a kernel."""
import ctypes
import os
import subprocess
import sys

import pytest

import kaldi_amd.hip as h

INVALID, TOO_LARGE = 100001, 100004
P = 4096  # a pointer that no refused call follows


def adapters(num=2, max_rank=8, rows=16, begin=P, scale=P, down=P, lddown=32, up=P, ldup=48):
    return h.Adapters(num, max_rank, rows, begin, scale, down, lddown, up, ldup)


FORWARD = dict(s=None, act=0, N=4, O=48, I=32, in_=P, ldin=32, W=P, ldw=32, bias=P, ad=None, row_adapter=P, order=None, t=P,
               ldt=8, out=2 * P, ldout=48)
BACKWARD = dict(s=None, N=4, O=48, I=32, e=P, lde=48, in_=P, ldin=32, W=P, ldw=32, ad=None, row_adapter=P, order=P, row_begin=P,
                t=P, ldt=8, u=2 * P, ldu=8, y=None, ldy=0, eout=3 * P, ldeout=32, gdown=4 * P, ldgdown=32, gup=5 * P, ldgup=48)
DISTILL = dict(s=None, x=P, d=(4, 100, 128), idx=P, ldidx=8, val=P, ldval=8, K=8, label=P, weight=P, temperature=2.0, hard=0.5,
               diff=P, lddiff=128, row_loss=P, loss=P)
TOP = dict(s=None, mat=P, d=(4, 100, 128), K=8, idx=P, ldidx=8, val=P, ldval=8, lse=P)
PLAN = dict(s=None, row_adapter=P, N=4, num=2, order=P, row_begin=P)


def status(name, base, **changes):
    a = dict(base, **{k: v for k, v in changes.items() if k in base})
    assert set(changes) <= set(base)
    if "ad" in a and a["ad"] is None:
        a["ad"] = adapters()
    args = [ctypes.byref(v) if isinstance(v, h.Adapters) else h.MatrixDim(*v) if k == "d" else v for k, v in a.items()]
    return getattr(h.lib, name)(*args)


@pytest.mark.parametrize("change", [
    dict(act=3), dict(act=-1), dict(N=-1), dict(O=-1), dict(I=-1), dict(ldin=31), dict(ldw=31), dict(ldout=47), dict(ldt=7),
    dict(in_=None), dict(W=None), dict(out=None), dict(out=P), dict(t=None), dict(row_adapter=None),
    dict(ad=adapters(num=-1)), dict(ad=adapters(max_rank=0)), dict(ad=adapters(rows=-1)), dict(ad=adapters(begin=None)),
    dict(ad=adapters(down=None)), dict(ad=adapters(up=None)), dict(ad=adapters(lddown=31)), dict(ad=adapters(ldup=47))])
def test_adapter_forward_refuses(change):
    assert status("hipF_adapter_forward", FORWARD, **change) == INVALID
    assert b"hipF_adapter_forward" in h.lib.hipK_error_string(INVALID) or b"check_adapters" in h.lib.hipK_error_string(INVALID)


def test_adapter_rank_too_large():
    ad = adapters(max_rank=h.MAX_ADAPTER_RANK + 1)
    assert status("hipF_adapter_forward", FORWARD, ad=ad, ldt=256) == TOO_LARGE
    assert status("hipF_adapter_backward", BACKWARD, ad=ad, ldt=256, ldu=256) == TOO_LARGE
    assert b"129" in h.lib.hipK_error_string(TOO_LARGE)


def test_adapter_without_struct():
    for name, base in (("hipF_adapter_forward", FORWARD), ("hipF_adapter_backward", BACKWARD)):
        args = [None if k == "ad" else v for k, v in base.items()]
        assert getattr(h.lib, name)(*args) == INVALID


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(O=-1), dict(I=-1), dict(e=None), dict(lde=47), dict(W=None), dict(ldw=31), dict(ldeout=31), dict(eout=P),
    dict(y=P, ldy=31), dict(u=None), dict(ldu=7), dict(u=P), dict(row_begin=None), dict(order=None), dict(in_=None), dict(ldin=31),
    dict(t=None), dict(ldt=7), dict(ldgdown=31), dict(ldgup=47), dict(row_adapter=None), dict(ad=adapters(begin=None))])
def test_adapter_backward_refuses(change):
    assert status("hipF_adapter_backward", BACKWARD, **change) == INVALID


@pytest.mark.parametrize("change", [dict(N=-1), dict(num=-1), dict(row_adapter=None), dict(order=None), dict(row_begin=None)])
def test_adapter_plan_refuses(change):
    assert status("hipI32_adapter_plan", PLAN, **change) == INVALID


@pytest.mark.parametrize("change", [
    dict(d=(-1, 100, 128)), dict(d=(4, -1, 128)), dict(d=(4, 100, 99)), dict(K=0), dict(K=-3), dict(ldidx=7), dict(ldval=7),
    dict(mat=None), dict(idx=None), dict(val=None)])
def test_row_top_refuses(change):
    assert status("hipF_row_top", TOP, **change) == INVALID


@pytest.mark.parametrize("change", [
    dict(d=(-1, 100, 128)), dict(d=(4, 100, 99)), dict(K=0), dict(ldidx=7), dict(ldval=7), dict(x=None), dict(idx=None),
    dict(val=None), dict(label=None), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
    dict(temperature=float("inf")), dict(hard=-0.1), dict(hard=1.1), dict(hard=float("nan")), dict(lddiff=99), dict(lddiff=127),
    dict(row_loss=None)])
def test_distill_refuses(change):
    assert status("hipF_distill_eval", DISTILL, **change) == INVALID


def test_outputs_over_each_other():
    assert status("hipF_adapter_forward", FORWARD, t=2 * P) == INVALID
    assert status("hipF_adapter_backward", BACKWARD, y=3 * P, ldy=32) == INVALID
    assert status("hipF_adapter_backward", BACKWARD, eout=2 * P) == INVALID


def test_too_many():
    rows = 2 ** 26 + 1
    assert status("hipF_adapter_forward", FORWARD, N=rows) == TOO_LARGE
    assert b"67108865" in h.lib.hipK_error_string(TOO_LARGE)
    assert status("hipF_adapter_backward", BACKWARD, N=rows) == TOO_LARGE
    assert status("hipF_adapter_forward", FORWARD, N=rows, ad=adapters(num=0)) == TOO_LARGE
    assert status("hipI32_adapter_plan", PLAN, num=2 ** 21 + 1) == TOO_LARGE
    assert b"2097153" in h.lib.hipK_error_string(TOO_LARGE)
    wide = 2 ** 30 + 1
    assert status("hipF_adapter_forward", FORWARD, I=wide, ldin=wide, ldw=wide, ad=adapters(lddown=wide)) == TOO_LARGE
    assert status("hipF_adapter_backward", BACKWARD, O=wide, lde=wide, ad=adapters(ldup=wide)) == TOO_LARGE
    assert status("hipF_row_top", TOP, d=(4, wide, wide)) == TOO_LARGE
    assert status("hipF_distill_eval", DISTILL, d=(4, wide, wide), lddiff=wide) == TOO_LARGE
    assert b"1073741825" in h.lib.hipK_error_string(TOO_LARGE)
    # one workgroup per adapter and 32 columns
    assert status("hipF_adapter_backward", BACKWARD, ad=adapters(num=2 ** 22)) == TOO_LARGE
    assert b"48 columns" in h.lib.hipK_error_string(TOO_LARGE)


@pytest.mark.parametrize("first", ["kaldi_amd.hip", "kaldi_amd.nnet"])
def test_torch_behind_the_library(first):
    """A program that uses both, in this order, ends as it should."""
    env = {k: v for k, v in os.environ.items() if k != "KALDI_AMD_HIP_LIB"}
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    assert subprocess.run([sys.executable, "-c", "import %s, torch" % first], env=env, cwd=root, timeout=300).returncode == 0


def test_k_too_large():
    big = h.MAX_TOP + 1
    assert status("hipF_row_top", TOP, K=big, ldidx=256, ldval=256) == TOO_LARGE
    assert status("hipF_distill_eval", DISTILL, K=big, ldidx=256, ldval=256) == TOO_LARGE
