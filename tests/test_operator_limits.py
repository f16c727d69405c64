"""More of what the adapter, top-logit and distillation entry points refuse (see test_operator_refusals.py): no GPU is needed, a
refused call never reaches a kernel."""
import pytest

import kaldi_amd.hip as h
from test_operator_refusals import BACKWARD, FORWARD, INVALID, PLAN, TOO_LARGE, status


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
