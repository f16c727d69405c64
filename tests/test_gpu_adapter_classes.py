"""The adapter classes where a call goes wrong or has nothing to do (tests/fuzz/adapter_edges_walk.cc)."""
import subprocess

import pytest

from test_adapter_classes import BAD, WALK

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", sorted(BAD))
def test_adapters_in_use_survive_a_refused_file(tmp_path, what):
    f = tmp_path / "adapters"
    f.write_text(BAD[what])
    r = subprocess.run([WALK, "reread", str(f)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[:2] == ["refused 1 adapters 3 12 -> 9", "same 1"]


def test_adapters_of_a_file_have_no_gradients_yet(tmp_path):
    """What the adapters before the file left behind (gradients, the narrow products of a forward pass) is not theirs."""
    r = subprocess.run([WALK, "stale", str(tmp_path / "adapters")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[:4] == ["update refused 1", "weights same 1", "backpropagate refused 1", "as fresh ones 1"]


def test_a_bunch_without_rows(tmp_path):
    """... has outputs without rows and gradients of zeros, in front of a bunch with rows and behind one."""
    r = subprocess.run([WALK, "empty"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[:4] == ["out 0 below 0 gradients zero 1", "out 37 below 37 gradients zero 0"] * 2


def test_outputs_that_are_inputs(tmp_path):
    """... are refused before they are resized: the inputs are still there."""
    r = subprocess.run([WALK, "inplace"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[:6] == ["propagate refused 1", "backpropagate refused 1 1 1", "row top refused 1", "distill refused 1",
                                        "inputs same 1", "in place 1"]
