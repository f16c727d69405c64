"""Adapters files that are refused (tests/fuzz/adapter_edges_walk.cc), without a GPU: what is wrong with a file is found before
anything of it is taken over."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WALK = os.path.join(ROOT, "kaldi_amd", "bin", "adapter_edges_walk")


def matrix(rows, cols):
    return " [\n" + "\n".join("  " + " ".join("0.5" for _ in range(cols)) for _ in range(rows)) + " ]\n"


def adapters_file(ranks, down, up, dims=(5, 4), scales=None):
    """An <adapters> file in text: dims = output, input; down, up = rows and columns of the stacks."""
    scale = " [ " + " ".join("1" for _ in range(len(ranks) if scales is None else scales)) + " ]\n"
    return "<adapters> %d %d [ %s ]\n" % (*dims, " ".join(map(str, ranks))) + scale + matrix(*down) + matrix(*up)


BAD = {
    "a rank of 129": adapters_file([129], (129, 4), (129, 5)),
    "a rank of 200 among others": adapters_file([2, 200, 1], (203, 4), (203, 5)),
    "a negative rank that another balances": adapters_file([-1, 3], (2, 4), (2, 5)),
    "ranks far apart that add up": adapters_file([2 ** 31 - 1, -2 ** 31 + 3], (2, 4), (2, 5)),
    "rows that the ranks do not add up to": adapters_file([1, 2], (4, 4), (3, 5)),
    "stacks of other columns": adapters_file([1, 2], (3, 4), (3, 6)),
    "scales of other adapters": adapters_file([1, 2], (3, 4), (3, 5), scales=3),
    "no inputs": adapters_file([1, 2], (3, 4), (3, 5), dims=(5, 0)),
}


@pytest.mark.parametrize("what", sorted(BAD))
def test_refused_into_empty_adapters(tmp_path, what):
    f = tmp_path / "adapters"
    f.write_text(BAD[what])
    r = subprocess.run([WALK, "read", str(f)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[0] == "refused 1 adapters 0 0 -> 0", r.stderr
