"""The adapter, top-logit and distillation entry points at the ends of what their interface allows, against the same oracles and
tolerances as test_gpu_adapters.py and test_gpu_distill.py."""
import numpy as np
import pytest

from test_gpu_distill import check_distill, table

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
