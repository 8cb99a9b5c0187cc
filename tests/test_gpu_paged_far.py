"""Decode attention under a bound far above most lengths, whose parts are
longer, against the definition (tests/test_gpu_paged.py has the tolerances)."""
import numpy as np
import pytest

import guanaco_amd.hip as H
from paged import BF16, F32, I8, World, dec
from test_gpu_paged import attend, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_many_sequences_under_a_far_bound(ctx, cache, xt):
    r = np.random.default_rng(40)
    lens = r.integers(0, 300, 700)
    lens[[3, 650]] = 5000, 1
    w = World(41, [n - 1 for n in lens], [1] * 700, 8, 64, cache, 64)
    w.max_len = 100000
    w.table = np.pad(w.table, ((0, 0), (0, -(-w.max_len // 64) - w.stride)), constant_values=-1)
    w.stride = w.table.shape[1]
    w.upload(ctx, H, with_first=False)
    q, got = attend(ctx, w, 16, xt, "paged_decode_dev")
    check_attention(w, q, dec(got, xt), [0, 3, 649, 650, 699, *r.integers(0, 700, 30)], xt, False)
    w.free()
