"""Sampling where a row has more than 131072 tokens: weights are whole numbers of
2^-S with S = 62 - ceil(log2 vocab) there, each off by one at most, so that a
running sum and the share of a sum that it is compared with are off by vocab *
2^-S of the largest weight each.  Draws and borders lie further apart here."""
import numpy as np
import pytest

from test_gpu_sample_rows import logits, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [131073, 262145, 1 << 20])
def test_draws_and_borders(ctx, V):
    S = 62 - (V - 1).bit_length()
    x = logits(6, V, 90 + V % 7)
    for n, (T, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (2.0, V // 3, 0.8, 0.0), (0.7, 500, 0.95, 0.02), (5.0, V - 1, 0.5, 0.2)]):
        u = np.random.default_rng(91 + n).random(6, np.float32)
        tok, lp = run(ctx, x, np.float32(T), k, np.float32(p), np.float32(m), u)
        for i in range(6):
            t, want, far = reference(x[i], np.float32(T), k, np.float32(p), np.float32(m), u[i])
            assert far > 2 * V * 2.0 ** -S, "the draw is too near to a border to say"
            assert tok[i] == t and abs(lp[i] - want) <= 2.0 ** -24 * abs(want) + V * 2.0 ** -S
