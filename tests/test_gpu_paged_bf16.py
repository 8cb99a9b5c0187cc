"""Attention under bf16 queries at the bounds of what the kernels round, with the
units of tests/test_gpu_paged.py: u = 2^-24, w = 2^-8 (bf16, half a step), M =
sum p |v| / sum p, S = the largest sum |q k| / sqrt(hd).

  all: scores and sums in fp32, (2 (hd / 4 + 8) S + 256) u M, and the result's
    rounding, w |y|.
  prompts: every probability rounded to bf16 (over int8: times V's scale), w M.
    bf16 values and int8 codes are exact.  An fp32 value x of 2^e .. 2^(e + 1)
    is two bf16 numbers: the first leaves 2^(e - 8) at most, and half a step of
    the second is 2^(e - 17) then, 2^-17 x.  Scores are off by 2^-17 S,
    probabilities by twice that relative to their sum, V by 2^-17: (2 S + 1) w^2 /
    2 M.
  decode: over bf16 and int8 probabilities are two bf16 numbers: 2^-17 M, which
    the 256 u M has in it.

In the 2-norm of many values, roundings that fall anywhere within half a step
(of at most w |x|) are w / sqrt(3) at most: one of them for decode, two
independent ones for prompts, w sqrt(2 / 3) = 0.0032.  Values of an fp32 or int8
cache rounded to one bf16 number each come to 0.0039."""
import numpy as np
import pytest

import guanaco_amd.hip as H
from paged import BF16, F32, I8, World, dec
from test_gpu_paged import DECODES, PROMPTS, U, W, attend, some_rows

pytestmark = pytest.mark.gpu


def check(w, q, got, rows, prompt):
    nh, hd = q.shape[1], w.hd
    num = den = 0.0
    for t in rows:
        y, mag, top = w.attention(q[t].astype(np.float64), t)
        tol = (2 * (hd / 4 + 8) * top + 256) * U * mag + W * np.abs(y)
        if prompt:
            tol = tol + W * mag
            if w.cache == F32:
                tol = tol + (2 * top + 1) * W ** 2 / 2 * mag
        off = np.abs(got[t].reshape(nh, hd) - y)
        assert (off <= tol + 1e-30).all(), (t, w.at[t], float((off - tol).max()), float(off.max()))
        num, den = num + float((off ** 2).sum()), den + float((y ** 2).sum())
    assert (num / den) ** 0.5 < W * ((2 if prompt else 1) / 3) ** 0.5, (num / den) ** 0.5


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("case", PROMPTS)
def test_prompt(ctx, case, cache):
    nh, nkv, hd, page, hist, new, holes = case
    w = World(60, hist, new, nkv, hd, cache, page, holes=holes).upload(ctx, H)
    q, got = attend(ctx, w, nh, BF16, "paged_prompt_dev")
    check(w, q, dec(got, BF16), range(len(w.at)), True)
    w.free()


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("hist,new", [([7001, 30, 0], [5, 130, 1]), ([500], [2000])])
def test_prompt_in_parts_and_in_large_tiles(ctx, hist, new, cache):
    w = World(61, hist, new, 4, 128, cache, 64).upload(ctx, H)
    q, got = attend(ctx, w, 16, BF16, "paged_prompt_dev")
    check(w, q, dec(got, BF16), some_rows(w, 30), True)
    w.free()


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("case", DECODES)
def test_decode(ctx, case, cache):
    nh, nkv, hd, page, lens, holes = case
    w = World(62, [n - 1 for n in lens], [1] * len(lens), nkv, hd, cache, page, holes=holes).upload(ctx, H, with_first=False)
    q, got = attend(ctx, w, nh, BF16, "paged_decode_dev")
    check(w, q, dec(got, BF16), range(len(lens)), False)
    w.free()
