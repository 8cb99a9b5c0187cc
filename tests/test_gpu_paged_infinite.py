"""Infinities and NaN of V, and scales of int8 rows that are none, wherever their
position lies in a tile, a block or a part: the outputs that see them are NaN
in V's dimensions, and every other output is what it is without them, bit for
bit."""
import numpy as np
import pytest

import guanaco_amd.hip as H
from paged import BF16, F32, I8, World, dec, enc
from test_gpu_paged import attend

pytestmark = pytest.mark.gpu


def poisoned(ctx, args, kw, cache, xt, nh, entry, at, value, head, dim, scale):
    """outputs with the value at position `at` of sequence 0"""
    w = World(*args, **kw)
    if at is not None:
        g, o = w.slot(0, at)
        if cache == I8:
            w.pools[1][1][g, head, o] = value
        else:
            w.pools[1][0][g, head, o, dim] = enc(np.array([value], np.float32), cache)[0]
    w.upload(ctx, H)
    got = attend(ctx, w, nh, xt, entry, scale=scale)[1]
    w.free()
    return dec(got, xt).reshape(-1, nh, args[4])


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("entry,nh,nkv,hd,page,hist,new,places", [
    # one part; sixteen; and heads of their own
    ("paged_decode_dev", 8, 2, 128, 32, [130, 5], [1, 1], [0, 17, 64, 130]),
    ("paged_decode_dev", 16, 1, 64, 64, [4095], [1], [0, 1000, 2049, 4095]),
    ("paged_decode_dev", 4, 4, 64, 16, [300, 2], [3, 1], [5, 255, 302]),
    # blocks that all rows see whole, that some do, and the last; parts
    ("paged_prompt_dev", 8, 2, 64, 16, [70, 0], [90, 40], [0, 65, 80, 128, 159]),
    ("paged_prompt_dev", 16, 8, 128, 64, [300], [150], [10, 299, 310, 449]),
    ("paged_prompt_dev", 12, 1, 128, 32, [5000, 300], [2, 130], [0, 2500, 4999, 5001]),
    ("paged_prompt_dev", 16, 4, 128, 64, [100], [1500], [3, 700, 1599]),
])
def test_one_answer_wherever_they_lie(ctx, entry, nh, nkv, hd, page, hist, new, places, cache, xt):
    args, kw, G = (50, hist, new, nkv, hd, cache, page), dict(pad=1), nh // nkv
    clean = {s: poisoned(ctx, args, kw, cache, xt, nh, entry, None, 0, 0, 0, s) for s in (1.5, 30.0)}
    for n, at in enumerate(places):
        for value in (np.inf, -np.inf, np.nan):
            scale = (1.5, 30.0)[n % 2]  # softmaxes that leave some weights above 0, and few
            head, dim = n % nkv, (37 * n + 5) % hd
            got = poisoned(ctx, args, kw, cache, xt, nh, entry, at, value, head, dim, scale)
            hit = np.zeros(got.shape, bool)
            first = max(0, at - hist[0]) if entry == "paged_prompt_dev" else new[0] - 1
            hit[first:new[0], head * G:(head + 1) * G, slice(None) if cache == I8 else dim] = True
            assert np.isnan(got[hit]).all(), (at, value, got[hit][~np.isnan(got[hit])][:4])
            assert np.array_equal(got[~hit], clean[scale][~hit]), (at, value)


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("entry", ["paged_decode_dev", "paged_prompt_dev"])
def test_both_infinities(ctx, entry, cache):
    """+ and - infinity in one dimension, before and behind each other."""
    for first, second in ((3, 200), (200, 3)):
        w = World(51, [255], [1], 2, 64, cache, 16)
        for at, v in ((first, np.inf), (second, -np.inf)):
            g, o = w.slot(0, at)
            if cache == I8:
                w.pools[1][1][g, 1, o] = v
            else:
                w.pools[1][0][g, 1, o, 7] = enc(np.array([v], np.float32), cache)[0]
        w.upload(ctx, H)
        got = attend(ctx, w, 4, F32, entry)[1].reshape(4, 64)
        w.free()
        hit = np.zeros(got.shape, bool)
        hit[2:, slice(None) if cache == I8 else 7] = True
        assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
