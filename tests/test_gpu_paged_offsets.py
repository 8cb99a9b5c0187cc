"""Offsets that pass 32 bits: pools of more than 2^32 values with the sequences'
pages at their end, and packed rows 2^24 elements apart.  Every result is bit for
bit that of small pools and dense rows."""
import numpy as np
import pytest

import guanaco_amd.hip as H
import paged as P
from paged import BF16, F32, I8

pytestmark = pytest.mark.gpu
NH, NKV, HD, PAGE, HIST, NEW = 8, 2, 128, 64, [0, 300], [330, 20]


def serve(ctx, cache, xt, n_pages, stride):
    """q as rotated, rows read back, prompt's and decode's outputs"""
    r = np.random.default_rng(90)
    size, width = P.itemsize(xt), (NH + 2 * NKV) * HD
    table = n_pages - 1 - r.permutation(12).reshape(2, 6).astype(np.int32)
    n = sum(NEW)
    values = n_pages * NKV * PAGE * HD
    pools = [ctx.alloc(values * P.itemsize(cache)) for _ in range(2)]
    scales = [ctx.alloc(4 * values // HD) if cache == I8 else None for _ in range(2)]
    tb, first = ctx.upload(table), np.concatenate([[0], np.cumsum(NEW)]).astype(np.int32)
    fb, zero, pos = ctx.upload(first), ctx.upload(np.zeros(2, np.int32)), ctx.upload(np.array(HIST, np.int32))
    pages = H.GqPages(pools[0].ptr, pools[1].ptr, *(s.ptr if s else None for s in scales), cache, n_pages, PAGE, NKV, HD)
    rope = ctx.upload(P.rope_table(384, HD))
    rows, out = ctx.alloc(n * stride * size), ctx.alloc(n * stride * size)
    at = lambda b, i, c=0: type("B", (), {"ptr": b.ptr + (i * stride + c) * size})  # noqa: E731

    def put(b, x):
        x = P.enc(x, xt)
        for i in range(len(x)):
            row = np.ascontiguousarray(x[i])
            ctx.check(H.lib.gq_hip_h2d(ctx.h, at(b, i).ptr, row.ctypes.data, row.nbytes), "h2d")

    def get(b, m, cols):
        got = np.empty((m, cols), P.np_type(xt))
        for i in range(m):
            ctx.check(H.lib.gq_hip_d2h(ctx.h, got[i].ctypes.data, at(b, i).ptr, got[i].nbytes), "d2h")
        return got

    append = lambda batch: ctx.paged_append_dev(pages, batch, xt, NH, rows, stride, rows, stride, at(rows, 0, NH * HD), stride,  # noqa: E731
                                                at(rows, 0, (NH + NKV) * HD), stride, rope, 384)
    put(rows, r.standard_normal((300, width)).astype(np.float32))  # the second sequence's history
    append(H.GqBatch(tb.ptr + 4 * 6, zero.ptr, ctx.upload(np.array([0, 300], np.int32)).ptr, 1, 6, 300, 384))
    put(rows, r.standard_normal((n, width)).astype(np.float32))
    batch = H.GqBatch(tb.ptr, pos.ptr, fb.ptr, 2, 6, n, 384)
    append(batch)
    got = [get(rows, n, NH * HD)]
    ctx.paged_read_dev(pages, batch, xt, out, stride, at(out, 0, NKV * HD), stride)
    got.append(get(out, n, 2 * NKV * HD))
    ctx.paged_prompt_dev(pages, batch, xt, NH, rows, stride, out, stride)
    got.append(get(out, n, NH * HD))
    ctx.paged_decode_dev(pages, batch, xt, NH, rows, stride, out, stride)
    got.append(get(out, n, NH * HD)[first[1:] - 1])
    for b in (*pools, *scales, tb, fb, zero, pos, rope, rows, out):
        if b:
            b.free()
    return got


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_as_in_small_ones(ctx, cache, xt):
    width = (NH + 2 * NKV) * HD
    small = serve(ctx, cache, xt, 12, width)
    pools = serve(ctx, cache, xt, (1 << 32) // (NKV * PAGE * HD) + 5, width)
    rows = serve(ctx, cache, xt, 12, 1 << 24)  # 350 of them: 2^32 elements and more
    for a, b, c in zip(small, pools, rows):
        assert np.array_equal(a, b) and np.array_equal(a, c)
    assert all(np.isfinite(P.dec(a, xt)).all() and P.dec(a, xt).any() for a in small)
