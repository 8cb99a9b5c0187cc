"""Sampling for a batch against the definition in float64 with exact sums
(fractions of the weights): the token of every draw, borders and ties included.

A weight is rounded by at most 2^-46 of the largest (half a unit of 2^-S, S at
least 45 up to 131072 tokens), so a sum over the vocabulary and a share of one
by vocab * 2^-46 each: a draw that falls within vocab * 2^-45 of the largest
weight of a border may pick the neighbour, and a filter's border likewise; the
draws here are checked to lie further away, except where the sums are exact
(equal logits), where there is nothing to move.  min-p compares one weight, not
a sum: 2^-45 away is enough.
logprobs: the float32 rounding of a float64 value, 2^-24 relative, and 1e-12."""
import numpy as np
import pytest

import guanaco_amd.hip as H

pytestmark = pytest.mark.gpu


def reference(x, T, k, p, m, u):
    """(token, logprob, distance of the nearest border in units of the largest weight)"""
    x = x.astype(np.float64)
    ok = ~np.isnan(x) & (x > -np.inf)
    if not ok.any():
        return -1, -np.inf, 1.0
    top = x[ok].max()
    if not T > 0:
        return int(np.flatnonzero(ok & (x == top))[0]), 0.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(ok, np.where(x == top, 1.0, np.exp((x - top) / np.float64(T))), 0.0)
    order = np.flatnonzero(ok)[np.argsort(-x[ok], kind="stable")]
    far = 1.0
    if p <= 0:
        k, p = 1, 1.0
    if k > 0:
        order = order[:k]
    ws = w[order]
    if p < 1:
        c = np.cumsum(ws)
        t = np.float64(np.float32(p)) * c[-1]
        n = int(np.searchsorted(c, t)) + 1
        far = min(far, float(np.abs(c - t).min()))
        order, ws = order[:n], ws[:n]
    m = min(max(np.float64(np.float32(m)), 0.0), 1.0)
    if m > 0:
        far = min(far, len(x) * float(np.abs(ws[ws < 1] - m).min()) if (ws < 1).any() else 1.0)  # one weight against 2^-45
        order = order[ws >= m]
    order = np.sort(order)
    c = np.cumsum(w[order])
    t = np.float64(np.float32(u)) * c[-1]
    i = int(np.searchsorted(c, t, side="right"))
    far = min(far, float(np.abs(c - t).min()))
    if not i < len(c):
        i = int(np.flatnonzero(w[order])[-1])
    return int(order[i]), float(np.log(w[order[i]] / c[-1])), far


def run(ctx, x, T, k, p, m, u, stride=None, nulls=()):
    rows, V = x.shape
    stride = stride or V
    a = np.full((rows, stride), 99.0, np.float32)  # above every logit
    a[:, :V] = x
    f = lambda v, t=np.float32: ctx.upload(np.broadcast_to(np.asarray(v, t), rows).copy())  # noqa: E731
    b = [ctx.upload(a), f(T), f(k, np.int32), f(p), f(m), f(u), ctx.upload(np.full(rows, -7, np.int32)), ctx.upload(np.full(rows, 7, np.float32))]
    c = [None if i in nulls else v for i, v in enumerate(b)]
    ctx.sample_rows_dev(c[0], rows, V, stride, *c[1:])
    tok, lp = b[6].download(np.int32), b[7].download()
    for v in b:
        v.free()
    return tok, lp


def check(ctx, x, T, k, p, m, u, exact=False, **kw):
    rows = len(x)
    full = [np.broadcast_to(np.asarray(v), rows) for v in (T, k, p, m, u)]
    tok, lp = run(ctx, x, T, k, p, m, u, **kw)
    for i in range(rows):
        t, l, far = reference(x[i], *(np.float32(v[i]) if n != 1 else int(v[i]) for n, v in enumerate(full)))
        if not exact:
            assert far > x.shape[1] * 2.0 ** -45, "the draw is too near to a border to say"
        assert tok[i] == t, (i, tok[i], t, far, [v[i] for v in full])
        assert lp[i] == l or abs(lp[i] - l) <= 2.0 ** -24 * abs(l) + 1e-12, (lp[i], l)


def logits(rows, V, seed, kind="normal"):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, V)) * 2.2
    if kind == "ties":
        x = np.round(x * 2) / 2
    if kind == "peaked":
        x[:, r.integers(0, V, 3)] += 25
    if kind == "flat":
        x *= 0.01
    return x.astype(np.float32)


FILTERS = [(0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (40, 0.95, 0.05), (1000, 0.5, 0.0), (1, 1.0, 0.0), (0, 0.0, 0.0),
           (0, 0.999, 0.001), (5, 0.99, 0.9)]


@pytest.mark.parametrize("V", [1, 2, 63, 65, 1000, 4097, 50257])
@pytest.mark.parametrize("kind", ["normal", "ties", "peaked", "flat"])
def test_filters(ctx, V, kind):
    r = np.random.default_rng(V)
    for n, (k, p, m) in enumerate(FILTERS):
        x = logits(6, V, 100 + n, kind)
        T = r.choice([0.3, 0.7, 1.0, 1.5], 6).astype(np.float32)
        check(ctx, x, T, k, p, m, r.random(6, np.float32), stride=V + n)


def test_rows_of_their_own(ctx):
    """128 rows of the 8B vocabulary, each with its own parameters"""
    r = np.random.default_rng(1)
    x = logits(128, 128256, 2)
    k, p, m = (np.array(v) for v in zip(*[FILTERS[r.integers(len(FILTERS))] for _ in range(128)]))
    T = r.choice([0.0, 0.5, 0.8, 1.2], 128).astype(np.float32)
    check(ctx, x, T, k.astype(np.int32), p.astype(np.float32), m.astype(np.float32), r.random(128, np.float32))


def test_many_draws_of_one_row(ctx):
    """Every token of a small vocabulary is drawn where its share of [0, 1) is."""
    x = np.repeat(logits(1, 300, 3), 2000, 0)
    u = ((np.arange(2000) + 0.5) / 2000).astype(np.float32)
    for k, p, m in [(0, 1.0, 0.0), (50, 0.8, 0.01)]:
        check(ctx, x, 1.0, k, p, m, u)


def test_equal_logits(ctx):
    """Sums that are exact, and so borders that can be hit: the lowest indexes."""
    x = np.full((8, 4096), -3.25, np.float32)
    u = np.array([0, 0.25, 0.5, 0.75, 0.99999994, 1 / 4096, 0.125, 0.3], np.float32)
    for k, p, m in [(0, 1.0, 0.0), (1024, 1.0, 0.0), (0, 0.5, 0.0), (2048, 0.25, 1.0), (0, 0.0625, 0.0), (0, 1.0, 1.0)]:
        check(ctx, x, 0.7, k, p, m, u, exact=True)
    two = np.where(np.arange(4096) % 3 == 0, np.float32(2), np.float32(-60)).astype(np.float32)[None].repeat(8, 0)
    for k, p in [(0, 1.0), (700, 1.0), (0, 0.5), (3000, 0.5)]:
        check(ctx, two, 0.5, k, p, 0.0, u, exact=True)


def test_large_vocabularies_of_equal_logits(ctx):
    x = np.zeros((2, 1 << 20), np.float32)
    check(ctx, x, 1.0, 0, 0.5, 0.0, np.array([0.5, 0.99], np.float32), exact=True)
    check(ctx, x, 1.0, 700001, 0.75, 0.0, np.array([0.0, 0.5], np.float32), exact=True)


def test_values_that_are_no_numbers(ctx):
    x = logits(9, 500, 5)
    x[0, 10:20] = np.nan
    x[1, :] = -np.inf
    x[2, :] = np.nan
    x[3, 5:] = -np.inf
    x[4, 7] = x[4, 400] = np.inf
    x[5, :499] = np.nan
    x[6, ::2] = -np.inf
    x[7, :] = 0.0
    x[7, ::3] = -0.0
    x[8, 3] = 3e38
    x[8, 4] = -3e38
    u = np.full(9, 0.37, np.float32)
    for T in (0.0, -1.0, np.nan, 1e-30, 0.8, 50.0):
        for k, p, m in [(0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.6, 0.0), (4, 0.9, 0.1), (499, 0.3, 0.0)]:
            check(ctx, x, np.float32(T), k, p, m, u, exact=True)


def test_parameters_out_of_range(ctx):
    x = logits(4, 700, 6)
    u = np.array([0.1, 0.4, 0.6, 0.9], np.float32)
    base = run(ctx, x, 1.0, 0, 1.0, 0.0, u)
    for k, p, m in [(-5, 1.0, 0.0), (700, 1.0, 0.0), (10 ** 9, 2.0, -1.0), (0, np.nan, np.nan)]:
        got = run(ctx, x, 1.0, k, p, m, u)
        assert np.array_equal(got[0], base[0]) and np.array_equal(got[1], base[1])
    assert np.array_equal(run(ctx, x, 9.0, 3, 0.1, 0.5, u, nulls=(1, 2, 3, 4))[0], base[0])  # all off, temperature 1
    assert np.array_equal(run(ctx, x, 1.0, 0, 1.0, 0.0, u, nulls=(7,))[0], base[0])
    top = run(ctx, x, 1.0, 0, 1.0, 2.0, u)  # min_p above 1: the largest alone
    assert np.array_equal(top[0], x.argmax(1)) and np.array_equal(top[1], np.zeros(4, np.float32))
    # rnd of 1 or more, and NaN: the last token that is kept; below 0: the first
    for v, first in [(1.0, False), (7.0, False), (np.nan, False), (-0.5, True)]:
        got = run(ctx, x, 1.0, 20, 1.0, 0.0, np.float32(v))[0]
        kept = np.sort(np.argsort(-x, 1, kind="stable")[:, :20], 1)
        assert np.array_equal(got, kept[:, 0 if first else -1])


def test_repeated_calls_give_the_same(ctx):
    x = logits(16, 128256, 7, "flat")
    u = np.random.default_rng(8).random(16, np.float32)
    a = run(ctx, x, 1.0, 0, 0.97, 0.0, u)
    for _ in range(3):
        b = run(ctx, x, 1.0, 0, 0.97, 0.0, u)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("rows", [1, 3, 70, 300, 600])
def test_rows_shared_by_workgroups(ctx, rows):
    """From one row to more than a launch takes: 16 parts a row to one, lists
    that hold all before top-k's border, lists that do not fit, none."""
    V = 66000 if rows < 100 else 9001
    r = np.random.default_rng(rows)
    f = [(3000, 0.9, 0.0), (6000, 0.9, 0.0), (6000, 0.999, 0.001), (8990, 0.5, 0.2), (50, 1.0, 0.0), (0, 0.97, 0.0), (0, 1.0, 0.0), (V, 0.3, 0.01)]
    k, p, m = (np.array(v) for v in zip(*[f[(i + rows) % len(f)] for i in range(rows)]))
    x = logits(rows, V, rows + 20)
    check(ctx, x, r.choice([0.6, 1.0, 1.7], rows).astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32),
          r.random(rows, np.float32), stride=V + 3)


@pytest.mark.parametrize("at", [0, 3, 30000])
def test_border_tokens_side_by_side(ctx, at):
    """9000 neighbours share the border's bin: more than fit a list, and all of
    them those of few waves; and 700, more than one wave's share of it."""
    for n in (700, 9000):
        x = logits(4, 128256, n + at) - 20
        x[:, at:at + n] = 3 + 1e-4 * np.random.default_rng(n).random((4, n))
        x[:, at + n + 5] = 4
        x = x.astype(np.float32)
        u = np.array([0.01, 0.3, 0.6, 0.99], np.float32)
        for k, p, m in [(n // 2, 1.0, 0.0), (0, 0.7, 0.0), (n - 50, 0.6, 0.2), (n // 2, 0.9, 0.9)]:
            check(ctx, x, 1.0, k, p, m, u)


def test_one_call_of_many_rows_is_many_calls(ctx):
    """A row's token does not depend on how many workgroups share its row."""
    x = logits(33, 50257, 9)
    u = np.random.default_rng(10).random(33, np.float32)
    a = run(ctx, x, 0.9, 400, 0.93, 0.001, u)
    for i in (0, 7, 32):
        b = run(ctx, x[i:i + 1], 0.9, 400, 0.93, 0.001, u[i:i + 1])
        assert a[0][i] == b[0][0] and a[1][i] == b[1][0]


@pytest.mark.parametrize("T", [np.inf, 3e38, 1e-42, 1e-37])
def test_temperatures_at_the_ends(ctx, T):
    x = logits(4, 5000, 12)
    x[1] *= 1e37
    x[2, :3] = 3.4e38
    x[3] *= 1e-38
    u = np.array([0.13, 0.5, 0.77, 0.91], np.float32)
    for k, p, m in [(0, 1.0, 0.0), (33, 1.0, 0.0), (0, 0.7, 0.0), (2500, 0.51, 0.3)]:
        check(ctx, x, np.float32(T), k, p, m, u, exact=True)


def test_the_largest_vocabulary(ctx):
    """2^20 tokens, a stride of their number and one: rows that start 4-byte
    aligned, borders in bins of more tokens than a list holds."""
    x = logits(3, 1 << 20, 13)
    u = np.array([0.2, 0.55, 0.9], np.float32)
    for T, k, p, m in [(1.0, 0, 0.9, 0.0), (3.0, 100000, 0.95, 0.01), (20.0, 0, 0.5, 0.0), (1.0, 50, 0.9, 0.0)]:
        check(ctx, x, np.float32(T), k, p, m, u, stride=(1 << 20) + 1)


def test_many_rows_of_the_largest_vocabulary(ctx):
    """Parts of more than 2^18 tokens, which are drawn from in larger groups;
    offsets past 2^28 elements."""
    rows, V = 300, 1 << 20
    x, on = logits(3, V, 14), [0, 151, 299]
    b = ctx.alloc(4 * rows * V)
    small = ctx.upload(np.zeros(V, np.float32))
    for i in range(rows):
        src = ctx.upload(x[on.index(i)]) if i in on else small
        assert H.lib.gq_hip_copy_dev(ctx.h, b.ptr + 4 * V * i, src.ptr, 4 * V) == 0
        ctx.sync()
        if i in on:
            src.free()
    u = np.random.default_rng(15).random(rows, np.float32)
    ub, tok = ctx.upload(u), ctx.upload(np.full(rows, -7, np.int32))
    f = lambda v, t: ctx.upload(np.full(rows, v, t))  # noqa: E731
    k, p, m = f(70000, np.int32), f(0.8, np.float32), f(0.001, np.float32)
    for with_filters in (False, True):
        ctx.sample_rows_dev(b, rows, V, V, None, k if with_filters else None, p if with_filters else None, m if with_filters else None, ub, tok)
        got = tok.download(np.int32)
        for j, i in enumerate(on):
            t, _, far = reference(x[j], np.float32(1), 70000 if with_filters else 0, 0.8 if with_filters else 1.0, 0.001 if with_filters else 0.0, u[i])
            assert far > V * 2.0 ** -44 and got[i] == t, (i, got[i], t, far)
        n = int(np.ceil(np.float64(np.float32(0.8)) * 70000)) if with_filters else V  # equal logits: the first n
        for i in (1, 150, 298):
            assert got[i] == int(np.float64(u[i]) * n)
    for v in (b, small, ub, tok, k, p, m):
        v.free()
