"""The paged cache's entry points against their definitions in float64
(tests/paged.py).

Append and read are exact: rotated rows bit for bit, bf16 rows rounded to
nearest even, int8 codes and scales as the definition gives them, everything
else in the pools as it was.

Attention, per output value, with u = 2^-24 (fp32), w = 2^-8 (bf16, half a
step), M = sum p |v| / sum p and S = the largest sum |q k| / sqrt(hd):
  fp32 throughout: scores are sums of hd products over at most hd / 4 + 8
    roundings, so off by at most (hd / 4 + 8) u S, and a probability by twice
    that relative to its sum; the outputs' own sums add at most 64 roundings per
    part of the keys (they are summed 16 or 32 at a time and rescaled): 256 u M.
    Together (2 (hd / 4 + 8) S + 256) u M, and 1e-5 in the 2-norm of all, the
    bar of the single-sequence attention.
  bf16 rows: the result's rounding w |y|, beside that.
  bf16 prompts: every probability rounded to bf16 besides: w M; and over an fp32
    or int8 cache K's and V's values too: scores off by w S, probabilities by
    twice that relative to their sum, 2 w S M, and w M from V.
"""
import numpy as np
import pytest

import guanaco_amd.hip as H
import paged as P
from paged import BF16, F32, I8, World, dec, enc

pytestmark = pytest.mark.gpu
U, W = 2.0 ** -24, 2.0 ** -8


def rows_buf(ctx, x, t, stride):
    """rows of x at a stride of `stride` elements, NaN between them"""
    a = np.full((len(x), stride), np.nan, np.float32)
    a[:, :x.shape[1]] = x
    return ctx.upload(enc(a, t))


LAYOUTS = [
    # heads, KV heads, head_dim, page, positions before, new tokens
    (32, 8, 128, 64, [4000, 0, 63, 64, -1, 130], [1, 1, 1, 1, 1, 1]),
    (32, 4, 64, 16, [0, 15, 301], [77, 1, 33]),
    (8, 8, 64, 32, [0], [1]),
    (6, 2, 128, 256, [5, 0, 0, 300], [3, 0, 41, 2]),
    (16, 1, 64, 128, [127, 1], [2, 5]),
    (28, 4, 128, 16, [17, -1, 0, 31], [1, 2, 16, 1]),
]


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_append(ctx, layout, cache, xt):
    nh, nkv, hd, page, hist, new = layout
    w = World(1, hist, new, nkv, hd, cache, page, holes=[(0, 0)] if len(hist) > 4 else [], pad=2).upload(ctx, H)
    r = np.random.default_rng(2)
    width = (nh + 2 * nkv) * hd
    x = dec(enc(r.standard_normal((w.rows, width)).astype(np.float32), xt), xt)
    cs = P.rope_table(w.max_len, hd)
    xb, rb = rows_buf(ctx, x, xt, width + 8), ctx.upload(cs)
    qo = ctx.upload(np.full((w.rows, nh * hd), 7, P.np_type(xt)))
    at = lambda n: type("B", (), {"ptr": xb.ptr + n * P.itemsize(xt)})  # noqa: E731
    ctx.paged_append_dev(w.pages, w.batch, xt, nh, xb, width + 8, qo, nh * hd, at(nh * hd), width + 8, at((nh + nkv) * hd),
                         width + 8, rb, w.max_len)
    q_exp = np.full((w.rows, nh * hd), 7, P.np_type(xt))
    exp = [(c.copy(), None if d is None else d.copy()) for c, d in w.pools]
    for t, (s, p) in enumerate(w.at):
        where = w.slot(s, p)
        if where is None:
            continue
        y = x[t].reshape(-1, hd)
        rot = P.rotate(y[:nh + nkv], cs[p][None])
        q_exp[t] = enc(rot[:nh], xt).reshape(-1)
        for i, v in ((0, rot[nh:]), (1, y[nh + nkv:])):
            if cache == I8:
                exp[i][0][where[0], :, where[1]], exp[i][1][where[0], :, where[1]] = P.quantise(v)
            else:
                exp[i][0][where[0], :, where[1]] = enc(v, cache)
    assert np.array_equal(qo.download(P.np_type(xt)).reshape(q_exp.shape), q_exp)
    for i in range(2):
        c, d = w.download(i)
        assert c.tobytes() == exp[i][0].tobytes()
        if d is not None:
            assert np.array_equal(d, exp[i][1], equal_nan=True)
    w.free()


def test_append_in_place_without_queries_and_without_rotation(ctx):
    w = World(3, [10, 0], [4, 9], 2, 128, BF16, 16).upload(ctx, H)
    x = w.r.standard_normal((w.rows, 10 * 128)).astype(np.float32)
    cs = P.rope_table(w.max_len, 128)
    xb, rb = ctx.upload(x), ctx.upload(cs)
    at = lambda n: type("B", (), {"ptr": xb.ptr + 4 * n})  # noqa: E731
    ctx.paged_append_dev(w.pages, w.batch, F32, 6, xb, 1280, xb, 1280, at(768), 1280, at(1024), 1280, rb, w.max_len)
    got = xb.download().reshape(x.shape)
    for t, (s, p) in enumerate(w.at):
        assert np.array_equal(got[t, :768].reshape(6, 128), P.rotate(x[t, :768].reshape(6, 128), cs[p][None]))
    assert np.array_equal(got[:, 768:], x[:, 768:])
    ctx.paged_append_dev(w.pages, w.batch, F32, 0, None, 0, None, 0, at(768), 1280, at(1024), 1280, None, 0)
    k, _ = w.download(0)
    for t, (s, p) in enumerate(w.at):
        g, o = w.slot(s, p)
        assert np.array_equal(k[g, :, o], P.to_bf16(x[t, 768:1024].reshape(2, 128)))
    w.free()


@pytest.mark.parametrize("hd", [64, 128])
def test_int8_rows_where_rounding_is_hard(ctx, hd):
    """Ties, borders, zeros, the smallest and largest magnitudes, infinities."""
    r = np.random.default_rng(5)
    x = np.zeros((40, hd), np.float32)
    x[1, :9] = [127, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5, 63.5]  # scale 1: ties to even
    x[2] = r.integers(-254, 255, hd) / np.float32(2)
    x[2, 5] = -127
    for i in range(3, 20):  # halves of the scale and their neighbours
        x[i, 0] = np.float32(r.uniform(0.5, 3) * 10.0 ** r.integers(-30, 30))
        d = np.float32(x[i, 0].astype(np.float64) / 127)
        h = (r.integers(-126, 126, hd - 1) + 0.5) * np.float64(d)
        x[i, 1:] = h.astype(np.float32)
        x[i, 1:] = np.nextafter(x[i, 1:], r.choice(np.array([-np.inf, np.inf], np.float32), hd - 1)) if i % 2 else x[i, 1:]
    x[20] = r.standard_normal(hd) * 1e-38
    x[21] = r.standard_normal(hd) * 1e37
    x[22, 3], x[23, 3], x[24, 3] = np.inf, -np.inf, np.nan
    x[25:] = r.standard_normal((15, hd))
    w = World(4, [0], [40], 1, hd, I8, 64).upload(ctx, H)
    xb = ctx.upload(x)
    ctx.paged_append_dev(w.pages, w.batch, F32, 0, None, 0, None, 0, xb, hd, xb, hd, None, 0)
    codes, scale = P.quantise(x)
    for i in range(2):
        c, d = w.download(i)
        g = w.table[0, 0]
        assert np.array_equal(d[g, 0, :40], scale, equal_nan=True)
        bad = np.argwhere(c[g, 0, :40] != codes)
        assert not len(bad), (bad[:4], x[tuple(bad[0])], scale[bad[0][0]])
    out = ctx.alloc(4 * 40 * hd)
    ctx.paged_read_dev(w.pages, w.batch, F32, out, hd, out, hd)
    y = out.download().reshape(40, hd)
    assert np.isnan(y[22:25]).all() and np.array_equal(y[:22], codes[:22] * scale[:22, None])
    w.free()


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_read(ctx, layout, cache, xt):
    nh, nkv, hd, page, hist, new = layout
    w = World(6, hist, new, nkv, hd, cache, page, holes=[(1, 0)], pad=3).upload(ctx, H)
    stride = nkv * hd + 16
    kb, vb = (ctx.upload(np.full((w.rows, stride), 9, P.np_type(xt))) for _ in range(2))
    ctx.paged_read_dev(w.pages, w.batch, xt, kb, stride, vb, stride)
    for i, b in ((0, kb), (1, vb)):
        exp = np.full((w.rows, stride), 9, P.np_type(xt))
        for t, (s, p) in enumerate(w.at):
            where = w.slot(s, p)
            exp[t, :nkv * hd] = 0 if where is None else enc(w.values(i, *where), xt).reshape(-1)
        got = b.download(P.np_type(xt)).reshape(exp.shape)
        assert np.array_equal(dec(got, xt), dec(exp, xt))
    w.free()


def check_attention(w, q, got, rows, xt, prompt):
    """got [rows of the call, heads * hd] against the definition at `rows`"""
    nh, hd = q.shape[1], w.hd
    num = den = 0.0
    for t in rows:
        y, mag, top = w.attention(q[t].astype(np.float64), t)
        tol = (2 * (hd / 4 + 8) * top + 256) * U * mag
        if xt == BF16:
            tol = tol + W * np.abs(y)
            if prompt:
                tol = tol + W * mag
                if w.cache != BF16:
                    tol = tol + (2 * W * top + W) * mag
        off = np.abs(got[t].reshape(nh, hd) - y)
        assert np.isfinite(got[t]).all(), (t, w.at[t])
        assert (off <= tol + 1e-30).all(), (t, w.at[t], float((off - tol).max()), float(off.max()))
        num, den = num + float((off ** 2).sum()), den + float((y ** 2).sum())
    if den:
        assert (num / den) ** 0.5 < (1e-5 if xt == F32 else 4 * W), (num / den) ** 0.5


def attend(ctx, w, nh, xt, entry, seed=8, extra=8, scale=1.5):
    """(q, outputs) of a call over the world's rows; the gaps of out stay as they were"""
    r = np.random.default_rng(seed)
    q = dec(enc(r.standard_normal((w.rows, nh * w.hd)).astype(np.float32) * np.float32(scale), xt), xt)
    stride = nh * w.hd + extra
    qb, ob = rows_buf(ctx, q, xt, stride), ctx.upload(np.full((w.rows, stride), 5, P.np_type(xt)))
    getattr(ctx, entry)(w.pages, w.batch, xt, nh, qb, stride, ob, stride)
    got = ob.download(P.np_type(xt)).reshape(w.rows, stride)
    if extra:
        assert (got[:, -extra:] == 5).all()
    qb.free(), ob.free()
    return q.reshape(w.rows, nh, w.hd), got[:, :nh * w.hd]


DECODES = [
    # heads, KV heads, head_dim, page, lengths (the token's own position included; 0: idle), holes
    (32, 8, 128, 64, [1, 2, 15, 16, 17, 64, 65, 300, 0], []),
    (32, 4, 64, 16, [301], []),
    (8, 8, 128, 32, [33, 128, 129, 31], [(0, 0), (1, 2)]),
    (8, 1, 64, 256, [513, 1, 0, 255], [(3, 0)]),  # a token that sees nothing at all
    (16, 1, 128, 16, [1000, 999], []),
    (6, 2, 128, 128, [4500, 3, 2049], []),
    (28, 4, 64, 64, [700, 5], []),
]


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("case", DECODES)
def test_decode(ctx, case, cache, xt):
    nh, nkv, hd, page, lens, holes = case
    w = World(7, [n - 1 for n in lens], [1] * len(lens), nkv, hd, cache, page, holes=holes, pad=2).upload(ctx, H, with_first=False)
    q, got = attend(ctx, w, nh, xt, "paged_decode_dev")
    check_attention(w, q, dec(got, xt), range(len(lens)), xt, False)
    assert (got[len(lens):] == 5).all()
    w.free()


@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_decode_takes_the_last_token_of_packed_rows(ctx, cache):
    w = World(9, [100, 0, 5, -1], [7, 0, 1, 2], 2, 64, cache, 32, pad=1).upload(ctx, H)
    q, got = attend(ctx, w, 8, F32, "paged_decode_dev")
    check_attention(w, q, got, [6, 7, 9], F32, False)
    assert (got[[0, 1, 2, 3, 4, 5, 8, 10]] == 5).all()
    w.free()


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("n", [8192, 70000])
def test_decode_of_one_long_sequence(ctx, cache, n):
    w = World(10, [n - 1, 130], [1, 1], 2, 128, cache, 128).upload(ctx, H, with_first=False)
    q, got = attend(ctx, w, 8, F32, "paged_decode_dev")
    check_attention(w, q, got, [0, 1], F32, False)
    w.free()


PROMPTS = [
    # heads, KV heads, head_dim, page, positions before, new tokens, holes
    (32, 8, 128, 64, [0, 0, 0], [1, 130, 64], []),
    (32, 4, 64, 16, [301, 165, 77], [77, 51, 7], []),
    (8, 8, 128, 32, [0, 40, -1, 9], [70, 0, 3, 33], []),
    (16, 1, 64, 128, [0, 500], [19, 9], []),
    (6, 2, 128, 256, [0, 1000], [200, 43], []),
    (28, 4, 128, 16, [63, 0], [66, 5], [(0, 1), (1, 0)]),  # the second one's tokens see nothing
    (16, 8, 64, 64, [700], [257], [(0, 3)]),
]


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("case", PROMPTS)
def test_prompt(ctx, case, cache, xt):
    nh, nkv, hd, page, hist, new, holes = case
    w = World(11, hist, new, nkv, hd, cache, page, holes=holes, pad=3).upload(ctx, H)
    q, got = attend(ctx, w, nh, xt, "paged_prompt_dev")
    check_attention(w, q, dec(got, xt), range(len(w.at)), xt, True)
    assert (got[len(w.at):] == 5).all()
    w.free()


@pytest.mark.parametrize("entry", ["paged_decode_dev", "paged_prompt_dev"])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_peaked_and_equal_scores(ctx, entry, cache):
    """Softmaxes that one key takes, and that all share (queries of zeros)."""
    for scale in (30.0, 0.0):
        w = World(12, [600, 20], [1, 1], 2, 128, cache, 32).upload(ctx, H)
        q, got = attend(ctx, w, 8, F32, entry, scale=scale)
        check_attention(w, q, got, [0, 1], F32, entry == "paged_prompt_dev")
        w.free()


def test_positions_past_max_len_do_not_exist(ctx):
    """Device lengths above the host's bound: read up to it, written nowhere."""
    for cache in (F32, BF16, I8):
        w = World(13, [199, 40], [1, 1], 2, 64, cache, 16).upload(ctx, H, with_first=False)
        w.batch.max_len = w.max_len = 100
        q, got = attend(ctx, w, 4, F32, "paged_decode_dev")
        w.at = [(0, 99), (1, 40)]
        check_attention(w, q, got, [0, 1], F32, False)
        x = ctx.upload(np.ones((2, 128), np.float32))
        before = w.download(0)[0]
        ctx.paged_append_dev(w.pages, w.batch, F32, 0, None, 0, None, 0, x, 128, x, 128, None, 0)
        after, (g, o) = w.download(0)[0], w.slot(1, 40)
        after[g, :, o] = before[g, :, o]
        assert after.tobytes() == before.tobytes()
        w.free()


@pytest.mark.parametrize("hd", [64, 128])
def test_paged_run_equals_the_contiguous_cache(ctx, hd):
    """Prompts of two sequences and then decode steps, appended and attended to
    together over pages, against the single-sequence entry points over the fp32
    slab: the same rows bit for bit, attention within the bar of both."""
    nh, nkv, page, hist, steps = 8, 2, 16, [37, 70], 5
    ms = 128
    ctx.kv_init(2, nkv, hd, ms, 500000.0)  # layer s: sequence s
    w = World(14, [0, 0], hist, nkv, hd, F32, page)
    w.table = np.arange(16).reshape(2, 8)[:, ::-1].copy()
    w.n_pages, w.stride = 16, 8
    w.pools = [(np.zeros((16, nkv, page, hd), np.float32), None) for _ in range(2)]
    w.max_len = ms
    r = np.random.default_rng(15)
    rb = ctx.upload(P.rope_table(ms, hd))

    def call(pos, new):
        w.hist, w.new = pos, new
        w.first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        w.rows = int(w.first[-1])
        w.upload(ctx, H)
        x = r.standard_normal((w.rows, (nh + 2 * nkv) * hd)).astype(np.float32)
        xb, qo, out = ctx.upload(x), ctx.alloc(4 * w.rows * nh * hd), ctx.alloc(4 * w.rows * nh * hd)
        at = lambda n: type("B", (), {"ptr": xb.ptr + 4 * n})  # noqa: E731
        width = x.shape[1]
        ctx.paged_append_dev(w.pages, w.batch, F32, nh, xb, width, qo, nh * hd, at(nh * hd), width, at((nh + nkv) * hd), width, rb, ms)
        (ctx.paged_decode_dev if new == [1, 1] else ctx.paged_prompt_dev)(w.pages, w.batch, F32, nh, qo, nh * hd, out, nh * hd)
        got, q = out.download().reshape(w.rows, -1), qo.download().reshape(w.rows, -1)
        w.pools = [w.download(0), w.download(1)]
        kb, vb = ctx.alloc(4 * w.rows * nkv * hd), ctx.alloc(4 * w.rows * nkv * hd)
        ctx.paged_read_dev(w.pages, w.batch, F32, kb, nkv * hd, vb, nkv * hd)
        back = kb.download().reshape(w.rows, nkv, hd)
        w.free()
        for s in range(2):
            a, b = w.first[s], w.first[s + 1]
            qs, ks, vs = (np.ascontiguousarray(m) for m in (q[a:b], back[a:b], x[a:b, (nh + nkv) * hd:]))
            for i in range(b - a):
                assert ctx.kv_append(s, pos[s] + i, ks[i], vs[i]) == 0
                ob = ctx.alloc(4 * nh * hd)
                assert ctx.attention_dev(s, pos[s] + i, nh, ctx.upload(qs[i]), ob) == 0
                ref = ob.download()
                assert np.linalg.norm(got[a + i] - ref) < 1e-5 * np.linalg.norm(ref)

    call([0, 0], hist)
    for i in range(steps):
        call([h + i for h in hist], [1, 1])


@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("entry", ["paged_decode_dev", "paged_prompt_dev"])
def test_repeated_calls_give_the_same_bits(ctx, entry, cache):
    w = World(16, [3000, 900, 77], [1, 3, 40] if entry == "paged_prompt_dev" else [1, 1, 1], 4, 128, cache, 64).upload(ctx, H)
    a = attend(ctx, w, 16, BF16, entry)[1]
    for _ in range(3):
        assert np.array_equal(attend(ctx, w, 16, BF16, entry)[1], a)
    w.free()


def test_empty_batches(ctx):
    w = World(17, [0, 0], [0, 0], 2, 64, F32, 16, pad=2).upload(ctx, H)
    for entry in ("paged_decode_dev", "paged_prompt_dev"):
        assert (attend(ctx, w, 4, F32, entry)[1] == 5).all()
    w.batch.n_seqs = 0
    assert (attend(ctx, w, 4, F32, "paged_decode_dev")[1] == 5).all()
    w.free()


@pytest.mark.parametrize("pos", [2 ** 31 - 1, 2 ** 31 - 3, 1 << 30])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_positions_near_the_end_of_int32(ctx, cache, pos):
    """Device positions whose sum with a token's number passes 31 bits: past
    max_len all the same."""
    w = World(18, [93, 40], [7, 3], 2, 64, cache, 16)
    w.hist[0] = pos
    w.upload(ctx, H)
    w.at = [(0, 99)] * 7 + [(1, 40 + i) for i in range(3)]
    for entry, rows in (("paged_decode_dev", [6, 9]), ("paged_prompt_dev", range(10))):
        q, got = attend(ctx, w, 4, F32, entry)
        check_attention(w, q, got, rows, F32, entry == "paged_prompt_dev")
    x = ctx.upload(np.ones((10, 128), np.float32))
    before = w.download(0)[0]
    ctx.paged_append_dev(w.pages, w.batch, F32, 0, None, 0, None, 0, x, 128, x, 128, None, 0)
    after = w.download(0)[0]
    for i in range(3):
        g, o = w.slot(1, 40 + i)
        after[g, :, o] = before[g, :, o]
    assert after.tobytes() == before.tobytes()
    ctx.paged_read_dev(w.pages, w.batch, F32, x, 128, x, 128)
    assert (x.download().reshape(10, 128)[:7] == 0).all()
    w.free()


ODD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("case", [(8, 2, 64, 16, [5, 0], [90, 40]), (16, 8, 128, 64, [70, 1], [150, 3]), (12, 1, 128, 32, [0, 300], [33, 130]),
                                  (4, 4, 64, 128, [1000, 0], [300, 64])])
def test_values_that_are_no_numbers_stay_in_their_future(ctx, case, cache, xt):
    """K and V rows with an infinity or NaN at one of a prompt's own positions:
    the tokens before it are as if they were not there, bit for bit, those from
    it on are no numbers in V's dimensions (in all of them for K's and for a row
    of int8 codes, whose scale is NaN then)."""
    nh, nkv, hd, page, hist, new = case
    clean = World(21, hist, new, nkv, hd, cache, page, pad=1).upload(ctx, H)
    q, ref = attend(ctx, clean, nh, xt, "paged_prompt_dev")
    clean.free()
    for which in (0, 1):
        for n, t in enumerate([0, 1, new[0] // 2, new[0] - 1]):
            w = World(21, hist, new, nkv, hd, cache, page, pad=1)
            g, o = w.slot(0, hist[0] + t)
            head, dim, v = n % nkv, (37 * n + 5) % hd, np.float32(ODD[n % 3])
            if cache == I8:
                w.pools[which][1][g, head, o] = np.nan
            else:
                w.pools[which][0][g, head, o, dim] = enc(np.array([v]), cache)[0]
            w.upload(ctx, H)
            got = attend(ctx, w, nh, xt, "paged_prompt_dev")[1]
            w.free()
            a, b = dec(got, xt).reshape(-1, nh, hd), dec(ref, xt).reshape(-1, nh, hd)
            G = nh // nkv
            hit = np.zeros(a.shape, bool)
            if cache == I8:
                hit[t:new[0], head * G:(head + 1) * G] = True
            else:
                hit[t:new[0], head * G:(head + 1) * G, dim if which else slice(None)] = True
            assert np.array_equal(a[~hit], b[~hit]), (which, t)
            if which or cache == I8 or np.isnan(v):  # an infinite score may also weigh nothing
                assert not np.isfinite(a[hit]).any(), (which, t)


def some_rows(w, n=40, seed=30):
    """the first and last token of a few sequences, and others"""
    r = np.random.default_rng(seed)
    ends = [t for s in r.permutation(len(w.new))[:8] if w.new[s] for t in (w.first[s], w.first[s + 1] - 1)]
    return sorted({*ends, *r.integers(0, len(w.at), n)})


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_prompts_of_many_sequences(ctx, cache, xt):
    """150 sequences, more than a wave looks through at once, longest first."""
    r = np.random.default_rng(31)
    hist, new = r.integers(-1, 200, 150), r.integers(0, 40, 150)
    w = World(32, hist.tolist(), new.tolist(), 2, 64, cache, 16, pad=5).upload(ctx, H)
    q, got = attend(ctx, w, 8, xt, "paged_prompt_dev")
    check_attention(w, q, dec(got, xt), some_rows(w), xt, True)
    idle = [t for t, (s, p) in enumerate(w.at) if p < 0]
    assert idle and not dec(got[idle], xt).any() and (got[len(w.at):] == 5).all()
    w.free()


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("hist,new", [([9000], [1]), ([7001, 30, 0], [5, 130, 1]), ([500], [2000]), ([0, 0, 100], [1500, 1, 999])])
def test_prompts_in_parts_and_in_large_tiles(ctx, hist, new, cache, xt):
    """Few tokens over many keys, whose parts are joined, beside sequences of
    fewer parts; and enough of them for the larger tiles."""
    w = World(33, hist, new, 4, 128, cache, 64, pad=2).upload(ctx, H)
    q, got = attend(ctx, w, 16, xt, "paged_prompt_dev")
    check_attention(w, q, dec(got, xt), some_rows(w, 12), xt, True)
    again = attend(ctx, w, 16, xt, "paged_prompt_dev")[1]
    assert np.array_equal(got, again) and (got[len(w.at):] == 5).all()
    w.free()
