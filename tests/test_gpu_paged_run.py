"""Generation for a batch as a server runs it: three sequences' prompts
appended, attended to and sampled from, then one token of each a step, against
the same in float64 on the host.  Attention is within 1e-5 of the definition, a
logit (|x| < 10) within 1e-4 then and a weight at temperature 0.8 within 1.3e-4
of itself: the sum of 20 kept ones moves by less than 3e-3 of the largest, and
the draws lie 1e-2 from the next border."""
import numpy as np
import pytest

import guanaco_amd.hip as H
import paged as P
from paged import BF16, F32, World
from test_gpu_sample_rows import reference


VOCAB, NH, NKV, HD, PAGE, MAX = 97, 4, 2, 64, 16, 64
PARAMS = (np.float32(0.8), 20, np.float32(0.9), np.float32(0.01))


def model(seed):
    r = np.random.default_rng(seed)
    rows = r.standard_normal((VOCAB, (NH + 2 * NKV) * HD)).astype(np.float32)
    head = (r.standard_normal((NH * HD, VOCAB)) * 0.25).astype(np.float32)
    prompts = [list(r.integers(0, VOCAB, n)) for n in (21, 1, 34)]
    return rows, head, prompts, r.random((4, 3)).astype(np.float32)


def by_definition(seed, cache):
    """tokens drawn in every step, and the nearest border to any draw"""
    rows, head, seqs, u = model(seed)
    seqs = [list(s) for s in seqs]
    rope, drawn, near = P.rope_table(MAX, HD), [], 1.0
    for step in u:
        new = []
        for s, seq in enumerate(seqs):
            x = rows[seq]
            cs = rope[:len(seq), None]
            q = P.rotate(x[-1, :NH * HD].reshape(NH, HD), cs[-1]).astype(np.float64)
            k = P.rotate(x[:, NH * HD:(NH + NKV) * HD].reshape(-1, NKV, HD), cs)
            v = x[:, (NH + NKV) * HD:].reshape(-1, NKV, HD)
            k, v = (P.dec(P.enc(a, cache), cache).astype(np.float64) for a in (k, v))
            out = np.empty((NH, HD))
            for h in range(NH):
                z = k[:, h * NKV // NH] @ q[h] / 8
                w = np.exp(z - z.max())
                out[h] = w @ v[:, h * NKV // NH] / w.sum()
            t, _, far = reference((out.ravel() @ head.astype(np.float64)).astype(np.float32), *PARAMS, step[s])
            near = min(near, far)
            new.append(t)
        for seq, t in zip(seqs, new):
            seq.append(t)
        drawn.append(new)
    return drawn, near


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [F32, BF16])
def test_generation(ctx, cache, seed=19):
    want, near = by_definition(seed, cache)
    assert near > 1e-2
    rows, head, seqs, u = model(seed)
    w = World(1, [0, 0, 0], [1, 1, 1], NKV, HD, cache, PAGE)
    w.n_pages, w.stride, w.max_len = 12, 4, MAX
    w.table = np.random.default_rng(seed).permutation(12).reshape(3, 4)
    w.pools = [(np.full((12, NKV, PAGE, HD), P.enc(np.float32([np.nan]), cache)[0]), None) for _ in range(2)]
    rope = ctx.upload(P.rope_table(MAX, HD))
    f = [ctx.upload(np.full(3, v)) for v in (PARAMS[0], np.int32(PARAMS[1]), PARAMS[2], PARAMS[3])]
    new, pos = [list(s) for s in seqs], [0, 0, 0]
    for step, draws in zip(u, want):
        w.hist, w.new = pos, [len(n) for n in new]
        w.first = np.concatenate([[0], np.cumsum(w.new)]).astype(np.int32)
        w.rows = int(w.first[-1])
        w.upload(ctx, H)
        x = rows[np.concatenate(new)]
        width, n = x.shape[1], len(x)
        xb, out = ctx.upload(x), ctx.alloc(4 * n * NH * HD)
        at = lambda c: type("B", (), {"ptr": xb.ptr + 4 * c})  # noqa: E731
        ctx.paged_append_dev(w.pages, w.batch, F32, NH, xb, width, xb, width, at(NH * HD), width, at((NH + NKV) * HD), width, rope, MAX)
        (ctx.paged_decode_dev if n == 3 else ctx.paged_prompt_dev)(w.pages, w.batch, F32, NH, xb, width, out, NH * HD)
        o = out.download().reshape(n, -1)[w.first[1:] - 1].astype(np.float64)
        lb, ub, tb = ctx.upload((o @ head.astype(np.float64)).astype(np.float32)), ctx.upload(step), ctx.alloc(12)
        ctx.sample_rows_dev(lb, 3, VOCAB, VOCAB, *f, ub, tb)
        got = tb.download(np.int32)
        assert list(got) == draws
        w.pools = [w.download(0), w.download(1)]
        for b in (xb, out, lb, ub, tb):
            b.free()
        w.free()
        pos, new = [p + len(s) for p, s in zip(pos, new)], [[t] for t in got]
    rope.free()
