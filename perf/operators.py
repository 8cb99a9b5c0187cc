"""Serving several sequences at once, as measurable cases: a paged K/V cache
(written, read back and attended to) and sampling for a batch.

A case is one call of a public entry point (include/gq_hip.h as guanaco_amd.hip
exposes it), or the two calls that write new rows and read them back.  `run`
computes it in plain torch operations, or through the framework where `own` is
set; `exact` evaluates the definition in float64.  Inputs are made on the GPU
from a seed.

Head layouts and vocabularies are those of guanaco_amd.spec's 8B and 1.1B
shapes (32 over 8 heads of 128, 32 over 4 of 64; 128256 and 32000 tokens), and
of other Llama-family models in the drawn cases.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
THETA = 500000.0
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}


# -------------------------------------------------------------------- cases
def listed():
    h8b, h1b = dict(heads=32, kv_heads=8, hd=128), dict(heads=32, kv_heads=4, hd=64)
    return [
        # one new token for each of 32 conversations goes into an int8 cache: a decode step's append
        dict(name="append_step_i8", kind="append", **h8b, cache="i8", x="f32", page=64, seqs=32, new=1, hist=4000, mix=1),
        # a batch of prompts of different lengths goes into a bf16 cache
        dict(name="append_prompts_bf16", kind="append", **h8b, cache="bf16", x="bf16", page=64, seqs=7, new=2048, hist=0, mix=2),
        # a long conversation's rows are read back (to be saved, or moved to a contiguous cache)
        dict(name="read_long_i8", kind="read", **h8b, cache="i8", x="f32", page=64, seqs=1, len=32000, mix=3),
        # one short chat of the 1.1B model on an fp32 cache: the smallest decode there is
        dict(name="decode_1b_f32", kind="decode", **h1b, cache="f32", x="f32", page=16, seqs=1, len=301, idle=0, mix=4),
        # 64 conversations of the 8B model, up to 8192 positions each, two slots idle
        dict(name="decode_8b_64", kind="decode", **h8b, cache="bf16", x="f32", page=64, seqs=64, len=8192, idle=2, mix=5),
        # one conversation over a very long int8 cache: the split over its length
        dict(name="decode_long_i8", kind="decode", **h8b, cache="i8", x="bf16", page=128, seqs=1, len=131072, idle=0, mix=6),
        # three short turns of the 1.1B model in the framework's own precision, fp32 throughout
        dict(name="prompt_turns_f32", kind="prompt", **h1b, cache="f32", x="f32", page=16, seqs=3, new=77, hist=301, pad=3, mix=7),
        # fresh prompts of different lengths, 8B heads, bf16
        dict(name="prompt_8b_bf16", kind="prompt", **h8b, cache="bf16", x="bf16", page=64, seqs=4, new=4096, hist=0, pad=0, mix=8),
        # chunks of 512 tokens of prompts that have got a long way already, over an int8 cache
        dict(name="prompt_chunks_i8", kind="prompt", **h8b, cache="i8", x="bf16", page=64, seqs=4, new=512, hist=7500, pad=0, mix=9),
        # fp32 queries of a whole prompt over a bf16 cache
        dict(name="prompt_f32_over_bf16", kind="prompt", **h8b, cache="bf16", x="f32", page=32, seqs=2, new=1500, hist=600, pad=5, mix=10),
        # one conversation's next token from the 8B vocabulary, every filter on
        dict(name="sample_one", kind="sample", vocab=128256, rows=1, mode="all", mix=11),
        # a batch's next tokens, each row with parameters of its own
        dict(name="sample_128", kind="sample", vocab=128256, rows=128, mode="mixed", mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt", "sample"])
    mix = rng.randrange(1, 1 << 20)
    if kind == "sample":
        return dict(kind=kind, vocab=_log(rng, 1000, 131072), rows=_log(rng, 1, 128),
                    mode=rng.choice(["all", "mixed", "mixed", "top_p", "temperature"]), mix=mix)
    hd, group = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    kv = rng.choice([1, 2, 4, 8] if group > 1 else [4, 8, 16])
    c = dict(kind=kind, heads=kv * group, kv_heads=kv, hd=hd, cache=rng.choice(["f32", "bf16", "i8"]),
             x=rng.choice(["f32", "bf16"]), page=rng.choice([16, 32, 64, 128, 256]), mix=mix)
    if c["heads"] > 64:
        c["kv_heads"], c["heads"] = 4, 4 * group
    if kind == "append":
        c["seqs"] = _log(rng, 1, 64)
        return dict(c, new=_log(rng, 1, min(2048, 8192 // c["seqs"])), hist=rng.choice([0, _log(rng, 1, 6000)]))
    if kind == "read":
        c["seqs"] = _log(rng, 1, 16)
        return dict(c, len=_log(rng, 1, 32000 // c["seqs"]))
    if kind == "decode":
        c["seqs"] = _log(rng, 1, 128)
        return dict(c, len=_log(rng, 1, min(65536, 262144 // c["seqs"])), idle=rng.choice([0, 0, 1]) if c["seqs"] > 1 else 0)
    c["seqs"] = _log(rng, 1, 12)
    new, hist = _log(rng, 1, min(2500, 5000 // c["seqs"])), rng.choice([0, _log(rng, 1, 4000)])
    while c["seqs"] * new * (hist + new) * c["heads"] > 4e8:  # no more than the largest listed one costs
        new, hist = new * 2 // 3, hist * 2 // 3
    return dict(c, new=new, hist=hist, pad=rng.choice([0, 0, 3]))


def lens(case):
    """(positions there before, new tokens) of each sequence: the first has the
    most of both, the others less; an idle slot has -1 positions."""
    r, n = random.Random(case["mix"]), case["seqs"]
    if case["kind"] == "read":
        return [0] * n, [case["len"]] + [r.randint(1, case["len"]) for _ in range(n - 1)]
    if case["kind"] == "decode":
        hist = [case["len"] - 1] + [r.randrange(case["len"]) for _ in range(n - 1)]
        for i in range(case["idle"]):
            hist[n - 1 - 2 * i] = -1
        return hist, [1] * n
    hist = [case["hist"]] + [r.randrange(case["hist"] + 1) for _ in range(n - 1)]
    return hist, [case["new"]] + [r.randint(1, case["new"]) for _ in range(n - 1)]


# ------------------------------------------------------------------- inputs
def _gen(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + int(tag) * 7919 + 12345) % (1 << 62))
    return g


def _normal(shape, seed, tag, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed, tag), device=DEV) * scale).to(dtype)


def _pool(case, n_pages, seed, tag):
    """A pool of pages with rows everywhere, stale ones where no sequence is:
    N(0, 1) values; int8 rows with a scale each."""
    shape = (n_pages, case["kv_heads"], case["page"], case["hd"])
    if case["cache"] != "i8":
        return _normal(shape, seed, tag, TORCH[case["cache"]]), None
    codes = _normal(shape, seed, tag, scale=45.0).round().clamp(-127, 127).to(torch.int8)
    return codes, (0.5 + torch.rand(shape[:3], generator=_gen(seed, tag + 1), device=DEV)) / 45.0


def _rope_table(n, hd):
    """(cos, sin) of positions 0 .. n - 1: angles of the framework's fp32 frequencies"""
    f = (1.0 / THETA ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)).float()
    a = torch.arange(n, device=DEV, dtype=torch.float32)[:, None] * f[None]
    return torch.stack([a.double().cos(), a.double().sin()], -1).float().contiguous()


class Buf:
    """A torch tensor as the methods of guanaco_amd.hip take a buffer."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


class State:
    pass


def _sampling(case, seed):
    """(temperature, top_k, top_p, min_p) of each row"""
    r, n = random.Random(case["mix"] * 7 + 1), case["rows"]
    kinds = {"all": [(0.7, 40, 0.95, 0.05)], "top_p": [(1.0, 0, 0.9, 0.0)], "temperature": [(0.8, 0, 1.0, 0.0)],
             "mixed": [(0.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 0, 1.0, 0.1), (1.2, 200, 0.98, 0.02),
                       (0.6, 0, 0.95, 0.05), (1.0, 0, 1.0, 0.0)]}[case["mode"]]
    rows = [kinds[0] if len(kinds) == 1 else r.choice(kinds) for _ in range(n)]
    return [list(v) for v in zip(*rows)]


def prepare(case, seed):
    st = State()
    st.case, st.plan = case, None
    if case["kind"] == "sample":
        n, vocab = case["rows"], case["vocab"]
        # logits as a language model's: a broad body and a few likely tokens
        x = _normal((n, vocab), seed, 1, scale=2.2)
        top = torch.randint(0, vocab, (n, max(4, vocab // 2000)), generator=_gen(seed, 2), device=DEV)
        x.scatter_add_(1, top, 4.0 + 3.0 * torch.rand(top.shape, generator=_gen(seed, 3), device=DEV))
        st.logits = x
        t, k, p, m = _sampling(case, seed)
        f = lambda v: torch.tensor(v, device=DEV, dtype=torch.float32)  # noqa: E731
        st.temperature, st.top_p, st.min_p = f(t), f(p), f(m)
        st.top_k = torch.tensor(k, device=DEV, dtype=torch.int32)
        st.rnd = torch.rand((n,), generator=_gen(seed, 4), device=DEV)
        st.tokens = torch.zeros(n, device=DEV, dtype=torch.int32)
        st.logprobs = torch.zeros(n, device=DEV)
        return st
    hist, new = lens(case)
    nh, nkv, hd, ps = case["heads"], case["kv_heads"], case["hd"], case["page"]
    need = [-(-max(0, h + n) // ps) if h >= 0 else 0 for h, n in zip(hist, new)]
    st.stride, st.n_pages = max(need) + 1, sum(need) + 3
    order = torch.randperm(st.n_pages, generator=_gen(seed, 9), device=DEV).tolist()
    table = np.full((case["seqs"], st.stride), -1, np.int32)
    for s, n in enumerate(need):  # pages of one sequence lie anywhere in the pool
        for i in range(n):
            table[s, i] = order.pop()
    st.table = torch.from_numpy(table).to(DEV)
    st.k, st.ks = _pool(case, st.n_pages, seed, 10)
    st.v, st.vs = _pool(case, st.n_pages, seed, 12)
    st.pos = torch.tensor(hist, device=DEV, dtype=torch.int32)
    firsts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    st.n, st.max_len = int(firsts[-1]) + case.get("pad", 0), max(h + n for h, n in zip(hist, new))
    st.first = torch.from_numpy(firsts).to(DEV)
    # packed row, sequence and position of every new token
    st.seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
    st.at = torch.arange(len(st.seq), device=DEV) - st.first[:-1].long()[st.seq]
    x = TORCH[case["x"]]
    if case["kind"] == "append":  # q | k | v rows as one projection leaves them
        st.qkv = _normal((st.n, (nh + 2 * nkv) * hd), seed, 14, x)
        st.rope = _rope_table(st.max_len, hd)
    if case["kind"] in ("decode", "prompt"):
        st.q = _normal((st.n, nh * hd), seed, 14, x, 1.5)
        st.out = torch.zeros((st.n, nh * hd), device=DEV, dtype=x)
    else:
        st.q = torch.zeros((st.n, nh * hd), device=DEV, dtype=x)
        st.k_rows, st.v_rows = (torch.zeros((st.n, nkv * hd), device=DEV, dtype=x) for _ in range(2))
    return st


# ------------------------------------------------------------ the plain forms
def _values(pool, scale):
    return pool.float() if scale is None else pool.float() * scale[..., None]


def _plain_append(st):
    c = st.case
    nh, nkv, hd, ps = c["heads"], c["kv_heads"], c["hd"], c["page"]
    x = st.qkv.float().view(st.n, nh + 2 * nkv, hd)
    pos = st.pos.long()[st.seq] + st.at
    cs = st.rope[pos][:, None]
    e, o = x[:, :nh + nkv, 0::2], x[:, :nh + nkv, 1::2]
    r = torch.stack([e * cs[..., 0] - o * cs[..., 1], e * cs[..., 1] + o * cs[..., 0]], -1).reshape(st.n, nh + nkv, hd)
    page, slot = st.table.long()[st.seq, pos // ps], pos % ps
    rows = []
    for pool, scale, y in ((st.k, st.ks, r[:, nh:]), (st.v, st.vs, x[:, nh + nkv:])):
        if scale is None:
            pool[page, :, slot] = y.to(pool.dtype)
        else:
            d = y.abs().amax(-1) / 127.0
            code = torch.where(d[..., None] > 0, torch.round(y.double() / d.double()[..., None]), 0.0)
            pool[page, :, slot], scale[page, :, slot] = code.to(torch.int8), d
        rows.append(_plain_read(st, pool, scale, page, slot))
    return {"q": r[:, :nh].reshape(st.n, nh * hd).to(st.q.dtype), "k": rows[0], "v": rows[1]}


def _plain_read(st, pool, scale, page, slot):
    v = _values(pool[page, :, slot], None if scale is None else scale[page, :, slot])
    return v.reshape(len(page), -1).to(st.q.dtype)


def _plain_attention(st):
    c = st.case
    n, nh, nkv, hd, ps = c["seqs"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    g, T = nh // nkv, max(lens(c)[1])
    P = -(-st.max_len // ps)
    t = st.table[:, :P].long().clamp(min=0)
    q = torch.zeros((n, T, nkv, g, hd), device=DEV)
    m = len(st.seq)
    q[st.seq, st.at] = st.q[:m].float().view(m, nkv, g, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n * nkv, g * T, hd)
    rows = lambda pool, scale: _values(pool[t], None if scale is None else scale[t]).permute(0, 2, 1, 3, 4).reshape(n * nkv, P * ps, hd)  # noqa: E731
    s = torch.bmm(q, rows(st.k, st.ks).transpose(1, 2).contiguous()).view(n, nkv, g, T, P * ps)
    s *= 1.0 / math.sqrt(hd)
    last = st.pos.long()[:, None] + torch.arange(T, device=DEV)  # the last position that a token sees
    seen = torch.arange(P * ps, device=DEV) <= last[..., None]
    seen &= (st.pos >= 0)[:, None, None]
    seen = seen[:, None, None]
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    z = s.sum(-1, keepdim=True)
    o = torch.bmm(s.view(n * nkv, g * T, P * ps), rows(st.v, st.vs)).view(n, nkv, g, T, hd)
    o = torch.where(z > 0, o / z, 0.0).permute(0, 3, 1, 2, 4).reshape(n, T, nh * hd)
    out = st.out.clone()
    out[:m] = o[st.seq, st.at].to(out.dtype)
    return out


def _plain_sample(st):
    x, n, vocab = st.logits.double(), st.case["rows"], st.case["vocab"]
    T = st.temperature.double()[:, None]
    greedy = T <= 0
    top = x.amax(1, keepdim=True)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    w = torch.exp((x - top) / torch.where(greedy, 1.0, T))
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=DEV)[None]
    k = st.top_k.long()[:, None]
    ws = torch.where((k <= 0) | (rank < k), ws, 0.0)
    cum = ws.cumsum(1)
    p = st.top_p.double()[:, None]
    keep = (ws > 0) & ((p >= 1) | (cum - ws < p * cum[:, -1:])) & (ws >= st.min_p.double()[:, None])
    keep = torch.where(greedy, rank == 0, keep | (rank == 0))
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    mass = torch.where(kept, w, 0.0).cumsum(1)
    token = (mass > st.rnd.double()[:, None] * mass[:, -1:]).int().argmax(1)
    logp = torch.log(w.gather(1, token[:, None]) / mass[:, -1:])[:, 0]
    return {"tokens": token.int(), "logprobs": logp.float()}


# --------------------------------------------------------- the framework's own
_shared = []


def _ctx():
    """One context for all states, as one program has one: its calls run in
    order on one stream."""
    import guanaco_amd.hip as H
    if not _shared:
        _shared.append(H.Context(0))
    return _shared[0]


def _ready():
    """The context's stream waits for no other: what torch has been given to
    write is there before a state's first call."""
    torch.cuda.synchronize()


def _plan(st):
    """The descriptions of the cache and the batch that a program keeps."""
    _ready()
    import guanaco_amd.hip as H
    c = st.case
    code = {"f32": H.S.F32, "bf16": H.BF16, "i8": H.I8_ROWS}
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    pages = H.GqPages(ptr(st.k), ptr(st.v), ptr(st.ks), ptr(st.vs), code[c["cache"]], st.n_pages, c["page"], c["kv_heads"], c["hd"])
    batch = H.GqBatch(ptr(st.table), ptr(st.pos), None if c["kind"] == "decode" else ptr(st.first), c["seqs"], st.stride, st.n, st.max_len)
    return _ctx(), pages, batch, code[c["x"]]


def _own(st):
    c = st.case
    if c["kind"] == "sample":
        if not st.plan:
            _ready()
            st.plan = [Buf(t) for t in (st.logits, st.temperature, st.top_k, st.top_p, st.min_p, st.rnd, st.tokens, st.logprobs)]
        b = st.plan
        _ctx().sample_rows_dev(b[0], c["rows"], c["vocab"], c["vocab"], *b[1:])
        return {"tokens": st.tokens, "logprobs": st.logprobs}
    ctx, pages, batch, x = st.plan = st.plan or _plan(st)
    nh, nkv, hd = c["heads"], c["kv_heads"], c["hd"]
    if c["kind"] == "decode":
        ctx.paged_decode_dev(pages, batch, x, nh, Buf(st.q), nh * hd, Buf(st.out), nh * hd)
        return st.out
    if c["kind"] == "prompt":
        ctx.paged_prompt_dev(pages, batch, x, nh, Buf(st.q), nh * hd, Buf(st.out), nh * hd)
        return st.out
    if c["kind"] == "append":
        row = (nh + 2 * nkv) * hd
        ctx.paged_append_dev(pages, batch, x, nh, Buf(st.qkv), row, Buf(st.q), nh * hd, Buf(st.qkv[:, nh * hd:]), row,
                             Buf(st.qkv[:, (nh + nkv) * hd:]), row, Buf(st.rope), st.max_len)
    ctx.paged_read_dev(pages, batch, x, Buf(st.k_rows), nkv * hd, Buf(st.v_rows), nkv * hd)
    return {"q": st.q, "k": st.k_rows, "v": st.v_rows} if c["kind"] == "append" else {"k": st.k_rows, "v": st.v_rows}


def run(st):
    """One pass.  With `own` it runs on the context's stream: synchronise the
    device before the outputs are read or the state is dropped or written to."""
    if own:
        return _own(st)
    kind = st.case["kind"]
    if kind == "sample":
        return _plain_sample(st)
    if kind == "append":
        return _plain_append(st)
    if kind == "read":
        page, slot = st.table.long()[st.seq, st.at // st.case["page"]], st.at % st.case["page"]
        return {"k": _plain_read(st, st.k, st.ks, page, slot), "v": _plain_read(st, st.v, st.vs, page, slot)}
    return _plain_attention(st)


# ----------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": case["rows"] * case["vocab"]}
    hist, new = lens(case)
    nh, nkv, hd = case["heads"], case["kv_heads"], case["hd"]
    xb = {"f32": 4, "bf16": 2}[case["x"]]
    row = 2 * nkv * (hd * {"f32": 4, "bf16": 2, "i8": 1}[case["cache"]] + (4 if case["cache"] == "i8" else 0))
    n = sum(new)
    if case["kind"] == "append":  # in, rotated and written, and the rows once more on their way back
        return {"bytes": n * (xb * hd * (2 * nh + 4 * nkv) + 2 * row) + 4 * hd * n, "flops": 6 * n * hd * (nh + 2 * nkv)}
    if case["kind"] == "read":
        return {"bytes": n * (row + 2 * xb * hd * nkv), "flops": 2 * n * hd * nkv}
    there = [(h, m) for h, m in zip(hist, new) if h >= 0]
    pairs = sum(m * h + m * (m + 1) // 2 for h, m in there)
    return {"bytes": sum(h + m for h, m in there) * row + 2 * xb * n * nh * hd, "flops": 4 * hd * nh * pairs}


# ---------------------------------------------------------------------- exact
def _exact_rows(st, s, pool, scale, n):
    """Positions 0 .. n - 1 of sequence s in float64: kv_heads x n x hd"""
    at = torch.arange(n, device=DEV)
    page, slot = st.table[s].long()[at // st.case["page"]], at % st.case["page"]
    v = pool[page, :, slot].double()
    return (v if scale is None else v * scale[page, :, slot].double()[..., None]).transpose(0, 1).contiguous()


def _exact_attention(st, hist, new):
    c = st.case
    nh, nkv, hd = c["heads"], c["kv_heads"], c["hd"]
    out, r = torch.zeros((st.n, nh, hd), device=DEV, dtype=torch.float64), 0
    for s, (h, m) in enumerate(zip(hist, new)):
        if h >= 0:
            k, v = (_exact_rows(st, s, p, d, h + m) for p, d in ((st.k, st.ks), (st.v, st.vs)))
            hidden = torch.arange(h + m, device=DEV)[None] > h + torch.arange(m, device=DEV)[:, None]
            for a in range(nh):
                q = st.q[r:r + m, a * hd:(a + 1) * hd].double()
                z = (q @ k[a * nkv // nh].T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[r:r + m, a] = torch.softmax(z, 1) @ v[a * nkv // nh]
        r += m
    return out.view(st.n, nh * hd)


def _exact_append(st):
    """Rotated rows are fp32, each product rounded and then their sum or
    difference; an int8 row's scale is fp32."""
    c = st.case
    nh, nkv, hd = c["heads"], c["kv_heads"], c["hd"]
    f32 = lambda t: t.float().double()  # noqa: E731
    x = st.qkv.double()
    cs = st.rope.double()[st.pos.long()[st.seq] + st.at]
    cos, sin = (cs[..., i].repeat(1, nh + nkv) for i in (0, 1))
    a, b = x[:, :(nh + nkv) * hd:2], x[:, 1:(nh + nkv) * hd:2]
    y = torch.empty((st.n, (nh + nkv) * hd), device=DEV, dtype=torch.float64)
    y[:, 0::2], y[:, 1::2] = f32(f32(a * cos) - f32(b * sin)), f32(f32(a * sin) + f32(b * cos))

    def held(v):
        if c["cache"] != "i8":
            return v.to(TORCH[c["cache"]]).double()
        v = v.reshape(st.n, nkv, hd)
        d = f32(v.abs().max(-1, keepdim=True).values / 127)
        return (torch.round(v / torch.where(d > 0, d, 1.0)) * d).reshape(st.n, nkv * hd)

    return {"q": y[:, :nh * hd], "k": held(y[:, nh * hd:]), "v": held(x[:, (nh + nkv) * hd:])}


def _exact_logprobs(st):
    x, out = st.logits.double().cpu().numpy(), []
    par = [t.double().cpu().numpy() for t in (st.temperature, st.top_k, st.top_p, st.min_p, st.rnd)]
    for i in range(len(x)):
        T, k, p, m, u = (v[i] for v in par)
        if T <= 0:
            out.append(0.0)
            continue
        order = np.argsort(-x[i], kind="stable")
        order = order[:int(k)] if k > 0 else order
        w = np.exp((x[i][order] - x[i][order[0]]) / T)
        if p < 1:
            cut = int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1
            order, w = order[:cut], w[:cut]
        order, w = order[w >= m], w[w >= m]
        by = np.argsort(order)
        c = np.cumsum(w[by])
        out.append(math.log(w[by][min(int(np.searchsorted(c, u * c[-1], side="right")), len(c) - 1)] / c[-1]))
    return torch.tensor(out, dtype=torch.float64)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "sample":
        return {"tokens": None, "logprobs": _exact_logprobs(st)}
    hist, new = lens(case)
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "read":
        rows = lambda p, d: torch.cat([_exact_rows(st, s, p, d, n).transpose(0, 1).reshape(n, -1) for s, n in enumerate(new)])  # noqa: E731
        return {"k": rows(st.k, st.ks), "v": rows(st.v, st.vs)}
    return _exact_attention(st, hist, new)
