"""Sizes at the ends of what the paged entry points take, on the CPU
(tests/test_paged_host.py's stand-in for the context and HIP)."""
import pytest

from test_paged_host import A, BF16, F32, I8, append, batch, decode, lib, pages, prompt, read, sample  # noqa: F401

BIG = dict(table_stride=1 << 20)


def one_head(**kw):
    return pages(dtype=BF16, n_kv_heads=1, head_dim=64, page_size=1024, **kw)


@pytest.mark.parametrize("call,p,fits,past,kw", [
    # 16 rows of 64 values a wave: 2^22 waves less one workgroup's, and all
    (append, one_head(), batch(n_tokens=(1 << 29) - 32), batch(n_tokens=1 << 29), dict(q=None, qo=None, rope=None)),
    (read, one_head(), batch(n_tokens=(1 << 29) - 32), batch(n_tokens=1 << 29), {}),
    # a workgroup a sequence and KV head (one part each), 2^24 of them are too many
    (decode, pages(), batch(n_seqs=(1 << 21) - 1, n_tokens=1 << 21, max_len=64), batch(n_seqs=1 << 21, n_tokens=1 << 21, max_len=64), {}),
    # 512 threads a tile of 256 / 16 tokens, and a tile more for the sequence
    (prompt, one_head(), batch(n_seqs=1, n_tokens=(1 << 27) - 32, max_len=1 << 28, **BIG), batch(n_seqs=1, n_tokens=1 << 27, max_len=1 << 28, **BIG),
     dict(nh=16)),
])
def test_launches_of_less_than_2_to_the_32_threads(lib, call, p, fits, past, kw):  # noqa: F811
    """HIP refuses a launch of 2^32 threads and more: such a batch is refused
    before anything runs, the one below it is taken."""
    lib.fake_reset(0)
    assert call(lib, p, fits, BF16, **kw) == 0, lib.fake_error()
    assert lib.fake_launches() >= 1
    lib.fake_reset(0)
    assert call(lib, p, past, BF16, **kw) == -1
    assert lib.fake_launches() == 0 and lib.fake_error()


@pytest.mark.parametrize("nkv,heads,hd,cache", [(8, 32, 128, BF16), (8, 32, 128, I8), (1, 16, 64, F32), (4, 4, 64, I8)])
@pytest.mark.parametrize("seqs,max_len", [(1, 1 << 30), (16, 1 << 20), (128, 131072), (128, 32768), (1024, 1 << 20), (5000, 4096), (40000, 1000000)])
def test_decode_workspace_is_bounded(lib, seqs, max_len, nkv, heads, hd, cache):  # noqa: F811
    """A far bound on the length costs no more than 64 workgroups a CU (of 256)
    and their results: parts are longer instead."""
    lib.fake_reset(0)
    p = pages(n_kv_heads=nkv, head_dim=hd, dtype=cache, page_size=1024, n_pages=1 << 20)
    assert decode(lib, p, batch(n_seqs=seqs, n_tokens=seqs, max_len=max_len, table_stride=1 << 20, first=None), nh=heads) == 0, lib.fake_error()
    most = max(64 * 256, seqs * nkv)
    assert lib.fake_ws() <= most * (heads // nkv) * (hd + 2) * 4
    assert lib.fake_blocks() <= most + seqs * heads * (hd // 32)


@pytest.mark.parametrize("call", [append, read, decode, prompt])
@pytest.mark.parametrize("what", [dict(table=A + 2), dict(pos=A + 1), dict(first=A + 3), dict(n_seqs=(1 << 30) + 1, n_tokens=1 << 30)])
def test_batches_refused(lib, call, what):  # noqa: F811
    lib.fake_reset(0)
    assert call(lib, b=batch(**what)) == -1
    assert lib.fake_launches() == 0 and lib.fake_error()


@pytest.mark.parametrize("call", [append, read, decode, prompt])
def test_batches_of_words_anywhere(lib, call):  # noqa: F811
    """table, pos and first need no more than the alignment of their words."""
    lib.fake_reset(0)
    assert call(lib, b=batch(table=A + 4, pos=A + 8, first=A + 12)) == 0 and lib.fake_launches()


@pytest.mark.parametrize("rows", [1, 16, 17, 255, 256, 257, 511, 512, 5000])
@pytest.mark.parametrize("vocab", [1000, 128256, 1 << 20])
def test_sampling_workspace_is_bounded(lib, rows, vocab):  # noqa: F811
    lib.fake_reset(0)
    assert sample(lib, rows=rows, vocab=vocab, stride=vocab) == 0
    assert 0 < lib.fake_ws() < 43.1e6


@pytest.mark.parametrize("nkv,heads,hd", [(8, 32, 128), (1, 16, 64), (8, 8, 64), (8, 128, 128)])
@pytest.mark.parametrize("cache", [F32, BF16, I8])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_prompt_workspace_is_bounded(lib, nkv, heads, hd, cache, xt):  # noqa: F811
    """However many tokens and whatever the bound; few tokens over many keys still
    come in parts."""
    p = pages(n_kv_heads=nkv, head_dim=hd, dtype=cache, page_size=1024, n_pages=1 << 20)
    for seqs in (1, 16, 256):
        for n in (seqs, 1000, 8000, 64000, 1000000):
            for max_len in (1000, 32000, 131072, 1 << 30):
                lib.fake_reset(0)
                b = batch(n_seqs=seqs, n_tokens=n, max_len=max_len, table_stride=1 << 20)
                assert prompt(lib, p, b, xt, nh=heads, qs=1 << 15, os=1 << 15) == 0, lib.fake_error()
                assert lib.fake_ws() <= 512 << 20
                assert seqs > 1 or n > 1 or max_len < 32000 or lib.fake_launches() == 2
