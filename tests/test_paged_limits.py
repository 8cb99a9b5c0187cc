"""Sizes at the ends of what the paged entry points take, on the CPU
(tests/test_paged_host.py's stand-in for the context and HIP)."""
import pytest

from test_paged_host import A, F32, BF16, append, batch, decode, lib, pages, prompt, read  # noqa: F401

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
