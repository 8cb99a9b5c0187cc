"""Which packed rows belong to a sequence, alike in every entry point."""
import numpy as np
import pytest

import guanaco_amd.hip as H
from paged import BF16, F32, I8, World
from test_gpu_paged import attend, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_a_sequence_that_passes_the_rows_has_none(ctx, cache):
    """Three sequences of which the last one's rows end past n_tokens: nothing of
    it is appended, read or attended to, and its rows stay as they were."""
    w = World(80, [20, 3, 50], [4, 5, 7], 2, 64, cache, 16).upload(ctx, H)
    w.batch.n_tokens = 13  # its rows would be 9 .. 15
    x = ctx.upload(np.ones((w.rows, 128), np.float32))
    before = [w.download(i) for i in range(2)]
    ctx.paged_append_dev(w.pages, w.batch, F32, 0, None, 0, None, 0, x, 128, x, 128, None, 0)
    for i in range(2):
        after = w.download(i)
        for t in range(9):
            s, p = w.at[t]
            g, o = w.slot(s, p)
            for a, b in zip(after, before[i]):
                if a is not None:
                    a[g, :, o] = b[g, :, o]
        assert all(a is None or a.tobytes() == b.tobytes() for a, b in zip(after, before[i]))
    x.upload(np.full((w.rows, 128), 7, np.float32))
    ctx.paged_read_dev(w.pages, w.batch, F32, x, 128, x, 128)
    assert (x.download().reshape(-1, 128)[9:] == 7).all()
    w.pools = [w.download(0), w.download(1)]
    for entry, rows in (("paged_decode_dev", [3, 8]), ("paged_prompt_dev", range(9))):
        q, got = attend(ctx, w, 4, F32, entry)
        check_attention(w, q, got, rows, F32, entry == "paged_prompt_dev")
        assert (got[9:] == 5).all()
    w.free()


@pytest.mark.parametrize("cache", [F32, BF16, I8])
def test_prompts_without_first(ctx, cache):
    """One token a sequence, row s of it: the prompt's entry and the decode's agree
    with the definition, more rows than sequences."""
    w = World(81, [0, 130, -1, 4000, 64], [1] * 5, 2, 128, cache, 64, pad=3).upload(ctx, H, with_first=False)
    for entry in ("paged_decode_dev", "paged_prompt_dev"):
        q, got = attend(ctx, w, 8, F32, entry)
        check_attention(w, q, got, range(5), F32, entry == "paged_prompt_dev")
        assert (got[5:] == 5).all()
    w.free()
