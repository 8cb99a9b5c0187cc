"""Parts of the paged kernels that a CPU can check: tests/native/paged_parts.cpp
compiled for the host."""
import ctypes as C
import os

import pytest

from test_paged_host import HIPCC, ROOT, build


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    return C.CDLL(build(tmp_path_factory.mktemp("parts"), os.path.join(ROOT, "tests", "native", "paged_parts.cpp")))


def test_flags_of_the_prompt_kernel_outlive_the_exchange(parts):
    """The waves' flags are read after the same barrier that lets the second
    half of the waves write the exchange, which starts at 0: no byte of one is a
    byte of the other, or of what lies before the flags."""
    out = (C.c_int * 256)()
    n = parts.parts_prompt_lds(out)
    rows = [out[i:i + 7] for i in range(0, n, 7)]
    assert len(rows) == 18
    for rg, qlo, scl, used, exchange, odd, total in rows:
        assert (exchange > 0) == (rg == 4)
        assert 0 < qlo <= scl <= used <= odd and exchange <= odd and odd + 8 * 4 <= total <= 160 * 1024


@pytest.mark.parametrize("max_len", [0, 1, 100, (1 << 30) - 1, 1 << 30])
def test_positions_that_exist(parts, max_len):
    """min(before + n, max_len) without the sum's 32nd bit: both are 2^30 at
    most where they count, and `before` is any number of the caller's."""
    for before in (-2 ** 31, -1, 0, 1, 57, max_len - 1, max_len, 1 << 30, 2 ** 31 - 1):
        for n in (0, 1, 2, 99, (1 << 30) - 1, 1 << 30):
            assert parts.parts_len(before, n, max_len) == (min(before + n, max_len) if before >= 0 else 0), (before, n)
