"""The workspace that the paged entry points and the batch sampler have of their
context, on a CPU (tests/test_runtime_host.py's device)."""
import ctypes as C

import pytest

import guanaco_amd.hip as H
from test_runtime_host import GB, SMALL, built, copies, dev, prompt  # noqa: F401


@pytest.fixture
def ws(dev):  # noqa: F811
    f = dev._Z15gq_ctx_paged_wsP6gq_ctxm
    f.restype, f.argtypes = C.c_void_p, [C.c_void_p, C.c_size_t]
    return f


def test_requests_take_the_workspace_back(dev, ws):  # noqa: F811
    """Between calls it is room that a request may need, as the prompts'
    workspaces are: one that fits with it gets it, one that would not fit even
    so leaves it, and the bf16 copies of the weights stay while it is enough."""
    dev.fake_reset(GB)
    with H.Context(0) as ctx:
        dm = H.DeviceModel(ctx, SMALL, 512)
        first = prompt(dm, 300)
        p = ws(ctx.h, 200 << 20)
        assert p and ws(ctx.h, 100 << 20) == p
        used = dev.fake_used()
        with pytest.raises(H.HipError):
            ctx.alloc(GB)
        assert dev.fake_used() == used and ws(ctx.h, 200 << 20) == p
        room = ctx.alloc(GB - 256 - used + (100 << 20))
        assert dev.gq_hip_prefill_copy_bytes(ctx.h) == copies(SMALL)
        assert not ws(ctx.h, 200 << 20)  # no room for it now, whatever is taken back
        room.free()
        assert ws(ctx.h, 200 << 20)
        assert prompt(dm, 300) == first


def test_the_workspace_makes_room_for_itself(dev, ws):  # noqa: F811
    """A larger one is asked for once the smaller is gone; refused, a smaller
    one can be had again."""
    dev.fake_reset(GB)
    with H.Context(0) as ctx:
        assert ws(ctx.h, 600 << 20) and ws(ctx.h, 700 << 20)
        assert not ws(ctx.h, 2 * GB)
        assert ws(ctx.h, 700 << 20)
