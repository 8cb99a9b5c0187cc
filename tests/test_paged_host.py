"""The host side of the paged entry points and of the batch sampler on a CPU:
gq_paged.hip and gq_sample_rows.hip linked with
tests/native/fake_paged.cpp, which stands for the HIP runtime and the context
and counts launches.  What is refused launches nothing; what is taken runs on
the context's device and leaves the caller's current."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import guanaco_amd.hip as H
from paged import BF16, F32, I8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def build(d, *sources):
    flags = ["--offload-arch=gfx950", "--offload-host-only", "-O1", "-fPIC", "-std=c++17", "-I",
             os.path.join(ROOT, "guanaco_amd", "csrc")]
    objs = []
    for src in sources:
        objs.append(str(d / (os.path.basename(src) + ".o")))
        subprocess.run([HIPCC, *flags, "-x", "hip", "-c", src, "-o", objs[-1]], check=True)
    # the device code that the host objects register is not there
    stub = d / "fatbin.c"
    names = [w for o in objs for w in subprocess.run(["nm", "-u", o], capture_output=True, text=True, check=True).stdout.split()
             if w.startswith("__hip_fatbin")]
    stub.write_text("".join(f"char {w}[64];\n" for w in names))
    so = str(d / "libfake.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", so, *objs, "-x", "c++", str(stub)], check=True)
    return so


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    src = [os.path.join(ROOT, "guanaco_amd", "csrc", n) for n in ("gq_paged.hip", "gq_paged_prompt.hip", "gq_sample_rows.hip")]
    src.append(os.path.join(ROOT, "tests", "native", "fake_paged.cpp"))
    lib = C.CDLL(build(tmp_path_factory.mktemp("fake_paged"), *src))
    for n in (n for n in H.EXPORTS if hasattr(lib, n)):
        f, g = getattr(lib, n), getattr(H.lib, n)
        f.restype, f.argtypes = g.restype, g.argtypes
    lib.fake_ctx.restype = C.c_void_p
    lib.fake_error.restype = C.c_char_p
    lib.fake_blocks.restype = C.c_ulonglong
    lib.fake_ws.restype = C.c_size_t
    return lib


A = 1 << 20  # an aligned address that nothing reads


def pages(**kw):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, dtype=I8, n_pages=100, page_size=64, n_kv_heads=8, head_dim=128)
    d.update(kw)
    return H.GqPages(*[d[n] for n, _ in H.GqPages._fields_])


def batch(**kw):
    d = dict(table=A, pos=A, first=A, n_seqs=4, table_stride=10, n_tokens=40, max_len=600)
    d.update(kw)
    return H.GqBatch(*[d[n] for n, _ in H.GqBatch._fields_])


def append(lib, p=None, b=None, xtype=F32, nh=32, q=A, qs=4096, qo=A, qos=4096, k=A, ks=1024, v=A, vs=1024, rope=A, n_rope=600):
    return lib.gq_hip_paged_append_dev(lib.fake_ctx(), C.byref(p or pages()), C.byref(b or batch()), xtype, nh, q, qs, qo, qos, k,
                                       ks, v, vs, rope, n_rope)


def read(lib, p=None, b=None, xtype=F32, k=A, ks=1024, v=A, vs=1024):
    return lib.gq_hip_paged_read_dev(lib.fake_ctx(), C.byref(p or pages()), C.byref(b or batch()), xtype, k, ks, v, vs)


def decode(lib, p=None, b=None, xtype=F32, nh=32, q=A, qs=4096, out=A, os=4096):
    return lib.gq_hip_paged_decode_dev(lib.fake_ctx(), C.byref(p or pages()), C.byref(b or batch()), xtype, nh, q, qs, out, os)


def prompt(lib, p=None, b=None, xtype=F32, nh=32, q=A, qs=4096, out=A, os=4096):
    return lib.gq_hip_paged_prompt_dev(lib.fake_ctx(), C.byref(p or pages()), C.byref(b or batch()), xtype, nh, q, qs, out, os)


ENTRIES = [append, read, decode, prompt]


@pytest.mark.parametrize("call", ENTRIES)
def test_taken_and_run_on_the_contexts_device(lib, call):
    for p in (pages(), pages(dtype=F32, k_scale=None, v_scale=None), pages(dtype=BF16, head_dim=64, page_size=16, n_pages=1000)):
        for x in (F32, BF16):
            lib.fake_reset(0)
            lib.fake_set_device(1)
            b = batch(max_len=160) if p.page_size == 16 else batch()
            assert call(lib, p, b, x) == 0, lib.fake_error()
            assert lib.fake_launches() >= 1 and lib.fake_device() == 1


@pytest.mark.parametrize("call", ENTRIES)
@pytest.mark.parametrize("what,rc", [
    (dict(p=pages(dtype=2)), -1), (dict(p=pages(dtype=4)), -1), (dict(xtype=I8), -1), (dict(xtype=1), -1),
    (dict(p=pages(k=None)), -1), (dict(p=pages(v=None)), -1), (dict(p=pages(k=A + 4)), -1), (dict(p=pages(v=A + 8)), -1),
    (dict(p=pages(k_scale=None)), -1), (dict(p=pages(v_scale=A + 4)), -1),
    (dict(p=pages(head_dim=96)), -1), (dict(p=pages(head_dim=256)), -1), (dict(p=pages(head_dim=0)), -1),
    (dict(p=pages(n_kv_heads=0)), -1), (dict(p=pages(n_pages=0)), -1),
    (dict(p=pages(page_size=8)), -1), (dict(p=pages(page_size=48)), -1), (dict(p=pages(page_size=2048)), -1),
    (dict(p=pages(page_size=0)), -1), (dict(p=pages(page_size=-64)), -1),
    (dict(b=batch(table=None)), -1), (dict(b=batch(pos=None)), -1), (dict(b=batch(n_seqs=-1)), -1),
    (dict(b=batch(n_tokens=-1)), -1), (dict(b=batch(table_stride=0)), -1), (dict(b=batch(max_len=-1)), -1),
    (dict(b=batch(first=None, n_tokens=3)), -1), (dict(b=batch(max_len=(1 << 30) + 1, table_stride=1 << 25)), -1), (dict(b=batch(max_len=641)), -5), (dict(b=batch(n_tokens=(1 << 30) + 1)), -1),
])
def test_refused_by_every_entry(lib, call, what, rc):
    lib.fake_reset(0)
    assert call(lib, **what) == rc
    assert lib.fake_launches() == 0 and lib.fake_error()


@pytest.mark.parametrize("call,what,rc", [
    (append, dict(nh=0), -1), (append, dict(qs=4095), -1), (append, dict(qs=4000), -1), (append, dict(q=A + 2), -1),
    (append, dict(qo=None), -1), (append, dict(qos=4088), -1), (append, dict(k=None), -1), (append, dict(ks=1016), -1),
    (append, dict(ks=1028), -1), (append, dict(v=A + 4), -1), (append, dict(vs=8), -1), (append, dict(rope=A + 8), -1),
    (append, dict(n_rope=599), -5),
    (read, dict(k=None), -1), (read, dict(v=None), -1), (read, dict(ks=1000), -1), (read, dict(vs=1025), -1), (read, dict(k=A + 8), -1),
    (decode, dict(nh=30), -1), (decode, dict(nh=0), -1), (decode, dict(nh=-8), -1), (decode, dict(nh=136, qs=1 << 15, os=1 << 15), -1),
    (decode, dict(q=None), -1), (decode, dict(out=None), -1), (decode, dict(qs=4088), -1), (decode, dict(os=4100), -1),
    (decode, dict(q=A + 4), -1), (decode, dict(out=A + 8), -1),
    (prompt, dict(nh=30), -1), (prompt, dict(nh=136, qs=1 << 15, os=1 << 15), -1), (prompt, dict(q=None), -1),
    (prompt, dict(out=A + 8), -1), (prompt, dict(os=64), -1),
])
def test_refused(lib, call, what, rc):
    lib.fake_reset(0)
    assert call(lib, **what) == rc
    assert lib.fake_launches() == 0 and lib.fake_error()


@pytest.mark.parametrize("call", ENTRIES)
def test_null_arguments(lib, call):
    lib.fake_reset(0)
    f = getattr(lib, {append: "gq_hip_paged_append_dev", read: "gq_hip_paged_read_dev", decode: "gq_hip_paged_decode_dev",
                      prompt: "gq_hip_paged_prompt_dev"}[call])
    rest = [0] * (len(f.argtypes) - 3)
    rest = [None if t is C.c_void_p else 0 for t in f.argtypes[3:]]
    assert f(None, C.byref(pages()), C.byref(batch()), *rest) == -1
    assert f(lib.fake_ctx(), None, C.byref(batch()), *rest) == -1
    assert f(lib.fake_ctx(), C.byref(pages()), None, *rest) == -1
    assert lib.fake_launches() == 0


@pytest.mark.parametrize("call", ENTRIES)
def test_nothing_to_do_launches_nothing(lib, call):
    lib.fake_reset(0)
    assert call(lib, b=batch(n_seqs=0, table=None, pos=None)) == 0
    assert call(lib, b=batch(n_tokens=0)) == 0
    assert lib.fake_launches() == 0


def sample(lib, logits=A, rows=4, vocab=1000, stride=1000, t=A, k=A, p=A, m=A, rnd=A, tokens=A, logprobs=A):
    return lib.gq_hip_sample_rows_dev(lib.fake_ctx(), logits, rows, vocab, stride, t, k, p, m, rnd, tokens, logprobs)


@pytest.mark.parametrize("what", [dict(), dict(t=None, k=None, p=None, m=None, logprobs=None), dict(vocab=1 << 20, stride=1 << 20),
                                  dict(vocab=1, stride=7), dict(logits=A + 4, rnd=A + 8)])
def test_sampling_taken(lib, what):
    lib.fake_reset(0)
    lib.fake_set_device(2)
    assert sample(lib, **what) == 0 and lib.fake_launches() >= 1 and lib.fake_device() == 2


@pytest.mark.parametrize("what", [dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 20) + 1, stride=1 << 21), dict(stride=999),
                                  dict(logits=None), dict(rnd=None), dict(tokens=None), dict(logits=A + 2), dict(k=A + 1),
                                  dict(logprobs=A + 3)])
def test_sampling_refused(lib, what):
    lib.fake_reset(0)
    assert sample(lib, **what) == -1
    assert lib.fake_launches() == 0 and lib.fake_error()
    assert lib.gq_hip_sample_rows_dev(None, A, 1, 10, 10, A, A, A, A, A, A, A) == -1


def test_sampling_of_no_rows(lib):
    lib.fake_reset(0)
    assert sample(lib, rows=0, logits=None) == 0 and lib.fake_launches() == 0


def test_workspace_refused(lib):
    """A call that needs workspace and gets none: -4, nothing launched."""
    long = dict(p=pages(page_size=128, n_pages=4000), b=batch(n_seqs=1, n_tokens=1, table_stride=1000, max_len=100000))
    for call, kw in ((decode, long), (prompt, long), (sample, {})):
        lib.fake_reset(1)
        assert call(lib, **kw) == -4
        assert lib.fake_launches() == 0 and lib.fake_ws() > 0
        lib.fake_reset(0)
        assert call(lib, **kw) == 0 and lib.fake_launches() > 1


def test_workspace_and_launches_follow_the_batch(lib):
    """One part needs neither workspace nor a second launch; sampling runs many
    rows in launches of 512."""
    for call in (decode, prompt):
        lib.fake_reset(0)
        assert call(lib, b=batch(n_seqs=1, n_tokens=1, max_len=60)) == 0 and lib.fake_launches() == 1
    lib.fake_reset(0)
    assert sample(lib, rows=512, vocab=50257, stride=50257) == 0
    one, ws = lib.fake_launches(), lib.fake_ws()
    lib.fake_reset(0)
    assert sample(lib, rows=1025, vocab=50257, stride=50257) == 0
    assert lib.fake_launches() == 3 * one and lib.fake_ws() == ws < 64 << 20
