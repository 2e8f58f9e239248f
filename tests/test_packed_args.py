"""Arguments that the packed-batch entries refuse, and the rotary frequencies.
CPU only: arguments are checked before the device is opened, so a call with
good arguments gets -7 where there is none."""
import ctypes as C

import numpy as np
import pytest

import slate_amd
from tests import packed_ref as pr

A = 1 << 20          # an address, aligned, never read by these calls


@pytest.fixture
def lib():
    lb = slate_amd.load_library()
    lb.slate_hip_clear_error()
    yield lb
    lb.slate_hip_clear_error()


def rope_cfg(**kw):
    d = dict(layout=0, rot_dim=64, scaling=0, orig_ctx=4096, theta_base=10000.0, factor=4.0, low=1.0, high=4.0,
             magnitude=0.0)
    d.update(kw)
    return slate_amd.RopeConfig(**d)


CONFIGS = [dict(), dict(layout=1, rot_dim=6), dict(scaling=1, factor=2.5), dict(scaling=2, theta_base=500000.0),
           dict(scaling=2, rot_dim=512, factor=32.0), dict(scaling=3, factor=16.0, high=32.0),
           dict(scaling=3, orig_ctx=1), dict(scaling=3, factor=0.5), dict(scaling=3, magnitude=0.75),
           dict(rot_dim=2), dict(scaling=3, rot_dim=100, factor=40.0, low=0.5, high=0.6)]


@pytest.mark.parametrize("kw", CONFIGS)
def test_rope_frequencies(lib, kw):
    c = rope_cfg(**kw)
    w, m = (C.c_double * (c.rot_dim // 2))(), C.c_double()
    assert lib.slate_hip_rope_frequencies(w, C.byref(m), C.byref(c)) == 0
    want, mag = pr.rope_frequencies(c.layout, c.rot_dim, c.scaling, c.theta_base, c.factor, c.low, c.high, c.orig_ctx,
                                    c.magnitude)
    # powers and logarithms of two libraries: a few units of 2^-52 each
    np.testing.assert_allclose(np.array(w), want, rtol=2.0 ** -46, atol=0)
    assert abs(m.value - mag) <= 2.0 ** -48 * mag


BAD_ROPE = [dict(layout=2), dict(layout=-1), dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=514), dict(scaling=4),
            dict(scaling=-1), dict(theta_base=0.0), dict(theta_base=float("nan")), dict(theta_base=float("inf")),
            dict(scaling=1, factor=0.0), dict(scaling=1, factor=-2.0), dict(scaling=2, factor=float("inf")),
            dict(scaling=2, orig_ctx=0), dict(scaling=2, low=4.0), dict(scaling=2, low=0.0),
            dict(scaling=3, high=float("nan")), dict(scaling=3, theta_base=1.0), dict(magnitude=float("nan"))]


@pytest.mark.parametrize("kw", BAD_ROPE)
def test_rope_refuses_configurations(lib, kw):
    c = rope_cfg(**kw)
    w, m = (C.c_double * 512)(), C.c_double()
    assert lib.slate_hip_rope_frequencies(w, C.byref(m), C.byref(c)) == -1
    assert lib.slate_hip_rope_scaled(A, A, A, 4, 2, 512, 1024, C.byref(c)) == -1
    assert "rope" in slate_amd.last_error()


@pytest.mark.parametrize("kw", [dict(scaling=1, factor=5e-324), dict(theta_base=1e-322, rot_dim=512),
                                dict(scaling=3, factor=1e-320), dict(scaling=1, factor=1e-300), dict(magnitude=1e39),
                                dict(magnitude=-1e300)])
def test_rope_refuses_what_overflows(lib, kw):
    """Frequencies whose angles, or a magnitude that, would be infinite."""
    c = rope_cfg(**kw)
    w, m = (C.c_double * 512)(), C.c_double()
    assert lib.slate_hip_rope_frequencies(w, C.byref(m), C.byref(c)) == -1
    assert lib.slate_hip_rope_scaled(A, A, A, 4, 2, 512, 1024, C.byref(c)) == -1
    assert "out of range" in slate_amd.last_error()


def good(lib, rc):
    """A call with these arguments passes the checks (it must not be made where it would run)."""
    assert rc == -7, slate_amd.last_error()


@pytest.fixture
def no_device(lib):
    import os
    if os.path.exists("/dev/kfd"):
        pytest.skip("a device is present: accepted calls would run on made-up addresses")
    return lib


def rope_args(**kw):
    d = dict(y=A, x=A, pos=A, rows=4, heads=2, hd=128, ld=256)
    d.update(kw)
    return [d[k] for k in ("y", "x", "pos", "rows", "heads", "hd", "ld")] + [C.byref(rope_cfg())]


@pytest.mark.parametrize("kw", [dict(y=None), dict(x=None), dict(pos=None), dict(rows=0), dict(heads=0), dict(hd=0),
                                dict(hd=62), dict(ld=255), dict(y=A + 4), dict(y=A + 4 * (3 * 256 + 255))])
def test_rope_refuses_arguments(lib, kw):
    assert lib.slate_hip_rope_scaled(*rope_args(**kw)) == -1
    assert lib.slate_hip_rope_scaled(A, A, A, 4, 2, 128, 256, None) == -1


def test_rope_accepts(no_device):
    good(no_device, no_device.slate_hip_rope_scaled(*rope_args()))
    good(no_device, no_device.slate_hip_rope_scaled(*rope_args(y=A + 4 * 4 * 256)))


def kv_args(load=False, **kw):
    d = dict(Kq=A, Ks=A, Vq=A, Vs=A, k=A, v=A, ld=256, tok_off=A, pos0=A, kv_base=A, B=2, T=5, heads=2, hd=128,
             stride=128 * 64, max_seq=64)
    d.update(kw)
    first = ["k", "v", "ld", "Kq", "Ks", "Vq", "Vs"] if load else ["Kq", "Ks", "Vq", "Vs", "k", "v", "ld"]
    return [d[k] for k in first + ["tok_off", "pos0", "kv_base", "B", "T", "heads", "hd", "stride", "max_seq"]]


BAD_KV = [{n: None} for n in ("Kq", "Ks", "Vq", "Vs", "k", "v", "tok_off", "pos0", "kv_base")] + \
         [{n: A + 8} for n in ("Kq", "Ks", "Vq", "Vs", "k", "v")] + \
         [dict(B=0), dict(B=1025), dict(T=0), dict(heads=0), dict(max_seq=0), dict(hd=48, ld=96, stride=48 * 64),
          dict(hd=544, ld=2048, stride=544), dict(ld=255), dict(ld=257), dict(stride=100), dict(stride=-128)]


@pytest.mark.parametrize("kw", BAD_KV)
def test_kv_refuses_arguments(lib, kw):
    assert lib.slate_hip_kv_store_q8(*kv_args(**kw)) == -1
    assert lib.slate_hip_kv_load_q8(*kv_args(True, **kw)) == -1
    assert "kv_" in slate_amd.last_error()


def test_kv_accepts(no_device):
    for kw in (dict(), dict(ld=260), dict(hd=512, ld=1024, stride=512), dict(hd=32, B=1024)):
        good(no_device, no_device.slate_hip_kv_store_q8(*kv_args(**kw)))
        good(no_device, no_device.slate_hip_kv_load_q8(*kv_args(True, **kw)))


def attn_call(lib, kind, **kw):
    d = dict(out=A, q=A + (1 << 24), K=A, V=A, Kq=A, Ks=A, Vq=A, Vs=A, tok_off=A, pos0=A, kv_base=A, parent=A, B=2,
             T=5, max_new=3, Hq=8, Hkv=2, hd=128, stride=128 * 64, max_seq=64, ws=None, ws_bytes=0)
    d.update(kw)
    pools = ["K", "V"] if kind == "tree" else ["Kq", "Ks", "Vq", "Vs"]
    names = ["out", "q"] + pools + ["tok_off", "pos0", "kv_base"] + ([] if kind == "ragged_q8" else ["parent"]) + \
        ["B", "T", "max_new", "Hq", "Hkv", "hd", "stride", "max_seq", "ws", "ws_bytes"]
    return getattr(lib, "slate_hip_attention_" + kind)(*[d[n] for n in names])


KINDS = ("ragged_q8", "tree", "tree_q8")
BAD_ATTN = [dict(out=None), dict(q=None), dict(tok_off=None), dict(pos0=None), dict(kv_base=None), dict(B=0),
            dict(B=1025), dict(T=0), dict(max_new=0), dict(max_seq=0), dict(Hq=9), dict(Hkv=0), dict(Hq=1),
            dict(hd=24), dict(hd=528), dict(stride=-128), dict(q=A), dict(q=A + 4 * (5 * 8 * 128 - 1)),
            dict(ws=A + 8, ws_bytes=1 << 40), dict(B=1000, T=100000, max_seq=1 << 30),
            dict(T=1 << 28, Hq=16, q=A + (1 << 45))]
BAD_Q8 = [{n: None} for n in ("Kq", "Ks", "Vq", "Vs")] + [{n: A + 8} for n in ("Kq", "Ks", "Vq", "Vs")] + \
         [dict(stride=100), dict(hd=48, stride=48)]


@pytest.mark.parametrize("kind", KINDS)
def test_attention_refuses_arguments(lib, kind):
    bad = BAD_ATTN + (BAD_Q8 if kind != "tree" else [dict(K=None), dict(V=None), dict(hd=40)])
    bad += [dict(parent=None), dict(max_new=1025)] if kind != "ragged_q8" else []
    for kw in bad:
        assert attn_call(lib, kind, **kw) == -1, kw
    assert "attention_" + kind in slate_amd.last_error()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_accepts(no_device, kind):
    for kw in (dict(), dict(hd=512, stride=512), dict(Hq=7, Hkv=1), dict(B=1024)):
        good(no_device, attn_call(no_device, kind, **kw))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_accepts_long_prompts(no_device, kind):
    """Whole prompts and wide steps of long contexts stay far inside the 32 bits that the kernels count in."""
    far = dict(q=A + (1 << 45))
    for kw in (dict(T=131072, Hq=64, Hkv=8, max_seq=131072, max_new=131072 if kind == "ragged_q8" else 1024, **far),
               dict(T=131072, Hq=64, Hkv=8, max_seq=1 << 20, max_new=1024, **far),
               dict(T=16384, B=1024, Hq=64, Hkv=8, max_seq=1 << 17, max_new=16, **far)):
        good(no_device, attn_call(no_device, kind, **kw))
    assert attn_call(no_device, kind, T=131072, Hq=64, Hkv=8, max_seq=1 << 22, max_new=1024, **far) == -1


def test_workspace_bytes(lib):
    f = lib.slate_hip_attention_packed_bytes
    assert f(32, 8, 128) >= 0 and f(7, 1, 16) >= 0
    for bad in ((0, 1, 128), (8, 0, 128), (9, 2, 128), (8, 2, 8), (8, 2, 528), (8, 2, 40)):
        assert f(*bad) == -1
    need = f(8, 2, 128)
    if need:
        for kind in KINDS:
            assert attn_call(lib, kind, ws=A, ws_bytes=need - 1) == -1
