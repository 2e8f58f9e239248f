"""Arguments that the entries of the cache in pages and of the verification
refuse.  CPU only: arguments are checked before the device is opened, so a
call with good arguments gets -7 where there is none."""
import ctypes as C
import os

import pytest

import slate_amd

A = 1 << 20          # an address, aligned, never read by these calls


@pytest.fixture
def lib():
    lb = slate_amd.load_library()
    lb.slate_hip_clear_error()
    yield lb
    lb.slate_hip_clear_error()


@pytest.fixture
def no_device(lib):
    if os.path.exists("/dev/kfd"):
        pytest.skip("a device is present: accepted calls would run on made-up addresses")
    return lib


def pages(**kw):
    d = dict(table=A, held=A, free_pages=A, n_free=A, n_slots=4, max_pages=10, n_pages=30, page_size=16)
    d.update({k: v for k, v in kw.items() if k in d})
    return slate_amd.Pages(*d.values())


def paged_kv(**kw):
    d = dict(K=A, V=A, dtype=1, n_kv_heads=2, head_dim=64, page_stride=2048, head_stride=1024, row_stride=64)
    d.update({k: v for k, v in kw.items() if k in d})
    return slate_amd.PagedKv(*d.values())


def call(lib, entry, **kw):
    d = dict(slot=A, pos0=A, n_new=A, B=2, T_cap=5, tok_off=A, tok2seq=A, tok_pos=A, tok_row=A, last_tok=A, status=A,
             length=A, k=A, v=A, ld=128, T=5, out=A, q=A + (1 << 40), max_new=3, Hq=8, ws=None, ws_bytes=0,
             n_acc=A, out_tok=A, out_row=A, logits=A, zld=100, token=A, parent=None, probs=A, pld=100,
             temperature=A, u=A, u_next=A, V=100)
    d.update({k: v for k, v in kw.items() if k in d})
    pg = None if kw.get("no_pages") else C.byref(pages(**kw))
    kv = None if kw.get("no_kv") else C.byref(paged_kv(**kw))
    names = {"pages_reset": [], "pages_extend": "slot pos0 n_new B T_cap tok_off tok2seq tok_pos tok_row last_tok status",
             "pages_trim": "slot length B status", "kv_store_paged": "k v ld tok_row T",
             "attention_paged": "slot tok_off pos0 B T max_new Hq ws ws_bytes",
             "verify_drafts": "n_acc out_tok out_row logits zld token parent probs pld temperature u u_next tok_off B T V "
                              "ws ws_bytes"}[entry]
    args = [d[n] for n in (names.split() if names else [])]
    first = {"kv_store_paged": [kv, pg], "attention_paged": [d["out"], d["q"], kv, pg], "verify_drafts": []}
    return getattr(lib, "slate_hip_" + entry)(*first.get(entry, [pg]), *args)


BAD_PAGES = [dict(no_pages=True)] + [{n: None} for n in ("table", "held", "free_pages", "n_free")] + \
            [{n: 0} for n in ("n_slots", "max_pages", "n_pages", "page_size")] + \
            [dict(n_pages=1 << 20, page_size=2048), dict(max_pages=(1 << 31) - 1, page_size=1),
             dict(page_size=(1 << 31) - 1, n_pages=1, max_pages=1)]
BAD_KV = [dict(no_kv=True), dict(K=None), dict(V=None), dict(K=A + 8), dict(V=A + 8), dict(dtype=3), dict(dtype=-1),
          dict(n_kv_heads=0), dict(n_kv_heads=65536), dict(head_dim=0), dict(head_dim=20),
          dict(head_dim=264, row_stride=264), dict(page_stride=-8), dict(page_stride=4), dict(head_stride=-8),
          dict(head_stride=12), dict(row_stride=56), dict(row_stride=68), dict(row_stride=(1 << 26) + 8)]
BAD = {
    "pages_reset": BAD_PAGES,
    "pages_extend": BAD_PAGES + [{n: None} for n in ("slot", "pos0", "n_new", "tok_off", "tok2seq", "tok_pos", "tok_row",
                                                     "last_tok", "status")] +
    [dict(B=0), dict(B=1025), dict(T_cap=-1)],
    "pages_trim": BAD_PAGES + [{n: None} for n in ("slot", "length", "status")] + [dict(B=0), dict(B=1025)],
    "kv_store_paged": BAD_PAGES + BAD_KV + [{n: None} for n in ("k", "v", "tok_row")] +
    [dict(k=A + 8), dict(v=A + 4), dict(T=0), dict(ld=124), dict(ld=130)],
    "attention_paged": BAD_PAGES + BAD_KV + [{n: None} for n in ("out", "q", "slot", "tok_off", "pos0")] +
    [dict(B=0), dict(B=1025), dict(T=0), dict(max_new=0), dict(Hq=9), dict(Hq=0), dict(Hq=65536, n_kv_heads=1),
     dict(q=A), dict(q=A + 4 * (5 * 8 * 64 - 1)), dict(ws=A + 8, ws_bytes=1 << 40), dict(T=1 << 28, Hq=16),
     dict(B=1000, T=100000, n_pages=1 << 20, max_pages=1 << 20, page_size=1024)],
    "verify_drafts": [{n: None} for n in ("n_acc", "out_tok", "logits", "token", "u", "u_next", "tok_off")] +
    [dict(B=0), dict(B=1025), dict(T=0), dict(V=0), dict(zld=99), dict(pld=99), dict(parent=A),
     dict(ws=A + 8, ws_bytes=1 << 40)],
}
GOOD = {
    "pages_reset": [{}, dict(page_size=1), dict(page_size=48, n_pages=1 << 20)],
    "pages_extend": [{}, dict(B=1024), dict(T_cap=0)],
    "pages_trim": [{}, dict(B=1024)],
    "kv_store_paged": [{}, dict(dtype=0), dict(dtype=2, ld=132), dict(head_dim=256, ld=512, row_stride=256),
                       dict(head_dim=8, row_stride=1 << 26), dict(page_stride=1 << 40)],
    "attention_paged": [{}, dict(Hq=14), dict(head_dim=40), dict(head_dim=256, row_stride=512), dict(B=1024, T=1024),
                        dict(T=131072, max_new=131072, Hq=64, n_kv_heads=8, max_pages=8192),
                        dict(B=1024, T=16384, max_new=16, Hq=64, n_kv_heads=8, max_pages=8192)],
    "verify_drafts": [{}, dict(out_row=None), dict(temperature=None), dict(probs=None), dict(probs=None, parent=A),
                      dict(zld=101, pld=1000)],
}


@pytest.mark.parametrize("entry", list(BAD))
def test_refused(lib, entry):
    for kw in BAD[entry]:
        assert call(lib, entry, **kw) == -1, kw
        assert entry in slate_amd.last_error(), kw
        lib.slate_hip_clear_error()


@pytest.mark.parametrize("entry", list(GOOD))
def test_accepted(no_device, entry):
    for kw in GOOD[entry]:
        assert call(no_device, entry, **kw) == -7, (kw, slate_amd.last_error())


def test_workspace_bytes(lib):
    f = lib.slate_hip_attention_paged_bytes
    assert f(32, 8, 128) >= 0 and f(7, 1, 8) >= 0 and f(8, 8, 256) >= 0
    for bad in ((0, 1, 128), (8, 0, 128), (9, 2, 128), (8, 2, 4), (8, 2, 264), (8, 2, 36), (65536, 1, 64)):
        assert f(*bad) == -1
    if f(8, 2, 64):
        assert call(lib, "attention_paged", ws=A, ws_bytes=f(8, 2, 64) - 1) == -1
    g = lib.slate_hip_verify_drafts_bytes
    assert g(1, 1, 1) >= 0 and g(1024, 1 << 20, 1 << 20) >= 0
    for bad in ((0, 1, 1), (1025, 1, 1), (1, 0, 1), (1, 1, 0)):
        assert g(*bad) == -1
    if g(2, 5, 100):
        assert call(lib, "verify_drafts", ws=A, ws_bytes=g(2, 5, 100) - 1) == -1


def test_structures_match_the_header(lib):
    """Sizes and offsets of the two structures, as C lays them out."""
    P, K = slate_amd.Pages, slate_amd.PagedKv
    assert C.sizeof(P) == 48 and P.n_slots.offset == 32 and P.page_size.offset == 44
    assert C.sizeof(K) == 56 and K.dtype.offset == 16 and K.page_stride.offset == 32 and K.row_stride.offset == 48
