"""The cache in pages and the verification of drafts at values, scores and sizes far from the ordinary ones.

Tolerances as in test_gpu_paged.py: outputs are held in the 2-norm to 2^-18, here each group of columns by itself (a
score is off by about 2^-22 and a weight by as much, so what a weight adds to an output is too; 2^-18 leaves 16 times
that); what a value must not change is equal bit for bit.
"""
import ctypes as C

import numpy as np
import pytest

import slate_amd
from tests import paged_ref as pr
from tests import test_gpu_packed as packed
from tests.test_gpu_paged import (BF16, F16, F32, NORM_TOL, Attend, Cache, DevicePages, Drafts, dev, lib, of_type, ok,
                                  same_pages, to_type)

pytestmark = pytest.mark.gpu
WILD = (np.nan, np.inf, -np.inf)


def put(c, name, b, x):
    """Sequence b's K or V rows x [rows, Hkv, hd] on the host; upload() sends them."""
    c.values[name][b] = to_type(np.asarray(x, np.float32), c.dtype)
    c.pools[name][c.where(b, np.arange(len(x)))] = c.values[name][b]


def upload(c):
    c.k.upload(c.pools["K"])
    c.v.upload(c.pools["V"])


def with_value(c, name, b, row, col, value):
    """The pool of K or V (kv head 0) with one more value, for an upload."""
    pool = c.pools[name].copy()
    pool[c.where(b, np.array([row]))[0, 0, col]] = to_type(np.array([value], np.float32), c.dtype)[0]
    return pool


# -- values that are not finite ------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("p", [50, 3000])
@pytest.mark.parametrize("hd,G", [(64, 32), (128, 40), (128, 71), (40, 64), (256, 16), (256, 20)])
def test_a_draft_does_not_reach_the_tokens_before_it(hip, hd, G, p, dtype):
    """Groups of query heads as large as the kernels' tiles, so that a tile's rows are all one token's."""
    n = 3
    c = Cache([(p, n), (33, 1)], 1, hd, 16, dtype, 0, 7)
    r = Attend(c, G)
    r.call()
    r.check()
    clean = r.result()
    for at in range(1, n):
        for what in WILD:
            c.v.upload(with_value(c, "V", 0, p + at, 5, what))
            r.call()
            got = r.result()
            assert np.array_equal(got[:at], clean[:at]), (at, what)
            assert np.array_equal(got[n:], clean[n:]), (at, what)
            assert not np.isfinite(got[at:n, :, 5]).any()
            assert np.array_equal(np.delete(got[at:n], 5, 2), np.delete(clean[at:n], 5, 2))
    c.v.upload(c.pools["V"])


def hot(c, r, b, row, score):
    """K's row of kv head 0 gets about this score from every query of the batch, the others stay around 0."""
    rng = np.random.default_rng(3)
    base = rng.normal(0, 1, c.hd)
    r.q = (base + 0.1 * rng.normal(0, 1, r.q.shape)).astype(np.float32)
    r.qd.upload(r.q)
    K = of_type(c.values["K"][b], c.dtype)
    K[row, 0] = score * c.hd ** 0.5 * base / (base @ base)
    put(c, "K", b, K)
    upload(c)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("p,top,low", [(700, 5, 40), (700, 690, 70), (20000, 5, 15000), (20000, 19990, 70)])
@pytest.mark.parametrize("n,G", [(1, 4), (3, 8), (8, 8)])
def test_a_value_reaches_every_token_that_sees_it(hip, n, G, p, top, low, dtype):
    """A key that takes all of the weight does not hide a NaN or an infinity in another part of the cache."""
    c = Cache([(p, n)], 1, 64, 16, dtype, 0, 8)
    r = Attend(c, G)
    hot(c, r, 0, top, 300.0)
    r.call()
    clean = r.result()[:n]
    assert np.isfinite(clean).all()
    for what in WILD:
        c.v.upload(with_value(c, "V", 0, low, 7, what))
        r.call()
        got = r.result()[:n]
        assert not np.isfinite(got[:, :, 7]).any(), what
        assert np.array_equal(np.delete(got, 7, 2), np.delete(clean, 7, 2)), what
    c.v.upload(c.pools["V"])
    c.k.upload(with_value(c, "K", 0, low, 7, np.nan))
    r.call()
    assert np.isnan(r.result()[:n]).all()


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("top,low", [(5, 15000), (19990, 70), (70, 100), (100, 70)])
def test_a_tree_sees_a_value_beside_a_key_that_takes_all(hip, top, low, n):
    """The same over the slots of f32 rows, whose parts are joined in the kernel and whose ranges by the same one."""
    p, hd, G = 20000, 64, 2
    rng = np.random.default_rng(5)
    bt = packed.Batch([(p, n), (50, 2)], 1, hd, p + 100, rng)
    pools = packed.fill_f32(bt, 3)
    base = rng.normal(0, 1, hd)
    at = bt.row(0, 0, top)
    pools["K"][at:at + hd] = 300.0 * hd ** 0.5 * base / (base @ base)
    at = bt.row(0, 0, low)
    pools["V"][at:at + hd] = np.nan
    r = packed.Run(bt, G, False, 3, packed.random_parents(bt, rng, "random"), pools=pools)
    r.q = (base + 0.1 * rng.normal(0, 1, r.q.shape)).astype(np.float32)
    r.qd.upload(r.q)
    r.call()
    out = r.result()
    assert np.isnan(out[:n]).all()
    assert np.isfinite(out[n:]).all()


# -- f16 below its normal numbers -----------------------------------------------------
def columns_good(r, b, columns):
    c, (p, n) = r.c, r.c.seqs[b]
    tk = np.arange(c.off[b], c.off[b + 1])
    for h in range(c.Hkv):
        q = r.q[tk][:, h * r.G:(h + 1) * r.G].astype(np.float64)
        want, _, _ = pr.attend(q, c.rows(b, "K", h), c.rows(b, "V", h), p, c.hd)
        got = r.result()[tk][:, h * r.G:(h + 1) * r.G]
        err = np.linalg.norm((got - want)[..., columns]) / np.linalg.norm(want[..., columns])
        assert err <= NORM_TOL, (h, err)


@pytest.mark.parametrize("scale", [2.0 ** -16, 2.0 ** -19, 2.0 ** -21])
@pytest.mark.parametrize("hd,G,seq", [(64, 4, (12, 1)), (128, 4, (900, 1)), (128, 4, (900, 5)), (128, 8, (3000, 8)),
                                      (256, 4, (330, 6)), (80, 3, (500, 2))])
def test_small_columns_of_f16(hip, hd, G, seq, scale):
    """Columns of V around and below the smallest normal number, beside ordinary ones, are as good as those."""
    c = Cache([seq, (40, 1)], 2, hd, 16, F16, 0, 11)
    small = np.zeros(hd, bool)
    small[8:16] = small[hd - 3] = small[33] = True
    for b in range(2):
        x = of_type(c.values["V"][b], F16)
        x[..., small] *= scale
        put(c, "V", b, x)
    upload(c)
    r = Attend(c, G)
    r.call()
    r.check()
    for b in range(2):
        columns_good(r, b, small)
        columns_good(r, b, ~small)


@pytest.mark.parametrize("value", [1.0, 6.2e-5, -60000.0])
@pytest.mark.parametrize("p,n,G", [(50, 5, 4), (1000, 3, 8), (20, 2, 40)])
def test_a_draft_does_not_change_small_values_before_it(hip, p, n, G, value):
    """V below the normal numbers, a later draft's above: the tokens before it stay as they were, bit for bit."""
    c = Cache([(p, n)], 1, 128, 16, F16, 0, 12)
    put(c, "V", 0, of_type(c.values["V"][0], F16) * 2.0 ** -21)
    upload(c)
    r = Attend(c, G)
    r.call()
    clean = r.result()
    c.v.upload(with_value(c, "V", 0, p + n - 1, 5, value))
    r.call()
    got = r.result()
    assert np.array_equal(got[:n - 1], clean[:n - 1])
    assert np.array_equal(np.delete(got[n - 1], 5, 1), np.delete(clean[n - 1], 5, 1))


@pytest.mark.parametrize("size,some", [(2.0 ** 16, False), (2.0 ** 20, False), (2.0 ** 22, False), (2.0 ** 16, True)])
@pytest.mark.parametrize("hd,G,seq", [(128, 4, (900, 1)), (128, 4, (900, 5)), (64, 8, (3000, 8)), (256, 4, (330, 6))])
def test_small_keys_of_f16(hip, hd, G, seq, size, some):
    """K below the normal numbers under large queries: scores as good as any.  `some`: in two of three columns; the
    other queries, `size` smaller, are off by at most 2^-38 of the row's largest (4 size), 2^-20 of themselves."""
    c = Cache([seq], 2, hd, 16, F16, 0, 13)
    small = np.ones(hd, bool)
    if some:
        small[::3] = False
    K = of_type(c.values["K"][0], F16)
    K[..., small] /= size
    put(c, "K", 0, K)
    upload(c)
    r = Attend(c, G)
    r.q[..., small] *= np.float32(size)
    r.qd.upload(r.q)
    r.call()
    r.check()


# -- scores of any size ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("p,n,G", [(300, 1, 4), (300, 5, 8), (5000, 3, 4)])
def test_scores_next_to_the_largest(hip, p, n, G, dtype):
    """Sums of |q k| just below 2^126: the key with the largest score is all that counts, so an output is its V."""
    hd = 64
    c = Cache([(p, n)], 1, hd, 16, dtype, 0, 14)
    r = Attend(c, G)
    for seed in range(20):
        rng = np.random.default_rng(seed)
        K = rng.normal(0, 1, (p + n, 1, hd)) * 2.0 ** 60
        put(c, "K", 0, K)
        K = c.rows(0, "K", 0)
        q = rng.normal(0, 1, (n, G, hd))
        most = (np.abs(q) @ np.abs(K).T).max()
        r.q[:n] = (q * (0.99 * 2.0 ** 126 / most)).astype(np.float32)
        s = r.q[:n].astype(np.float64) @ K.T
        for i in range(n):
            s[i, :, p + i + 1:] = -np.inf
        two = np.sort(s, 2)[..., -2:]
        if ((two[..., 1] - two[..., 0]) > 2.0 ** -16 * 2.0 ** 126).all():      # hd 2^-24 of 2^126 is 2^-18 of it
            break
    else:
        raise AssertionError("no inputs away from ties")
    upload(c)
    r.qd.upload(r.q)
    r.call()
    assert np.array_equal(r.result()[:n], c.rows(0, "V", 0)[s.argmax(2)].astype(np.float32))


# -- pages ------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [-1, 25, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("at", [(0, 2), (3, 0), (5, 9)])
def test_trim_refuses_what_is_no_page(hip, at, bad):
    """An entry among those that would go back names no page: refused, and nothing is given back."""
    d, h = DevicePages(6, 10, 25, 4), pr.Pages(6, 10, 25, 4)
    d.reset()
    assert d.extend([3, 0, 5], [0, 0, 0], [9, 12, 40], 99)[0] == 0
    assert h.extend([3, 0, 5], [0, 0, 0], [9, 12, 40], 99)[0] == 0
    table, held, free, n = d.state()
    broken = table.copy()
    broken[at] = bad
    d.load(broken, held, free[:n])
    before = d.state()
    assert d.trim([1, 5, 3, 0], [0, 0, 0, 0]) == -1
    for a, b in zip(before, d.state()):
        assert np.array_equal(a, b)
    keep = [40 if s == at[0] else 4 for s in (5, 3, 0)]        # the entry stays where it is: as before
    assert d.trim([5, 3, 0], keep) == 0 == h.trim([5, 3, 0], keep)
    h.table[at] = bad
    same_pages(d, h)


@pytest.mark.parametrize("B,n", [(1, 100000), (3, 40001), (300, 333)])
def test_trim_of_many_pages(hip, B, n):
    """More pages than the workgroup takes in a round."""
    d, h = DevicePages(B, n // 16 + 1, 9000, 16), pr.Pages(B, n // 16 + 1, 9000, 16)
    d.reset()
    slot = list(range(B))[::-1]
    for p, k in ((0, [n - b % 7 for b in range(B)]), (16, [b % 40 for b in range(B)])):
        assert d.extend(slot, [p] * B, k, 1 << 20)[0] == 0 == h.extend(slot, [p] * B, k, 1 << 20)[0]
        keep = [b % 3 * 16 + b % 2 for b in range(B)]
        assert d.trim(slot, keep) == 0 == h.trim(slot, keep)
        same_pages(d, h)


def test_rows_stored_to_the_same_place(hip):
    """Tokens with one cache row: each of its elements is one of theirs, and nothing else changes."""
    T, Hkv, hd, ps = 40, 3, 64, 4
    d = DevicePages(1, 2, 2, ps)
    pools = [dev(np.zeros(2 * Hkv * ps * hd, np.float32)) for _ in range(2)]
    kv = slate_amd.PagedKv(pools[0].ptr, pools[1].ptr, F32, Hkv, hd, Hkv * ps * hd, ps * hd, hd)
    x = [np.random.default_rng(k).normal(0, 1, (T, Hkv, hd)).astype(np.float32) for k in range(2)]
    rows, src = dev(np.full(T, 5), np.int32), [dev(v) for v in x]
    ok(lib().slate_hip_kv_store_paged(C.byref(kv), d.ref, src[0].p, src[1].p, Hkv * hd, rows.p, T))
    for pool, v in zip(pools, x):
        got = pool.to_array(np.float32, (2, Hkv, ps, hd))
        assert (got[1, :, 1] == v).any(0).all()
        got[1, :, 1] = 0
        assert not got.any()


# -- large vocabularies --------------------------------------------------------------------
@pytest.mark.parametrize("kind,V,chunks", [("probs", 560000, 256), ("plain", 1060000, 512), ("tree", 1060000, 512)])
def test_verify_more_chunks_than_threads(hip, kind, V, chunks):
    """Vocabularies whose chunks of 1024 are summed in several rounds: the next token in the first, a middle and the
    last round, at both ends of u_next, and behind chunks that have no weight."""
    end = np.float32(1.0 - 2.0 ** -24)

    def edit(d, rng):
        for b, place in enumerate((9, chunks * 1024 + 5, V - 2)):
            t = int(d.off[b])
            d.z[t, place:place + 2] = d.z[t].max() + np.float32(6.0)
            d.r[b] = 0.4
        t = int(d.off[3])
        d.z[t, V - 3 * 1024:] = -np.inf
        d.r[3] = end
        t = int(d.off[4])
        d.z[t, :chunks * 1024 + 700] = -np.inf
        d.r[4] = 0.0
        if kind == "probs":
            d.token[t + 1] = 0                         # a banned one: p has gone to the others
        d.u[d.off[:5] + 1] = end                       # drafts are turned down
    d = Drafts([2, 2, 2, 3, 2, 1], V, kind, 15, edit=edit, temps=[1.0] * 6)
    assert [w[1] // (chunks * 1024) for w in d.want[:5]][:3] == [0, 1, (V - 2) // (chunks * 1024)]
    assert d.want[4][1] >= chunks * 1024 + 700 and d.want[3][1] < V - 3 * 1024
    assert all(len(w[0]) == 0 for w in d.want[:5])
    d.call().check()
    d.call(own_ws=True).check()
