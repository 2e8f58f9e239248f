"""The K/V cache in pages: pages taken and given back, rows stored, attention
over them; and the verification of drafted tokens; against 64-bit references
on the host (tests/paged_ref.py).

Tolerances, from the arithmetic of the kernels:
* pages: whole numbers, equal.  Store: the nearest value of the type, equal.
* attention: a score is off by at most (2^-21 + hd 2^-24) A, A the largest sum
  |q_i k_i| / sqrt(hd) (q in 22 bits or more; f32 sums), and by 2^-22 of itself
  when scaled; a weight by twice that and the exponential's 2^-22; sums over
  keys by keys * 2^-24.  Times max |V|.  These are worst cases; the whole
  output is held to 2^-18 in the 2-norm too, as an operand that lost its lower
  half (2^-12) would show there.
* verification: whole numbers, equal, where the reference's decisions are at
  least 2^-18 of their size from their borders and its sums 2^-40 of the whole (an
  exponential is good to 2^-42 of itself, a sum of V to 2^-52 V^(1/2)); inputs are drawn
  until that holds for every sequence.
"""
import ctypes as C
import threading

import numpy as np
import pytest

import slate_amd
from slate_amd import DeviceBuffer
from tests import paged_ref as pr

pytestmark = pytest.mark.gpu
NORM_TOL = 2.0 ** -18
SENTINEL = np.float32(-77.25)
MARK = -777
F32, F16, BF16 = 0, 1, 2
SIZE = {F32: 4, F16: 2, BF16: 2}


def lib():
    return slate_amd.load_library()


def ok(rc, what="call"):
    slate_amd.check(rc, what)


def dev(a, dtype=None):
    return DeviceBuffer.from_array(np.asarray(a, dtype))


def to_type(x, dtype):
    """float32 values as the type's bits, to nearest, ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == F32:
        return x
    if dtype == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def of_type(b, dtype):
    if dtype == BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


# -- pages ------------------------------------------------------------------------
class DevicePages:
    def __init__(self, n_slots, max_pages, n_pages, page_size):
        self.shape, self.n_pages = (n_slots, max_pages), n_pages
        self.t, self.h, self.f, self.n = (DeviceBuffer(4 * k) for k in (n_slots * max_pages, n_slots, n_pages, 1))
        self.c = slate_amd.Pages(self.t.ptr, self.h.ptr, self.f.ptr, self.n.ptr, n_slots, max_pages, n_pages, page_size)

    @property
    def ref(self):
        return C.byref(self.c)

    def reset(self):
        ok(lib().slate_hip_pages_reset(self.ref))

    def state(self):
        return (self.t.to_array(np.int32, self.shape), self.h.to_array(np.int32, self.shape[:1]),
                self.f.to_array(np.int32, self.n_pages), int(self.n.to_array(np.int32, 1)[0]))

    def load(self, table, held, free):
        self.t.upload(table.astype(np.int32))
        self.h.upload(held.astype(np.int32))
        f = np.zeros(self.n_pages, np.int32)
        f[:len(free)] = free
        self.f.upload(f)
        self.n.upload(np.array([len(free)], np.int32))

    def extend(self, slot, pos0, n_new, T_cap, T=None):
        """status and descriptors; the outputs keep MARK where nothing is written."""
        B, T = len(slot), sum(n_new) if T is None else T
        ins = [dev(a, np.int32) for a in (slot, pos0, n_new)]
        outs = [dev(np.full(k, MARK), np.int32) for k in (B + 1, T + 3, T + 3, T + 3, B, 1)]
        ok(lib().slate_hip_pages_extend(self.ref, *[i.p for i in ins], B, T_cap, *[o.p for o in outs]), "extend")
        got = [o.to_array(np.int32, o.nbytes // 4) for o in outs]
        return int(got[5][0]), got[:5]

    def trim(self, slot, length):
        ins, st = [dev(a, np.int32) for a in (slot, length)], dev([MARK], np.int32)
        ok(lib().slate_hip_pages_trim(self.ref, ins[0].p, ins[1].p, len(slot), st.p), "trim")
        return int(st.to_array(np.int32, 1)[0])


def same_pages(d, h):
    table, held, free, n = d.state()
    assert np.array_equal(table, h.table)
    assert np.array_equal(held, h.held)
    assert n == len(h.free) and list(free[:n]) == h.free


def check_extend(d, h, slot, pos0, n_new, cap=1 << 20):
    total = sum(max(0, n) for n in n_new)
    status, got = d.extend(slot, pos0, n_new, cap, total if total <= cap else 0)
    want, desc = h.extend(slot, pos0, n_new, cap)
    assert status == want
    if want:
        assert all((g == MARK).all() for g in got)
    else:
        T = sum(n_new)
        for g, w in zip(got, desc):
            assert np.array_equal(g[:len(w)], w)
        assert all((g[T:] == MARK).all() for g in got[1:4])
    same_pages(d, h)
    return status


@pytest.mark.parametrize("page,n_slots,max_pages,n_pages", [(1, 5, 40, 100), (16, 70, 20, 700), (7, 3, 300, 500),
                                                            (48, 1, 9, 4), (64, 1100, 12, 9000), (256, 33, 64, 2000)])
def test_pages_life(hip, page, n_slots, max_pages, n_pages):
    """Requests come, grow and go; every state and every status as the host's."""
    rng = np.random.default_rng(page)
    d, h = DevicePages(n_slots, max_pages, n_pages, page), pr.Pages(n_slots, max_pages, n_pages, page)
    d.reset()
    same_pages(d, h)
    length = np.zeros(n_slots, np.int64)
    seen = set()
    for step in range(12):
        B = int(rng.integers(1, min(n_slots, 1024) + 1))
        slot = rng.permutation(n_slots)[:B]
        most = max_pages * page - length[slot]
        big = rng.random(B) < 0.1
        n = np.where(big, rng.integers(0, most + 1), np.minimum(rng.integers(0, 2 * page + 2, B), most))
        if step == 5:
            n[-1] = most[-1] + 1
        st = check_extend(d, h, slot.tolist(), length[slot].tolist(), n.tolist())
        seen.add(st)
        if st == 0:
            length[slot] += n
        gone = rng.permutation(n_slots)[:max(1, min(n_slots, 1024) // 2)]
        keep = np.where(rng.random(len(gone)) < 0.5, 0, rng.integers(0, length[gone] + 1))
        assert d.trim(gone.tolist(), keep.tolist()) == h.trim(gone.tolist(), keep.tolist()) == 0
        length[gone] = np.minimum(length[gone], keep)
        same_pages(d, h)
    assert seen >= {0, -2}


def test_pages_refusals(hip):
    d, h = DevicePages(6, 10, 25, 4), pr.Pages(6, 10, 25, 4)
    d.reset()
    assert check_extend(d, h, [3, 0, 5], [0, 0, 0], [9, 0, 40]) == 0
    for slot, pos0, n in (([3, 3], [9, 9], [1, 1]), ([6], [0], [1]), ([-1], [0], [1]), ([1], [-1], [2]),
                          ([1], [0], [-1]), ([0, 1, 2, 3, 4, 0], [0] * 6, [0] * 6)):
        assert check_extend(d, h, slot, pos0, n) == -1
    for slot, pos0, n in (([1], [0], [41]), ([1], [2147483647], [2147483647]), ([1, 2], [0, 0], [40, 13]),
                          ([0, 1, 2], [2147483647, 0, 5], [1, 2147483647, 2147483647])):
        assert check_extend(d, h, slot, pos0, n) == -2
    assert check_extend(d, h, [1, 2], [0, 0], [5, 6], 10) == -2                  # T_cap
    assert check_extend(d, h, [1, 2], [0, 0], [5, 6], 11) == 0
    assert check_extend(d, h, [1, 2], [5, 6], [0, 0], 0) == 0
    for slot, n in (([3, 3], [1, 1]), ([6], [0]), ([-1], [0]), ([0], [-1])):
        assert d.trim(slot, n) == h.trim(slot, n) == -1
        same_pages(d, h)
    assert d.trim([0, 3, 5], [5, 2147483647, 39]) == 0                           # longer than held, nothing, nothing
    same_pages(d, h)
    # state that cannot be: refused, nothing written
    table, held, free, n = d.state()
    for what, v in ((d.n, [-1]), (d.n, [26]), (d.h, [11, 0, 0, 0, 0, 0]), (d.h, [-1, 0, 0, 0, 0, 0])):
        d.load(table, held, free[:n])
        what.upload(np.array(v, np.int32))
        assert d.extend([0], [0], [1], 9)[0] == -1
        assert d.trim([0], [0]) == -1
    # a stack that would hold more pages than there are
    d.load(table, held, np.arange(25))
    assert d.trim([3], [0]) == -1
    # an entry that names no page: its rows are -1
    d.load(np.where(table < 0, table, 25), held, free[:n])
    st, got = d.extend([3], [1], [4], 9)
    assert st == 0 and list(got[3][:4]) == [-1] * 4


def test_pages_extend_then_trim_restores(hip):
    d = DevicePages(70, 30, 900, 16)
    rng = np.random.default_rng(1)
    d.load(np.full((70, 30), -1), np.zeros(70), rng.permutation(900))
    pos = rng.integers(0, 200, 64)
    slot = rng.permutation(70)[:64]
    assert d.extend(slot, [0] * 64, pos, 1 << 20)[0] == 0
    before = d.state()
    assert d.extend(slot, pos, rng.integers(0, 60, 64), 1 << 20)[0] == 0
    assert d.trim(slot, pos) == 0
    after = d.state()
    for a, b in zip(before, after):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("B,n", [(1, 100000), (3, 40001), (1024, 100)])
def test_pages_many_tokens(hip, B, n):
    d, h = DevicePages(B, n // 16 + 1, 9000, 16), pr.Pages(B, n // 16 + 1, 9000, 16)
    d.reset()
    assert check_extend(d, h, list(range(B))[::-1], [0] * B, [n - b % 7 for b in range(B)]) == 0


def test_pages_without_a_limit_on_tokens(hip):
    """T_cap as large as it can be: the call takes what the tokens need."""
    d, h = DevicePages(3, 400, 900, 16), pr.Pages(3, 400, 900, 16)
    d.reset()
    assert check_extend(d, h, [2, 0], [0, 0], [5000, 37], 2 ** 31 - 1) == 0
    assert check_extend(d, h, [2, 1], [5000, 0], [0, 0], 2 ** 31 - 1) == 0


def test_pages_of_a_slot_in_one(hip):
    """One page that is as long as a slot can be: counts of rows next to 2^31."""
    most = 2 ** 31 - 1024
    d = DevicePages(2, 1, 1, most)
    d.load(np.full((2, 1), -1), np.zeros(2), [0])
    assert d.extend([1], [most - 3], [4], 9, 4)[0] == -2
    st, got = d.extend([1], [most - 3], [3], 9, 3)
    assert st == 0 and list(got[3][:3]) == [most - 3, most - 2, most - 1]
    table, held, free, n = d.state()
    assert table[1, 0] == 0 and list(held) == [0, 1] and n == 0
    assert d.trim([1], [2 ** 31 - 1]) == 0 and d.state()[3] == 0
    assert d.trim([1], [0]) == 0 and d.state()[3] == 1


# -- a cache ------------------------------------------------------------------------
class Cache:
    """Pools of n_pages pages in shuffled order behind a table; rows that no sequence has cached hold NaN and
    infinities.  layout 0: [page, head, row], 1: [page, row, head], 2: [head, page, row] with gaps."""

    def __init__(self, seqs, Hkv, hd, page, dtype, layout, seed, spare=2, scale=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.Hkv, self.hd, self.ps, self.dtype = seqs, Hkv, hd, page, dtype
        B = self.B = len(seqs)
        need = [-(-(p + n) // page) for p, n in seqs]
        self.n_pages = sum(need) + 3
        most = max(max(need), 1) + spare
        self.d = DevicePages(B + 2, most, self.n_pages, page)
        self.slot = rng.permutation(B + 2)[:B].astype(np.int32)
        self.table = np.full((B + 2, most), -1, np.int32)
        order = rng.permutation(self.n_pages)
        at = 0
        for s, k in zip(self.slot, need):
            self.table[s, :k] = order[at:at + k]
            at += k
        self.d.load(self.table, np.zeros(B + 2), order[at:])
        self.strides = {0: (Hkv * page * hd, page * hd, hd), 1: (Hkv * page * hd, hd, Hkv * hd),
                        2: (page * (hd + 8) + 16, self.n_pages * (page * (hd + 8) + 16) + 24, hd + 8)}[layout]
        ps_, hs_, rs_ = self.strides
        self.elems = (self.n_pages - 1) * ps_ + (Hkv - 1) * hs_ + (page - 1) * rs_ + hd
        self.off = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        self.T = int(self.off[-1])
        self.pools, self.values = {}, {}
        for name in "KV":
            raw = rng.choice(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), self.elems)
            buf = to_type(raw, dtype)
            vals = []
            for b, (p, n) in enumerate(seqs):
                x = to_type(rng.normal(0, scale, (p + n, Hkv, hd)).astype(np.float32), dtype)
                vals.append(x)
                buf[self.where(b, np.arange(p + n))] = x
            self.pools[name], self.values[name] = buf, vals
        self.upload()

    def where(self, b, rows):
        """Elements [rows, Hkv, hd] of a sequence's cache rows."""
        ps_, hs_, rs_ = self.strides
        page = self.table[self.slot[b], rows // self.ps].astype(np.int64)
        first = page * ps_ + rows % self.ps * rs_
        return first[:, None, None] + np.arange(self.Hkv)[:, None] * hs_ + np.arange(self.hd)

    def upload(self):
        self.k, self.v = (DeviceBuffer.from_array(self.pools[n]) for n in "KV")
        self.kv = slate_amd.PagedKv(self.k.ptr, self.v.ptr, self.dtype, self.Hkv, self.hd, *self.strides)
        self.d_slot, self.d_off = dev(self.slot), dev(self.off)
        self.d_pos = dev([p for p, _ in self.seqs], np.int32)

    def rows(self, b, name, h):
        return of_type(self.values[name][b][:, h], self.dtype)


class Attend:
    def __init__(self, c, G, behind=2, seed=1):
        self.c, self.G, self.T = c, G, c.T + behind
        rng = np.random.default_rng(seed)
        self.q = rng.normal(0, 1, (self.T, c.Hkv * G, c.hd)).astype(np.float32)
        self.qd, self.out = DeviceBuffer.from_array(self.q), DeviceBuffer.from_array(np.full_like(self.q, SENTINEL))
        self.need = lib().slate_hip_attention_paged_bytes(c.Hkv * G, c.Hkv, c.hd)
        self.ws = DeviceBuffer(max(self.need, 16))

    def call(self, own_ws=False, max_new=None):
        c = self.c
        mx = max_new or max(1, max(n for _, n in c.seqs))
        ok(lib().slate_hip_attention_paged(self.out.p, self.qd.p, C.byref(c.kv), c.d.ref, c.d_slot.p, c.d_off.p,
                                           c.d_pos.p, c.B, self.T, mx, c.Hkv * self.G,
                                           self.ws.p if own_ws else None, max(self.need, 16)), "attention_paged")

    def result(self):
        return self.out.to_array(np.float32, self.q.shape)

    def check(self, left_out=(), norm=True):
        c, G, out = self.c, self.G, self.result()
        owned = np.zeros(self.T, bool)
        num = den = 0.0
        for b, (p, n) in enumerate(c.seqs):
            tk = np.arange(c.off[b], c.off[b + 1])
            if b in left_out or n == 0:
                continue
            owned[tk] = True
            for h in range(c.Hkv):
                K, V = c.rows(b, "K", h), c.rows(b, "V", h)
                want, A, top = pr.attend(self.q[tk][:, h * G:(h + 1) * G].astype(np.float64), K, V, p, c.hd)
                got = out[tk][:, h * G:(h + 1) * G].astype(np.float64)
                tol = 2 * ((2.0 ** -21 + c.hd * 2.0 ** -24) * A + 2.0 ** -22 * top) + 2.0 ** -22 + (p + n) * 2.0 ** -24
                assert np.isfinite(got).all(), (b, h)
                err = np.abs(got - want).max() / np.abs(V).max()
                assert err <= tol, (b, h, err, tol)
                num += ((got - want) ** 2).sum()
                den += (want ** 2).sum()
        if norm and den:
            assert (num / den) ** 0.5 <= NORM_TOL, (num / den) ** 0.5
        assert np.all(out[~owned] == SENTINEL)


# -- store ----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("Hkv,hd,page,T", [(1, 8, 1, 5), (8, 128, 16, 77), (3, 80, 7, 130), (2, 256, 64, 33),
                                           (5, 64, 48, 1100)])
def test_store(hip, dtype, layout, Hkv, hd, page, T):
    rng = np.random.default_rng(hd + T)
    c = Cache([(T + 9, 0), (3, 1)], Hkv, hd, page, dtype, layout, 3)
    ld = Hkv * hd + 4
    x = {}
    for name in "KV":
        # all magnitudes: subnormals and overflow of the types, ties, both zeros, NaN, infinities
        v = rng.normal(0, 1, (T, ld)) * 2.0 ** rng.integers(-30, 30, (T, ld))
        v[rng.random((T, ld)) < 0.05] = rng.choice([0.0, -0.0, np.nan, np.inf, -np.inf, 65519.9, 65520.0, 2.0 ** -25, 3e38,
                                                    1 + 2.0 ** -9, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11])
        x[name] = v.astype(np.float32)
    at = rng.permutation(T + 9)[:T]                    # cache rows of the first sequence, in any order
    row = c.table[c.slot[0], at // page] * page + at % page
    skip = rng.random(T) < 0.2
    row = np.where(skip, rng.choice([-1, -2 ** 31, c.n_pages * page, 2 ** 31 - 1], T), row).astype(np.int32)
    bufs = [dev(x["K"]), dev(x["V"]), dev(row)]
    ok(lib().slate_hip_kv_store_paged(C.byref(c.kv), c.d.ref, bufs[0].p, bufs[1].p, ld, bufs[2].p, T))
    for name, buf in (("K", c.k), ("V", c.v)):
        want = c.pools[name].copy()
        cells = c.where(0, at[~skip])
        want[cells] = to_type(x[name][~skip][:, :Hkv * hd].reshape(-1, Hkv, hd), dtype)
        got = buf.to_array(want.dtype, want.shape)
        if dtype == BF16:
            got, want = ((a.astype(np.uint32) << 16).view(np.float32) for a in (got, want))
        both = np.isnan(got) & np.isnan(want)
        assert np.all(both | (got.view(np.uint16 if dtype == F16 else np.uint32) ==
                              want.view(np.uint16 if dtype == F16 else np.uint32)))


def test_store_more_rows_than_workgroups(hip):
    T, hd = 70001, 8
    rng = np.random.default_rng(4)
    d = DevicePages(1, 1, 40, 2048)
    pools = [dev(np.zeros(40 * 2048 * hd, np.uint16)) for _ in range(2)]
    kv = slate_amd.PagedKv(pools[0].ptr, pools[1].ptr, BF16, 1, hd, 2048 * hd, 0, hd)
    x = [rng.normal(0, 1, (T, hd)).astype(np.float32) for _ in range(2)]
    row = rng.permutation(40 * 2048)[:T].astype(np.int32)
    bufs = [dev(x[0]), dev(x[1]), dev(row)]
    ok(lib().slate_hip_kv_store_paged(C.byref(kv), d.ref, bufs[0].p, bufs[1].p, hd, bufs[2].p, T))
    for pool, v in zip(pools, x):
        want = np.zeros((40 * 2048, hd), np.uint16)
        want[row] = to_type(v, BF16)
        assert np.array_equal(pool.to_array(np.uint16, want.shape), want)


# -- attention --------------------------------------------------------------------------
DECODE = [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (31, 1), (32, 1), (33, 1), (127, 1), (255, 1), (256, 1), (700, 1),
          (1299, 1)]
DRAFTS = [(0, 1), (0, 5), (27, 5), (30, 4), (31, 2), (0, 0), (126, 5), (127, 3), (128, 5), (600, 1), (1290, 5)]
CHUNKS = [(0, 70), (5, 15), (0, 16), (17, 17), (300, 33), (64, 1), (650, 130), (3, 0), (0, 5)]
SHAPES = [(64, 2, 4), (128, 2, 4), (128, 1, 8), (128, 1, 7), (128, 2, 1), (256, 1, 4), (32, 2, 1), (8, 1, 3), (80, 2, 3),
          (96, 1, 2), (200, 1, 5), (128, 1, 16), (64, 1, 20), (40, 1, 40)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,Hkv,G", SHAPES)
@pytest.mark.parametrize("kind", ["decode", "drafts", "chunks"])
def test_attention(hip, hd, Hkv, G, dtype, kind):
    seqs = {"decode": DECODE, "drafts": DRAFTS, "chunks": CHUNKS}[kind]
    pages = {"decode": 16, "drafts": 32, "chunks": 64}
    r = Attend(Cache(seqs, Hkv, hd, pages[kind], dtype, (hd // 8 + dtype) % 3, hd + G), G)
    r.call()
    r.check()
    r.out.upload(np.full_like(r.q, SENTINEL))
    r.call(own_ws=True)
    r.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [1, 3, 8, 12, 16, 24, 40, 48, 64, 100, 128, 1000])
@pytest.mark.parametrize("layout", [0, 1, 2])
def test_attention_page_sizes(hip, page, dtype, layout):
    r = Attend(Cache(DRAFTS, 2, 64, page, dtype, layout, page), 3)
    r.call()
    r.check()


@pytest.mark.parametrize("B", [1, 64, 65, 200, 1024])
def test_attention_many_sequences(hip, B):
    rng = np.random.default_rng(B)
    seqs = [(int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(B - 1)] + [(37, 2)]
    r = Attend(Cache(seqs, 1, 64, 8, BF16, 0, B), 4)
    r.call()
    r.check()


@pytest.mark.parametrize("dtype,page", [(F32, 16), (F16, 64), (BF16, 16), (BF16, 20)])
@pytest.mark.parametrize("hd,n", [(128, 1), (128, 7), (64, 3), (256, 1)])
def test_attention_long(hip, dtype, page, hd, n):
    """One long context beside short ones: the long ones are split over workgroups and joined."""
    r = Attend(Cache([(20000, n), (3, 1), (0, 1), (9001, n), (513, n)], 2, hd, page, dtype, 0, 1), 4)
    r.call()
    r.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_left_out(hip, dtype):
    """Sequences whose numbers do not fit, and queries behind the last one, stay as they are."""
    seqs = [(40, 2), (100, 3), (7, 1), (0, 2), (300, 2), (55, 1)]
    r = Attend(Cache(seqs, 2, 128, 16, dtype, 0, 5), 4, behind=5)
    c = r.c
    slot, pos = c.slot.copy(), np.array([p for p, _ in seqs], np.int32)
    slot[0], pos[1], pos[4] = len(c.table), -1, c.table.shape[1] * 16 - 1
    c.d_slot.upload(slot)
    c.d_pos.upload(pos)
    r.call(max_new=2)
    r.check(left_out=(0, 1, 4))
    slot[0], slot[2] = c.slot[0], -1
    c.d_slot.upload(slot)
    r.call(max_new=3)
    r.check(left_out=(1, 4))                           # the third sequence keeps what it had
    # a fall of tok_off: what lies before it is answered
    off = c.off.copy()
    off[4] = 3
    c.d_off.upload(off)
    c.d_slot.upload(c.slot)
    c.d_pos.upload(np.array([p for p, _ in seqs], np.int32))
    r.out.upload(np.full_like(r.q, SENTINEL))
    r.call(max_new=3)
    got = r.result()
    r.c.d_off.upload(c.off)
    r.out.upload(np.full_like(r.q, SENTINEL))
    r.call(max_new=3)
    assert np.array_equal(got[:6], r.result()[:6])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page,n", [(16, 1), (16, 6), (64, 6), (12, 3)])
def test_attention_bad_pages(hip, dtype, page, n):
    """Keys in pages that the table does not name count as not seen; a token that sees none gets zeros."""
    seqs = [(200, n), (30, n), (0, n), (1000, n)]
    c = Cache(seqs, 2, 64, page, dtype, 0, 6)
    r = Attend(c, 2)
    bad = c.table.copy()
    holes = {0: [1, 3], 1: list(range(c.table.shape[1])), 3: [0, 7]}
    for b, pages in holes.items():
        bad[c.slot[b], pages] = [(-1, c.n_pages, -2 ** 31, 2 ** 31 - 1)[i % 4] for i in range(len(pages))]
    c.d.t.upload(bad)
    r.call()
    out = r.result()
    for b, (p, n_) in enumerate(seqs):
        seen = np.array([i // page not in holes.get(b, []) for i in range(p + n_)])
        for i in range(n_):
            for h in range(2):
                got = out[c.off[b] + i, 2 * h:2 * h + 2].astype(np.float64)
                rows = np.nonzero(seen[:p + i + 1])[0]
                if not len(rows):
                    assert np.all(got == 0)
                    continue
                K, V = c.rows(b, "K", h)[rows], c.rows(b, "V", h)[rows]
                q = r.q[c.off[b] + i, 2 * h:2 * h + 2].astype(np.float64)[None]
                want, A, top = pr.attend(q, K, V, len(rows) - 1, 64)
                tol = 2 * ((2.0 ** -21 + 64 * 2.0 ** -24) * A + 2.0 ** -22 * top) + 2.0 ** -22 + len(rows) * 2.0 ** -24
                assert np.abs(got - want[0]).max() <= tol * np.abs(V).max()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("p,n,G", [(50, 5, 1), (0, 6, 4), (127, 9, 3), (1000, 4, 8)])
def test_attention_values_not_finite(hip, dtype, what, p, n, G):
    """A draft's K or V that is not finite does not reach the tokens before it, and reaches its own and later ones."""
    c = Cache([(p, n), (33, 1)], 1, 64, 16, dtype, 0, 7)
    r = Attend(c, G)
    r.call()
    clean = r.result()
    at = n // 2
    for name, buf in (("K", c.k), ("V", c.v)):
        pool = c.pools[name].copy()
        pool[c.where(0, np.array([p + at]))[0, 0, 5]] = to_type(np.array([what], np.float32), dtype)[0]
        buf.upload(pool)
        r.call()
        got = r.result()
        assert np.array_equal(got[:at], clean[:at]), name
        assert np.array_equal(got[n:], clean[n:]), name
        late = got[at:n]
        if name == "V":
            assert not np.isfinite(late[:, :, 5]).any()
            assert np.array_equal(np.delete(late, 5, 2), np.delete(clean[at:n], 5, 2))
        elif np.isnan(what):
            assert np.isnan(late).all()
        buf.upload(c.pools[name])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("row", [0, 5, 200, 511, 900])
def test_attention_committed_value_not_finite(hip, dtype, row):
    c = Cache([(900, 3)], 1, 128, 16, dtype, 1, 8)
    r = Attend(c, 4)
    r.call()
    clean = r.result()
    pool = c.pools["V"].copy()
    pool[c.where(0, np.array([row]))[0, 0, 77]] = to_type(np.array([np.nan], np.float32), dtype)[0]
    c.v.upload(pool)
    r.call()
    got = r.result()[:3]
    assert np.isnan(got[:, :, 77]).all()
    assert np.array_equal(np.delete(got, 77, 2), np.delete(clean[:3], 77, 2))


@pytest.mark.parametrize("dtype,scale", [(F32, 1e-30), (F32, 1e18), (F16, 2e-7), (F16, 6000.0), (BF16, 1e-30),
                                         (BF16, 1e18)])
@pytest.mark.parametrize("n", [1, 6])
def test_attention_v_of_any_size(hip, dtype, scale, n):
    """V far from 1, and rows of it far from each other: the outputs go by the weights, whatever V's size is."""
    c = Cache([(700, n), (12, n)], 1, 128, 16, dtype, 0, 9)
    for b in range(2):
        x = of_type(c.values["V"][b], dtype) * scale
        x[::3] *= 2.0 ** -6
        c.values["V"][b] = to_type(x.astype(np.float32), dtype)
        c.pools["V"][c.where(b, np.arange(sum(c.seqs[b])))] = c.values["V"][b]
    c.v.upload(c.pools["V"])
    r = Attend(c, 4)
    r.call()
    r.check()


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("scale", [1e-7, 1e-6, 1e-5, 1e-4])
@pytest.mark.parametrize("seq", [(12, 1), (330, 5), (1700, 1), (700, 16)])
def test_attention_v_below_normal(hip, seq, scale, seed):
    """V in f16 around and below its normal numbers: as good as any, each sequence by itself."""
    c = Cache([seq], 2, 128, 16, F16, 0, seed)
    c.values["V"][0] = to_type((of_type(c.values["V"][0], F16) * scale).astype(np.float32), F16)
    c.pools["V"][c.where(0, np.arange(sum(seq)))] = c.values["V"][0]
    c.v.upload(c.pools["V"])
    r = Attend(c, 4)
    r.call()
    r.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [1.0, 2.0 ** -20])
@pytest.mark.parametrize("score", [8.0, 12.3, 13.6, 15.1])
def test_attention_many_small_weights(hip, dtype, v, score):
    """One key far above 16000 that weigh alike: their weights' roundings all go the same way."""
    c = Cache([(16000, 1)], 1, 128, 16, dtype, 0, 4)
    r = Attend(c, 1)
    q = r.q[0, 0].astype(np.float64)
    K, V = np.zeros((16001, 1, 128)), np.full((16001, 1, 128), v)
    K[5, 0] = score * 128 ** 0.5 * q / (q @ q)
    V[5, 0] = -3 * v
    for name, x in (("K", K), ("V", V)):
        c.values[name][0] = to_type(x.astype(np.float32), dtype)
        c.pools[name][c.where(0, np.arange(16001))] = c.values[name][0]
    c.k.upload(c.pools["K"])
    c.v.upload(c.pools["V"])
    r.call()
    r.check()


@pytest.mark.parametrize("spare", [0, 1])
@pytest.mark.parametrize("dtype,Hkv,hd,G,n,B", [(BF16, 8, 64, 1, 1, 70), (F16, 2, 128, 4, 1, 3), (F32, 1, 64, 8, 5, 9),
                                                (BF16, 1, 256, 4, 9, 5), (F16, 16, 64, 2, 1, 50)])
def test_attention_slots_of_1024_rows(hip, dtype, Hkv, hd, G, n, B, spare):
    """Slots of 1024 rows and of a page more, full and nearly empty ones, more blocks than workgroups and fewer."""
    rng = np.random.default_rng(B)
    seqs = [(1024 - n, n)] + [(int(rng.choice([0, 1, 127, 128, 900, 1024 - n])), n) for _ in range(B - 1)]
    r = Attend(Cache(seqs, Hkv, hd, 16, dtype, 0, 3, spare=spare), G)
    assert r.c.d.shape[1] == 64 + spare
    r.call()
    r.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [2.0 ** -12, 30.0])
def test_attention_scores_of_any_size(hip, dtype, scale):
    """Scores near 0 (all weights alike) and in the hundreds (one key takes all)."""
    c = Cache([(700, 5), (12, 2), (4000, 1)], 2, 128, 16, dtype, 0, 10)
    r = Attend(c, 4)
    r.q *= np.float32(scale)
    r.qd.upload(r.q)
    r.call()
    r.check(norm=scale < 1)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_attention_small_columns(hip, dtype):
    """Columns of V 2^-12 of the largest: each is good to the weights' 2^-34 of the largest weight times itself."""
    c = Cache([(900, 5)], 1, 64, 16, dtype, 0, 11)
    x = of_type(c.values["V"][0], dtype)
    x[..., 8:16] *= 2.0 ** -12
    c.values["V"][0] = to_type(x.astype(np.float32), dtype)
    c.pools["V"][c.where(0, np.arange(905))] = c.values["V"][0]
    c.v.upload(c.pools["V"])
    r = Attend(c, 4)
    r.call()
    r.check()
    want, A, top = pr.attend(r.q[:5].astype(np.float64), c.rows(0, "K", 0), c.rows(0, "V", 0), 900, 64)
    err = np.abs(r.result()[:5, :, 8:16] - want[..., 8:16]).max()
    tol = 2 * ((2.0 ** -21 + 64 * 2.0 ** -24) * A + 2.0 ** -22 * top) + 2.0 ** -22 + 905 * 2.0 ** -24
    assert err <= tol * np.abs(c.rows(0, "V", 0)[:, 8:16]).max()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_offsets_past_32_bits(hip, dtype):
    """Pages 2^29 elements apart: the last one starts past 2^31 elements (and 2^32 bytes)."""
    ps, hd, Hkv, G, n_pages = 32, 64, 2, 4, 6
    stride = 1 << 29
    rng = np.random.default_rng(12)
    pools = [DeviceBuffer(SIZE[dtype] * (stride * (n_pages - 1) + Hkv * ps * hd)) for _ in range(2)]
    d = DevicePages(1, n_pages, n_pages, ps)
    d.load(rng.permutation(n_pages)[None], np.array([n_pages]), [])
    table = d.state()[0][0]
    L = ps * n_pages - 3
    vals = [rng.normal(0, 1, (L, Hkv, hd)).astype(np.float32) for _ in range(2)]
    kv = slate_amd.PagedKv(pools[0].ptr, pools[1].ptr, dtype, Hkv, hd, stride, ps * hd, hd)
    rows = dev(table[np.arange(L) // ps] * ps + np.arange(L) % ps, np.int32)
    src = [dev(v) for v in vals]
    ok(lib().slate_hip_kv_store_paged(C.byref(kv), d.ref, src[0].p, src[1].p, Hkv * hd, rows.p, L))
    q = rng.normal(0, 1, (2, Hkv * G, hd)).astype(np.float32)
    qd, out = dev(q), DeviceBuffer(q.nbytes)
    bufs = [dev([0], np.int32), dev([0, 2], np.int32), dev([L - 2], np.int32)]
    ok(lib().slate_hip_attention_paged(out.p, qd.p, C.byref(kv), d.ref, *[b.p for b in bufs], 1, 2, 2, Hkv * G, None, 0))
    got = out.to_array(np.float32, q.shape)
    for h in range(Hkv):
        K, V = (of_type(to_type(v[:, h], dtype), dtype) for v in vals)
        want, A, top = pr.attend(q[:, h * G:(h + 1) * G].astype(np.float64), K, V, L - 2, hd)
        assert np.abs(got[:, h * G:(h + 1) * G] - want).max() <= 2.0 ** -17 * np.abs(V).max()


def test_attention_shared_pages(hip):
    """Two sequences over the same slot, and two slots that share a prefix's pages."""
    c = Cache([(100, 1), (100, 1), (64, 2)], 2, 64, 16, F16, 0, 13)
    c.slot[1] = c.slot[0]
    c.table[c.slot[2], :4] = c.table[c.slot[0], :4]
    c.d.t.upload(c.table)
    c.d_slot.upload(c.slot)
    c.values["K"][1], c.values["V"][1] = c.values["K"][0], c.values["V"][0]
    for name, buf in (("K", c.k), ("V", c.v)):
        c.values[name][2][:64] = c.values[name][0][:64]
    r = Attend(c, 4)
    r.call()
    r.check()


def test_attention_workspace_content(hip):
    c = Cache([(5000, 3), (40, 1)], 2, 128, 16, BF16, 0, 14)
    r = Attend(c, 4)
    for fill in (0, 255, 127):
        r.ws.upload(np.full(max(r.need, 16), fill, np.uint8))
        r.out.upload(np.full_like(r.q, SENTINEL))
        r.call(own_ws=True)
        r.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_is_the_same_every_time(hip, dtype):
    """The order of sums goes by the lengths alone; and several threads call it at once."""
    c = Cache([(5000, 5), (40, 1), (0, 3), (777, 2)], 2, 128, 16, dtype, 0, 21)
    r = Attend(c, 8)
    r.call()
    r.check()
    first = r.result()
    others = [Attend(c, 8) for _ in range(3)]

    def work(o):
        for _ in range(8):
            o.call()
    threads = [threading.Thread(target=work, args=(o,)) for o in others]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for o in others:
        assert np.array_equal(o.result().view(np.uint32), first.view(np.uint32))


# -- verification -----------------------------------------------------------------------
class Drafts:
    """A batch of drafts on host and device; near() says how far the reference keeps from its borders."""

    def __init__(self, counts, V, kind, seed, ld=None, temps=None, edit=None, scale=3.0):
        self.counts, self.V, self.kind, self.ld = counts, V, kind, ld or V
        self.off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.T, self.B = int(self.off[-1]), len(counts)
        for attempt in range(50):
            self.make(np.random.default_rng([seed, attempt]), temps, edit, scale)
            self.want = [self.one(b) for b in range(self.B)]
            if all(w is None or (w[2][0] > 2.0 ** -18 and w[2][1] > 2.0 ** -40) for w in self.want):
                break
        else:
            raise AssertionError("no inputs away from the borders")

    def make(self, rng, temps, edit, scale):
        T, V, B = self.T, self.V, self.B
        self.z = rng.normal(0, scale, (T, V)).astype(np.float32)
        self.z[np.arange(T)[:, None], rng.integers(0, V, (T, 3))] += np.float32(4 * scale)
        self.parent = np.full(T, -1, np.int32)
        for b, k in enumerate(self.counts):
            for i in range(1, k):
                self.parent[self.off[b] + i] = rng.integers(max(0, i - 3), i) if self.kind == "tree" else i - 1
        up = np.maximum(self.parent, 0) + np.repeat(self.off[:-1], self.counts)
        guess = self.z[up] + rng.normal(0, 0.3 * scale, (T, V)).astype(np.float32)
        e = np.exp(guess - guess.max(1, keepdims=True))
        self.q = (e / e.sum(1, keepdims=True)).astype(np.float32)
        self.token = np.array([rng.choice(V, p=p / p.sum()) for p in self.q.astype(np.float64)], np.int32)
        self.temps = np.array(temps if temps is not None else rng.choice([0.0, 0.5, 0.8, 1.0, 1.0, 2.0], B), np.float32)
        self.u, self.r = rng.random(T).astype(np.float32), rng.random(B).astype(np.float32)
        if edit:
            edit(self, rng)

    def one(self, b):
        k, t = self.counts[b], int(self.off[b])
        if k == 0:
            return None
        s = slice(t, t + k)
        return pr.verify(self.z[s], self.token[s], self.parent[s], self.q[s] if self.kind == "probs" else None,
                         self.temps[b], self.u[s], self.r[b])

    def call(self, own_ws=False, rows=True, behind=2):
        T = self.T + behind
        zp = np.full((T, self.ld), np.nan, np.float32)
        zp[:self.T, :self.V] = self.z
        qp = np.full((T, self.ld), np.nan, np.float32)
        qp[:self.T, :self.V] = self.q
        self.bufs = [dev(zp), dev(np.concatenate([self.token, np.zeros(behind, np.int32)])),
                     dev(np.concatenate([self.parent, np.zeros(behind, np.int32)])), dev(qp), dev(self.temps),
                     dev(np.concatenate([self.u, np.zeros(behind, np.float32)])), dev(self.r), dev(self.off)]
        z, tok, par, q, temp, u, r, off = [x.p for x in self.bufs]
        self.outs = [dev(np.full(k, MARK), np.int32) for k in (self.B, T, T)]
        need = lib().slate_hip_verify_drafts_bytes(self.B, T, self.V)
        self.ws = DeviceBuffer(max(need, 16))
        self.fn = lambda ws: ok(lib().slate_hip_verify_drafts(
            self.outs[0].p, self.outs[1].p, self.outs[2].p if rows else None, z, self.ld, tok,
            par if self.kind == "tree" else None, q if self.kind == "probs" else None, self.ld, temp, u, r, off,
            self.B, T, self.V, ws, max(need, 16)), "verify_drafts")
        self.fn(self.ws.p if own_ws else None)
        return self

    def check(self, rows=True):
        n_acc, tok, row = (o.to_array(np.int32, o.nbytes // 4) for o in self.outs)
        for b, w in enumerate(self.want):
            t, k = int(self.off[b]), self.counts[b]
            if w is None:
                assert n_acc[b] == -1
                continue
            path, nxt = w[0], w[1]
            m = len(path)
            assert n_acc[b] == m, (b, n_acc[b], path)
            assert list(tok[t:t + k]) == [self.token[t + i] for i in path] + [nxt] + [-1] * (k - m - 1), b
            if rows:
                assert list(row[t:t + k]) == path + [-1] * (k - m), b
        assert np.all(tok[self.T:] == MARK) and np.all(row[self.T if rows else 0:] == MARK)


SIZES = [1, 2, 5, 63, 64, 65, 255, 257, 1000, 1024, 4095, 4097, 16385, 32000]


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
@pytest.mark.parametrize("V", SIZES)
def test_verify(hip, V, kind):
    d = Drafts([5, 1, 0, 3, 9, 2, 1, 6], V, kind, V)
    d.call().check()
    d.call(own_ws=True, rows=False).check(rows=False)


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
def test_verify_large_vocabulary(hip, kind):
    Drafts([5, 4, 5, 1, 8, 3], 128256, kind, 5).call().check()


@pytest.mark.parametrize("kind", ["probs", "tree"])
@pytest.mark.parametrize("B", [1, 64, 65, 300, 1024])
def test_verify_many_sequences(hip, B, kind):
    rng = np.random.default_rng(B)
    Drafts([int(k) for k in rng.integers(0, 5, B - 1)] + [4], 97, kind, B).call().check()


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
def test_verify_one_long_draft(hip, kind):
    Drafts([300, 2], 50, kind, 6).call().check()


def test_verify_most_drafts(hip):
    """1024 drafts are taken, one more is not."""
    d = Drafts([1025, 2, 1026, 3], 12, "plain", 14, scale=0.3, temps=[3, 1, 1, 1],
               edit=lambda d, rng: d.u.__imul__(np.float32(0.02)))
    d.want[2] = None
    d.call().check()
    assert len(d.want[0][0]) > 70                      # over more than a wave's lanes
    d = Drafts([1025, 1], 12, "tree", 14, scale=0.3, temps=[3, 1])
    d.call().check()


def test_verify_at_the_border(hip):
    """u q equal to p turns a draft down: two tokens of 1/2 each, q 1/2 and 1 (numbers without rounding)."""
    V, B = 2, 4
    z = dev(np.zeros((2 * B, V), np.float32))
    tok = dev(np.tile([0, 1], B), np.int32)
    q = dev(np.tile(np.array([[0.5, 0.5], [0.0, 1.0]], np.float32), (B, 1)))
    u = np.zeros(2 * B, np.float32)
    u[1::2] = [0.5, np.nextafter(np.float32(0.5), np.float32(0)), 0.25, 0.0]
    r = dev(np.full(B, 0.9, np.float32))
    ud, off = dev(u), dev(np.arange(0, 2 * B + 1, 2), np.int32)
    for probs in (q.p, None):
        outs = [DeviceBuffer(4 * B), DeviceBuffer(8 * B)]
        ok(lib().slate_hip_verify_drafts(outs[0].p, outs[1].p, None, z.p, V, tok.p, None, probs, V, None, ud.p, r.p, off.p,
                                         B, 2 * B, V, None, 0))
        assert list(outs[0].to_array(np.int32, B)) == [0, 1, 1, 1]
        assert list(outs[1].to_array(np.int32, (B, 2))[0]) == [0, -1]      # what is left is the other token


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
@pytest.mark.parametrize("extra", [1, 2, 3, 61])
def test_verify_rows_apart(hip, kind, extra):
    Drafts([3, 4, 1, 2], 1001, kind, 7, ld=1001 + extra).call().check()


def masks(d, rng):
    """Banned tokens, NaN, rows with one token, none, and infinite logits; drafts outside the vocabulary."""
    V, T = d.V, d.T
    d.z[rng.random((T, V)) < 0.3] = -np.inf
    d.z[rng.random((T, V)) < 0.05] = np.nan
    d.z[rng.random((T, V)) < 0.05] = np.finfo(np.float32).min
    for b in range(d.B):
        t, k = int(d.off[b]), d.counts[b]
        at = t + int(rng.integers(0, max(1, k)))
        if b % 5 == 1:
            d.z[at] = -np.inf
        elif b % 5 == 2:
            d.z[at] = np.nan
        elif b % 5 == 3:
            d.z[at] = -np.inf
            d.z[at, rng.integers(0, V)] = rng.choice([-3e38, 0.0, 3e38])
        elif b % 5 == 4:
            d.z[at, rng.integers(0, V, 3)] = np.inf
    out = rng.random(T) < 0.1
    d.token[out] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31], out.sum())


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
@pytest.mark.parametrize("V", [1, 3, 40, 5000])
def test_verify_masks(hip, V, kind):
    Drafts([4, 5, 3, 6, 2, 1, 7, 4, 4, 1, 3, 2, 2, 5, 1], V, kind, V + 1, edit=masks).call().check()


def repeated(d, rng):
    """All drafts of a sequence hang on its first row and have few different tokens."""
    for b in range(d.B):
        t, k = int(d.off[b]), d.counts[b]
        d.parent[t + 1:t + k] = 0
        likely = np.argsort(-d.z[t])[:3]
        d.token[t:t + k] = rng.choice(likely, k)
        d.z[t, likely] = d.z[t].max() - np.float32(rng.random(3))


@pytest.mark.parametrize("V", [3, 50, 3001])
def test_verify_repeated_siblings(hip, V):
    Drafts([9, 2, 6, 12, 4, 1, 5, 9], V, "tree", V, edit=repeated).call().check()


def edges(d, rng):
    d.r[:] = rng.choice(np.array([0.0, 1.0 - 2.0 ** -24, 7.0, -1.0, 0.5], np.float32), d.B)
    d.u[:] = rng.choice(np.array([0.0, 1.0 - 2.0 ** -24, 2.0, -1.0, 0.5], np.float32), d.T)
    ban = rng.random(d.V) < 0.3                        # the ends of the vocabulary among them
    ban[[0, 1, -1]] = True
    ban[d.V // 2] = False
    d.z[:, ban] = -np.inf


@pytest.mark.parametrize("kind", ["probs", "plain", "tree"])
@pytest.mark.parametrize("V", [20, 5000])
def test_verify_random_numbers_at_their_ends(hip, V, kind):
    Drafts([4, 5, 3, 6, 2, 1, 7, 4, 4, 1, 3, 2], V, kind, V + 2, edit=edges).call().check()


def test_verify_parents_outside(hip):
    """Rows whose parent is no earlier row belong to no path."""
    def edit(d, rng):
        own = np.arange(d.T) - np.repeat(d.off[:-1], d.counts)
        for t in range(d.T):
            if rng.random() < 0.4:
                d.parent[t] = rng.choice([-1, -5, 2 ** 31 - 1, -2 ** 31, own[t], own[t] + 1, own[t] + 3])
    d = Drafts([6, 9, 3, 12, 5, 7], 60, "tree", 8, edit=edit, temps=[1, 0, 1, 0.7, 1, 1])
    d.call().check()


def test_verify_without_temperature(hip):
    d = Drafts([4, 5, 1], 500, "probs", 9, temps=[1, 1, 1])
    d.call()
    z, tok, _, q, _, u, r, off = [x.p for x in d.bufs]
    ok(lib().slate_hip_verify_drafts(d.outs[0].p, d.outs[1].p, d.outs[2].p, z, d.ld, tok, None, q, d.ld, None, u, r, off,
                                     d.B, d.T + 2, d.V, None, 0))
    d.check()


@pytest.mark.parametrize("temp", [-1.0, np.nan, -np.inf, 1e-30, 1e30, np.inf])
def test_verify_temperatures(hip, temp):
    def edit(d, rng):
        d.z[:, 3] = -np.inf
        d.z[:, 5] = d.z[:, 7] = d.z.max(1) + 1         # equal largest logits: the lower token
    Drafts([4, 5, 1, 3], 500, "probs", 10, temps=[temp] * 4, edit=edit).call().check()


def test_verify_left_out(hip):
    """Sequences whose tok_off does not fit, and those behind a fall of it, get -1, and nothing of them is written."""
    d = Drafts([3, 4, 2, 5], 100, "probs", 11)
    d.call()
    off = d.off.copy()
    for bad, who in (([0, 3, 2, 9, 14], (1, 2, 3)), ([-1, 3, 7, 9, 14], (0,)), ([0, 3, 7, 9, 1000], (3,)),
                     ([0, 3, 7, 9, 8], (3,))):
        d.bufs[7].upload(np.array(bad, np.int32))
        for o in d.outs:
            o.upload(np.full(o.nbytes // 4, MARK, np.int32))
        d.fn(None)
        n_acc, tok, _ = (o.to_array(np.int32, o.nbytes // 4) for o in d.outs)
        for b in range(4):
            t0, t1 = bad[b], bad[b + 1]
            if b in who:
                assert n_acc[b] == -1
            else:
                assert (t0, t1) == (off[b], off[b + 1]) and n_acc[b] == len(d.want[b][0])
        if who == (3,):
            assert np.all(tok[9:] == MARK)


def test_verify_keeps_the_target(hip):
    """Tokens come out distributed as the target says, whatever the draft is: the first token's shares over a grid of
    random numbers, 64 for the draft (whose probabilities are whole 64ths, so it has its shares), 64 to accept it, 16
    for the next token, each at the middle of its step.  A threshold is off by at most half a step, 1/128, of a draft's
    share, so what is accepted of a token and what is left to the next one by 1/128 each; each of its two borders
    moves a token's part of that (R in all) by half of 1/16."""
    V, N, M = 4, 64, 16
    z = np.array([0.3, -0.5, 0.9, 0.1], np.float32)
    p = np.exp(z.astype(np.float64)) / np.exp(z.astype(np.float64)).sum()
    q = np.array([6, 32, 10, 16], np.float32) / N
    draft = np.repeat(np.arange(V), (q * N).astype(int)).astype(np.int32)
    B = 1024
    zs, qs = dev(np.tile(z, (2 * B, 1))), dev(np.tile(q, (2 * B, 1)))
    off = dev(np.arange(0, 2 * B + 1, 2), np.int32)
    shares = np.zeros(V)
    for m in range(M):
        r = dev(np.full(B, (m + 0.5) / M, np.float32))
        for part in range(N * N // B):
            grid = np.arange(part * B, (part + 1) * B)
            tok, u = np.zeros(2 * B, np.int32), np.zeros(2 * B, np.float32)
            tok[1::2], u[1::2] = draft[grid // N], (grid % N + 0.5) / N
            ins, outs = [dev(tok), dev(u)], [DeviceBuffer(4 * B), DeviceBuffer(8 * B)]
            ok(lib().slate_hip_verify_drafts(outs[0].p, outs[1].p, None, zs.p, V, ins[0].p, None, qs.p, V, None,
                                             ins[1].p, r.p, off.p, B, 2 * B, V, None, 0))
            shares += np.bincount(outs[1].to_array(np.int32, (B, 2))[:, 0], minlength=V)
    shares /= shares.sum()
    R = np.maximum(q - p, 0).sum()
    assert np.abs(shares - p).max() <= 2 / 128 + R / 16


# -- together ---------------------------------------------------------------------------
class _Graph:
    """A captured call on the backend stream (HIP runtime through ctypes)."""

    def __init__(self, fn):
        self.rt = C.CDLL("libamdhip64.so")
        self.stream = C.c_void_p(lib().slate_hip_stream())
        self.graph, self.exe = C.c_void_p(), C.c_void_p()
        assert self.rt.hipStreamBeginCapture(self.stream, 2) == 0
        try:
            self.error = None
            fn()
        except slate_amd.HipError as e:
            self.error = str(e)
        assert self.rt.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0
        if self.error is None:
            assert self.rt.hipGraphInstantiate(C.byref(self.exe), self.graph, None, None, C.c_size_t(0)) == 0

    def launch(self):
        assert self.rt.hipGraphLaunch(self.exe, self.stream) == 0

    def free(self):
        if self.exe:
            self.rt.hipGraphExecDestroy(self.exe)
        self.rt.hipGraphDestroy(self.graph)


def test_captured_calls(hip):
    """Captured calls with a workspace each, replayed between eager ones, on new inputs."""
    rng = np.random.default_rng(15)
    runs = [Attend(Cache([(2000 + 700 * k, n), (50, 2)], 1, 128, 16, k, 0, 50 + k), 4) for k, n in enumerate((3, 5, 1))]
    for r in runs:
        r.call(own_ws=True)
    refused = _Graph(lambda: runs[0].call())
    if runs[0].need:
        assert refused.error and "workspace" in refused.error
    refused.free()
    d = Drafts([5, 3, 1, 4], 3001, "probs", 15)
    d.call(own_ws=True)
    pages = DevicePages(8, 40, 300, 16)
    pages.reset()
    host = pr.Pages(8, 40, 300, 16)
    slot, pos = np.array([2, 5, 7], np.int32), np.zeros(3, np.int32)
    n = np.array([9, 17, 1], np.int32)
    ins = [dev(slot), dev(pos), dev(n)]
    outs = [dev(np.zeros(64), np.int32) for _ in range(6)]
    graphs = [_Graph(lambda r=r: r.call(own_ws=True)) for r in runs]
    graphs.append(_Graph(lambda: d.fn(d.ws.p)))
    graphs.append(_Graph(lambda: ok(lib().slate_hip_pages_extend(pages.ref, *[i.p for i in ins], 3, 64,
                                                                 *[o.p for o in outs]))))
    assert all(g.error is None for g in graphs)
    for rep in range(4):
        for r in runs:
            r.q = rng.normal(0, 1, r.q.shape).astype(np.float32)
            r.qd.upload(r.q)
            r.out.upload(np.full_like(r.q, SENTINEL))
        for o in d.outs:
            o.upload(np.full(o.nbytes // 4, MARK, np.int32))
        ins[1].upload(pos)
        for g in graphs:
            g.launch()
        lib().slate_hip_sync()
        for r in runs:
            r.check()
            r.call()                                   # eager, on the backend's own workspace
            r.check()
        d.check()
        d.fn(None)
        d.check()
        status, desc = host.extend(slot.tolist(), pos.tolist(), n.tolist(), 64)
        assert status == 0 and int(outs[5].to_array(np.int32, 1)[0]) == 0
        assert np.array_equal(outs[3].to_array(np.int32, len(desc[3])), desc[3])
        same_pages(pages, host)
        pos = pos + n
    for g in graphs:
        g.free()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_serving_loop_with_drafts(hip, dtype):
    """Steps of a server: pages for the new tokens, their K/V stored, attention, drafts verified, pages of those that
    did not stand given back; requests end and new ones come.  Against the host's cache of every sequence."""
    Hkv, G, hd, ps, V, users = 2, 4, 64, 8, 40, 5
    rng = np.random.default_rng(16)
    d, h = DevicePages(users, 30, 60, ps), pr.Pages(users, 30, 60, ps)
    d.reset()
    pools = [dev(np.full(60 * Hkv * ps * hd, 0x7fff if dtype else np.nan, np.uint16 if dtype else np.float32))
             for _ in range(2)]
    kv = slate_amd.PagedKv(pools[0].ptr, pools[1].ptr, dtype, Hkv, hd, Hkv * ps * hd, ps * hd, hd)
    cached = [[np.zeros((0, Hkv, hd))] * 2 for _ in range(users)]
    for step in range(14):
        slot = rng.permutation(users)[:int(rng.integers(1, users + 1))]
        p0 = [len(cached[s][0]) for s in slot]
        n = [int(rng.integers(4, 20)) if p == 0 else int(rng.integers(1, 6)) for p in p0]
        T = sum(n)
        ins = [dev(a, np.int32) for a in (slot, p0, n)]
        outs = [DeviceBuffer(4 * (T + 9)) for _ in range(6)]
        ok(lib().slate_hip_pages_extend(d.ref, *[i.p for i in ins], len(slot), T, *[o.p for o in outs]))
        assert h.extend(slot.tolist(), p0, n, T)[0] == 0 == int(outs[5].to_array(np.int32, 1)[0])
        k, v = (rng.normal(0, 1, (T, Hkv, hd)).astype(np.float32) for _ in range(2))
        bufs = [dev(k), dev(v)]
        ok(lib().slate_hip_kv_store_paged(C.byref(kv), d.ref, bufs[0].p, bufs[1].p, Hkv * hd, outs[3].p, T))
        q = rng.normal(0, 1, (T, Hkv * G, hd)).astype(np.float32)
        qd, out = dev(q), DeviceBuffer(q.nbytes)
        ok(lib().slate_hip_attention_paged(out.p, qd.p, C.byref(kv), d.ref, ins[0].p, outs[0].p, ins[1].p, len(slot), T,
                                           max(n), Hkv * G, None, 0))
        got, t = out.to_array(np.float32, q.shape), 0
        for b, s in enumerate(slot):
            for i, x in enumerate((k, v)):
                cached[s][i] = np.concatenate([cached[s][i], of_type(to_type(x[t:t + n[b]], dtype), dtype)])
            for g in range(Hkv):
                K, W = (cached[s][i][:, g] for i in range(2))
                want, A, top = pr.attend(q[t:t + n[b], g * G:(g + 1) * G].astype(np.float64), K, W, p0[b], hd)
                assert np.abs(got[t:t + n[b], g * G:(g + 1) * G] - want).max() <= 2.0 ** -16 * np.abs(W).max()
            t += n[b]
        dr = Drafts(n, V, "probs", 100 + step, scale=1.0)
        dr.call(behind=0).check()
        keep = [p + 1 + len(w[0]) if p else p + k for p, k, w in zip(p0, n, dr.want)]
        for s, m in zip(slot, keep):
            cached[s] = [x[:m] for x in cached[s]]
        gone = [s for s in range(users) if len(cached[s][0]) > 60]
        for s in gone:
            cached[s] = [x[:0] for x in cached[s]]
        all_slots = list(range(users))
        length = [len(cached[s][0]) for s in all_slots]
        assert d.trim(all_slots, length) == h.trim(all_slots, length) == 0
        same_pages(d, h)
