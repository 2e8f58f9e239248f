"""Rotary variants, the 8-bit K/V cache and the attention of packed batches
over it and over trees of drafted tokens, against 64-bit references on the
host (tests/packed_ref.py).

Tolerances, from the arithmetic of the kernels:
* rope: cos and sin within 2 units in the last place and the reduced angle
  within half of one (1 + pi/4 units of 2^-23 in all), the products, the
  magnitude and the sum rounded once each: below 4 * 2^-23 of
  m (|x_j| + |x_k|).
* cache: exact (steps, codes and values).
* attention: a score is off by at most (2^-21 + hd 2^-24) A, A the largest
  sum |q_i k_i| / sqrt(hd) (q as two halves of 11 bits, or three of 8; f32
  sums), and by 2^-22 of itself when scaled; a weight by twice that and the
  exponential's 2^-22; sums over keys by keys * 2^-24.  Times max |V|.
  These are worst cases.  Roundings of independent sign add up to about
  sqrt(hd) 2^-25 of the partial sums, 4e-7, so the whole output is held to
  2^-18 in the 2-norm too: an operand that lost its lower half (2^-12) shows
  there.
"""
import ctypes as C
import threading

import numpy as np
import pytest

import slate_amd
from slate_amd import DeviceBuffer
from tests import packed_ref as pr

pytestmark = pytest.mark.gpu
NORM_TOL = 2.0 ** -18
SENTINEL = np.float32(-77.25)


def lib():
    return slate_amd.load_library()


def ok(rc, what="call"):
    slate_amd.check(rc, what)


# -- rope -----------------------------------------------------------------------
ROPES = [
    # rows, heads, hd, extra ld, farthest, config
    (1, 1, 32, 0, 10, dict(layout=0, rot_dim=32)),
    (3, 5, 128, 0, 1 << 20, dict(layout=0, rot_dim=128, scaling=2, factor=8.0, theta_base=500000.0)),
    (16, 40, 128, 12, 131072, dict(layout=1, rot_dim=64, scaling=3, factor=16.0, high=32.0)),
    (7, 3, 80, 3, 5000, dict(layout=0, rot_dim=20)),
    (7, 3, 80, 0, 5000, dict(layout=1, rot_dim=22, scaling=1)),
    (2, 2, 512, 0, 1 << 30, dict(layout=0, rot_dim=512)),
    (2, 3, 512, 1, 1000, dict(layout=1, rot_dim=510)),
    (600, 2, 64, 0, 4096, dict(layout=0, rot_dim=64, magnitude=0.5)),
    (5, 9, 33, 0, 100, dict(layout=0, rot_dim=2)),
    (515, 11, 96, 5, 1 << 17, dict(layout=1, rot_dim=96)),
    (3, 40000, 16, 0, 3000, dict(layout=0, rot_dim=16)),
    (4, 7, 2056, 0, 900, dict(layout=1, rot_dim=512)),
    (9, 6, 116, 1, 900, dict(layout=1, rot_dim=42)),
    (520, 3, 29, 0, 900, dict(layout=0, rot_dim=22)),
    (520, 2, 25, 2, 900, dict(layout=1, rot_dim=22)),
    (3, 2, 2083, 0, 900, dict(layout=0, rot_dim=64)),
]


@pytest.mark.parametrize("rows,heads,hd,extra,far,kw", ROPES)
@pytest.mark.parametrize("inplace", [False, True])
def test_rope(hip, rows, heads, hd, extra, far, kw, inplace):
    rng = np.random.default_rng(rows * 1000 + hd)
    cfg = dict(orig_ctx=4096, theta_base=10000.0, scaling=0, factor=4.0, low=1.0, high=4.0, magnitude=0.0)
    cfg.update(kw)
    ld = heads * hd + extra
    x = rng.normal(0, 1, (rows, ld)).astype(np.float32)
    x[0, 0] = 0.0
    pos = rng.integers(-far, far, rows).astype(np.int32)
    pos[0] = far - 1
    xd, pd = DeviceBuffer.from_array(x), DeviceBuffer.from_array(pos)
    yd = xd if inplace else DeviceBuffer.from_array(np.full_like(x, SENTINEL))
    ok(lib().slate_hip_rope_scaled(yd.p, xd.p, pd.p, rows, heads, hd, ld, C.byref(slate_amd.RopeConfig(**cfg))), "rope")
    got = yd.to_array(np.float32, x.shape)
    w, m = pr.rope_frequencies(cfg["layout"], cfg["rot_dim"], cfg["scaling"], cfg["theta_base"], cfg["factor"],
                               cfg["low"], cfg["high"], cfg["orig_ctx"], cfg["magnitude"])
    body = x[:, :heads * hd].reshape(rows, heads, hd).astype(np.float64)
    want = pr.rope(body, pos, cfg["layout"], cfg["rot_dim"], w, m)
    g = got[:, :heads * hd].reshape(rows, heads, hd)
    r = cfg["rot_dim"]
    a = np.abs(body[..., :r])
    pair = a[..., :r // 2] + a[..., r // 2:] if cfg["layout"] == 0 else a[..., 0::2] + a[..., 1::2]
    bound = 4 * 2.0 ** -23 * m * (np.concatenate([pair, pair], 2) if cfg["layout"] == 0 else np.repeat(pair, 2, 2))
    # the frequencies are 64-bit: at 2^30 turns of the fastest pair they leave 2^-22 of a radian
    bound = bound + np.abs(pos).max() * 2.0 ** -50 * a.max() * m
    assert np.all(np.abs(g[..., :r] - want[..., :r]) <= bound)
    assert np.array_equal(g[..., r:], body[..., r:].astype(np.float32))
    gap = got[:, heads * hd:]
    assert np.array_equal(gap, x[:, heads * hd:] if inplace else np.full_like(gap, SENTINEL))


def test_rope_matches_rope_rows_and_undoes_itself(hip):
    """Layout 0 without scaling is rope_rows; the negated positions turn back, which is also the gradient."""
    rng = np.random.default_rng(3)
    rows, heads, hd = 9, 4, 64
    x = rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)
    pos = rng.integers(0, 50, rows).astype(np.int32)
    c = slate_amd.RopeConfig(layout=0, rot_dim=hd, theta_base=10000.0)
    a, b, p, n = (DeviceBuffer.from_array(v) for v in (x, x, pos, -pos))
    ok(lib().slate_hip_rope_scaled(a.p, a.p, p.p, rows, heads, hd, heads * hd, C.byref(c)))
    ok(hip.rope_rows(b.p, p.p, rows, heads, hd, 10000.0, 64))
    ya, yb = a.to_array(np.float32, x.shape), b.to_array(np.float32, x.shape)
    assert np.abs(ya - yb).max() <= 50 * 2.0 ** -22 * np.abs(x).max()       # rope_rows' angles are f32 products
    # differences: <R x, g> changes with x as R^T g says
    g = rng.normal(0, 1, x.shape).astype(np.float32)
    gd = DeviceBuffer.from_array(g)
    ok(lib().slate_hip_rope_scaled(gd.p, gd.p, n.p, rows, heads, hd, heads * hd, C.byref(c)))
    dx = rng.normal(0, 1, x.shape).astype(np.float32)
    d = DeviceBuffer.from_array(dx)
    ok(lib().slate_hip_rope_scaled(d.p, d.p, p.p, rows, heads, hd, heads * hd, C.byref(c)))
    lhs = (d.to_array(np.float32, x.shape).astype(np.float64) * g).sum()
    rhs = (gd.to_array(np.float32, x.shape).astype(np.float64) * dx).sum()
    assert abs(lhs - rhs) <= 8 * 2.0 ** -23 * np.abs(dx).sum() * np.abs(g).max()
    ok(lib().slate_hip_rope_scaled(a.p, a.p, n.p, rows, heads, hd, heads * hd, C.byref(c)))
    assert np.abs(a.to_array(np.float32, x.shape) - x).max() <= 16 * 2.0 ** -23 * np.abs(x).max()


# -- packed batches ---------------------------------------------------------------
class Batch:
    """Descriptors and pools of a batch on host and device.  seqs: (pos0, n) each; `bad` sequences get numbers
    that do not fit."""

    def __init__(self, seqs, Hkv, hd, max_seq, rng, behind=0, bad=(), odd=0):
        self.seqs, self.Hkv, self.hd, self.max_seq, self.rng = seqs, Hkv, hd, max_seq, rng
        self.B = len(seqs)
        self.off = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        self.T = int(self.off[-1]) + behind
        self.pos0 = np.array([p for p, _ in seqs], np.int32)
        for b in bad:
            self.pos0[b] = max_seq - seqs[b][1] + 1
        self.bad = set(bad)
        self.head_stride = max_seq * hd + (3 if odd else 0)
        self.slot = Hkv * self.head_stride
        self.first = rng.permutation(self.B).astype(np.int64) * self.slot + odd      # each sequence's first element
        self.base = self.first.copy()
        self.elems = self.B * self.slot + odd
        self.d_off, self.d_pos, self.d_base = (DeviceBuffer.from_array(a) for a in (self.off, self.pos0, self.base))

    def desc(self):
        return self.d_off.p, self.d_pos.p, self.d_base.p

    def tokens(self, b):
        return range(self.off[b], self.off[b + 1]) if b not in self.bad else range(0)

    def row(self, b, h, p):
        """Element where row p of head h starts."""
        return int(self.first[b]) + h * self.head_stride + p * self.hd


def fill_q8(bt, seed):
    """8-bit pools: quantised rows up to each sequence's last token, elsewhere codes of any value under NaN steps."""
    rng = np.random.default_rng(seed)
    pools = {}
    for name in "KV":
        q = rng.integers(-127, 128, bt.elems).astype(np.int8)
        s = np.full(bt.elems // 32, np.nan, np.float16)
        for b, (p, n) in enumerate(bt.seqs):
            for h in range(bt.Hkv):
                at = bt.row(b, h, 0)
                cq, cs = pr.quantise(rng.normal(0, 1, (min(p + n, bt.max_seq), bt.hd)).astype(np.float32))
                q[at:at + cq.size] = cq.reshape(-1)
                s[at // 32:at // 32 + cs.size] = cs.reshape(-1)
        pools[name] = (q, s)
    return pools


def fill_f32(bt, seed):
    rng = np.random.default_rng(seed)
    pools = {}
    for name in "KV":
        x = np.full(bt.elems, np.nan, np.float32)
        for b, (p, n) in enumerate(bt.seqs):
            for h in range(bt.Hkv):
                at = bt.row(b, h, 0)
                r = rng.normal(0, 1, min(p + n, bt.max_seq) * bt.hd).astype(np.float32)
                x[at:at + r.size] = r
        pools[name] = x
    return pools


def host_rows(bt, pool, b, h, rows):
    at = bt.row(b, h, 0)
    if isinstance(pool, tuple):
        q, s = pool
        return pr.values(q[at:at + rows * bt.hd].reshape(rows, bt.hd),
                         s[at // 32:(at + rows * bt.hd) // 32].reshape(rows, -1))
    return pool[at:at + rows * bt.hd].reshape(rows, bt.hd).astype(np.float64)


def check_attention(bt, pools, q, out, G, parent=None, norm=True):
    """out [T, Hq, hd] against the reference; rows that no sequence owns keep the sentinel."""
    hd = bt.hd
    owned = np.zeros(bt.T, bool)
    num = den = 0.0
    for b, (p, n) in enumerate(bt.seqs):
        tk = list(bt.tokens(b))
        if not tk:
            continue
        owned[tk] = True
        sees = np.ones((n, p + n), bool)
        sees[:, p:] = np.tril(np.ones((n, n), bool)) if parent is None else pr.ancestors(parent[tk])
        for h in range(bt.Hkv):
            K, V = host_rows(bt, pools["K"], b, h, p + n), host_rows(bt, pools["V"], b, h, p + n)
            want, A, top = pr.attend(q[tk][:, h * G:(h + 1) * G].astype(np.float64), K, V, sees, hd)
            got = out[tk][:, h * G:(h + 1) * G].astype(np.float64)
            tol = 2 * ((2.0 ** -21 + hd * 2.0 ** -24) * A + 2.0 ** -22 * top) + 2.0 ** -22 + (p + n) * 2.0 ** -24
            assert np.isfinite(got).all(), (b, h)
            err = np.abs(got - want).max() / np.abs(V).max()
            assert err <= tol, (b, h, err, tol)
            num += ((got - want) ** 2).sum()
            den += (want ** 2).sum()
    if norm and den:
        assert (num / den) ** 0.5 <= NORM_TOL, (num / den) ** 0.5
    assert np.all(out[~owned] == SENTINEL)


class Run:
    """Device side of one attention call over a batch."""

    def __init__(self, bt, G, q8, seed, parent=None, pools=None, offset=0):
        self.bt, self.G, self.q8, self.parent = bt, G, q8, parent
        rng = np.random.default_rng(seed + 1)
        self.pools = pools or (fill_q8(bt, seed) if q8 else fill_f32(bt, seed))
        self.q = rng.normal(0, 1, (bt.T, bt.Hkv * G, bt.hd)).astype(np.float32)
        self.qd = DeviceBuffer.from_array(self.q)
        self.out = DeviceBuffer.from_array(np.full_like(self.q, SENTINEL))
        flat = [a for n in "KV" for a in (self.pools[n] if q8 else (self.pools[n],))]
        self.pd = [DeviceBuffer.from_array(a) for a in flat]
        self.par = DeviceBuffer.from_array(parent) if parent is not None else None
        need = lib().slate_hip_attention_packed_bytes(bt.Hkv * G, bt.Hkv, bt.hd)
        self.need = need
        self.ws = DeviceBuffer(max(need, 16))

    def call(self, own_ws=False, max_new=None):
        bt = self.bt
        name = "slate_hip_attention_" + ("ragged_q8" if self.par is None else "tree_q8" if self.q8 else "tree")
        mx = max_new or max(1, max(n for _, n in bt.seqs))
        rc = getattr(lib(), name)(self.out.p, self.qd.p, *[d.p for d in self.pd], *bt.desc(),
                                  *([self.par.p] if self.par else []), bt.B, bt.T, mx, bt.Hkv * self.G, bt.Hkv, bt.hd,
                                  bt.head_stride, bt.max_seq, self.ws.p if own_ws else None, max(self.need, 16))
        ok(rc, name)

    def result(self):
        return self.out.to_array(np.float32, self.q.shape)

    def check(self, norm=True):
        check_attention(self.bt, self.pools, self.q, self.result(), self.G, self.parent, norm)


DECODE = [(0, 1), (1, 1), (30, 1), (31, 1), (32, 1), (33, 1), (127, 1), (255, 1), (256, 1), (700, 1), (1299, 1)]
CHUNKS = [(0, 1), (0, 2), (5, 15), (0, 16), (17, 17), (300, 33), (0, 70), (64, 1), (650, 130), (3, 0), (0, 5)]
SHAPES = [(32, 2, 1), (32, 1, 8), (64, 2, 4), (64, 1, 3), (128, 2, 4), (128, 1, 8), (128, 1, 7), (128, 2, 1),
          (96, 1, 2), (256, 1, 4), (128, 1, 16), (64, 1, 20), (512, 1, 2)]


@pytest.mark.parametrize("hd,Hkv,G", SHAPES)
@pytest.mark.parametrize("kind", ["decode", "chunks"])
def test_ragged_q8(hip, hd, Hkv, G, kind):
    rng = np.random.default_rng(hd + G)
    bt = Batch(DECODE if kind == "decode" else CHUNKS, Hkv, hd, 1301, rng, behind=3, bad=(4,))
    r = Run(bt, G, True, 7)
    r.call()
    r.check()
    r.call(own_ws=True)
    r.check()


@pytest.mark.parametrize("hd", [64, 96])
@pytest.mark.parametrize("n", [1, 25])
@pytest.mark.parametrize("kind", ["ragged", "tree_q8", "tree"])
def test_no_limit_on_the_context(hip, kind, n, hd):
    """max_seq = INT32_MAX, as a program without a limit passes it: blocks are cut and joined as with the true one."""
    rng = np.random.default_rng(17)
    bt = Batch([(5000, n), (700, 1)], 1, hd, 5100, rng)
    r = Run(bt, 4, kind != "tree", 6, None if kind == "ragged" else random_parents(bt, rng, "random"))
    bt.max_seq = 2 ** 31 - 1
    r.call()
    r.check()


@pytest.mark.parametrize("B", [1, 65, 200])
def test_ragged_q8_many_sequences(hip, B):
    rng = np.random.default_rng(B)
    seqs = [(int(rng.integers(0, 40)), int(rng.integers(0, 3))) for _ in range(B - 1)] + [(37, 2)]
    bt = Batch(seqs, 1, 64, 50, rng, behind=1)
    r = Run(bt, 4, True, B)
    r.call()
    r.check()


def test_ragged_q8_long(hip):
    """One long context beside short ones: the long one is split over workgroups and joined."""
    bt = Batch([(20000, 1), (3, 1), (0, 1), (9001, 1)], 2, 128, 20005, np.random.default_rng(1))
    r = Run(bt, 4, True, 1)
    r.call()
    r.check()


@pytest.mark.parametrize("G,seqs", [(8, [(300, 1100), (0, 1)]), (3, [(40, 2800)]), (130, [(0, 70), (513, 3)]),
                                    (1, [(0, 600), (2000, 129), (0, 9000)])])
def test_prompts_of_many_blocks(hip, G, seqs):
    """More blocks of 128 query rows than a wave has lanes; blocks that begin and end inside a token's heads."""
    bt = Batch(seqs, 1, 32, max(p + n for p, n in seqs) + 1, np.random.default_rng(G))
    r = Run(bt, G, True, 9)
    r.call()
    r.check()


def test_prompt_of_131072_tokens(hip):
    """A whole long prompt in one call, 64 heads: a few of its rows against the reference.

    With N(0, 1) values and weights of one size the sum over t keys is a random walk: its partial sums are at most
    about as large as the result.  Each of the 2 t / 32 products that are added to it rounds it by up to 2^-24, with
    independent signs sqrt(2 t / 32) 2^-24 in all (5.4e-6 for 131072 keys), besides what NORM_TOL stands for."""
    n, hd, Hkv, G = 131072, 32, 8, 8
    rng = np.random.default_rng(18)
    bt = Batch([(0, n)], Hkv, hd, n, rng)
    pools = fill_q8(bt, 6)
    part = rng.normal(0, 1, (4096, Hkv * G, hd)).astype(np.float32)
    q = np.concatenate([part] * (n // 4096))
    flat = [DeviceBuffer.from_array(a) for name in "KV" for a in pools[name]]
    qd, out = DeviceBuffer.from_array(q), DeviceBuffer(q.nbytes)
    ok(lib().slate_hip_attention_ragged_q8(out.p, qd.p, *[d.p for d in flat], *bt.desc(), 1, n, n, Hkv * G, Hkv, hd,
                                           bt.head_stride, n, None, 0))
    got = out.to_array(np.float32, q.shape).astype(np.float64)
    for h in range(Hkv):
        K, V = (host_rows(bt, pools[name], 0, h, n) for name in "KV")
        for t in (0, 1, 4095, 65536 + 17 * h, n - 1):
            want, _, _ = pr.attend(q[t:t + 1, h * G:(h + 1) * G].astype(np.float64), K[:t + 1], V[:t + 1],
                                   np.ones((1, t + 1), bool), hd)
            err = np.linalg.norm(got[t, h * G:(h + 1) * G] - want) / np.linalg.norm(want)
            assert err <= NORM_TOL + (2 * (t + 1) / 32) ** 0.5 * 2.0 ** -24, (h, t, err)


def test_ragged_q8_bound_on_tokens(hip):
    """A sequence with more tokens than max_new is left out; the others are computed."""
    bt = Batch([(10, 1), (20, 5), (30, 2)], 1, 64, 64, np.random.default_rng(1))
    r = Run(bt, 2, True, 5)
    r.call(max_new=2)
    bt.bad = {1}
    r.check()


def test_empty_batch(hip):
    """Sequences without tokens, or with numbers that do not fit: nothing is written, cut entries of an earlier call
    are not taken for this one's."""
    rng = np.random.default_rng(2)
    bt = Batch([(9000, 1), (3000, 1)], 1, 64, 9002, rng)
    r = Run(bt, 4, True, 5)
    r.call(own_ws=True)
    r.check()
    for off, pos in (([0, 0, 0], [5, 5]), ([0, 1, 0], [9002, 0]), ([0, -1, -1], [0, 0]), ([2, 3, 4], [0, 0]),
                     ([0, 1, 2], [-1, 1 << 30])):
        bt.d_off.upload(np.array(off, np.int32))
        bt.d_pos.upload(np.array(pos, np.int32))
        r.out.upload(np.full_like(r.q, SENTINEL))
        r.call(own_ws=True)
        assert np.all(r.result() == SENTINEL), (off, pos)


@pytest.mark.parametrize("q8", [False, True])
def test_workspace_content_does_not_matter(hip, q8):
    """A workspace full of NaN and of large numbers, as another call may leave it."""
    rng = np.random.default_rng(3)
    for n in (5, 40):
        bt = Batch([(5000, n), (700, 3), (0, 1)], 1, 128, 5100, rng)
        r = Run(bt, 4, q8, 31, random_parents(bt, rng, "random"))
        for fill in (np.float32(np.nan), np.float32(3e38)):
            r.ws.upload(np.full(r.need // 4, fill, np.float32))
            r.call(own_ws=True)
            r.check()


def test_more_sequences_than_fit_a_wave(hip):
    rng = np.random.default_rng(4)
    seqs = [(int(rng.integers(0, 90)), int(rng.integers(0, 2))) for _ in range(1023)] + [(2000, 1)]
    bt = Batch(seqs, 1, 32, 2001, rng)
    r = Run(bt, 2, True, 4)
    r.call()
    r.check()


def test_sequences_that_share_cached_rows(hip):
    """Two sequences over one slot, as beams over a shared prompt read it."""
    rng = np.random.default_rng(14)
    bt = Batch([(800, 1), (800, 1), (300, 1)], 2, 64, 801, rng)
    bt.first[1] = bt.first[0]
    bt.d_base.upload(bt.first)
    r = Run(bt, 4, True, 6)
    r.call()
    r.check()


def test_base_is_rounded_down_to_a_row(hip):
    rng = np.random.default_rng(15)
    bt = Batch([(40, 2), (100, 1)], 1, 64, 128, rng)
    r = Run(bt, 4, True, 6)
    bt.d_base.upload(bt.first + np.array([63, 17]))
    r.call()
    r.check()
    bt.d_base.upload(np.array([-1, bt.first[1]]))
    bt.bad = {0}
    r.out.upload(np.full_like(r.q, SENTINEL))
    r.call()
    r.check()


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("first", [2, 70])
def test_token_offsets_that_fall(hip, q8, n, first):
    """Offsets that go back over the same tokens again and again: the sequences before the first fall are computed,
    the others may be left out, and no count of keys passes 32 bits."""
    seqs = [(50 + b, n) for b in range(first)]
    B = 1000
    rng = np.random.default_rng(first)
    bt = Batch(seqs, 1, 64, 4000, rng)
    parent = random_parents(bt, rng, "chain")
    r = Run(bt, 2, q8, 21, parent)
    off = np.zeros(B + 1, np.int32)
    off[:first + 1] = bt.off
    off[first + 1::2] = 0
    off[first + 2::2] = bt.T
    pos0 = np.zeros(B, np.int32)
    pos0[:first] = bt.pos0
    base = np.zeros(B, np.int64)
    base[:first] = bt.base
    bt.d_off, bt.d_pos, bt.d_base = (DeviceBuffer.from_array(a) for a in (off, pos0, base))
    bt.B = B
    r.call(max_new=min(bt.T, 1024))
    bt.B = first
    r.check()


@pytest.mark.parametrize("order", ["mixed", "rising", "falling"])
@pytest.mark.parametrize("hd,G,n", [(128, 4, 1), (128, 4, 40), (64, 8, 33), (32, 2, 70)])
def test_q8_steps_of_all_sizes(hip, hd, G, n, order):
    """V steps that differ by up to 2^26 from block to block and key to key, some of them 0 or below f16's normal
    range."""
    rng = np.random.default_rng(n)
    bt = Batch([(600, n), (0, n), (77, max(1, n - 3))], 2, hd, 700, rng)
    pools = fill_q8(bt, 8)
    q, st = pools["V"]
    for b, (p, m) in enumerate(bt.seqs):
        for h in range(bt.Hkv):
            at, rows = bt.row(b, h, 0) // 32, p + m
            by = rng.integers(-13, 14, (rows, hd // 32)).astype(np.float64)
            if order != "mixed":
                by = np.clip(np.sort(by[:, 0])[::-1 if order == "falling" else 1][:, None] + by / 8, -13, 13)
            v = st[at:at + rows * (hd // 32)].reshape(rows, -1).astype(np.float64) * 2.0 ** np.rint(by)
            v[rng.random(v.shape) < 0.05] = 0
            st[at:at + v.size] = v.astype(np.float16).reshape(-1)
    r = Run(bt, G, True, 8, pools=pools)
    r.call()
    r.check()


# committed rows whose V is 0: the first 32 keys, a whole stage of 64, one half of a stage, both halves of two
# stages that meet, a row alone, and drafts
ZERO_ROWS = [(0, 32), (128, 192), (288, 320), (416, 480), (500, 501), (608, 610)]


def zero_v_rows(bt, pools, drop, scale):
    """V by `scale`, and 0 in the rows `drop` (first, past the last) of every sequence."""
    v = pools["V"][1] if isinstance(pools["V"], tuple) else pools["V"]
    v[:] = (v.astype(np.float64) * scale).astype(v.dtype)
    per = 32 if isinstance(pools["V"], tuple) else 1
    for b, (p, n) in enumerate(bt.seqs):
        for h in range(bt.Hkv):
            at = bt.row(b, h, 0)
            for lo, hi in drop:
                lo, hi = min(lo, p + n), min(hi, p + n)
                v[(at + lo * bt.hd) // per:(at + hi * bt.hd) // per] = 0


@pytest.mark.parametrize("scale", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("kind", ["causal", "tree"])
@pytest.mark.parametrize("hd,Hkv,G,n", [(32, 2, 2, 70), (64, 1, 8, 40), (128, 2, 4, 40), (128, 1, 4, 1)])
def test_q8_rows_of_zero_steps(hip, hd, Hkv, G, n, kind, scale):
    """V steps of 0 in all of 32 and of 64 neighbouring keys that every token sees, as zeroed cache rows have them and
    as the store leaves where a step rounds to 0; blocks of 128 query rows and of fewer (which share the keys)."""
    rng = np.random.default_rng(hd + n)
    bt = Batch([(600, n), (64, max(1, n - 3)), (450, max(1, n // 8)), (0, n)], Hkv, hd, 700, rng)
    pools = fill_q8(bt, 8)
    zero_v_rows(bt, pools, ZERO_ROWS, scale)
    r = Run(bt, G, True, 8, random_parents(bt, rng, "random") if kind == "tree" else None, pools=pools)
    r.call()
    check_beside_zero_rows(r)


def check_beside_zero_rows(r):
    """As Run.check; a sequence whose V is 0 in every row gets zeros (its error has no largest V to go by)."""
    bt, out = r.bt, r.result()
    for b, (p, n) in enumerate(bt.seqs):
        if not any(host_rows(bt, r.pools["V"], b, h, p + n).any() for h in range(bt.Hkv)):
            tk = list(bt.tokens(b))
            assert np.all(out[tk] == 0)
            out[tk] = SENTINEL
            bt.bad.add(b)
    check_attention(bt, r.pools, r.q, out, r.G, r.parent)


def test_q8_all_steps_zero(hip):
    """Nothing but zeros in V: the output is 0."""
    rng = np.random.default_rng(1)
    for n in (1, 40):
        bt = Batch([(300, n), (0, 2)], 1, 64, 400, rng)
        pools = fill_q8(bt, 8)
        zero_v_rows(bt, pools, [(0, 400)], 1.0)
        r = Run(bt, 4, True, 8, pools=pools)
        r.call()
        check_beside_zero_rows(r)


@pytest.mark.parametrize("scale", [1.0, 1e-2, 1e-4, 2.0 ** -20, 2.0 ** -60])
@pytest.mark.parametrize("drop", [[(0, 1)], [(77, 78)], [(299, 300)], [(310, 312)], ZERO_ROWS, [(0, 64), (301, 340)]])
def test_tree_rows_of_zeros(hip, drop, scale):
    """V rows of zeros, committed and drafted, among small ones in f32 pools: the others keep their bits."""
    rng = np.random.default_rng(3)
    bt = Batch([(300, 40), (64, 3), (600, 12)], 2, 64, 640, rng)
    pools = fill_f32(bt, 5)
    zero_v_rows(bt, pools, drop, scale)
    r = Run(bt, 4, False, 5, random_parents(bt, rng, "random"), pools=pools)
    r.call()
    check_beside_zero_rows(r)


@pytest.mark.parametrize("hd,n", [(32, 33), (128, 5)])
def test_tree_all_rows_zero(hip, hd, n):
    rng = np.random.default_rng(4)
    bt = Batch([(700, n), (0, 2)], 1, hd, 800, rng)
    pools = fill_f32(bt, 5)
    zero_v_rows(bt, pools, [(0, 800)], 1.0)
    r = Run(bt, 4, False, 5, random_parents(bt, rng, "random"), pools=pools)
    r.call()
    check_beside_zero_rows(r)


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -20, 2.0 ** -41, 2.0 ** -70, 2.0 ** 80])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_tree_weights_do_not_go_by_the_size_of_v(hip, hd, scale):
    """Few keys of small scores, where the bound on a weight is a few 2^-22: it holds at any size of V."""
    rng = np.random.default_rng(hd)
    bt = Batch([(2, 6), (0, 3), (5, 1), (0, 12), (1, 4), (3, 2)] * 8, 2, hd, 16, rng)
    pools = fill_f32(bt, 5)
    pools["K"] *= np.float32(2.0 ** -8)
    pools["V"] *= np.float32(scale)
    r = Run(bt, 3, False, 5, random_parents(bt, rng, "random"), pools=pools)
    r.call()
    r.check()


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -6, 2.0 ** -14, 2.0 ** -17, 2.0 ** 10])
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_q8_weights_do_not_go_by_the_size_of_v(hip, hd, n, scale):
    """The same over the 8-bit cache, whose steps end at 2^-24."""
    rng = np.random.default_rng(hd)
    few = [(1, 1), (1, 1), (2, 1), (3, 1)] * 8
    bt = Batch(few + [(2, min(n, 5)), (0, min(n, 3)), (5, 1), (70, 1), (1, min(n, 4)), (35, n)] * 4, 2, hd, 80, rng)
    pools = fill_q8(bt, 5)
    for name, by in (("K", 2.0 ** -8), ("V", scale)):
        st = pools[name][1]
        st[:] = (st.astype(np.float64) * by).astype(np.float16)
    for parent in (None, random_parents(bt, rng, "random")):
        r = Run(bt, 3, True, 5, parent, pools=pools)
        r.call()
        r.check()


@pytest.mark.parametrize("ratio", [2.0 ** 6, 2.0 ** 10])
@pytest.mark.parametrize("hd,G,n", [(128, 4, 1), (128, 4, 40), (64, 8, 33), (32, 2, 12)])
def test_large_v_rows_without_weight(hip, hd, G, n, ratio):
    """One key in ten has V `ratio` times as large and, by its K, a weight below 2^-60: what the others give is still
    held to 2^-18 of itself.  Each weight is resolved to 2^-33 of the largest weight times the largest V seen: 2^-23 of
    the others here, and their errors are independent."""
    rng = np.random.default_rng(n)
    bt = Batch([(600, n), (0, n), (77, max(1, n - 3))], 2, hd, 700, rng)
    for kind in ("ragged", "tree_q8", "tree"):
        q8 = kind != "tree"
        pools = fill_f32(bt, 8)
        for b, (p, m) in enumerate(bt.seqs):
            for h in range(bt.Hkv):
                at, rows = bt.row(b, h, 0), p + m
                K, V = (pools[x][at:at + rows * hd].reshape(rows, hd) for x in "KV")
                big = rng.random(rows) < 0.1
                big[:max(1, p)][0] = False             # a root sees a key with weight
                big[p:] = False
                K[:, 0] = np.where(big, -6 * np.sqrt(hd), 0.0)
                V[big] *= np.float32(ratio)
        if q8:
            full = fill_q8(bt, 8)
            for x in "KV":
                for b, (p, m) in enumerate(bt.seqs):
                    for h in range(bt.Hkv):
                        at, size = bt.row(b, h, 0), (p + m) * hd
                        cq, cs = pr.quantise(pools[x][at:at + size].reshape(-1, hd))
                        full[x][0][at:at + size] = cq.reshape(-1)
                        full[x][1][at // 32:(at + size) // 32] = cs.reshape(-1)
            pools = full
        r = Run(bt, G, q8, 8, None if kind == "ragged" else random_parents(bt, rng, "random"), pools=pools)
        r.q[:, :, 0] = 9.0
        r.qd.upload(r.q)
        r.call()
        r.check()


@pytest.mark.parametrize("kind", ["ragged", "tree_q8", "tree"])
@pytest.mark.parametrize("hd,G,n", [(64, 8, 1), (128, 4, 40), (64, 8, 33)])
def test_small_columns_beside_large_ones(hip, hd, G, n, kind):
    """32 columns of V 2^16 times as large as the others.  A value is resolved to 2^-24 of the largest around it (f32:
    2^-22 of itself or far less), what a key adds to 2^-33 of the largest V; the weights' own errors count against the
    column.  So a small column is off by at most 2^-23 of the largest V and the usual bound times its own values."""
    rng = np.random.default_rng(n)
    bt = Batch([(300, n), (64, max(1, n - 3))], 1, hd, 400, rng)
    q8 = kind != "tree"
    pools = (fill_q8 if q8 else fill_f32)(bt, 8)
    x = pools["V"][1] if q8 else pools["V"]
    for b, (p, m) in enumerate(bt.seqs):
        at, per = bt.row(b, 0, 0) // (32 if q8 else 1), hd // 32 if q8 else hd
        v = x[at:at + (p + m) * per].reshape(p + m, per)
        large = slice(0, 1) if q8 else slice(0, 32)
        v[:] = (v.astype(np.float64) * 2.0 ** -6).astype(x.dtype)
        v[:, large] = (v[:, large].astype(np.float64) * 2.0 ** 16).astype(x.dtype)
    parent = None if kind == "ragged" else random_parents(bt, rng, "random")
    r = Run(bt, G, q8, 8, parent, pools=pools)
    r.call()
    r.check()
    out = r.result().astype(np.float64)
    for b, (p, m) in enumerate(bt.seqs):
        tk = list(bt.tokens(b))
        sees = np.ones((m, p + m), bool)
        sees[:, p:] = np.tril(np.ones((m, m), bool)) if parent is None else pr.ancestors(parent[tk])
        K, V = (host_rows(bt, pools[name], b, 0, p + m) for name in "KV")
        want, A, top = pr.attend(r.q[tk].astype(np.float64), K, V, sees, hd)
        tol = 2 * ((2.0 ** -21 + hd * 2.0 ** -24) * A + 2.0 ** -22 * top) + 2.0 ** -22 + (p + m) * 2.0 ** -24
        err = np.abs(out[tk] - want)[:, :, 32:].max()
        assert err <= 2.0 ** -23 * np.abs(V).max() + tol * np.abs(V[:, 32:]).max(), (b, err)


@pytest.mark.parametrize("order", ["mixed", "rising", "falling", "one"])
@pytest.mark.parametrize("hd,G,n", [(128, 4, 5), (128, 4, 40), (64, 8, 33), (32, 2, 70)])
def test_tree_rows_of_all_sizes(hip, hd, G, n, order):
    """V rows of f32 pools that differ by up to 2^26 from key to key; one row in each ten far above the others, at
    any place among its neighbours."""
    rng = np.random.default_rng(n)
    bt = Batch([(600, n), (0, n), (77, max(1, n - 3))], 2, hd, 700, rng)
    pools = fill_f32(bt, 8)
    for b, (p, m) in enumerate(bt.seqs):
        for h in range(bt.Hkv):
            at, rows = bt.row(b, h, 0), p + m
            by = rng.integers(-13, 14, rows)
            if order in ("rising", "falling"):
                by = np.sort(by)[::-1 if order == "falling" else 1]
            if order == "one":
                by = np.where(rng.random(rows) < 0.1, 13, 0)
            pools["V"][at:at + rows * hd] *= np.repeat(2.0 ** by, hd).astype(np.float32)
    r = Run(bt, G, False, 8, random_parents(bt, rng, "random"), pools=pools)
    r.call()
    r.check()


@pytest.mark.parametrize("scale", [2.0 ** 96, 2.0 ** -60, 2.0 ** -85, 2.0 ** -105, 2.0 ** -130])
def test_tree_values_far_from_one(hip, scale):
    """f32 values up to 2^99, far below 1, and queries that are all but 0: nothing over- or underflows into NaN."""
    rng = np.random.default_rng(3)
    for name in ("K", "V", "q"):
        bt = Batch([(40, 12), (0, 40), (300, 3)], 2, 64, 400, rng)
        pools = fill_f32(bt, 5)
        if name != "q":
            pools[name] *= np.float32(scale)
        r = Run(bt, 4, False, 5, random_parents(bt, rng, "random"), pools=pools)
        if name == "q":
            r.q *= np.float32(scale)
            r.qd.upload(r.q)
        r.call()
        if name != "V" or scale >= 2.0 ** -85:
            r.check()
            continue
        # below 2^-92 a value is kept to 2^-114: half a step of the lower half at the scale 2^90, and products add
        # at most the weights' own rounding
        out = r.result().astype(np.float64)
        exact = Run(bt, 4, False, 5, r.parent, pools=dict(pools, V=pools["V"] / np.float32(scale)))
        exact.call()
        exact.check()
        want = exact.result().astype(np.float64) * scale
        assert np.abs(out - want).max() <= 2.0 ** -113 + 2.0 ** -20 * np.abs(want).max()


@pytest.mark.parametrize("G,n", [(1, 32), (1, 33), (3, 26), (3, 27), (3, 32), (4, 20), (4, 21), (4, 24), (4, 25), (16, 5),
                                 (16, 6), (16, 7), (80, 1), (81, 1), (96, 1), (97, 1)])
def test_rows_around_the_kernels_border(hip, G, n):
    """80 query rows per kv head and 32 tokens are where one kernel hands over to the other."""
    rng = np.random.default_rng(16)
    bt = Batch([(700, n), (31, max(1, n - 1)), (5, 1)], 1, 64, 800, rng)
    for kind in ("causal", "tree"):
        r = Run(bt, G, True, 6, random_parents(bt, rng, "random") if kind == "tree" else None)
        r.call()
        r.check()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("G,n", [(3, 16), (3, 17), (4, 12), (4, 13), (12, 4), (7, 6), (7, 7), (16, 3), (16, 4), (48, 1),
                                 (49, 1), (1, 31), (2, 24), (2, 25)])
def test_rows_around_48(hip, G, n, hd):
    """Up to 48 query rows per kv head (and 32 tokens) one kernel takes a batch, from there on another."""
    rng = np.random.default_rng(19)
    bt = Batch([(700, n), (31, max(1, n - 1)), (5, 1)], 1, hd, 800, rng)
    for kind in ("causal", "tree"):
        r = Run(bt, G, True, 6, random_parents(bt, rng, "random") if kind == "tree" else None)
        r.call()
        r.check()


def random_parents(bt, rng, kind):
    out = np.full(bt.T, -1, np.int32)
    for b in range(bt.B):
        for i, t in enumerate(range(bt.off[b], bt.off[b + 1])):
            if i == 0:
                continue
            out[t] = {"random": int(rng.integers(max(0, i - 4), i)), "chain": i - 1, "star": 0, "forest": -1,
                      "odd": int(rng.choice([i, i + 1, -5, 1 << 30, i - 1, -(1 << 31)]))}[kind]
    return out


DRAFTS = [(0, 1), (0, 17), (1, 8), (31, 3), (32, 33), (100, 64), (290, 70), (640, 12), (7, 0), (1200, 16)]
TREE_SHAPES = [(32, 2, 1), (64, 1, 4), (64, 1, 3), (128, 2, 4), (128, 1, 8), (128, 1, 7), (96, 1, 2), (256, 1, 2)]


@pytest.mark.parametrize("kind", ["random", "chain", "star", "forest", "odd"])
@pytest.mark.parametrize("q8", [False, True])
def test_tree_kinds(hip, kind, q8):
    rng = np.random.default_rng(11)
    bt = Batch(DRAFTS, 1, 64, 1230, rng, behind=2, bad=(3,), odd=0 if q8 else 5)
    r = Run(bt, 4, q8, 21, random_parents(bt, rng, kind))
    r.call()
    r.check()


@pytest.mark.parametrize("hd,Hkv,G", TREE_SHAPES + [(16, 2, 2), (48, 1, 4)])
@pytest.mark.parametrize("q8", [False, True])
def test_tree_shapes(hip, hd, Hkv, G, q8):
    if q8 and hd % 32:
        pytest.skip("8-bit pools have head_dim in blocks of 32")
    rng = np.random.default_rng(hd + G)
    bt = Batch(DRAFTS, Hkv, hd, 1230, rng, behind=2, odd=0 if q8 else 4)
    r = Run(bt, G, q8, 22, random_parents(bt, rng, "random"))
    r.call()
    r.check()
    r.call(own_ws=True)
    r.check()


@pytest.mark.parametrize("q8", [False, True])
def test_tree_large(hip, q8):
    """As many drafts as a sequence may bring, and a long context that is split."""
    rng = np.random.default_rng(12)
    bt = Batch([(40, 1024), (9000, 20)], 1, 64, 9100, rng)
    r = Run(bt, 2, q8, 23, random_parents(bt, rng, "random"))
    r.call()
    r.check()


@pytest.mark.parametrize("q8", [False, True])
def test_tree_values_a_token_does_not_see(hip, q8):
    """Infinities and NaN in K and V rows of drafts reach the tokens that see them and no others."""
    rng = np.random.default_rng(5)
    bt = Batch([(40, 24), (0, 10)], 1, 64, 80, rng)
    parent = random_parents(bt, rng, "random")
    pools = (fill_q8 if q8 else fill_f32)(bt, 3)
    dirty = {(0, 5): "V", (0, 9): "K", (1, 4): "V", (1, 7): "V"}
    for (b, i), name in dirty.items():
        at = bt.row(b, 0, bt.seqs[b][0] + i)
        if q8:
            pools[name][1][at // 32:at // 32 + 2] = np.inf if i == 4 else np.nan
        else:
            pools[name][at:at + bt.hd] = np.inf if i == 4 else np.nan
    r = Run(bt, 4, q8, 3, parent, pools)
    r.call()
    out = r.result()
    for b, (p, n) in enumerate(bt.seqs):
        tk = list(bt.tokens(b))
        sees = pr.ancestors(parent[tk])
        hit = np.array([[sees[i, j] for (bb, j) in dirty if bb == b] for i in range(n)]).any(1)
        assert 0 < hit.sum() < n
        for i in range(n):
            assert np.isfinite(out[tk[i]]).all() == (not hit[i]), (b, i)
        clean = [i for i in range(n) if not hit[i]]
        full = np.concatenate([np.ones((n, p), bool), sees], 1)
        K, V = (np.nan_to_num(host_rows(bt, pools[x], b, 0, p + n), posinf=0, neginf=0) for x in "KV")
        want, _, _ = pr.attend(r.q[tk].astype(np.float64), K, V, full, bt.hd)
        err = np.linalg.norm(out[tk][clean] - want[clean]) / np.linalg.norm(want[clean])
        assert err <= NORM_TOL


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("row", [0, 31, 35, 39])
def test_tree_committed_values_that_are_not_finite(hip, n, row):
    """A committed V row that is not finite reaches every token of its sequence and kv head, and no other, wherever
    it lies among the drafts' keys."""
    rng = np.random.default_rng(row)
    bt = Batch([(40, n), (50, 2)], 2, 64, 100, rng)
    pools = fill_f32(bt, 3)
    at = bt.row(0, 1, row)
    pools["V"][at:at + 64] = np.nan
    r = Run(bt, 2, False, 3, random_parents(bt, rng, "random"), pools=pools)
    r.call()
    out = r.result()
    assert np.isnan(out[:n, 2:]).all()
    assert np.isfinite(out[:n, :2]).all() and np.isfinite(out[n:]).all()


def test_attention_large_scores(hip):
    """Scores of thousands (a channel of K far above the others) and queries and keys far from 1."""
    rng = np.random.default_rng(9)
    bt = Batch([(500, 1), (60, 20)], 1, 128, 600, rng)
    for q8, scale in ((True, 1.0), (True, 2.0 ** 20), (True, 2.0 ** -30), (False, 1.0), (False, 2.0 ** 20),
                      (False, 2.0 ** -30)):
        parent = random_parents(bt, rng, "chain")
        pools = (fill_q8 if q8 else fill_f32)(bt, 3)
        r = Run(bt, 4, q8, 3, parent, pools)
        r.q *= np.float32(40.0 * scale)
        if q8:
            for n, f in (("K", 1.0 / scale if scale < 1 else 1.0), ("V", 2.0 ** -12)):
                r.pools[n][1][:] = (r.pools[n][1].astype(np.float64) * min(f, 2.0 ** 14)).astype(np.float16)
        else:
            r.pools["K"][:] *= np.float32(1.0 / scale)
            r.pools["V"][:] *= np.float32(2.0 ** 100)
        if q8 and scale > 1:
            r.q /= np.float32(scale / 8)
        r.qd.upload(r.q)
        for d, a in zip(r.pd, [a for n in "KV" for a in (r.pools[n] if q8 else (r.pools[n],))]):
            d.upload(a)
        r.call()
        r.check(norm=False)


# -- cache ------------------------------------------------------------------------
def store_load(bt, k, v, ld, extra=0):
    Hkv, hd = bt.Hkv, bt.hd
    kd, vd = DeviceBuffer.from_array(k), DeviceBuffer.from_array(v)
    pools = {n: (DeviceBuffer.from_array(np.full(bt.elems, 99, np.int8)),
                 DeviceBuffer.from_array(np.full(bt.elems // 32, 7.0, np.float16))) for n in "KV"}
    ps = [d.p for n in "KV" for d in pools[n]]
    size = (bt.B, bt.T, Hkv, hd, bt.head_stride, bt.max_seq)
    ok(lib().slate_hip_kv_store_q8(*ps, kd.p, vd.p, ld, *bt.desc(), *size), "store")
    back = [DeviceBuffer.from_array(np.full((bt.T, ld), SENTINEL)) for _ in "KV"]
    ok(lib().slate_hip_kv_load_q8(back[0].p, back[1].p, ld, *ps, *bt.desc(), *size), "load")
    host = {n: (pools[n][0].to_array(np.int8, bt.elems), pools[n][1].to_array(np.float16, bt.elems // 32))
            for n in "KV"}
    return host, [b.to_array(np.float32, (bt.T, ld)) for b in back]


@pytest.mark.parametrize("hd,Hkv,extra", [(32, 1, 0), (64, 3, 4), (128, 8, 0), (96, 2, 32), (256, 2, 0), (512, 1, 8)])
def test_kv_store_and_load(hip, hd, Hkv, extra):
    rng = np.random.default_rng(hd)
    bt = Batch([(0, 1), (5, 7), (19, 0), (3, 33), (0, 40), (39, 1)], Hkv, hd, 40, rng, behind=3, bad=(3,))
    ld = Hkv * hd + extra
    k, v = (rng.normal(0, 1, (bt.T, ld)).astype(np.float32) for _ in "KV")
    t = bt.off[1]
    k[t + 1, :32] = 0.0
    k[t + 2, :32] = np.linspace(-127, 127, 32)                   # step 1: halves are ties
    k[t + 2, 3:7] = [0.5, 1.5, -2.5, 126.5]
    k[t, :32] = 2.0 ** -24 * np.arange(32)                      # steps below f16's normal range
    v[t, :32] = 1e-9                                             # a step that rounds to zero
    v[t + 1, :32] = np.linspace(-3e38, 3e38, 32)                 # above the largest step
    v[t + 2, :32] = np.nan
    v[t + 3, 3], v[t + 3, 4], v[t + 3, 5] = np.nan, np.inf, -np.inf
    v[t + 4, :32] = np.float32(127.0) * np.nextafter(np.float32(1), np.float32(2))
    host, (kb, vb) = store_load(bt, k, v, ld)
    for name, x, back in (("K", k, kb), ("V", v, vb)):
        q, s = np.full(bt.elems, 99, np.int8), np.full(bt.elems // 32, 7.0, np.float16)
        want = np.full((bt.T, ld), SENTINEL)
        for b, (p, n) in enumerate(bt.seqs):
            for i, t in enumerate(bt.tokens(b)):
                cq, cs = pr.quantise(x[t, :Hkv * hd].reshape(Hkv, hd))
                want[t, :Hkv * hd] = pr.values(cq, cs).reshape(-1).astype(np.float32)
                for h in range(Hkv):
                    at = bt.row(b, h, p + i)
                    q[at:at + hd] = cq[h]
                    s[at // 32:(at + hd) // 32] = cs[h]
        assert np.array_equal(host[name][0], q)
        assert np.array_equal(host[name][1].view(np.uint16), s.view(np.uint16))
        assert np.array_equal(back, want)


def test_kv_many_tokens(hip):
    """More tokens than one per workgroup, more sequences than lanes, rows left out among them."""
    rng = np.random.default_rng(7)
    for B, most in ((9, 400), (80, 40)):
        seqs = [(int(rng.integers(0, 30)), int(rng.integers(0, most))) for _ in range(B)]
        bt = Batch(seqs, 2, 64, 460, rng, behind=5, bad=(2,))
        k, v = (rng.normal(0, 1, (bt.T, 128)).astype(np.float32) for _ in "KV")
        assert bt.T >= 1024
        _, back = store_load(bt, k, v, 128)
        for x, y in ((k, back[0]), (v, back[1])):
            want = pr.values(*pr.quantise(x)).astype(np.float32)
            owned = np.zeros(bt.T, bool)
            for b in range(B):
                owned[list(bt.tokens(b))] = True
            assert np.array_equal(y[owned], want[owned]) and np.all(y[~owned] == SENTINEL)


def test_kv_codes_at_every_tie(hip):
    """Elements at and next to each tie of the rounding, for many steps: the nearest code, ties to even."""
    rng = np.random.default_rng(2)
    n = 64
    k = np.zeros((n, 64), np.float32)
    for t in range(n):
        d = np.float32(np.float16(rng.uniform(2.0 ** -14, 4.0)))
        for blk in range(2):
            x = (rng.integers(0, 127, 32) + 0.5).astype(np.float32) * d
            x = np.where(rng.integers(0, 3, 32) == 1, np.nextafter(x, np.float32(1e9)), x)
            x = np.where(rng.integers(0, 3, 32) == 1, np.nextafter(x, np.float32(0)), x)
            x *= rng.choice([-1, 1], 32).astype(np.float32)
            x[blk] = 127 * d
            k[t, 32 * blk:32 * blk + 32] = x
    bt = Batch([(0, n)], 1, 64, n, rng)
    host, _ = store_load(bt, k, k, 64)
    cq, cs = pr.quantise(k)
    at = bt.row(0, 0, 0)
    assert np.array_equal(host["K"][0][at:at + n * 64], cq.reshape(-1))
    assert np.array_equal(host["K"][1][at // 32:at // 32 + 2 * n].view(np.uint16), cs.reshape(-1).view(np.uint16))


def test_kv_steps_next_to_ties(hip):
    """The step is f16(max / 127) with one rounding: maxima at and next to 127 times each kind of f16 tie (a quotient
    taken as a product with 1 / 127 lands on the wrong side of some, 1.9853441 among them)."""
    rng = np.random.default_rng(6)
    bits = np.concatenate([np.arange(1, 64), rng.integers(64, 0x7bfe, 1500), [0x7bfe]]).astype(np.uint16)
    low, high = (b.view(np.float16).astype(np.float64) for b in (bits, bits + np.uint16(1)))
    tie = 127.0 * (low + high) / 2                     # exact: 12 bits times 7
    tops, want = [], []
    for by in (-2, -1, 0, 1, 2):
        t = tie.astype(np.float32)
        for _ in range(abs(by)):
            t = np.nextafter(t, np.float32(np.inf) if by > 0 else np.float32(0))
        up = (t > tie) | ((t == tie) & (bits % 2 == 1))
        tops.append(t)
        want.append(bits + up.astype(np.uint16))
    more = np.array([1.9853441, 1.9892198, 3.9706881, 3.9939425], np.float32)
    tops = np.concatenate(tops + [more])
    want = np.concatenate(want + [(more.astype(np.float64) / 127).astype(np.float16).view(np.uint16)])
    n = -(-len(tops) // 2)
    k = np.zeros((n, 64), np.float32)
    k.reshape(-1, 32)[:len(tops), 7] = tops * rng.choice([-1, 1], len(tops)).astype(np.float32)
    k.reshape(-1, 32)[:len(tops), 20] = tops / np.float32(3)
    bt = Batch([(0, n)], 1, 64, n, rng)
    host, back = store_load(bt, k, k, 64)
    at = bt.row(0, 0, 0)
    for name in "KV":
        got = host[name][1][at // 32:at // 32 + len(tops)].view(np.uint16)
        assert np.array_equal(got, want), (tops[got != want][:5], got[got != want][:5], want[got != want][:5])
    cq, cs = pr.quantise(k)
    assert np.array_equal(host["K"][0][at:at + n * 64], cq.reshape(-1))
    assert np.array_equal(back[0], pr.values(cq, cs).astype(np.float32))


# -- offsets, streams, graphs, threads ----------------------------------------------
@pytest.mark.parametrize("q8", [False, True])
def test_offsets_past_32_bits(hip, q8):
    """Pools whose rows start past 2^31 elements (8-bit) and past 2^32 bytes (f32)."""
    rng = np.random.default_rng(4)
    hd, G = 64, 4
    bt = Batch([(33, 9), (70, 3)], 1, hd, 80, rng)
    parent = random_parents(bt, rng, "random")
    r = Run(bt, G, q8, 3, parent)
    far = (1 << 31) + (1 << 20) if q8 else (1 << 30) + (1 << 20)
    small, big = r.pd, []
    widths = (1, 2, 1, 2) if q8 else (4, 4)
    for d, w in zip(small, widths):
        at = far // 32 * 2 if w == 2 else far * w
        b = DeviceBuffer(at + d.nbytes)
        host = d.to_array(np.uint8, d.nbytes)
        lib().slate_hip_copy_h2d(b.ptr + at, host.ctypes.data_as(C.c_void_p), host.nbytes)
        big.append(b)
    bt.base = bt.base + far
    bt.d_base.upload(bt.base)
    r.pd = big
    r.call()
    bt.base = bt.base - far
    r.check()


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
    """Captured attention calls with a workspace each, replayed between eager calls, on new queries; one
    without a workspace is refused and leaves the stream usable."""
    rng = np.random.default_rng(6)
    runs = []
    for k, (q8, n) in enumerate(((True, 9), (True, 40), (False, 9))):
        bt = Batch([(2000 + 700 * k, n), (50, 5)], 1, 128, 4000, rng)
        runs.append(Run(bt, 4, q8, 40 + k, random_parents(bt, rng, "random")))
    for r in runs:
        r.call(own_ws=True)
    refused = _Graph(lambda: runs[0].call())
    assert refused.error and "workspace" in refused.error
    refused.free()
    graphs = [_Graph(lambda r=r: r.call(own_ws=True)) for r in runs]
    assert all(g.error is None for g in graphs)
    for rep in range(4):
        for r in runs:
            r.q = rng.normal(0, 1, r.q.shape).astype(np.float32)
            r.qd.upload(r.q)
            r.out.upload(np.full_like(r.q, SENTINEL))
        for g in graphs:
            g.launch()
        lib().slate_hip_sync()
        for r in runs:
            r.check()
            r.call()                                   # eager, on the backend's own workspace
            r.check()
    for g in graphs:
        g.free()


def test_calls_from_several_threads(hip):
    rng = np.random.default_rng(8)
    runs = []
    for k in range(4):
        bt = Batch([(100 * k + 40, 1), (1500, 1), (10 * k, 1)], 1, 64, 1600, rng)
        runs.append(Run(bt, 4, True, 50 + k))
    fail = []

    def work(r):
        try:
            for _ in range(8):
                r.call()
        except Exception as e:                         # reported by the main thread
            fail.append(e)
    ts = [threading.Thread(target=work, args=(r,)) for r in runs]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not fail
    for r in runs:
        r.check()


# -- together -----------------------------------------------------------------------
def test_a_serving_step_with_drafts(hip):
    """As a serving program runs them: pack_batch lays a batch out, q and k are rotated in one call, K and V go
    into the 8-bit cache, causal attention reads it; then the same with drafted trees, whose accepted tokens are
    stored again at their final rows and read by the next step."""
    rng = np.random.default_rng(13)
    Hq, Hkv, hd, max_seq, slots = 8, 2, 64, 96, 3
    G, width = Hq // Hkv, (Hq + 2 * Hkv) * hd
    L = lib()
    stride = Hkv * max_seq * hd
    pool = [DeviceBuffer.from_array(np.zeros(slots * stride, np.int8) if i % 2 == 0 else
                                    np.zeros(slots * stride // 32, np.float16)) for i in range(4)]
    cfg = dict(layout=1, rot_dim=32, scaling=2, orig_ctx=32, theta_base=10000.0, factor=4.0, low=1.0, high=4.0)
    w, m = pr.rope_frequencies(1, 32, 2, 10000.0, 4.0, 1.0, 4.0, 32)
    slot = np.array([2, 0, 1], np.int32)
    kept = [[np.zeros((0, Hkv, hd)), np.zeros((0, Hkv, hd))] for _ in range(3)]    # cached values per sequence

    def step(pos0, n_new, positions, parent):
        T = int(np.sum(n_new))
        d = {k: DeviceBuffer.from_array(np.asarray(v, np.int32)) for k, v in
             (("slot", slot), ("pos0", pos0), ("n", n_new), ("positions", positions))}
        o = {k: DeviceBuffer(8 * 64) for k in ("off", "t2s", "tpos", "base", "last", "status")}
        ok(L.slate_hip_pack_batch(d["slot"].p, d["pos0"].p, d["n"].p, 3, max_seq, stride, 64, o["off"].p, o["t2s"].p,
                                  o["tpos"].p, o["base"].p, o["last"].p, o["status"].p))
        qkv = rng.normal(0, 1, (T, width)).astype(np.float32)
        rot, x = DeviceBuffer(qkv.nbytes), DeviceBuffer.from_array(qkv)
        c = slate_amd.RopeConfig(**cfg)
        ok(L.slate_hip_rope_scaled(rot.p, x.p, d["positions"].p, T, Hq + Hkv, hd, width, C.byref(c)))
        qk = pr.rope(qkv[:, :(Hq + Hkv) * hd].reshape(T, -1, hd).astype(np.float64), np.asarray(positions), 1, 32, w, m)
        got = rot.to_array(np.float32, (T, width))[:, :(Hq + Hkv) * hd].reshape(T, -1, hd)
        assert np.abs(got - qk).max() <= 8 * 2.0 ** -23 * np.abs(qk).max()
        off = o["off"].to_array(np.int32, 4)
        kf, vf = C.c_void_p(rot.ptr + Hq * hd * 4), C.c_void_p(x.ptr + (Hq + Hkv) * hd * 4)
        size = (3, T, Hkv, hd, max_seq * hd, max_seq)
        ok(L.slate_hip_kv_store_q8(*[p.p for p in pool], kf, vf, width, o["off"].p, d["pos0"].p, o["base"].p, *size))
        q = np.ascontiguousarray(got[:, :Hq])
        qd, out = DeviceBuffer.from_array(q), DeviceBuffer(q.nbytes)
        args = (3, T, int(max(n_new)), Hq, Hkv, hd, max_seq * hd, max_seq, None, 0)
        if parent is None:
            ok(L.slate_hip_attention_ragged_q8(out.p, qd.p, *[p.p for p in pool], o["off"].p, d["pos0"].p, o["base"].p,
                                               *args))
        else:
            pd = DeviceBuffer.from_array(parent)
            ok(L.slate_hip_attention_tree_q8(out.p, qd.p, *[p.p for p in pool], o["off"].p, d["pos0"].p, o["base"].p,
                                             pd.p, *args))
        res = out.to_array(np.float32, q.shape)
        K = pr.values(*pr.quantise(got[:, Hq:]))
        V = pr.values(*pr.quantise(qkv[:, (Hq + Hkv) * hd:].reshape(T, Hkv, hd)))
        for b in range(3):
            s, p, n = slice(off[b], off[b + 1]), pos0[b], n_new[b]
            sees = np.ones((n, p + n), bool)
            sees[:, p:] = np.tril(np.ones((n, n), bool)) if parent is None else pr.ancestors(parent[s])
            for h in range(Hkv):
                Kh, Vh = (np.concatenate([kept[b][i][:p, h], x[s, h]]) for i, x in ((0, K), (1, V)))
                want, _, _ = pr.attend(q[s, h * G:(h + 1) * G].astype(np.float64), Kh, Vh, sees, hd)
                err = np.linalg.norm(res[s, h * G:(h + 1) * G] - want) / np.linalg.norm(want)
                assert err <= NORM_TOL
        return K, V, off, rot, x, d, o

    # prompts of different lengths
    n = [20, 3, 33]
    K, V, off, *_ = step([0, 0, 0], n, np.concatenate([np.arange(k) for k in n]), None)
    for b in range(3):
        kept[b] = [K[off[b]:off[b + 1]], V[off[b]:off[b + 1]]]
    # drafted trees: positions go by depth, rows by order
    nd = [5, 1, 7]
    parent = np.array([-1, 0, 0, 1, 2] + [-1] + [-1, -1, 0, 1, 2, 3, 4], np.int32)
    depth, at = [], 0
    for k in nd:
        dd = []
        for i in range(k):
            dd.append(0 if parent[at + i] < 0 else dd[parent[at + i]] + 1)
        depth += dd
        at += k
    p0 = np.repeat(n, nd)
    K, V, off, rot, x, d, o = step(n, nd, p0 + np.array(depth), parent)
    # accepted: draft 0, 2, 4 of the first sequence, 0 of the second, 1, 3 of the third
    accepted = [[0, 2, 4], [0], [1, 3]]
    rows = np.concatenate([off[b] + np.array(a) for b, a in enumerate(accepted)])
    kr = rot.to_array(np.float32, (sum(nd), width))[rows][:, Hq * hd:(Hq + Hkv) * hd]
    vr = x.to_array(np.float32, (sum(nd), width))[rows][:, (Hq + Hkv) * hd:]
    na = [len(a) for a in accepted]
    kd, vd, od = (DeviceBuffer.from_array(np.ascontiguousarray(a)) for a in
                  (kr, vr, np.concatenate([[0], np.cumsum(na)]).astype(np.int32)))
    ok(L.slate_hip_kv_store_q8(*[p.p for p in pool], kd.p, vd.p, Hkv * hd, od.p, d["pos0"].p, o["base"].p, 3, sum(na),
                               Hkv, hd, max_seq * hd, max_seq))
    at = 0
    for b in range(3):
        s = rows[at:at + na[b]]
        kept[b] = [np.concatenate([kept[b][0], K[s]]), np.concatenate([kept[b][1], V[s]])]
        at += na[b]
    # and the next decode step reads what was accepted
    total = [a + b for a, b in zip(n, na)]
    step(total, [1, 1, 1], np.array(total), None)
