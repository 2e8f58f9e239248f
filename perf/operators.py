"""Measured operators of serving with an 8-bit K/V cache and drafted tokens:

  rope       rotary positions: pairs in halves or interleaved, part of a head,
             frequencies rescaled for contexts longer than the trained one
  kv         new K/V rows quantised into the cache (blocks of 32 with an f16
             step, the values of Q8_0) and read back as f32
  ragged_q8  causal GQA attention of a packed batch over that cache: decode
             tokens, prompt chunks, both
  tree       attention of trees of drafted tokens over an f32 cache: a token
             sees its sequence's committed keys, its ancestors and itself
  tree_q8    the same over the 8-bit cache

A batch is B sequences, packed token-major: sequence b has the tokens
tok_off[b] .. tok_off[b+1]-1, pos0[b] rows of it are cached already, and its
token i belongs to cache row pos0[b] + i.  The row p of kv head h starts at
element kv_base[b] + h * head_stride + p * head_dim of the K and of the V pool;
the steps of an 8-bit pool are laid out alike, one for 32 elements.

Inputs: queries and cached rows N(0, 1), a few channels of K ten times as
large, as trained models have them; slots of the cache in a shuffled order.
"""
from __future__ import annotations

import ctypes
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 32


# -- cases --------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 users, q and k heads of the 8B shape in one call, context rescaled 8x
        {"name": "rope decode 16", "op": "rope", "rows": 16, "heads": 40, "hd": 128, "rot": 128, "layout": 0,
         "scaling": 2, "theta": 500000.0, "factor": 8.0, "low": 1.0, "high": 4.0, "orig": 8192, "far": 65536},
        # prompt chunks of the 70B shape's heads, half of each head rotated, interleaved pairs, far positions
        {"name": "rope chunk 4096", "op": "rope", "rows": 4096, "heads": 72, "hd": 128, "rot": 64, "layout": 1,
         "scaling": 3, "theta": 10000.0, "factor": 16.0, "low": 1.0, "high": 32.0, "orig": 4096, "far": 65536},
        # a decode step's 16 new rows go into the cache
        {"name": "kv decode 16", "op": "kv", "B": 16, "dec": 16, "n": 1, "L": 4096, "Hkv": 8, "hd": 128, "lens": 1},
        # five prompt chunks of odd lengths
        {"name": "kv chunks", "op": "kv", "B": 5, "dec": 0, "n": 1601, "L": 8192, "Hkv": 8, "hd": 128, "lens": 2},
        # one user, short context: latency
        {"name": "q8 one token", "op": "ragged_q8", "B": 1, "dec": 1, "n": 1, "L": 333, "Hkv": 8, "G": 4, "hd": 64,
         "lens": 3},
        # decode step of 16 users, 8B heads
        {"name": "q8 decode 16", "op": "ragged_q8", "B": 16, "dec": 16, "n": 1, "L": 4096, "Hkv": 8, "G": 4,
         "hd": 128, "lens": 4},
        # decode step of 64 users with contexts up to 16384
        {"name": "q8 decode 64", "op": "ragged_q8", "B": 64, "dec": 64, "n": 1, "L": 16384, "Hkv": 8, "G": 4,
         "hd": 128, "lens": 5},
        # a mixed step: 13 users decode, three bring prompt chunks
        {"name": "q8 chunks", "op": "ragged_q8", "B": 16, "dec": 13, "n": 1024, "L": 4096, "Hkv": 8, "G": 4,
         "hd": 128, "lens": 6},
        # one user's drafted tree
        {"name": "tree one", "op": "tree", "B": 1, "dec": 0, "n": 17, "L": 1000, "Hkv": 8, "G": 4, "hd": 128,
         "lens": 7},
        # sixteen users' trees over long f32 caches
        {"name": "tree 16", "op": "tree", "B": 16, "dec": 0, "n": 26, "L": 8192, "Hkv": 8, "G": 4, "hd": 128,
         "lens": 8},
        # small trees of sixteen users, 8-bit cache
        {"name": "tree q8 16", "op": "tree_q8", "B": 16, "dec": 0, "n": 8, "L": 4096, "Hkv": 8, "G": 4, "hd": 128,
         "lens": 9},
        # large trees over long contexts, 70B heads
        {"name": "tree q8 long", "op": "tree_q8", "B": 4, "dec": 0, "n": 64, "L": 16384, "Hkv": 8, "G": 8, "hd": 128,
         "lens": 10},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "kv", "ragged_q8", "ragged_q8", "tree", "tree_q8"])
    if op == "rope":
        hd = 2 * rng.randint(8, 128)
        heads = rng.choice([1, 5, 12, 40, 72])
        rows = _log(rng, 1, 4096 * 72 * 128 // (heads * hd))
        scaling = rng.randint(0, 3)
        return {"op": op, "rows": min(rows, 16384), "heads": heads, "hd": hd, "rot": 2 * rng.randint(4, hd // 2),
                "layout": rng.randint(0, 1), "scaling": scaling, "theta": rng.choice([10000.0, 500000.0, 1e6]),
                "factor": rng.uniform(1.5, 32.0), "low": 1.0, "high": rng.choice([4.0, 32.0]),
                "orig": rng.choice([2048, 4096, 8192]), "far": _log(rng, 64, 1 << 20)}
    hd = rng.choice([32, 64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    B = _log(rng, 1, 64)
    if op == "kv":
        n = _log(rng, 1, max(2, 6000 // B))
        return {"op": op, "B": B, "dec": rng.randint(0, B), "n": n, "L": n + _log(rng, 1, 8192), "Hkv": Hkv, "hd": hd,
                "lens": rng.randrange(1 << 20)}
    G = rng.choice([1, 2, 3, 4, 7, 8])
    if op == "ragged_q8":
        dec = rng.choice([B, rng.randint(0, B)])
        n = 1 if dec == B else _log(rng, 2, 1024)
        ctx = _log(rng, 1, 4096 if dec < B else 16384)
    else:
        dec, n, ctx = 0, _log(rng, 2, 64), _log(rng, 1, 16384)
    # at most the largest listed case's queries times keys, and cached bytes
    while (B - dec) * n * Hkv * G * (ctx + n) > 400_000_000 or B * (ctx + n) * Hkv * hd > 200_000_000:
        ctx, n = max(1, ctx // 2), (max(2, n // 2) if dec < B else 1)
        if ctx == 1:
            B = max(1, B // 2)
            dec = min(dec, B)
            if dec == B and op == "ragged_q8":
                n = 1
    return {"op": op, "B": B, "dec": dec, "n": n, "L": ctx + n, "Hkv": Hkv, "G": G, "hd": hd,
            "lens": rng.randrange(1 << 20)}


def _batch(case):
    """(tokens, cached rows) of each sequence: the first `dec` bring one token, the others up to n; contexts are
    ragged between a quarter of L and L, the first sequence's reaching it."""
    r = random.Random(case["lens"])
    n, p = [], []
    for b in range(case["B"]):
        k = 1 if b < case["dec"] else r.randint((case["n"] + 1) // 2, case["n"])
        total = case["L"] if b == 0 else r.randint(max(k, case["L"] // 4), max(k, case["L"]))
        n.append(k)
        p.append(max(0, total - k))
    return n, p


def _parents(case, n):
    """A tree per sequence: each drafted token hangs on one of the four before it, or on the last committed token."""
    r = random.Random(case["lens"] + 1)
    out = []
    for k in n:
        out += [-1 if i == 0 or r.random() < 0.1 else r.randint(max(0, i - 4), i - 1) for i in range(k)]
    return out


def work(case):
    if case["op"] == "rope":
        vals = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 8 * vals + 4 * case["rows"], "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    n, p = _batch(case)
    hd, Hkv, T = case["hd"], case["Hkv"], sum(n)
    row8 = hd + 2 * hd // BLOCK
    if case["op"] == "kv":
        return {"bytes": T * Hkv * 2 * (4 * hd + row8 + row8 + 4 * hd), "flops": T * Hkv * 2 * hd * 4}
    Hq = Hkv * case["G"]
    row = 4 * hd if case["op"] == "tree" else row8
    if case["op"] == "ragged_q8":
        seen = sum(k * q + k * (k + 1) // 2 for k, q in zip(n, p))
    else:
        par, seen, at = _parents(case, n), 0, 0
        for k, q in zip(n, p):
            depth = []
            for i in range(k):
                j = par[at + i]
                depth.append(1 + (depth[j] if j >= 0 else 0))
                seen += q + depth[-1]
            at += k
    keys = sum(n) + sum(p)
    return {"bytes": keys * Hkv * 2 * row + 2 * 4 * T * Hq * hd, "flops": 4 * seen * Hq * hd}


# -- inputs -------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _channels(case, g):
    """K's channels: a few are ten times as large as the others."""
    w = torch.ones(case["Hkv"], case["hd"], device=DEV)
    w[:, torch.randint(0, case["hd"], (max(1, case["hd"] // 32),), generator=g, device=DEV)] = 10.0
    return w


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "rope":
        rows, heads, hd = case["rows"], case["heads"], case["hd"]
        st = {"case": case, "x": torch.randn(rows, heads, hd, generator=g, device=DEV),
              "y": torch.empty(rows, heads, hd, device=DEV),
              "pos": torch.randint(0, case["far"], (rows,), generator=g, device=DEV, dtype=torch.int32)}
        torch.cuda.synchronize()
        return st
    n, p = _batch(case)
    B, Hkv, hd, T = case["B"], case["Hkv"], case["hd"], sum(n)
    cap = case["L"] + 5                        # rows of a slot: the capacity is no round number
    off = [0]
    for k in n:
        off.append(off[-1] + k)
    perm = torch.randperm(B, generator=g, device=DEV)
    st = {"case": case, "B": B, "T": T, "n_max": max(n), "L_max": max(a + b for a, b in zip(n, p)), "max_seq": cap,
          "head_stride": cap * hd, "tok_off": torch.tensor(off, dtype=torch.int32, device=DEV),
          "pos0": torch.tensor(p, dtype=torch.int32, device=DEV), "kv_base": perm * (Hkv * cap * hd)}
    rows = B * Hkv * cap
    if case["op"] == "kv":
        st["k"] = torch.randn(T, Hkv, hd, generator=g, device=DEV) * _channels(case, g)
        st["v"] = torch.randn(T, Hkv, hd, generator=g, device=DEV)
        for name in ("K", "V"):
            st[name + "q"] = torch.zeros(rows, hd, dtype=torch.int8, device=DEV)
            st[name + "s"] = torch.zeros(rows, hd // BLOCK, dtype=torch.float16, device=DEV)
        st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        torch.cuda.synchronize()
        return st
    Hq = Hkv * case["G"]
    st["q"] = torch.randn(T, Hq, hd, generator=g, device=DEV)
    st["out"] = torch.empty_like(st["q"])
    K = torch.randn(B, Hkv, cap, hd, generator=g, device=DEV) * _channels(case, g).view(1, Hkv, 1, hd)
    V = torch.randn(B, Hkv, cap, hd, generator=g, device=DEV)
    if case["op"] == "tree":
        st["K"], st["V"] = K.view(rows, hd), V.view(rows, hd)
    else:
        st["Kq"], st["Ks"] = _quantise(K.view(rows, hd))
        st["Vq"], st["Vs"] = _quantise(V.view(rows, hd))
    if case["op"] != "ragged_q8":
        st["parent"] = torch.tensor(_parents(case, n), dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    return st


# -- plain forms --------------------------------------------------------------
def _quantise(x):
    """Blocks of 32: step d = f16(max|x| / 127), codes x / d rounded to the nearest whole number, ties to even.  The
    quotient is taken in 64 bits: in 32 it can land on a tie that x is only next to."""
    b = x.reshape(-1, BLOCK)
    d = (b.abs().amax(1, keepdim=True) / 127.0).clamp(max=65504.0).half()
    q = torch.where(d > 0, b.double() / d.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    q = torch.round(q).clamp(-127, 127).to(torch.int8)
    return q.view(x.shape), d.view(x.shape[0], -1)


def _values(q, s):
    return (q.view(q.shape[0], -1, BLOCK).float() * s.float().unsqueeze(2)).view(q.shape)


def _frequencies(case):
    """Angle per position of each pair, in 64 bits, and the factor on the rotated elements."""
    rot, f = case["rot"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    w = torch.exp(i * (-2.0 / rot * math.log(case["theta"])))
    if case["scaling"] == 0:
        return w, 1.0
    if case["scaling"] == 1:
        return w / f, 1.0
    if case["scaling"] == 2:
        turns = case["orig"] * w / (2 * math.pi)
        keep = ((turns - case["low"]) / (case["high"] - case["low"])).clamp(0.0, 1.0)
        return w / f * (1 - keep) + w * keep, 1.0

    def pair(turns):
        return rot * math.log(case["orig"] / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))
    lo = max(0, math.floor(pair(case["high"])))
    hi = min(rot - 1, math.ceil(pair(case["low"])))
    slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return w / f * slow + w * (1 - slow), 0.1 * math.log(f) + 1.0


def _rope_plain(st):
    c, x = st["case"], st["x"]
    w, mag = _frequencies(c)
    ang = st["pos"].double().unsqueeze(1) * w
    cos, sin = (torch.cos(ang) * mag).float().unsqueeze(1), (torch.sin(ang) * mag).float().unsqueeze(1)
    rot = c["rot"]
    if c["layout"] == 0:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2)
    return torch.cat([y, x[..., rot:]], 2)


def _rows(st, h_rows):
    """Pool rows [T, Hkv] of the batch's tokens."""
    t = torch.arange(st["T"], device=DEV)
    seq = torch.searchsorted(st["tok_off"][1:].long(), t, right=True)
    row = st["kv_base"][seq] // st["case"]["hd"] + st["pos0"][seq] + t - st["tok_off"][seq]
    return row.unsqueeze(1) + h_rows


def _heads(st):
    return torch.arange(st["case"]["Hkv"], device=DEV) * st["max_seq"]


def _kv_plain(st):
    rows = _rows(st, _heads(st)).reshape(-1)
    out = []
    for name, x in (("K", st["k"]), ("V", st["v"])):
        q, s = _quantise(x.view(-1, st["case"]["hd"]))
        st[name + "q"][rows], st[name + "s"][rows] = q, s
        out.append(_values(st[name + "q"][rows], st[name + "s"][rows]).view(x.shape))
    return out


def _seen(st, lo, hi, n, keys):
    """[hi - lo, n, L]: whether token i of sequence b sees key j."""
    p = st["pos0"][lo:hi].view(-1, 1, 1)
    i = torch.arange(n, device=DEV).view(1, -1, 1)
    if "parent" not in st:
        return keys <= p + i
    # ancestors: the closure of the parent relation, by squaring
    tok = (st["tok_off"][lo:hi].view(-1, 1) + i.view(1, -1)).clamp(max=st["T"] - 1)
    par = st["parent"][tok].long()
    up = torch.zeros(hi - lo, n, n, device=DEV)
    up.scatter_(2, par.clamp(min=0).unsqueeze(2), (par >= 0).float().unsqueeze(2))
    up = up + torch.eye(n, device=DEV)
    for _ in range(max(1, (n - 1).bit_length())):
        up = (torch.matmul(up, up) > 0).float()
    j = (keys - p).expand(hi - lo, n, keys.shape[2])
    drafted = torch.gather(up, 2, j.clamp(0, n - 1)) > 0
    return (j < 0) | ((j < n) & drafted)


def _attention_part(st, lo, hi, n):
    """Sequences lo .. hi-1, each padded to n tokens."""
    c = st["case"]
    hd, Hkv, G, B, L = c["hd"], c["Hkv"], c["G"], hi - lo, st["L_max"]
    key = torch.arange(L, device=DEV)
    rows = ((st["kv_base"][lo:hi] // hd).view(-1, 1, 1) + _heads(st).view(1, -1, 1) + key).reshape(-1)
    if c["op"] == "tree":
        K, V = st["K"][rows], st["V"][rows]
    else:
        K, V = _values(st["Kq"][rows], st["Ks"][rows]), _values(st["Vq"][rows], st["Vs"][rows])
    K, V = K.view(B, Hkv, L, hd), V.view(B, Hkv, L, hd)
    tok = st["tok_off"][lo:hi].view(-1, 1) + torch.arange(n, device=DEV)
    real = tok < st["tok_off"][lo + 1:hi + 1].view(-1, 1)
    q = st["q"][tok.clamp(max=st["T"] - 1)].view(B, n, Hkv, G, hd).permute(0, 2, 1, 3, 4)
    s = torch.matmul(q.reshape(B, Hkv, n * G, hd) / math.sqrt(hd), K.transpose(2, 3).contiguous())
    s = s.view(B, Hkv, n, G, L)
    s = s.masked_fill(~_seen(st, lo, hi, n, key.view(1, 1, -1)).view(B, 1, n, 1, L), -math.inf)
    s = torch.exp(s - s.amax(4, keepdim=True))
    o = torch.matmul(s.view(B, Hkv, n * G, L), V) / s.sum(4).view(B, Hkv, n * G, 1)
    o = o.view(B, Hkv, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B, n, Hkv * G, hd)
    return o[real]


def _attention_plain(st):
    dec, B = st["case"]["dec"], st["B"]
    if dec == 0 or dec == B:
        return _attention_part(st, 0, B, st["n_max"])
    return torch.cat([_attention_part(st, 0, dec, 1), _attention_part(st, dec, B, st["n_max"])])


# -- the framework's operators ------------------------------------------------
def _lib():
    import slate_amd
    slate_amd.Backend()                        # raises where there is no device
    return slate_amd


_kept = []


def _own(st):
    if not _kept:
        _kept.append(_lib())
    sa = _kept[0]
    lib, c = sa.load_library(), st["case"]

    def p(name):
        return st[name].data_ptr()
    if c["op"] == "rope":
        r = sa.RopeConfig(layout=c["layout"], rot_dim=c["rot"], scaling=c["scaling"], orig_ctx=c["orig"],
                          theta_base=c["theta"], factor=c["factor"], low=c["low"], high=c["high"], magnitude=0.0)
        rc = lib.slate_hip_rope_scaled(p("y"), p("x"), p("pos"), c["rows"], c["heads"], c["hd"], c["heads"] * c["hd"],
                                       ctypes.byref(r))
        if rc:
            sa.check(rc, "rope_scaled")
        return st["y"]
    batch = (p("tok_off"), p("pos0"), p("kv_base"))
    if c["op"] == "kv":
        size = (st["B"], st["T"], c["Hkv"], c["hd"], st["head_stride"], st["max_seq"])
        pools = (p("Kq"), p("Ks"), p("Vq"), p("Vs"))
        ld = c["Hkv"] * c["hd"]
        rc = (lib.slate_hip_kv_store_q8(*pools, p("k"), p("v"), ld, *batch, *size) or
              lib.slate_hip_kv_load_q8(p("k_out"), p("v_out"), ld, *pools, *batch, *size))
        if rc:
            sa.check(rc, "kv_store_q8 / kv_load_q8")
        return [st["k_out"], st["v_out"]]
    size = (st["B"], st["T"], st["n_max"], c["Hkv"] * c["G"], c["Hkv"], c["hd"], st["head_stride"], st["max_seq"],
            None, 0)
    if c["op"] == "ragged_q8":
        rc = lib.slate_hip_attention_ragged_q8(p("out"), p("q"), p("Kq"), p("Ks"), p("Vq"), p("Vs"), *batch, *size)
    elif c["op"] == "tree_q8":
        rc = lib.slate_hip_attention_tree_q8(p("out"), p("q"), p("Kq"), p("Ks"), p("Vq"), p("Vs"), *batch,
                                             p("parent"), *size)
    else:
        rc = lib.slate_hip_attention_tree(p("out"), p("q"), p("K"), p("V"), *batch, p("parent"), *size)
    if rc:
        sa.check(rc, c["op"])
    return st["out"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _rope_plain(state) if op == "rope" else _kv_plain(state) if op == "kv" else _attention_plain(state)


# -- the definitions in 64 bits -----------------------------------------------
def _exact_rope(case, st):
    rot, half = case["rot"], case["rot"] // 2
    x, out = st["x"].double(), st["x"].double().clone()
    pos = st["pos"].double()
    mag = 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == 3 else 1.0
    for i in range(half):
        w = case["theta"] ** (-2.0 * i / rot)
        if case["scaling"] == 1:
            w /= case["factor"]
        elif case["scaling"] == 2:
            length = 2 * math.pi / w
            if length > case["orig"] / case["low"]:
                w /= case["factor"]
            elif length > case["orig"] / case["high"]:
                part = (case["orig"] / length - case["low"]) / (case["high"] - case["low"])
                w = (1 - part) * w / case["factor"] + part * w
        elif case["scaling"] == 3:
            a, b = (rot * math.log(case["orig"] / (t * 2 * math.pi)) / (2 * math.log(case["theta"]))
                    for t in (case["high"], case["low"]))
            a, b = max(0, math.floor(a)), min(rot - 1, math.ceil(b))
            part = min(1.0, max(0.0, (i - a) / (b - a if b > a else 0.001)))
            w = w / case["factor"] * part + w * (1 - part)
        j, k = (i, i + half) if case["layout"] == 0 else (2 * i, 2 * i + 1)
        co, si = torch.cos(pos * w).unsqueeze(1) * mag, torch.sin(pos * w).unsqueeze(1) * mag
        out[..., j] = x[..., j] * co - x[..., k] * si
        out[..., k] = x[..., k] * co + x[..., j] * si
    return out


def _exact_block(x):
    """x / d to the nearest code, and the code's value, in 64 bits (d itself is an f16 number by definition)."""
    b = x.double().view(x.shape[0], x.shape[1], -1, BLOCK)
    d = (b.abs().amax(3, keepdim=True) / 127.0).float().half().double()
    return (torch.nan_to_num(torch.round(b / d)).clamp(-127, 127) * d).view(x.shape)


def _exact_pool(st, name, lo, hi):
    if name in st:
        return st[name][lo:hi].double()
    q, s = st[name + "q"][lo:hi].double(), st[name + "s"][lo:hi].double()
    return q * s.repeat_interleave(BLOCK, 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, st)
    if case["op"] == "kv":
        return [_exact_block(st["k"]), _exact_block(st["v"])]
    hd, G, cap = case["hd"], case["G"], st["max_seq"]
    n, p = _batch(case)
    par = _parents(case, n)
    out, t = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV), 0
    for b, (k, ctx) in enumerate(zip(n, p)):
        sees = torch.ones(k, ctx + k, dtype=torch.bool)
        if case["op"] == "ragged_q8":
            sees[:, ctx:] = torch.tril(torch.ones(k, k, dtype=torch.bool))
        else:
            sees[:, ctx:] = False
            for i in range(k):
                j = i
                while j >= 0:
                    sees[i, ctx + j] = True
                    j = par[t + j]
        sees = sees.to(DEV)
        for h in range(case["Hkv"]):
            lo = int(st["kv_base"][b]) // hd + h * cap
            K, V = _exact_pool(st, "K", lo, lo + ctx + k), _exact_pool(st, "V", lo, lo + ctx + k)
            q = st["q"][t:t + k, h * G:(h + 1) * G].double().reshape(k * G, hd)
            s = (q @ K.t().contiguous()).view(k, G, ctx + k) * hd ** -0.5
            w = torch.softmax(torch.where(sees.view(k, 1, -1), s, -math.inf), 2)
            out[t:t + k, h * G:(h + 1) * G] = (w.view(k * G, -1) @ V).view(k, G, hd)
        t += k
    return out
