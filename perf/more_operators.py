"""Measured operators of serving with a paged K/V cache and drafted tokens:

  pages   pages of the cache taken for a step's new tokens, from the lengths of
          its requests, with the step's token descriptors and slot map; pages
          given back
  store   new K/V rows written into the pages by the slot map
  attend  attention of the new tokens (one of each sequence, or a few drafted
          ones) over the paged cache
  verify  which drafted tokens stand, from the target's logits, the draft's
          probabilities and given random numbers, and the token after them

A cache has n_pages pages of `page` rows.  table[slot, i] is the page of rows
i * page .. of that slot, held[slot] how many it has, free[0 .. n_free-1] are
the free ones, the last taken first.  A batch is B sequences, packed
token-major: sequence b has the tokens tok_off[b] .. tok_off[b+1]-1, pos0[b]
rows of it are cached already, and its token i belongs to its cache row
pos0[b] + i.  K/V pools lie [page, head, row, head_dim] (layout 0) or [page,
row, head, head_dim] (layout 1).

In `verify` a sequence's first row is the last committed token, the others are
drafts; parent[t] is the row, counted within the sequence, that row t continues.
Row t of the logits is the target's distribution after row t, row t of the
draft's probabilities the distribution that token t was drawn from.

Inputs: queries and cached rows N(0, 1), a few channels of K ten times as
large, as trained models have them; pages in shuffled order; logits N(0, 3)
with six likely tokens a row and one token in a hundred banned (-infinity),
drafts drawn from a noisy copy.
"""
from __future__ import annotations

import ctypes
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


# -- cases --------------------------------------------------------------------
def listed():
    return [
        # a decode step of 64 users: most have room in their last page, a few take one
        {"name": "pages decode 64", "op": "pages", "B": 64, "n": 1, "ctx": 4096, "page": 16, "lens": 1},
        # requests arrive and chunks of their prompts are placed: 37 sequences, odd lengths
        {"name": "pages prompts 37", "op": "pages", "B": 37, "n": 2048, "ctx": 2048, "page": 64, "lens": 2},
        # a decode step's new rows, 8B heads
        {"name": "store decode 16", "op": "store", "B": 16, "n": 1, "ctx": 4096, "page": 16, "Hkv": 8, "hd": 128,
         "type": 2, "layout": 0, "lens": 3},
        # five prompt chunks of odd lengths
        {"name": "store chunks", "op": "store", "B": 5, "n": 1601, "ctx": 4096, "page": 64, "Hkv": 8, "hd": 128,
         "type": 1, "layout": 1, "lens": 4},
        # one user, short context: latency
        {"name": "attend one token", "op": "attend", "B": 1, "n": 1, "ctx": 333, "page": 16, "Hkv": 8, "G": 4,
         "hd": 64, "type": 1, "layout": 0, "lens": 5},
        # decode step of 16 users, 8B heads, bf16 cache
        {"name": "attend bf16 16", "op": "attend", "B": 16, "n": 1, "ctx": 4096, "page": 16, "Hkv": 8, "G": 4,
         "hd": 128, "type": 2, "layout": 0, "lens": 6},
        # decode step of 64 users with contexts up to 16384, f16 cache
        {"name": "attend f16 64", "op": "attend", "B": 64, "n": 1, "ctx": 16384, "page": 64, "Hkv": 8, "G": 4,
         "hd": 128, "type": 1, "layout": 0, "lens": 7},
        # up to four drafts and the committed token of 16 users, f32 cache, token-major pages
        {"name": "attend f32 drafts 16", "op": "attend", "B": 16, "n": 5, "ctx": 8192, "page": 32, "Hkv": 8, "G": 4,
         "hd": 128, "type": 0, "layout": 1, "lens": 8},
        # up to seven drafts of eight users with long contexts, 70B heads
        {"name": "attend bf16 drafts 8", "op": "attend", "B": 8, "n": 8, "ctx": 16384, "page": 16, "Hkv": 8, "G": 8,
         "hd": 128, "type": 2, "layout": 0, "lens": 9},
        # one user's four drafts
        {"name": "verify one", "op": "verify", "B": 1, "n": 5, "V": 128256, "probs": True, "tree": False, "lens": 10},
        # 64 users with up to four drafts each, their probabilities kept
        {"name": "verify 64", "op": "verify", "B": 64, "n": 5, "V": 128256, "probs": True, "tree": False, "lens": 11},
        # trees of up to eight drafts of 16 users, guessed without probabilities
        {"name": "verify trees 16", "op": "verify", "B": 16, "n": 9, "V": 128256, "probs": False, "tree": True,
         "lens": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "store", "attend", "attend", "attend", "verify"])
    page = rng.choice([8, 16, 16, 32, 48, 64, 128, 256])
    lens = rng.randrange(1 << 20)
    if op == "pages":
        B = _log(rng, 1, 512)
        return {"op": op, "B": B, "n": _log(rng, 1, max(2, 65536 // B)), "ctx": _log(rng, 1, 16384), "page": page,
                "lens": lens}
    if op == "verify":
        V = rng.choice([256, 4999, 32000, 50257, 128256])
        tree = rng.random() < 0.4
        return {"op": op, "B": _log(rng, 1, 64 if V < 100000 else 40), "n": rng.randint(1, 8), "V": V,
                "probs": not tree and rng.random() < 0.7, "tree": tree, "lens": lens}
    c = {"op": op, "B": _log(rng, 1, 64), "page": page, "Hkv": rng.choice([1, 2, 4, 8]),
         "hd": rng.choice([32, 64, 80, 96, 128, 128, 128, 256]), "type": rng.randint(0, 2),
         "layout": rng.randint(0, 1), "lens": lens}
    if op == "store":
        c["n"], c["ctx"] = _log(rng, 1, max(2, 6000 // c["B"])), _log(rng, 1, 4096)
        return c
    c["n"], c["ctx"] = rng.choice([1, 1, rng.randint(2, 8)]), _log(rng, 1, 16384)
    c["G"] = rng.choice([1, 2, 3, 4, 7, 8])
    # at most the largest listed case's cached bytes
    while c["B"] * (c["ctx"] + c["n"]) * c["Hkv"] * c["hd"] * (4 if c["type"] == 0 else 2) > 1_500_000_000:
        c["ctx"] = max(1, c["ctx"] // 2)
    return c


def _batch(case):
    """(new tokens, cached rows) of each sequence: up to n, contexts ragged between a quarter of ctx and ctx, the
    first sequence's reaching it."""
    r, ctx = random.Random(case["lens"]), case.get("ctx", 1)
    n, p = [], []
    for b in range(case["B"]):
        n.append(r.randint((case["n"] + 1) // 2, case["n"]))
        p.append(ctx if b == 0 else r.randint(ctx // 4, ctx))
    return n, p


def _parents(case, n):
    """A tree per sequence: each draft continues one of the three rows before it; -1 for the first row."""
    r = random.Random(case["lens"] + 1)
    out = []
    for k in n:
        out += [i - 1 if not case["tree"] or i == 0 else r.randint(max(0, i - 3), i - 1) for i in range(k)]
    return out


def work(case):
    n, p = _batch(case)
    T, B = sum(n), case["B"]
    if case["op"] == "pages":
        ps = case["page"]
        fresh = sum(-(-(a + b) // ps) - -(-b // ps) for a, b in zip(n, p))
        # slot, pos0, n_new, held and lengths in; held, offsets, last rows, three numbers a token out; a page's
        # number from the stack to the table and back
        return {"bytes": 4 * (8 * B + 3 * T + 4 * fresh), "flops": 0}
    if case["op"] == "verify":
        return {"bytes": 4 * case["V"] * (T + (B if case["probs"] else 0)), "flops": 3 * T * case["V"]}
    e = 4 if case["type"] == 0 else 2
    rows = case["Hkv"] * case["hd"]
    if case["op"] == "store":
        return {"bytes": 2 * T * rows * (4 + e) + 4 * T, "flops": 0}
    Hq = case["Hkv"] * case["G"]
    seen = sum(k * q + k * (k + 1) // 2 for k, q in zip(n, p))
    return {"bytes": 2 * (sum(n) + sum(p)) * rows * e + 8 * T * Hq * case["hd"], "flops": 4 * seen * Hq * case["hd"]}


# -- inputs -------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _paged(case, n, p, g, with_new):
    """Table, held and free pages of a cache in which the sequences have the pages of their cached rows (of their
    new ones too, where with_new says so), shuffled; and the batch."""
    B, ps = case["B"], case["page"]
    n_slots = B + 3
    most = -(-max(a + b for a, b in zip(n, p)) // ps) + 2
    slot = torch.randperm(n_slots, generator=g, device=DEV)[:B]
    have = [-(-(q + (k if with_new else 0)) // ps) for k, q in zip(n, p)]
    n_pages = sum(-(-(a + b) // ps) for a, b in zip(n, p)) + 5
    order = torch.randperm(n_pages, generator=g, device=DEV)
    used = sum(have)
    table = torch.full((n_slots, most), -1, dtype=torch.int32, device=DEV)
    held = torch.zeros(n_slots, dtype=torch.int32, device=DEV)
    held[slot] = _i32(have)
    j = torch.arange(most, device=DEV)
    mine = torch.full((B, most), -1, dtype=torch.int32, device=DEV)
    mine[j < _i32(have).view(-1, 1)] = order[:used].int()
    table[slot] = mine
    free = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    free[:n_pages - used] = order[used:].int()
    off = [0]
    for k in n:
        off.append(off[-1] + k)
    return {"case": case, "B": B, "T": off[-1], "n_max": max(n), "ps": ps, "n_slots": n_slots, "max_pages": most,
            "n_pages": n_pages, "most_new": max(1, max(-(-(a + b) // ps) - -(-b // ps) for a, b in zip(n, p))),
            "L_max": max(a + b for a, b in zip(n, p)), "slot": slot.int(), "pos0": _i32(p), "n_new": _i32(n),
            "tok_off": _i32(off), "table": table, "held": held, "free": free, "n_free": _i32([n_pages - used])}


def _pool(st, x):
    """A pool of the pages' values x [n_pages, page, Hkv, hd] in the case's type and layout."""
    x = x.to(TYPES[st["case"]["type"]])
    return (x if st["case"]["layout"] else x.transpose(1, 2)).contiguous()


def _channels(case, g):
    """K's channels: a few are ten times as large as the others."""
    w = torch.ones(case["Hkv"], case["hd"], device=DEV)
    w[:, torch.randint(0, case["hd"], (max(1, case["hd"] // 32),), generator=g, device=DEV)] = 10.0
    return w


def _prepare_verify(case, seed, g):
    n, _ = _batch(case)
    B, V, T = case["B"], case["V"], sum(n)
    off = [0]
    for k in n:
        off.append(off[-1] + k)
    par = _parents(case, n)
    z = torch.randn(T, V, generator=g, device=DEV) * 3.0
    likely = torch.randint(0, V, (T, 6), generator=g, device=DEV)
    z.scatter_(1, likely, 16.0 + 2.0 * torch.randn(T, 6, generator=g, device=DEV))
    banned = torch.rand(V, generator=g, device=DEV) < 0.01
    banned[:2] = False
    z[:, banned] = -INF
    # the row whose distribution a draft was drawn from, as the drafting model sees it
    r = random.Random(case["lens"] + 2)
    temp = [r.choice([0.0, 0.7, 0.8, 1.0, 1.0, 1.2]) for _ in range(B)]
    up = _i32([off[b] + max(0, par[off[b] + i]) for b, k in enumerate(n) for i in range(k)]).long()
    temps = _i32([b for b, k in enumerate(n) for i in range(k)]).long()
    temps = torch.tensor(temp, device=DEV)[temps].view(-1, 1)
    guess = (z[up] + 0.7 * torch.randn(T, V, generator=g, device=DEV)) / torch.where(temps > 0, temps, 1.0)
    q = torch.softmax(guess, 1)
    tok = torch.where(temps.view(-1) > 0, torch.multinomial(q, 1, generator=g).view(-1), guess.argmax(1))
    st = {"case": case, "B": B, "T": T, "n_max": max(n), "logits": z, "token": tok.int(), "parent": _i32(par),
          "tok_off": _i32(off), "temperature": torch.tensor(temp, device=DEV),
          "u": torch.rand(T, generator=g, device=DEV), "r": torch.rand(B, generator=g, device=DEV),
          "n_acc": torch.empty(B, dtype=torch.int32, device=DEV)}
    if case["probs"]:
        st["q"] = q
    for name in ("out_tok", "out_row"):
        st[name] = torch.empty(T, dtype=torch.int32, device=DEV)
    return st


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "verify":
        st = _prepare_verify(case, seed, g)
        torch.cuda.synchronize()
        return st
    n, p = _batch(case)
    st = _paged(case, n, p, g, case["op"] != "pages")
    T, B, Hkv, hd = st["T"], case["B"], case.get("Hkv"), case.get("hd")
    if case["op"] == "pages":
        for name, size in (("o_off", B + 1), ("o_seq", T), ("o_pos", T), ("o_row", T), ("o_last", B), ("status", 1),
                           ("status2", 1)):
            st[name] = torch.empty(size, dtype=torch.int32, device=DEV)
    elif case["op"] == "store":
        st["k"] = torch.randn(T, Hkv, hd, generator=g, device=DEV) * _channels(case, g)
        st["v"] = torch.randn(T, Hkv, hd, generator=g, device=DEV)
        for name in ("K", "V"):
            st[name] = _pool(st, torch.zeros(st["n_pages"], case["page"], Hkv, hd, device=DEV))
        st["tok_row"] = _tokens(st)[2].int()
    else:
        st["q"] = torch.randn(T, Hkv * case["G"], hd, generator=g, device=DEV)
        st["out"] = torch.empty_like(st["q"])
        shape = (st["n_pages"], case["page"], Hkv, hd)
        st["K"] = _pool(st, torch.randn(shape, generator=g, device=DEV) * _channels(case, g))
        st["V"] = _pool(st, torch.randn(shape, generator=g, device=DEV))
    torch.cuda.synchronize()
    return st


# -- plain forms --------------------------------------------------------------
def _tokens(st):
    """Sequence, position and cache row of every new token."""
    t = torch.arange(st["T"], device=DEV)
    off = torch.cumsum(st["n_new"].long(), 0)
    seq = torch.searchsorted(off, t, right=True)
    pos = st["pos0"].long()[seq] + t - (off - st["n_new"])[seq]
    page = st["table"][st["slot"].long()[seq], pos // st["ps"]].long()
    return seq, pos, page * st["ps"] + pos % st["ps"]


def _scatter(to, at, real, values):
    """to[at] = values where real, in place and without asking the device how many that are."""
    flat = torch.cat([to.reshape(-1), torch.zeros(1, dtype=to.dtype, device=DEV)])
    flat.scatter_(0, torch.where(real, at, to.numel()).view(-1), values.reshape(-1).to(to.dtype))
    to.copy_(flat[:-1].view(to.shape))


def _pages_plain(st):
    ps, slot, j = st["ps"], st["slot"].long(), torch.arange(st["most_new"], device=DEV)
    have, n = st["held"].long()[slot].view(-1, 1), st["n_new"].long()
    need = (st["pos0"].long() + n + ps - 1).div(ps, rounding_mode="floor").view(-1, 1)
    new = (need - have).clamp(min=0)
    at = st["n_free"] - 1 - (torch.cumsum(new, 0) - new + j)
    cell = slot.view(-1, 1) * st["max_pages"] + have + j
    _scatter(st["table"], cell, j < new, st["free"][at.clamp(min=0)])
    st["held"][slot] = torch.maximum(have, need).view(-1).int()
    st["n_free"] -= new.sum().int()
    seq, pos, row = _tokens(st)
    end = torch.cumsum(n, 0)
    out = {"off": torch.cat([torch.zeros_like(end[:1]), end]).int(), "seq": seq.int(), "pos": pos.int(),
           "row": row.int(), "last": torch.where(n > 0, end - 1, -1).int()}
    # the drafts, or the requests, are gone again: pages behind pos0 go back
    have, keep = st["held"].long()[slot].view(-1, 1), (st["pos0"].long() + ps - 1).div(ps, rounding_mode="floor")
    keep = torch.minimum(keep.view(-1, 1), have)
    back = have - keep
    at = st["n_free"] + back.sum() - 1 - (torch.cumsum(back, 0) - back + j)
    cell = (slot.view(-1, 1) * st["max_pages"] + keep + j).clamp(max=st["table"].numel() - 1)
    pages = st["table"].view(-1)[cell]
    _scatter(st["free"], at, j < back, pages)
    _scatter(st["table"], cell, j < back, torch.full_like(pages, -1))
    st["held"][slot] = keep.view(-1).int()
    st["n_free"] += back.sum().int()
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    return {**out, "status": zero, "status2": zero, **{k: st[k] for k in ("table", "held", "free", "n_free")}}


def _store_plain(st):
    page = st["tok_row"].long().div(st["ps"], rounding_mode="floor").view(-1, 1)
    row, head = st["tok_row"].long().remainder(st["ps"]).view(-1, 1), torch.arange(st["case"]["Hkv"], device=DEV)
    for pool, x in ((st["K"], st["k"]), (st["V"], st["v"])):
        at = (page, row, head) if st["case"]["layout"] else (page, head, row)
        pool[at] = x.to(pool.dtype)
    return [st["K"], st["V"]]


def _attend_plain(st):
    """Every sequence padded to the longest context and the most new tokens."""
    c = st["case"]
    hd, Hkv, G, B, L, n = c["hd"], c["Hkv"], c["G"], st["B"], st["L_max"], st["n_max"]
    key = torch.arange(L, device=DEV)
    page = st["table"][st["slot"].long()][:, key // st["ps"]].long().clamp(min=0)      # [B, L]
    row = (key % st["ps"]).expand(B, L)

    def cached(pool):
        if c["layout"]:
            return pool[page, row].transpose(1, 2).float().contiguous()
        head = torch.arange(Hkv, device=DEV).view(1, -1, 1)
        return pool[page.unsqueeze(1), head, row.unsqueeze(1)].float()
    tok = st["tok_off"][:-1].long().view(-1, 1) + torch.arange(n, device=DEV)
    q = st["q"][tok.clamp(max=st["T"] - 1)].view(B, n, Hkv, G, hd).permute(0, 2, 1, 3, 4)
    s = torch.matmul(q.reshape(B, Hkv, n * G, hd) / math.sqrt(hd), cached(st["K"]).transpose(2, 3).contiguous())
    sees = key <= st["pos0"].view(-1, 1, 1) + torch.arange(n, device=DEV).view(1, -1, 1)       # [B, n, L]
    s = s.view(B, Hkv, n, G, L).masked_fill(~sees.view(B, 1, n, 1, L), -INF)
    s = torch.exp(s - s.amax(4, keepdim=True))
    o = torch.matmul(s.view(B, Hkv, n * G, L), cached(st["V"])) / s.sum(4).view(B, Hkv, n * G, 1)
    o = o.view(B, Hkv, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B * n, Hkv * G, hd)
    t = torch.arange(st["T"], device=DEV)
    seq = torch.searchsorted(st["tok_off"][1:].long(), t, right=True)
    return o[seq * n + t - st["tok_off"].long()[seq]]


def _probabilities(z, temperature):
    """Rows of p in 64 bits; all of it on the first largest logit where the temperature is 0."""
    w = torch.exp((z.double() - z.amax(1, keepdim=True)) / torch.where(temperature > 0, temperature, 1.0).double())
    return w / w.sum(1, keepdim=True)


def _verify_plain(st):
    B, T, n, V, probs = st["B"], st["T"], st["n_max"], st["case"]["V"], st["case"]["probs"]
    t0, count = st["tok_off"][:-1].long(), (st["tok_off"][1:] - st["tok_off"][:-1]).long()
    greedy = st["temperature"] <= 0
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(st["tok_off"][1:].long(), t, right=True)
    up = t0[seq] + st["parent"].long().clamp(min=0)
    temps = st["temperature"][seq].view(-1, 1)
    p, best = _probabilities(st["logits"], temps), st["logits"].argmax(1)
    token = st["token"].long()
    p_tok = torch.where(greedy[seq], (best[up] == token).double(), p[up, token])
    q_tok = st["q"][t, token].double() if probs else torch.ones_like(p_tok)
    u = torch.where(greedy[seq], 0.5, st["u"].double())
    i = torch.arange(n, device=DEV)
    rows = (t0.view(-1, 1) + i).clamp(max=T - 1)                        # [B, n]
    tried, node, rest = torch.zeros(B, n, dtype=torch.bool, device=DEV), torch.zeros_like(t0), torch.ones_like(p[:B, 0])
    accepted = torch.zeros(B, n, dtype=torch.bool, device=DEV)
    for k in range(1, n):                                               # a draft is decided before those behind it
        row = rows[:, k]
        child = (k < count) & (st["parent"][row] == node)
        again = (tried & (token[rows] == token[row].view(-1, 1))).any(1)
        p_row = torch.where(again, 0.0, p_tok[row])
        yes = child & (u[row] * q_tok[row] * rest < p_row)
        no = child & ~yes
        accepted[:, k] = yes
        node = torch.where(yes, k, node)
        rest = torch.where(yes, 1.0, torch.where(no, rest - p_row, rest)) if not probs else rest
        tried = torch.where(yes.view(-1, 1), False, tried | (no.view(-1, 1) & (i == k)))
    last = t0 + node
    w = p[last]
    if probs:
        turned = tried.any(1, keepdim=True)
        less = (w - st["q"][(t0 + tried.int().argmax(1)).clamp(max=T - 1)].double()).clamp(min=0)
        w = torch.where(turned & (less.sum(1, keepdim=True) > 0), less, w)
    else:
        out = torch.where(tried, token[rows], V)
        w = torch.cat([w, w[:, :1]], 1).scatter(1, out, 0.0)[:, :V]
    total = torch.cumsum(w, 1)
    nxt = torch.searchsorted(total, total[:, -1:] * st["r"].double().view(-1, 1), right=True).view(-1).clamp(max=V - 1)
    nxt = torch.where(greedy, best[last], nxt)
    n_acc = accepted.sum(1)
    # accepted rows first, in order, then the next token, then -1
    place = torch.where(accepted, torch.cumsum(accepted, 1) - 1, n)
    none = torch.full((B, n + 1), -1, dtype=torch.int64, device=DEV)
    out_row = none.scatter(1, place, i.expand(B, n).contiguous())
    out_tok = none.scatter(1, place, token[rows]).scatter(1, n_acc.view(-1, 1), nxt.view(-1, 1))
    out_row[:, n] = -1
    at = t - t0[seq]
    out_row = torch.where(at < n_acc[seq], out_row[seq, at], -1)
    out_tok = torch.where(at <= n_acc[seq], out_tok[seq, at], -1)
    return {"n_acc": n_acc.int(), "tok": out_tok.int(), "row": out_row.int()}


# -- the framework's operators ------------------------------------------------
_kept = []


def _lib():
    if not _kept:
        import slate_amd
        slate_amd.Backend()                    # raises where there is no device
        _kept.append(slate_amd)
    return _kept[0]


def _own(st):
    sa = _lib()
    lib, c = sa.load_library(), st["case"]

    def p(name):
        return st[name].data_ptr() if name in st else None
    if c["op"] == "verify":
        rc = lib.slate_hip_verify_drafts(p("n_acc"), p("out_tok"), p("out_row"), p("logits"), c["V"], p("token"),
                                         p("parent") if c["tree"] else None, p("q"), c["V"], p("temperature"), p("u"),
                                         p("r"), p("tok_off"), st["B"], st["T"], c["V"], None, 0)
        if rc:
            sa.check(rc, "verify_drafts")
        return {"n_acc": st["n_acc"], "tok": st["out_tok"], "row": st["out_row"]}
    if "pages" not in st:                      # the handles that a program keeps with its cache
        st["pages"] = sa.Pages(p("table"), p("held"), p("free"), p("n_free"), st["n_slots"], st["max_pages"],
                               st["n_pages"], st["ps"])
        if c["op"] != "pages":
            ps, H, hd = c["page"], c["Hkv"], c["hd"]
            head, row = (hd, H * hd) if c["layout"] else (ps * hd, hd)
            st["kv"] = sa.PagedKv(p("K"), p("V"), c["type"], H, hd, ps * H * hd, head, row)
    pages = ctypes.byref(st["pages"])
    if c["op"] == "pages":
        rc = (lib.slate_hip_pages_extend(pages, p("slot"), p("pos0"), p("n_new"), st["B"], st["T"], p("o_off"),
                                         p("o_seq"), p("o_pos"), p("o_row"), p("o_last"), p("status")) or
              lib.slate_hip_pages_trim(pages, p("slot"), p("pos0"), st["B"], p("status2")))
        if rc:
            sa.check(rc, "pages_extend / pages_trim")
        return {"off": st["o_off"], "seq": st["o_seq"], "pos": st["o_pos"], "row": st["o_row"], "last": st["o_last"],
                **{k: st[k] for k in ("status", "status2", "table", "held", "free", "n_free")}}
    kv = ctypes.byref(st["kv"])
    if c["op"] == "store":
        rc = lib.slate_hip_kv_store_paged(kv, pages, p("k"), p("v"), c["Hkv"] * c["hd"], p("tok_row"), st["T"])
        if rc:
            sa.check(rc, "kv_store_paged")
        return [st["K"], st["V"]]
    rc = lib.slate_hip_attention_paged(p("out"), p("q"), kv, pages, p("slot"), p("tok_off"), p("pos0"), st["B"],
                                       st["T"], st["n_max"], c["Hkv"] * c["G"], None, 0)
    if rc:
        sa.check(rc, "attention_paged")
    return st["out"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"pages": _pages_plain, "store": _store_plain, "attend": _attend_plain, "verify": _verify_plain}[op](state)


# -- the definitions in 64 bits, sequence by sequence -------------------------------
def _exact_pages(case, st):
    ps = case["page"]
    n, p = _batch(case)
    table, free = st["table"].tolist(), st["free"].tolist()
    left, slots = int(st["n_free"]), st["slot"].tolist()
    seq, pos, row, off, last = [], [], [], [0], []
    for b, s in enumerate(slots):
        for i in range(n[b]):
            at = p[b] + i
            page = table[s][at // ps]
            if page < 0:                       # the first row of a page that the slot does not have yet
                left -= 1
                page = table[s][at // ps] = free[left]
            seq.append(b)
            pos.append(at)
            row.append(page * ps + at % ps)
        off.append(len(seq))
        last.append(off[-1] - 1 if n[b] else -1)
    # all pages that were taken go back, so table, held and stack are those of before
    return {"off": _i32(off), "seq": _i32(seq), "pos": _i32(pos), "row": _i32(row), "last": _i32(last),
            "status": _i32([0]), "status2": _i32([0]), **{k: st[k] for k in ("table", "held", "free", "n_free")}}


def _exact_attend(case, st):
    hd, G, ps = case["hd"], case["G"], case["page"]
    n, p = _batch(case)
    out, t = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV), 0
    for b, (k, ctx) in enumerate(zip(n, p)):
        pages = st["table"][int(st["slot"][b])][:-(-(ctx + k) // ps)].long()

        def rows(pool):
            x = pool[pages].double()
            x = x if case["layout"] else x.transpose(1, 2)
            return x.reshape(-1, case["Hkv"], hd)[:ctx + k]
        K, V = rows(st["K"]), rows(st["V"])
        hidden = torch.ones(k, ctx + k, dtype=torch.bool, device=DEV).triu(ctx + 1)
        for h in range(case["Hkv"]):
            q = st["q"][t:t + k, h * G:(h + 1) * G].double().transpose(0, 1).reshape(G * k, hd)
            s = (q @ K[:, h].t().contiguous()).view(G, k, ctx + k) * hd ** -0.5
            w = torch.softmax(s.masked_fill(hidden, -INF), 2).view(G * k, -1)
            out[t:t + k, h * G:(h + 1) * G] = (w @ V[:, h].contiguous()).view(G, k, hd).transpose(0, 1)
        t += k
    return out


def _exact_verify(case, st):
    n, _ = _batch(case)
    par, tok = _parents(case, n), st["token"].tolist()
    u, r, temp = st["u"].tolist(), st["r"].tolist(), st["temperature"].tolist()
    n_acc, out_tok, out_row, t = [], [], [], 0
    for b, k in enumerate(n):
        def target(i):
            z = st["logits"][t + i].double()
            if temp[b] <= 0:
                return torch.nn.functional.one_hot(z.argmax(), case["V"]).double()
            return torch.softmax(z / temp[b], 0)
        node, path = 0, []
        left = target(0)
        while True:
            for c in [i for i in range(node + 1, k) if par[t + i] == node]:
                drafted = st["q"][t + c].double() if case["probs"] else None
                there = float(left[tok[t + c]])
                chance = there / float(drafted[tok[t + c]]) if case["probs"] else there
                if (there > 0.5) if temp[b] <= 0 else u[t + c] < chance:
                    path.append(c)
                    break
                if temp[b] <= 0:
                    continue
                if case["probs"]:              # what the target has more than the draft
                    left = torch.relu(left - drafted)
                else:                          # the target without this token
                    left[tok[t + c]] = 0.0
                left = left / left.sum()
            if not path or path[-1] == node:
                break
            node = path[-1]
            left = target(node)
        total = left.cumsum(0)
        nxt = int((total <= r[b] * float(total[-1])).sum().clamp(max=case["V"] - 1))
        if temp[b] <= 0:
            nxt = int(left.argmax())
        n_acc.append(len(path))
        out_row += path + [-1] * (k - len(path))
        out_tok += [tok[t + c] for c in path] + [nxt] + [-1] * (k - len(path) - 1)
        t += k
    return {"n_acc": _i32(n_acc), "tok": _i32(out_tok), "row": _i32(out_row)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "pages":
        return _exact_pages(case, st)
    if case["op"] == "attend":
        return _exact_attend(case, st)
    if case["op"] == "verify":
        return _exact_verify(case, st)
    # a value of the cache is the nearest one of its type: the difference to that is counted, so none is named here
    out = []
    for name, x in (("K", st["k"]), ("V", st["v"])):
        pool = st[name].double() if case["layout"] else st[name].double().transpose(1, 2)
        flat = pool.reshape(-1, case["Hkv"], case["hd"]).clone()
        flat[st["tok_row"].long()] = x.double()
        flat = flat.view(st["n_pages"], case["page"], case["Hkv"], case["hd"])
        out.append(flat if case["layout"] else flat.transpose(1, 2).contiguous())
    return out
