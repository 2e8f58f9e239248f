"""A K/V cache in pages, attention over it and the verification of drafted
tokens in 64 bits on the host (test infrastructure)."""
import math

import numpy as np


class Pages:
    """The page table's upkeep, token by token."""

    def __init__(self, n_slots, max_pages, n_pages, page_size):
        self.ps, self.n_pages = page_size, n_pages
        self.table = np.full((n_slots, max_pages), -1, np.int32)
        self.held = np.zeros(n_slots, np.int32)
        self.free = list(range(n_pages))[::-1]

    def extend(self, slot, pos0, n_new, T_cap):
        """status and the batch's descriptors (None where refused)."""
        if min(map(min, (slot, pos0, n_new))) < 0 or max(slot) >= len(self.held) or len(set(slot)) < len(slot):
            return -1, None
        need = [-(-(p + n) // self.ps) for p, n in zip(pos0, n_new)]
        fresh = sum(max(0, k - int(self.held[s])) for k, s in zip(need, slot))
        if max(need) > self.table.shape[1] or fresh > len(self.free) or sum(n_new) > T_cap or \
                any(p + n > self.table.shape[1] * self.ps for p, n in zip(pos0, n_new)):
            return -2, None
        off, seq, pos, row, last = [0], [], [], [], []
        for b, (s, p, n, k) in enumerate(zip(slot, pos0, n_new, need)):
            while self.held[s] < k:
                self.table[s, self.held[s]] = self.free.pop()
                self.held[s] += 1
            for i in range(p, p + n):
                seq.append(b)
                pos.append(i)
                page = int(self.table[s, i // self.ps])
                row.append(page * self.ps + i % self.ps if 0 <= page < self.n_pages else -1)
            off.append(len(seq))
            last.append(off[-1] - 1 if n else -1)
        return 0, [np.array(a, np.int32) for a in (off, seq, pos, row, last)]

    def trim(self, slot, length):
        if min(map(min, (slot, length))) < 0 or max(slot) >= len(self.held) or len(set(slot)) < len(slot):
            return -1
        back = []
        for s, n in zip(slot, length):
            keep = min(int(self.held[s]), -(-n // self.ps))
            back += [int(p) for p in self.table[s, keep:self.held[s]]]
            self.table[s, keep:] = -1
            self.held[s] = keep
        self.free += back[::-1]
        return 0


def attend(q, K, V, first, hd):
    """One kv head: q [n, G, hd], K, V [keys, hd] float64; token i sees keys 0 .. first + i.  Returns out, and the
    largest sum |q_i k_i| / sqrt(hd) and |score| of a seen key."""
    n, G = q.shape[:2]
    out, mag, top = np.zeros(q.shape), 0.0, 0.0
    for i in range(n):
        k, v = K[:first + i + 1], V[:first + i + 1]
        s = q[i] @ k.T / math.sqrt(hd)
        mag = max(mag, float((np.abs(q[i]) @ np.abs(k).T).max()) / math.sqrt(hd))
        top = max(top, float(np.abs(s).max()))
        p = np.exp(s - s.max(1, keepdims=True))
        out[i] = p @ v / p.sum(1, keepdims=True)
    return out, mag, top


def target(z, temperature):
    """A row's p; None where it has none."""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    top = z.max()
    if top == -np.inf:
        return None
    if not temperature > 0:
        p = np.zeros(len(z))
        p[int(np.argmax(z))] = 1.0
        return p
    if top == np.inf:
        p = (z == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            p = np.where(z == -np.inf, 0.0, np.exp((z - top) / float(temperature)))
        p[z == top] = 1.0
    return p / p.sum()


def verify(z, token, parent, q, temperature, u, r):
    """One sequence: z [n, V], token, parent [n], q [n, V] or None.  Returns the accepted rows, the next token, and
    how near a decision (of its p) and a sum (of the whole) came to its border."""
    n, V = z.shape
    node, path, near = 0, [], [1.0, 1.0]
    greedy = not temperature > 0
    while True:
        full = target(z[node], temperature)
        if full is None:
            return path, -1, near
        left, nxt = full.copy(), -1
        for c in range(node + 1, n):
            if parent[c] != node:
                continue
            x = int(token[c])
            p = float(left[x]) if 0 <= x < V else 0.0
            if greedy:
                yes = p > 0
            else:
                drafted = (float(q[c, x]) if 0 <= x < V else 1.0) if q is not None else left.sum()
                a = float(u[c]) * drafted
                yes = a < p
                if p > 0:
                    near[0] = min(near[0], abs(a - p) / p)
            if yes:
                nxt = c
                break
            if greedy:
                continue
            if q is not None:
                left = np.maximum(left - q[c].astype(np.float64), 0.0)
            elif 0 <= x < V:
                left[x] = 0.0
        if nxt < 0:
            break
        path.append(nxt)
        node = nxt
    if not left.sum() > 0:
        left = full
    total = np.cumsum(left)
    at = total[-1] * float(r)
    some = np.nonzero(left > 0)[0]
    past = some[total[some] > at]
    nxt = int(past[0]) if len(past) else int(some[-1])
    if not greedy:
        near[1] = float(np.abs(total[some] - at).min() / total[-1])
    return path, nxt, near
