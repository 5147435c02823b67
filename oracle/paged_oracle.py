"""Plain restatement of the paged KV cache and of tree attention: numpy, loops and 64-bit
arithmetic, one sequence after the other. Test infrastructure; nothing in the package uses it.

``PagedOracle`` keeps the same state as ``cab_attention.PagedKVCache`` (pages, table, lengths,
use counts, status) and must agree with it bit for bit. ``tree_attention`` returns the
attention's output and log-sum-exp, and with them the sums that error bounds need."""

from __future__ import annotations

import numpy as np

FULL, TABLE_FULL, BAD_ROW, BAD_ARG, BAD_TABLE = 1, 2, 4, 8, 16


class PagedOracle:
    def __init__(self, k, v, table, lens, refs):
        self.k, self.v = k.copy(), v.copy()            # [L, P, H, S, D]
        self.table, self.lens, self.refs = table.copy(), lens.copy(), refs.copy()
        self.status = 0
        self.P, self.S = k.shape[1], k.shape[3]
        self.R, self.W = table.shape

    def pages_of(self, tokens):
        return -(-int(tokens) // self.S)

    def update(self, pairs, copies=True):
        """``pairs``: dicts with src, dst, start (None: all), keep (list or None), grow."""
        if self.status:
            return
        err, seen, uses = 0, set(), {}
        for p in pairs:
            s, d = p["src"], p["dst"]
            if not (0 <= s < self.R and 0 <= d < self.R):
                err |= BAD_ROW
                continue
            keep, n = p.get("keep") or [], int(self.lens[s])
            a = n if p.get("start") is None else p["start"]
            if a < 0 or a > n or p.get("grow", 0) < 0 or p.get("short"):
                err |= BAD_ARG
            elif a + len(keep) + p.get("grow", 0) > self.W * self.S:
                err |= TABLE_FULL
            if d in seen:
                err |= BAD_ROW
            seen.add(d)
            uses[s] = uses.get(s, 0) + 1
        if err:
            self.status |= err
            return
        free = [int(x) for x in np.flatnonzero(self.refs == 0)]
        plans, need = [], 0
        for p in pairs:
            s, d, keep, n = p["src"], p["dst"], p.get("keep") or [], int(self.lens[p["src"]])
            a = n if p.get("start") is None else p["start"]
            if any(x < 0 or x >= n - a for x in keep):
                err |= BAD_ARG
            same = next((i for i, x in enumerate(keep) if x != i), len(keep))
            held = a + len(keep)
            stay = (a + same) // self.S
            if a + same == held and held % self.S and s == d:
                tail = int(self.table[s, held // self.S])
                if 0 <= tail < self.P and self.refs[tail] == 1 and uses[s] == 1:
                    stay += 1
                elif not copies:
                    err |= BAD_TABLE
            size = held + p.get("grow", 0)
            plans.append((s, d, a, keep, held, size, stay, need))
            need += self.pages_of(size) - stay
        if need > len(free):
            err |= FULL
        if err:
            self.status |= err
            return
        old_table, old_lens = self.table.copy(), self.lens.copy()
        for s, d, a, keep, held, size, stay, base in plans:
            have, now = self.pages_of(old_lens[d]), self.pages_of(size)
            row = [int(old_table[s, j]) if j < stay else free[base + j - stay] for j in range(now)]
            for j in range(have):
                self.refs[old_table[d, j]] -= 1
            for q in row:
                self.refs[q] += 1
            for pos in range(stay * self.S, held):
                frm = pos if pos < a else a + keep[pos - a]
                q, t = int(old_table[s, frm // self.S]), row[pos // self.S]
                self.k[:, t, :, pos % self.S] = self.k[:, q, :, frm % self.S]
                self.v[:, t, :, pos % self.S] = self.v[:, q, :, frm % self.S]
            self.table[d, :max(have, now)] = row + [-1] * (max(have, now) - now)
            self.lens[d] = size

    def write(self, layer, k, v, rows=None, num_new=None):
        if self.status:
            return
        n, _, T, _ = k.shape
        for i in range(n):
            r = i if rows is None else rows[i]
            m = T if num_new is None else num_new[i]
            for t in range(m):
                pos = int(self.lens[r]) - m + t
                q = int(self.table[r, pos // self.S])
                self.k[layer, q, :, pos % self.S] = k[i, :, t]
                self.v[layer, q, :, pos % self.S] = v[i, :, t]

    def tokens(self, layer, row):
        """K and V of a row's tokens, [H, len, D] each."""
        n = int(self.lens[row])
        q = [int(self.table[row, x // self.S]) for x in range(n)]
        s = [x % self.S for x in range(n)]
        return self.k[layer, q, :, s].transpose(1, 0, 2), self.v[layer, q, :, s].transpose(1, 0, 2)


def tree_sees(m, parents=None, mask=None):
    """[m, m] truth: node t sees node u."""
    if mask is not None:
        return np.asarray(mask)[:m, :m].astype(bool)
    sees = np.zeros((m, m), dtype=bool)
    for t in range(m):
        u = t
        while u >= 0:
            sees[t, u] = True
            up = u - 1 if parents is None else int(parents[u])
            u = up if up < u else -1
    return sees


def tree_attention(q, k, v, m, scale, parents=None, mask=None, there=None):
    """One sequence: q [Hq, T, D], k, v [Hkv, len, D] (the last m tokens are the nodes), ``there``
    [len] truth (default all). Returns out [Hq, T, D], lse [Hq, T], and per row what a bound on the
    error needs: sum_j p_j |v_j| / sum p [Hq, T, D] and max_j scale * sum_d |q_d k_jd| [Hq, T]."""
    Hq, T, D = q.shape
    H, n = k.shape[:2]
    out, lse = np.zeros((Hq, T, D)), np.full((Hq, T), -np.inf)
    absv, absqk = np.zeros((Hq, T, D)), np.zeros((Hq, T))
    sees = np.zeros((T, n), dtype=bool)
    sees[:m, :n - m] = True
    sees[:m, n - m:] = tree_sees(m, parents, mask)
    if there is not None:
        sees &= there
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for h in range(Hq):
        kk, vv = k[h // (Hq // H)], v[h // (Hq // H)]
        for t in range(T):
            at = np.flatnonzero(sees[t])
            if at.size == 0:
                continue
            s = scale * (kk[at] @ q[h, t])
            top = s.max()
            p = np.exp(s - top)
            out[h, t] = p @ vv[at] / p.sum()
            lse[h, t] = top + np.log(p.sum())
            absv[h, t] = p @ np.abs(vv[at]) / p.sum()
            absqk[h, t] = scale * (np.abs(kk[at]) @ np.abs(q[h, t])).max()
    return out, lse, absv, absqk
