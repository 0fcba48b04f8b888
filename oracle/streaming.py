"""The masked and the paged attention and the page operations of their cache, from their definitions in 64 bits
(numpy; no counterpart in the reference, whose inference is one clip at a time).

``masked_attention`` also returns how far a kernel may be off, element by element, from roundings that are counted:

* a score x_j is a dot product of 64 products in fp32: at most 64 * 2^-24 * sum_d |q_d k_jd| * scale off; forming it in the
  log2 domain with cap, bias and distance rounds it at most 8 more times, 2^-24 of its size (of the sizes of its terms) each;
  the cap's tanh is good to 2^-20 relative and 2^-21 absolute, times the cap;
* e^x then is off by that much relative, plus 2^-13 where 16-bit types allow a polynomial exponential (7.5e-5), 2^-21 for
  fp32;
* sums over the keys round 2^-24 per addition, at most keys / 16 + 128 in a row;
* 16-bit types round each probability (eps / 2) before the product with the values, and the result once (eps / 2);
  fp16 besides rounds to its smallest step 2^-24: the kernels keep a row's largest probability, before it is divided by the sum, above 2^3
  and round a probability at most four times (once, and once for each time that the maximum grows while its tile is in work), so a key
  loses at most 4 * 2^-25 / 2^3 of the row's largest, or what two roundings take of its own; the result rounds to 2^-25.
"""
from __future__ import annotations

import numpy as np

EPS_HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def masked_attention(q, k, v, bias=None, ranges=None, *, scale=0.125, softcap=None, slope=None, qpos=None, kpos=None, dtype="f32"):
    """q [B,H,Nq,64], k, v [B,Hkv,Nk,64] (values of ``dtype``), bias [Nk] or [B,Nk], ranges [Nq,2] or [B,Nq,2]
    -> (out float64, bound float64), both [B,H,Nq,64]."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1:3]
    out, bound = np.zeros((B, H, Nq, D)), np.zeros((B, H, Nq, D))
    if Nk == 0:
        return out, bound
    key = np.arange(Nk)
    u, half = 2.0 ** -24, EPS_HALF[dtype]
    for b in range(B):
        r = None if ranges is None else np.asarray(ranges)[b] if np.ndim(ranges) == 3 else np.asarray(ranges)
        see = np.ones((Nq, Nk), bool) if r is None else (key[None] >= r[:, :1]) & (key[None] < r[:, 1:])
        m = None if bias is None else np.asarray(bias, np.float64)[b] if np.ndim(bias) == 2 else np.asarray(bias, np.float64)
        if m is not None:
            see = see & ~np.isneginf(m)[None]
        at = lambda p, n, first: np.arange(first, first + n, dtype=np.float64) if p is None else np.asarray(  # noqa: E731
            p[b] if np.ndim(p) == 2 else p, np.float64)
        for h in range(H):
            kk, vv = k[b, h // (H // Hkv)], v[b, h // (H // Hkv)]
            with np.errstate(invalid="ignore", over="ignore"):
                x = scale * (q[b, h] @ kk.T)
                err = 64 * u * abs(scale) * (np.abs(q[b, h]) @ np.abs(kk).T) + 8 * u * np.abs(x)
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                    err += np.minimum(softcap * 2.0 ** -21, np.abs(x) * 2.0 ** -20)
                if m is not None:
                    x = x + m[None]
                    err += 8 * u * np.abs(m)[None]
                if slope is not None:
                    d = float(slope[h]) * np.abs(at(qpos, Nq, Nk - Nq)[:, None] - at(kpos, Nk, 0)[None])
                    x = x - d
                    err += 8 * u * np.abs(d)  # slopes may be negative
            x = np.where(see, x, -np.inf)
            top = x.max(1, keepdims=True)
            p = np.exp(x - np.where(np.isneginf(top), 0.0, top))
            total = p.sum(1, keepdims=True)
            some = total[:, 0] > 0
            p[some] /= total[some]
            err = np.where(see, err, 0.0) + 8 * u * np.where(np.isneginf(top), 0.0, np.abs(top)) + (
                2.0 ** -21 if dtype == "f32" else 2.0 ** -13) + u * (Nk / 16 + 128)
            hidden = ~see.any(0)
            vv = np.where(hidden[:, None], 0.0, vv)
            # a value that only other rows see takes no part: 0 * NaN is not formed
            bad = ~np.isfinite(vv).all(1)
            vz = np.where(bad[:, None], 0.0, vv)
            o = p @ vz
            for j in np.nonzero(bad)[0]:
                with np.errstate(invalid="ignore"):
                    o[see[:, j]] += p[see[:, j], j:j + 1] * vv[j:j + 1]
            size = p @ np.abs(vz)
            out[b, h] = o
            bound[b, h] = (p * err) @ np.abs(vz) + np.abs(o) * (p * err).sum(1, keepdims=True)
            if dtype != "f32":
                bound[b, h] += half * (size + np.abs(o)) * 1.01
            else:
                bound[b, h] += half * np.abs(o)
            if dtype == "f16":  # absolute step of small probabilities and of small results
                bound[b, h] += np.minimum(2 * p, 2.0 ** -26 * p.max(1, keepdims=True)) @ np.abs(vz) + 2.0 ** -25
    return out, bound


class Cache:
    """The page operations by hand: one token after the other, lists of pages per slot."""

    def __init__(self, k, v, mass, table, length, refs):
        self.k, self.v = (np.array(t) for t in (k, v))
        self.mass = None if mass is None else np.array(mass)
        self.held = [[int(p) for p in row if p >= 0] for row in np.asarray(table)]
        self.length, self.refs = [int(x) for x in length], [int(x) for x in refs]
        self.page, self.max_pages = self.k.shape[1], np.asarray(table).shape[1]

    def _rows(self):
        return [t for t in (self.k, self.v, self.mass) if t is not None]

    def table(self):
        return np.array([row + [-1] * (self.max_pages - len(row)) for row in self.held], np.int32).reshape(len(self.held), self.max_pages)

    def free(self, sequence):
        for s in sequence:
            if 0 <= s < len(self.held):
                for p in self.held[s]:
                    self.refs[p] -= 1
                self.held[s], self.length[s] = [], 0

    def fork(self, source, target):
        ok = [(s, t) for s, t in zip(source, target) if 0 <= s < len(self.held) and 0 <= t < len(self.held)]
        last = {t: s for s, t in ok}
        snap = {t: (list(self.held[s]), self.length[s]) for t, s in last.items()}
        for t, (pages, length) in snap.items():
            for p in pages:
                self.refs[p] += 1
            for p in self.held[t]:
                self.refs[p] -= 1
            self.held[t], self.length[t] = list(pages), length

    def append(self, sequence, offsets, k, v, mass=None):
        """True when the tokens were added (all or nothing)."""
        if any(b < a for a, b in zip(offsets, offsets[1:])) or offsets[0] < 0 or offsets[-1] > len(k):
            return False
        todo, seen = [], set()
        for i, s in enumerate(sequence):
            if 0 <= s < len(self.held) and s not in seen:
                seen.add(s)
                todo.append((s, range(offsets[i], offsets[i + 1])))
        shared = list(self.refs)
        copies = [bool(self.length[s] % self.page and len(r) and shared[self.held[s][-1]] > 1) for s, r in todo]
        free = [p for p, r in enumerate(shared) if r == 0]
        pages = [-(-(self.length[s] + len(r)) // self.page) for s, r in todo]
        need = sum(n - len(self.held[s]) + c for (s, r), n, c in zip(todo, pages, copies))
        if need > len(free) or any(n > self.max_pages for n in pages):
            return False
        taken = iter(free)
        for (s, r), copy in zip(todo, copies):
            if copy:
                old, new = self.held[s][-1], next(taken)
                for pool in self._rows():
                    pool[new, :self.length[s] % self.page] = pool[old, :self.length[s] % self.page]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.held[s][-1] = new
            for t in r:
                at = self.length[s] % self.page
                if at == 0:
                    self.held[s].append(next(taken))
                    self.refs[self.held[s][-1]] = 1
                p = self.held[s][-1]
                self.k[p, at], self.v[p, at] = k[t], v[t]
                if self.mass is not None:
                    self.mass[p, at] = 0.0 if mass is None else mass[t]
                self.length[s] += 1
        return True

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        to = dict(zip([p for p in live if p >= len(live)], [p for p in range(len(live)) if self.refs[p] == 0]))
        for a, b in to.items():
            for pool in self._rows():
                pool[b] = pool[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.held = [[to.get(p, p) for p in row] for row in self.held]
        return len(live)

    def tokens(self, slot):
        """(k, v, mass) of a slot, in order."""
        n = self.length[slot]
        rows = lambda t: t[self.held[slot]].reshape(-1, *t.shape[2:])[:n]  # noqa: E731
        return rows(self.k), rows(self.v), None if self.mass is None else rows(self.mass)
