"""Plain 64-bit restatements of the serving operators, for the tests.

Attention and its error bounds (numpy / torch float64), the paged cache's
bookkeeping as ordinary Python lists, and draft verification.
"""
import math

import numpy as np

EPS24 = 2.0 ** -24          # half a unit of f32
EPS11 = 2.0 ** -11          # half a unit of f16


def attention(q, k, v, limit):
    """q [R, 128], k, v [L, 128] (float64 torch), row r sees keys < limit[r].
    Returns the outputs and what their error bounds are made of: sum p |v|,
    the largest sum |q||k| / sqrt(128) of a seen key, sum |v| of the seen."""
    import torch
    n = k.shape[0]
    seen = torch.arange(n, device=q.device)[None] < limit[:, None]
    s = torch.where(seen, q @ k.T / math.sqrt(128.0), -math.inf)
    mx = s.amax(1, keepdim=True) if n else torch.zeros(q.shape[0], 1, dtype=q.dtype, device=q.device)
    mx = torch.where(torch.isinf(mx), 0.0, mx)
    e = torch.where(seen, torch.exp(s - mx), 0.0)
    den = e.sum(1, keepdim=True)
    p = torch.where(den > 0, e / den, 0.0)
    mag = torch.where(seen, q.abs() @ k.abs().T / math.sqrt(128.0), 0.0)
    big = mag.amax(1, keepdim=True) if n else torch.zeros_like(mx)
    return p @ v, p @ v.abs(), big, torch.where(seen, 1.0, 0.0).to(v.dtype) @ v.abs()


def attention_bound(out, pv, big, va, n, f16, out_f16):
    """How far a result may be off, by elements.

    A score is a sum of 128 products, each addition off by at most one f32
    unit (tensor cores may cut instead of rounding: 2 EPS24) of the running
    magnitude, plus its scaling, the subtraction of the maximum and the
    exponential (2 units each at most): |ds| <= (128 * 2 + 8) EPS24 * big + 8
    EPS24. A weight is off by a factor e^(2 ds) at most (its own score's error
    and the normaliser's), the sums over n keys by n units each of p |v| and of
    p. With f16, each weight is rounded: EPS11 of itself, or 2^-25 where it is
    subnormal (weights stand against a maximum of at least 1). The result is
    rounded once more to f16.
    """
    ds = (128 * 2 + 8) * EPS24 * big + 8 * EPS24
    b = pv * (2.1 * ds + (2 * n + 32) * 2 * EPS24)
    if f16:
        b = b + pv * EPS11 * 1.01 + 2.0 ** -25 * va
    b = b + out.abs() * 2 * EPS24 + 1e-37
    if out_f16:
        b = b + (out.abs() + b) * EPS11 + 2.0 ** -25
    return b


class PageModel:
    """The bookkeeping of sllm_cuda_kv_*, one slot after the other."""

    def __init__(self, n_pages, n_slots, width, page):
        self.n_pages, self.n_slots, self.width, self.page = n_pages, n_slots, width, page
        self.refs = [0] * n_pages
        self.tables = [[0] * width for _ in range(n_slots)]
        self.lens = [0] * n_slots

    def used(self, n):
        return -(-n // self.page)

    def _row_ok(self, s):
        if not 0 <= s < self.n_slots or not 0 <= self.lens[s] <= self.width * self.page:
            return False
        ids = self.tables[s][:self.used(self.lens[s])]
        return all(0 <= i < self.n_pages and self.refs[i] > 0 for i in ids)

    def fork(self, src, dst):
        if len(set(dst)) < len(dst) or not all(self._row_ok(s) for s in list(src) + list(dst)):
            return -1
        rows = [(self.tables[s][:self.used(self.lens[s])], self.lens[s]) for s in src]
        for ids, _ in rows:
            for i in ids:
                self.refs[i] += 1
        for d in dst:
            for i in self.tables[d][:self.used(self.lens[d])]:
                self.refs[i] -= 1
        for d, (ids, n) in zip(dst, rows):
            self.tables[d][:len(ids)] = ids
            self.lens[d] = n
        return 0

    def reserve(self, slots, new):
        """Status and the copies made: (source, destination, rows)."""
        if any(not 0 <= s < self.n_slots for s in slots) or len(set(slots)) < len(slots) or min(new, default=0) < 0:
            return -1, []
        for s, n in zip(slots, new):
            if self.lens[s] + n > self.width * self.page:
                return -36, []
        free = [i for i in range(self.n_pages) if self.refs[i] == 0]
        plan, refs, at = [], list(self.refs), 0
        for s, n in zip(slots, new):
            cur = self.lens[s]
            old = self.tables[s][cur // self.page] if n > 0 and cur % self.page else None
            cow = old is not None and refs[old] > 1
            if cow:
                refs[old] -= 1
            fresh = self.used(cur + n) - self.used(cur)
            plan.append((s, n, cur, old if cow else None, at, fresh))
            at += fresh + (1 if cow else 0)
        if at > len(free):
            return -2, []
        copies = []
        self.refs = refs
        for s, n, cur, old, a, fresh in plan:
            if old is not None:
                self.tables[s][cur // self.page] = free[a]
                self.refs[free[a]] = 1
                copies.append((old, free[a], cur % self.page))
                a += 1
            first = self.used(cur)
            for x in range(fresh):
                self.tables[s][first + x] = free[a + x]
                self.refs[free[a + x]] = 1
            self.lens[s] = cur + n
        return 0, copies

    def release(self, slots, new_len):
        new_len = [0] * len(slots) if new_len is None else new_len
        if len(set(slots)) < len(slots) or not all(self._row_ok(s) for s in slots):
            return -1
        if any(n < 0 or n > self.lens[s] for s, n in zip(slots, new_len)):
            return -1
        for s, n in zip(slots, new_len):
            for i in self.tables[s][self.used(n):self.used(self.lens[s])]:
                self.refs[i] -= 1
            self.lens[s] = n
        return 0

    def compact(self):
        if not all(self._row_ok(s) for s in range(self.n_slots)):
            return -1, []
        live = sum(r > 0 for r in self.refs)
        src = [i for i in range(live, self.n_pages) if self.refs[i] > 0]
        dst = [i for i in range(live) if self.refs[i] == 0]
        to = dict(zip(src, dst))
        for a, b in zip(src, dst):
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(self.n_slots):
            for j in range(self.used(self.lens[s])):
                self.tables[s][j] = to.get(self.tables[s][j], self.tables[s][j])
        return 0, [(a, b, self.page) for a, b in zip(src, dst)]


def verify(p, q, draft, nd, ua, us):
    """Draft verification in float64: tokens [n][k + 1], count [n], and each
    draw's distance to the nearest border of its running sum, over the sum."""
    n, k1, _ = p.shape
    toks = np.full((n, k1), -1, np.int64)
    cnt = np.zeros(n, np.int64)
    gap = np.full(n, np.inf)
    clean = lambda x: np.where((x > 0) & np.isfinite(x), x, 0.0).astype(np.float64)
    for b in range(n):
        r, refused = 0, None
        while r < nd[b]:
            x = int(draft[b, r])
            inside = 0 <= x < p.shape[2]
            qx = 1.0 if q is None else (clean(q[b, r])[x] if inside else 0.0)
            if not (inside and np.float64(ua[b, r]) * qx < clean(p[b, r])[x]):
                refused = x
                break
            toks[b, r] = x
            r += 1
        mass = clean(p[b, r])
        if refused is not None:
            if q is None:
                rest = mass.copy()
                if 0 <= refused < rest.size:
                    rest[refused] = 0.0
            else:
                rest = np.maximum(mass - clean(q[b, r]), 0.0)
            if rest.sum() > 0:
                mass = rest
        cnt[b] = r + 1
        cum = np.cumsum(mass)
        if cum[-1] > 0:
            target = np.float64(us[b]) * cum[-1]
            x = int(np.searchsorted(cum, target, side="right"))
            toks[b, r] = min(x, int(np.nonzero(mass)[0][-1]))
            gap[b] = np.abs(cum - target).min() / cum[-1]
    return toks, cnt, gap
