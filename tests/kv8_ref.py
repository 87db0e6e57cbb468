"""Plain restatements of the 8-bit cache and of beam selection, for the tests.

Quantisation follows the definition's own operations in float32 (numpy), value
by value, so codes and scales have to be equal; attention and selection are in
64 bits.
"""
import math

import numpy as np

BLOCK = 16
LEAST = np.float32(2.0 ** -100)


def rope(x, cos, sin):
    """x [heads][128] float32, rotated; each product and sum rounded once."""
    a, b = x[:, :64], x[:, 64:]
    return np.concatenate([a * cos - b * sin, a * sin + b * cos], 1).astype(np.float32)


def store_block(codes, scale, row0, rows, values):
    """One block of one head: codes int8 [16][128], its scale; `values` float32
    [len(rows)][128] go to `rows` (ascending, the first row0). Returns
    (codes, scale, whether a value was no finite number)."""
    codes = codes.copy()
    old = np.float32(scale) if row0 > 0 else np.float32(0)
    if not (old > 0 and np.isfinite(old)):
        old = np.float32(0)
    mag = np.abs(values)
    fine = np.isfinite(values)
    top = np.float32(np.where(fine, mag, 0).max(initial=0))
    s = old
    grows = top > np.float32(old * np.float32(127))
    if grows:
        s = max(np.float32(top / np.float32(127)), LEAST)
    inv = np.float32(1) / s if s > 0 else np.float32(0)
    if grows and row0 > 0:
        f = np.float32(old * inv)
        codes[:row0] = np.rint(codes[:row0].astype(np.float32) * f).astype(np.int8)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.where(np.isnan(values) | (inv == 0), np.float32(0), values * inv)
    codes[rows] = np.rint(np.clip(y, -127, 127)).astype(np.int8)
    return codes, s, not fine.all()


class Cache8:
    """An 8-bit cache on the host: the same arrays as the device's."""

    def __init__(self, pages, layers, heads, page, seed=None):
        shape = (pages, layers, heads, page, 128)
        r = np.random.default_rng(seed)
        if seed is None:
            self.codes = [np.zeros(shape, np.int8) for _ in range(2)]
            self.scales = [np.zeros(shape[:3] + (page // BLOCK,), np.float32) for _ in range(2)]
        else:                           # a used cache: every place holds something
            self.codes = [r.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.scales = [np.exp(r.normal(-3, 0.5, shape[:3] + (page // BLOCK,))).astype(np.float32) for _ in range(2)]
        self.page = page

    def append(self, layer, tables, lens, refs, slot, pos, k, v, cos, sin):
        """The tokens of the lists; returns (error, tokens that were left out)."""
        bad, left, i, n = False, set(), 0, len(slot)
        while i < n:
            if slot[i] < 0:
                i += 1
                continue
            j = i + 1
            while j < n and slot[j] == slot[i] and pos[j] >> 4 == pos[i] >> 4:
                j += 1
            run = [i]
            for t in range(i + 1, j):
                if pos[t] <= pos[t - 1]:
                    break
                run.append(t)
            left |= set(range(i, j)) - set(run)
            ok = 0 <= slot[i] < len(lens)
            limit = min(lens[slot[i]] if ok else 0, len(tables[0]) * self.page, len(cos))
            live = [t for t in run if 0 <= pos[t] < limit]
            left |= set(run) - set(live)
            if live:
                page = tables[slot[i]][pos[live[0]] // self.page]
                if 0 <= page < len(refs) and refs[page] == 1:
                    b = pos[live[0]] % self.page // BLOCK
                    rows = [pos[t] % BLOCK for t in live]
                    for h in range(k.shape[1]):
                        for w, x in enumerate((k, v)):
                            y = np.stack([rope(x[t, h:h + 1], cos[pos[t]], sin[pos[t]])[0] if w == 0 else x[t, h]
                                          for t in live])
                            at = (page, layer, h, slice(b * BLOCK, b * BLOCK + BLOCK))
                            c, s, odd = store_block(self.codes[w][at], self.scales[w][page, layer, h, b], rows[0], rows, y)
                            self.codes[w][at], self.scales[w][page, layer, h, b] = c, s
                            bad = bad or odd
                else:
                    left |= set(live)
            i = j
        return bad or bool(left), left

    def values(self, which, layer, table, n):
        """float64 [heads][n][128] of a slot's first n tokens."""
        pages = table[:-(-n // self.page)]
        x = self.codes[which][pages, layer].astype(np.float64)
        x *= np.repeat(self.scales[which][pages, layer], BLOCK, -1)[..., None].astype(np.float64)
        return x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, 128)[:, :n]


def beam_select(logits, score, done, eos, beams):
    """One request: logits [B][V], score [B] (float64), done [B]. Returns the best
    `beams` candidates (value, beam, logit, word), the best `beams` + 1 of weight, and all
    that can be among them."""
    cand = []
    for b in range(beams):
        x = np.where(logits[b] < np.inf, logits[b], -np.inf).astype(np.float64)
        sc = score[b] if score[b] < np.inf else -np.inf
        if done is not None and done[b]:
            cand.append((sc, b, -np.inf, eos))
            continue
        top = x.max()
        lse = top + math.log(np.exp(x - top).sum()) if top > -np.inf else -np.inf
        with np.errstate(invalid="ignore"):
            v = sc + (x - lse)
        v = np.where(v > -np.inf, v, -np.inf)
        keep = np.argsort(-v, kind="stable")[:4 * beams]
        low = np.flatnonzero(~(v > -np.inf))[:beams]
        for i in sorted(set(keep.tolist()) | set(low.tolist())):
            cand.append((v[i], b, x[i], i))
    # weight: value down, beam up, logit down, word up; without: beam, word
    live = sorted([c for c in cand if c[0] > -np.inf], key=lambda c: (-c[0], c[1], -c[2], c[3]))
    dead = sorted([c for c in cand if not c[0] > -np.inf], key=lambda c: (c[1], c[3]))
    return (live + dead)[:beams], live[:beams + 1], live + dead
