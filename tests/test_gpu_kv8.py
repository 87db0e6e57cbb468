"""The 8-bit paged cache on a GPU: stores, reading back, attention, and the page
operations over it, against plain restatements (kv8_ref.py, serving_ref.py).
Codes and scales have to be equal; attention's tolerance is derived below."""
import math

import numpy as np
import pytest

from kv8_ref import BLOCK, Cache8
from serving_ref import PageModel, attention, attention_bound

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16}[name]


def _i32(a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Eight:
    """A cache on the device beside its host model."""

    def __init__(self, cuda, pages, slots, width, page, layers, heads, seed=None):
        import torch
        self.cuda, self.m = cuda, PageModel(pages, slots, width, page)
        self.host = Cache8(pages, layers, heads, page, seed)
        self.k, self.v = (_t(x) for x in self.host.codes)
        self.ks, self.vs = (_t(x) for x in self.host.scales)
        self.refs, self.lens = _i32([0] * pages), _i32([0] * slots)
        self.tables = _i32(self.m.tables)
        self.p = cuda.KvPages(self.k, self.v, self.refs, self.tables, self.lens, self.ks, self.vs)
        self.work = torch.empty(self.p.work_bytes(), dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def take_status(self):
        v = int(self.status.item())
        self.status.zero_()
        return v

    def reserve(self, slots, new):
        self.p.reserve(_i32(slots), _i32(new), self.work, self.status)
        want, copies = self.m.reserve(slots, new)
        for a, b, rows in copies:
            self.copy(a, b, rows)
        return want

    def copy(self, a, b, rows):
        for c, s in zip(self.host.codes, self.host.scales):
            c[b, :, :, :rows] = c[a, :, :, :rows]
            blocks = -(-rows // BLOCK)
            s[b, :, :, :blocks] = s[a, :, :, :blocks]

    def place(self, lens, seed=0):
        """Slots of these lengths, in pages of no order."""
        r = np.random.default_rng(seed)
        ids = r.permutation(self.m.n_pages).tolist()
        for s, n in enumerate(lens):
            for j in range(self.m.used(n)):
                p = ids.pop()
                self.m.tables[s][j] = p
                self.m.refs[p] = 1
            self.m.lens[s] = n
        self.refs.copy_(_i32(self.m.refs))
        self.tables.copy_(_i32(self.m.tables))
        self.lens.copy_(_i32(self.m.lens))

    def same(self):
        got = [x.cpu().numpy() for x in (self.k, self.v, self.ks, self.vs)]
        want = self.host.codes + self.host.scales
        return [bool(np.array_equal(a, b)) for a, b in zip(got, want)]


def _angles(n):
    ang = np.arange(n)[:, None] * (500000.0 ** (-np.arange(64) / 64))[None]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _random_call(r, c, S, n_ctx):
    """Lists for one call: runs of several slots, some of them padded, wrong or out of order."""
    slot, pos = [], []
    for s in r.permutation(S):
        n = int(r.integers(0, 40))
        a = int(r.integers(0, max(1, c.m.lens[s] + 6)))
        slot += [int(s)] * n
        pos += list(range(a, a + n))
        if r.random() < 0.3:
            slot += [-1] * int(r.integers(1, 4))
            pos += [5] * (len(slot) - len(pos))
    if slot and r.random() < 0.5:                            # (between slots: a block's tokens stay together)
        i = int(r.choice([0] + [j for j in range(1, len(slot)) if slot[j] != slot[j - 1]]))
        slot.insert(i, S + 3)
        pos.insert(i, 0)
    if len(slot) > 3 and r.random() < 0.5:                   # one token twice, one position negative
        i = int(r.integers(len(slot)))
        slot.insert(i, slot[i])
        pos.insert(i, pos[i])
        slot.append(0)
        pos.append(-3)
    return slot, pos


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,layers", [((4, 4), 1), ((5, 1), 2), ((20, 5), 1), ((16, 2), 3)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_append8(cuda, page, heads, layers, out):
    """Several calls on one cache: blocks begun, gone on with, grown and written again; tokens out of order,
    wrong ones and padding among them. Codes and scales are equal to the definition's, whole pools."""
    import torch
    H, Hkv = heads
    S, n_ctx = 5, 150
    c = Eight(cuda, 60, S, -(-160 // page) + 1, page, layers, Hkv, seed=3)
    c.place([37, 150, 0, 64, 15], seed=page)
    cos, sin = _angles(n_ctx)
    r = np.random.default_rng(page + H)
    for step in range(6):
        layer = int(r.integers(layers))
        slot, pos = _random_call(r, c, S, n_ctx)
        T = len(slot)
        qkv = r.standard_normal((T, H + 2 * Hkv, 128)).astype(np.float32)
        qkv *= np.exp(r.normal(0, 1, (T, 1, 1))).astype(np.float32)
        d = _t(qkv)
        q, k, v = d[:, :H], d[:, H:H + Hkv], d[:, H + Hkv:]
        qo = torch.full((T, H, 128), 7.0, dtype=_dt(out), device="cuda")
        ko, vo = (torch.full((T, Hkv, 128), 7.0, dtype=_dt(out), device="cuda") for _ in range(2))
        c.p.append8(layer, _i32(slot), _i32(pos), q, k, v, _t(cos), _t(sin), qo, ko, vo, c.status)
        torch.cuda.synchronize()
        bad, left = c.host.append(layer, c.m.tables, c.m.lens, c.m.refs, slot, pos, qkv[:, H:H + Hkv], qkv[:, H + Hkv:],
                                  cos, sin)
        assert c.take_status() == (-1 if bad else 0)
        assert all(c.same()), (step, c.same())
        for t in range(T):
            if slot[t] < 0:
                assert bool((qo[t] == 7).all() and (ko[t] == 7).all() and (vo[t] == 7).all())
            elif t not in left:
                from kv8_ref import rope
                for got, x, rot in ((qo, qkv[t, :H], True), (ko, qkv[t, H:H + Hkv], True), (vo, qkv[t, H + Hkv:], False)):
                    want = rope(x, cos[pos[t]], sin[pos[t]]) if rot else x
                    assert np.array_equal(got[t].cpu().numpy(), want.astype(got[t].cpu().numpy().dtype))


def test_append8_odd_values(cuda):
    """Zeros, values too small or large for an ordinary scale, NaN and infinities."""
    import torch
    c = Eight(cuda, 6, 1, 6, 16, 1, 2, seed=1)
    c.place([96])
    cos, sin = np.ones((96, 64), np.float32), np.zeros((96, 64), np.float32)
    x = np.zeros((96, 2, 128), np.float32)
    x[16:32, 0, :5] = 1e-38                                  # below the least scale's step
    x[16:32, 1, 7] = 3e-30
    x[32:48, 0] = 3.3e38
    x[32, 1, 3], x[33, 1, 4], x[34, 1, 5], x[35, 1, 6] = np.nan, np.inf, -np.inf, 2.0
    x[48, :, 1], x[49, :, 2], x[60, :, 3] = 1e-20, 1.0, 1e30         # steps up by many orders
    x[64, 0, 0] = np.inf                                     # nothing finite but zeros
    x[80:] = np.random.default_rng(0).standard_normal((16, 2, 128))
    for a in range(0, 96, 1):                                # one token at a time
        d = _t(x[a:a + 1])
        c.p.append8(0, _i32([0]), _i32([a]), None, d, d, _t(cos), _t(sin), status=c.status)
        bad, _ = c.host.append(0, c.m.tables, c.m.lens, c.m.refs, [0], [a], x[a:a + 1], x[a:a + 1], cos, sin)
        assert c.take_status() == (-1 if bad else 0), a
    torch.cuda.synchronize()
    assert all(c.same())
    assert bool(torch.isfinite(c.ks).all() and torch.isfinite(c.vs).all())


def test_append8_leaves_shared_pages_alone(cuda):
    import torch
    c = Eight(cuda, 8, 3, 4, 16, 1, 1, seed=1)
    c.place([20, 0, 20])
    c.p.fork(_i32([0]), _i32([1]), c.work, c.status)
    c.m.fork([0], [1])
    cos, sin = _angles(64)
    x = np.random.default_rng(0).standard_normal((3, 1, 128)).astype(np.float32)
    d = _t(x)
    c.p.append8(0, _i32([0, 1, 2]), _i32([19, 19, 19]), None, d, d, _t(cos), _t(sin), status=c.status)
    torch.cuda.synchronize()
    bad, left = c.host.append(0, c.m.tables, c.m.lens, c.m.refs, [0, 1, 2], [19, 19, 19], x, x, cos, sin)
    assert left == {0, 1} and c.take_status() == -1 and all(c.same())


# ---------------------------------------------------------------------------
# read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("heads", [1, 3, 5, 8])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_read8(cuda, page, heads, out):
    """Tokens in any order, twice, wrong and padded: one product and one rounding a value."""
    import torch
    c = Eight(cuda, 40, 4, 9, page, 2, heads, seed=heads)
    c.place([100, 1, 0, 130], seed=2)
    r = np.random.default_rng(5)
    slot = r.integers(-1, 5, 300).tolist()
    pos = r.integers(-2, 140, 300).tolist()
    n = len(slot)
    ok = [0 <= s < 4 and 0 <= p < c.m.lens[s] for s, p in zip(slot, pos)]
    for which in ("kv", "k", "v"):
        ko = torch.full((n, heads, 128), 7.0, dtype=_dt(out), device="cuda") if "k" in which else None
        vo = torch.full((n, heads, 128), 7.0, dtype=_dt(out), device="cuda") if "v" in which else None
        c.p.read8(1, _i32(slot), _i32(pos), ko, vo, c.status)
        torch.cuda.synchronize()
        assert c.take_status() == -1
        for w, o in ((0, ko), (1, vo)):
            if o is None:
                continue
            got = o.cpu().numpy()
            for t in range(n):
                if not ok[t]:
                    assert (got[t] == 7).all()
                    continue
                pg, row = c.m.tables[slot[t]][pos[t] // page], pos[t] % page
                want = c.host.codes[w][pg, 1, :, row].astype(np.float32) * c.host.scales[w][pg, 1, :, row // BLOCK][:, None]
                assert np.array_equal(got[t], want.astype(got.dtype))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attn8_bound(o, pv, big, va, n, f16, out_f16):
    """serving_ref's bound, with the stored values as the exact inputs: code times scale is applied to sums of
    exact products (one more unit, inside its 8), f32 queries and weights are pairs of f16, 2^-22 of each
    lost at most: of a score 2^-22 big, so 2 * 2^-22 big of a weight, and 2^-22 of the weight itself. One half
    as much again for the products of the second with the first. Where the first of a pair is subnormal the
    second is rounded to 2^-25 of its own scale, 2^-36, on weights that are 2^15 at most: 2^-51 of the largest
    weight, which is at most 1."""
    b = attention_bound(o, pv, big, va, n, f16, out_f16)
    return b if f16 else b + 1.5 * pv * (2 * 2.0 ** -22 * big + 2.0 ** -22) + 2.0 ** -51 * va


def check_attn8(c, layer, q, out, slots, f16):
    import torch
    n, nq, H, _ = q.shape
    Hkv = c.host.codes[0].shape[2]
    for b, s in enumerate(slots):
        L = c.m.lens[s]
        k, v = (torch.from_numpy(c.host.values(w, layer, c.m.tables[s], L)).cuda() for w in range(2))
        for h in range(H):
            lim = torch.tensor([max(0, L - nq + 1 + j) for j in range(nq)], device="cuda")
            o, pv, big, va = attention(q[b, :, h].double(), k[h * Hkv // H], v[h * Hkv // H], lim)
            tol = attn8_bound(o, pv, big, va, L, f16, out.dtype == torch.float16)
            err = (out[b, :, h].double() - o).abs()
            assert bool((err <= tol).all()), (b, h, L, float((err / tol).nan_to_num(math.inf).max()))


def run_attn8(c, layer, q, slots, odt, stream=None):
    import torch
    n, nq, H, _ = q.shape
    out = torch.full(q.shape, 7.0, dtype=odt, device="cuda")
    work = torch.empty(c.p.attn8_work_bytes(n, nq, H), dtype=torch.uint8, device="cuda")
    c.p.attn8(layer, q, out, _i32(slots), work, c.status, stream=stream)
    torch.cuda.synchronize()
    return out


def _q(seed, n, nq, H, dt, scale=1.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((n, nq, H, 128), generator=g, device="cuda") * scale).to(dt)


# heads (query, key), query tokens, lengths
CASES = [
    ((1, 1), 1, [1]),
    ((8, 1), 1, [1, 15, 16, 17, 0, 63, 64, 65]),
    ((20, 5), 1, [300, 1, 128, 129]),
    ((4, 4), 3, [2, 3, 4, 70]),
    ((14, 2), 2, [127, 1, 33]),
    ((64, 8), 1, [513, 64]),
    ((6, 2), 16, [16, 15, 200, 1]),
    ((32, 4), 4, [77, 4, 260]),
    ((24, 1), 1, [190, 7]),
    ((40, 1), 2, [100, 65, 1]),
    ((128, 1), 1, [90, 257]),
    ((16, 2), 16, [300, 31]),
    ((66, 1), 3, [129, 2]),
    ((8, 8), 1, [1500, 0, 3]),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("types", [("f32", "f32"), ("f16", "f16"), ("f16", "f32")])
def test_attn8(cuda, case, page, types):
    (H, Hkv), nq, lens = case
    width = max(lens) // page + 2
    c = Eight(cuda, sum(x // page + 1 for x in lens) + 9, len(lens) + 2, width, page, 2, Hkv, seed=H + nq)
    c.place([9] + lens + [40 if width * page >= 40 else 1], seed=nq)
    slots = np.random.default_rng(H).permutation(np.arange(1, len(lens) + 1)).tolist()
    q = _q(H + nq, len(lens), nq, H, _dt(types[0]))
    out = run_attn8(c, 1, q, slots, _dt(types[1]))
    assert c.take_status() == 0
    check_attn8(c, 1, q, out, slots, types[0] == "f16")
    for b, s in enumerate(slots):                            # rows that see nothing are zeros
        for j in range(nq):
            if c.m.lens[s] - nq + 1 + j <= 0:
                assert bool((out[b, j] == 0).all())


@pytest.mark.parametrize("case", [x for x in CASES if x[0][0] // x[0][1] * x[1] > 16], ids=str)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_attn8_wide_tables(cuda, case, page, out):
    """Tables with room for many keys, as of long contexts: the form for much work of 17 rows and more."""
    (H, Hkv), nq, lens = case
    width = (1 << 20) // page // len(lens) + max(lens) // page
    c = Eight(cuda, sum(x // page + 1 for x in lens) + 9, len(lens) + 2, width, page, 2, Hkv, seed=H + nq)
    c.place([9] + lens + [40], seed=nq)
    slots = np.random.default_rng(H).permutation(np.arange(1, len(lens) + 1)).tolist()
    q = _q(H + nq, len(lens), nq, H, _dt("f16"))
    o = run_attn8(c, 1, q, slots, _dt(out))
    assert c.take_status() == 0
    check_attn8(c, 1, q, o, slots, True)
    for b, s in enumerate(slots):
        for j in range(nq):
            if c.m.lens[s] - nq + 1 + j <= 0:
                assert bool((o[b, j] == 0).all())
    # bad ones are reported, and the others come out right
    import torch
    c.lens[slots[0]] = -1
    bad = run_attn8(c, 1, q, slots, _dt(out))
    assert c.take_status() == -1
    assert bool(torch.allclose(bad[1:].float(), o[1:].float(), atol=2e-3))
    c.lens[slots[0]] = c.m.lens[slots[0]]
    c.tables[slots[0], 0] = 1 << 30
    bad = run_attn8(c, 1, q, slots, _dt(out))
    assert c.take_status() == (-1 if c.m.lens[slots[0]] > 0 else 0)
    assert torch.equal(bad[1:], o[1:])


@pytest.mark.parametrize("page", [16, 128])
def test_attn8_wide_long_and_short(cuda, page):
    """Much work of 17 rows and more: very different lengths, one row block and two, several times the same."""
    import torch
    r = np.random.default_rng(4)
    lens = [int(x) for x in np.exp(r.uniform(0, 6, 70))] + [20000, 0, 1]
    c = Eight(cuda, sum(x // page + 1 for x in lens) + 3, len(lens), max(lens) // page + 1, page, 1, 2, seed=8)
    c.place(lens, seed=1)
    slots = r.permutation(len(lens)).tolist()
    for nq, H in ((3, 16), (7, 14), (1, 130)):
        q = _q(3, len(lens), nq, H, torch.float16)
        out = run_attn8(c, 0, q, slots, torch.float16)
        assert c.take_status() == 0
        check_attn8(c, 0, q, out, slots, True)
        assert torch.equal(run_attn8(c, 0, q, slots, torch.float16), out)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("page", [16, 128])
def test_attn8_long_and_short(cuda, dt, page):
    """Many sequences of very different lengths, one of them far longer than the others."""
    r = np.random.default_rng(4)
    lens = [int(x) for x in np.exp(r.uniform(0, 6, 70))] + [20000, 0, 1]
    c = Eight(cuda, sum(x // page + 1 for x in lens) + 3, len(lens), max(lens) // page + 1, page, 1, 2, seed=8)
    c.place(lens, seed=1)
    slots = r.permutation(len(lens)).tolist()
    q = _q(3, len(lens), 2, 8, _dt(dt))
    out = run_attn8(c, 0, q, slots, _dt(dt))
    assert c.take_status() == 0
    check_attn8(c, 0, q, out, slots, dt == "f16")


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_attn8_one_slot_twice(cuda, dt):
    import torch
    c = Eight(cuda, 20, 2, 12, 16, 1, 2, seed=8)
    c.place([150, 33], seed=1)
    q = _q(3, 3, 1, 4, _dt(dt))
    q[2] = q[0]
    out = run_attn8(c, 0, q, [0, 1, 0], _dt(dt))
    check_attn8(c, 0, q, out, [0, 1, 0], dt == "f16")
    assert torch.equal(out[0], out[2])


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_attn8_peaked_rows(cuda, dt):
    """Scores up to some hundreds, the largest late, early, and alone; scales that differ by many orders
    between neighbouring blocks."""
    import torch
    lens = [700, 333]
    c = Eight(cuda, 70, 2, 45, 16, 1, 2, seed=2)
    c.place(lens, seed=3)
    r = np.random.default_rng(3)
    c.host.scales[0][:] = np.exp(r.uniform(-8, 1.5, c.host.scales[0].shape)).astype(np.float32)
    c.host.scales[1][:] = np.exp(r.uniform(-25, 25, c.host.scales[1].shape)).astype(np.float32)
    c.ks.copy_(_t(c.host.scales[0]))
    c.vs.copy_(_t(c.host.scales[1]))
    q = _q(5, 2, 2, 8, _dt(dt), 0.2)
    out = run_attn8(c, 0, q, [0, 1], torch.float32)
    check_attn8(c, 0, q, out, [0, 1], dt == "f16")


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_attn8_unseen_places_leave_no_trace(cuda, dt):
    """Codes, scales that are no numbers and page ids behind a sequence's end reach nothing."""
    import torch
    lens = [100, 7, 64]
    c = Eight(cuda, 30, 3, 12, 32, 1, 2, seed=2)
    c.place(lens, seed=3)
    q = _q(5, 3, 2, 8, _dt(dt))
    a = run_attn8(c, 0, q, [0, 1, 2], _dt(dt))
    seen = {(c.m.tables[s][t // 32], t % 32) for s in range(3) for t in range(lens[s])}
    blocks = {(p, row // BLOCK) for p, row in seen}
    for p in range(30):
        for b in range(2):
            if (p, b) not in blocks:
                c.ks[p, :, :, b], c.vs[p, :, :, b] = math.nan, math.inf
        for row in range(32):
            if (p, row) not in seen:
                c.k[p, :, :, row], c.v[p, :, :, row] = 127, -128
    for s in range(3):
        c.tables[s, -(-lens[s] // 32):] = 1 << 30
    b = run_attn8(c, 0, q, [0, 1, 2], _dt(dt))
    assert c.take_status() == 0 and torch.equal(a, b)


@pytest.mark.parametrize("rows", [(8, 1), (24, 1), (8, 4), (64, 1)])
@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("low,high", [(-24, 24), (-69, 80), (-40, -38)])
def test_attn8_scales_far_apart(cuda, dt, rows, low, high):
    """Value scales of e^low to e^high in neighbouring blocks, and blocks of scale 0 that hold codes.

    Where f16 weights are rounded together with their keys' scales, a product below 2^-14 of the range is off by
    2^-25 of it, and the largest of a row stands at 2^7 of it at least: an absolute 2^-32 of the row's largest
    product of weight and scale, times each key's code."""
    import torch
    H, nq = rows
    lens = [300, 1000, 17]
    c = Eight(cuda, 90, 3, 64 if dt == "f32" else 16384, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    r = np.random.default_rng(9)
    sv = np.exp(r.uniform(low, high, c.host.scales[1].shape)).astype(np.float32)
    sv[r.random(sv.shape) < 0.2] = 0
    c.host.scales[1][:] = sv
    c.vs.copy_(_t(sv))
    q = _q(5, 3, nq, H, _dt(dt), 0.4)
    out = run_attn8(c, 0, q, [0, 1, 2], torch.float32)
    assert c.take_status() == 0
    for b, L in enumerate(lens):
        k, v = (torch.from_numpy(c.host.values(w, 0, c.m.tables[b], L)).cuda()[0] for w in range(2))
        scale = torch.from_numpy(np.repeat(np.concatenate([sv[p, 0, 0] for p in c.m.tables[b][:c.m.used(L)]]), BLOCK)[:L]).cuda().double()
        for h in range(H):
            lim = torch.tensor([max(0, L - nq + 1 + j) for j in range(nq)], device="cuda")
            o, pv, big, va = attention(q[b, :, h].double(), k, v, lim)
            tol = attn8_bound(o, pv, big, va, L, dt == "f16", False)
            if dt == "f16":
                s = q[b, :, h].double() @ k.T / math.sqrt(128)
                s[torch.arange(L, device="cuda")[None] >= lim[:, None]] = -math.inf
                top = (torch.softmax(s, -1) * scale).amax(-1, keepdim=True)
                codes = torch.where(scale[:, None] > 0, v / scale[:, None], 0.).abs().sum(0)
                tol = tol + 2.0 ** -32 * 1.01 * top * codes
            err = (out[b, :, h].double() - o).abs()
            assert bool((err <= tol).all()), (b, h, float((err / tol).nan_to_num(math.inf).max()))


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("rows", [(8, 1), (16, 1), (24, 1), (64, 1)])
def test_attn8_a_wait_that_runs_out_is_reported(cuda, dt, rows):
    """With a limit of 1 ns a CTA's first wait runs out (all of them load at once, from memory): the kernels end,
    *status and the error word say so, and the next call is as good as ever. In a workspace that an earlier call has
    used, and in two of no good numbers."""
    import torch
    H, nq, n = 5 * rows[0], rows[1], 24
    c = Eight(cuda, 800, n, 33 if dt == "f32" else 1024, 16, 1, 5, seed=2)
    c.place([500] * n, seed=3)
    q = _q(5, n, nq, H, _dt(dt))
    good = run_attn8(c, 0, q, list(range(n)), _dt(dt))
    assert c.take_status() == 0 and cuda.attn_error() == 0
    out, slots = torch.empty_like(q), _i32(list(range(n)))
    size = c.p.attn8_work_bytes(n, nq, H)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    works = [torch.full((size // 4 + 1,), x, dtype=torch.int32, device="cuda").view(torch.uint8) for x in (0, 0x7f7f7f7f, 12345)]
    c.p.attn8(0, q, out, slots, works[0], c.status)
    cuda.set_attn_wait(1)
    try:
        for work in works:
            flush.zero_()
            c.p.attn8(0, q, out, slots, work, c.status)
        torch.cuda.synchronize()
    finally:
        cuda.set_attn_wait(0)
    assert c.take_status() == -61 and cuda.attn_error() != 0
    cuda.attn_error()                                       # (one word per file)
    assert torch.equal(run_attn8(c, 0, q, list(range(n)), _dt(dt)), good)
    assert c.take_status() == 0 and cuda.attn_error() == 0


def test_attn8_bad_sequences_are_reported(cuda):
    """Wrong slots, lengths and pages: *status says so, and the other sequences come out right."""
    import torch
    lens = [90, 40, 64, 200]
    c = Eight(cuda, 40, 4, 14, 16, 1, 2, seed=2)
    c.place(lens, seed=3)
    for dt in (torch.float32, torch.float16):
        q = _q(5, 4, 1, 8, dt)
        good = run_attn8(c, 0, q, [0, 1, 2, 3], dt)
        assert c.take_status() == 0
        for slots in ([0, 4, 2, 3], [0, -1, 2, 3]):
            out = run_attn8(c, 0, q, slots, dt)
            assert c.take_status() == -1
            for b in (0, 2, 3):
                assert torch.equal(out[b], good[b]) or bool(torch.allclose(out[b].float(), good[b].float(), atol=2e-3))
        for bad in (-1, 14 * 16 + 1):
            c.lens[1] = bad
            out = run_attn8(c, 0, q, [0, 1, 2, 3], dt)
            assert c.take_status() == -1
            assert bool(torch.allclose(out[[0, 2, 3]].float(), good[[0, 2, 3]].float(), atol=2e-3))
        c.lens[1] = 40
        for bad in (-1, 40, 1 << 30):
            keep = int(c.tables[1, 1])
            c.tables[1, 1] = bad
            out = run_attn8(c, 0, q, [0, 1, 2, 3], dt)
            assert c.take_status() == -1
            assert torch.equal(out[[0, 2, 3]], good[[0, 2, 3]])
            c.tables[1, 1] = keep
        assert torch.equal(run_attn8(c, 0, q, [0, 1, 2, 3], dt), good) and c.take_status() == 0


def test_attn8_same_result_every_time(cuda):
    import torch
    lens = [5000, 77, 300]
    c = Eight(cuda, 400, 3, 340, 16, 1, 2, seed=2)
    c.place(lens, seed=3)
    q = _q(5, 3, 1, 8, torch.float16)
    a = run_attn8(c, 0, q, [0, 1, 2], torch.float16)
    for _ in range(5):
        assert torch.equal(run_attn8(c, 0, q, [0, 1, 2], torch.float16), a)


# ---------------------------------------------------------------------------
# page operations, offsets, streams, graphs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64, 128])
def test_copies_take_the_scales_along(cuda, page):
    """Copy on write moves a page's live rows and their blocks' scales; compaction whole pages."""
    import torch
    c = Eight(cuda, 40, 6, 8, page, 3, 2, seed=4)
    c.place([page + page // 2 + 1, 3 * page, 5, 0, 0, 0], seed=1)
    for src, dst in (([0, 0, 2], [3, 4, 5]),):
        c.p.fork(_i32(src), _i32(dst), c.work, c.status)
        assert c.m.fork(src, dst) == 0
    want = c.reserve([0, 3, 4, 2, 5], [1, 2, 1, 1, page])
    assert c.take_status() == want == 0
    assert all(c.same())
    c.p.release(_i32([1, 3]), None, c.work, c.status)
    assert c.m.release([1, 3], None) == 0
    c.p.compact(c.work, c.status)
    rc, moves = c.m.compact()
    for a, b, rows in moves:
        c.copy(a, b, rows)
    assert c.take_status() == rc == 0 and len(moves) > 0
    assert all(c.same()) and torch.equal(c.tables.cpu()[0, :2], torch.tensor(c.m.tables[0][:2], dtype=torch.int32))


def test_offsets_beyond_32_bits(cuda):
    """Pools of more than 2^32 bytes: the last pages are stored to, read and attended over."""
    import torch
    heads, page, layers = 8, 128, 2
    n_pages = (1 << 32) // (layers * heads * page * 128) + 3
    k, v = (torch.zeros((n_pages, layers, heads, page, 128), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((n_pages, layers, heads, page // 16), device="cuda") for _ in range(2))
    tab = _i32([[n_pages - 1, n_pages - 3, 0]])
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[n_pages - 1] = refs[n_pages - 3] = 1
    lens, status = _i32([200]), _i32([0])
    p = cuda.KvPages(k, v, refs, tab, lens, ks, vs)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((200, 3 * heads, 128), generator=g, device="cuda")
    cos, sin = torch.ones((200, 64), device="cuda"), torch.zeros((200, 64), device="cuda")
    slot, pos = _i32([0] * 200), _i32(list(range(200)))
    p.append8(1, slot, pos, None, x[:, :heads], x[:, heads:2 * heads], cos, sin, status=status)
    ko, vo = (torch.empty((200, heads, 128), device="cuda") for _ in range(2))
    p.read8(1, slot, pos, ko, vo, status)
    q = x[199:, 2 * heads:].contiguous().view(1, 1, heads, 128)
    out = torch.empty_like(q)
    work = torch.empty(p.attn8_work_bytes(1, 1, heads), dtype=torch.uint8, device="cuda")
    p.attn8(1, q, out, _i32([0]), work, status)
    assert int(status.item()) == 0
    for got, want in ((ko, x[:, :heads]), (vo, x[:, heads:2 * heads])):
        blocks = want.abs().amax(-1)
        step = torch.stack([blocks[i // 16 * 16:min(200, i // 16 * 16 + 16)].amax(0) for i in range(200)])[..., None] / 127
        assert bool(((got - want).abs() <= step * 0.5001).all())
    for h in range(heads):
        o, pv, big, va = attention(q[0, :, h].double(), ko[:, h].double(), vo[:, h].double(), torch.tensor([200], device="cuda"))
        assert bool(((out[0, :, h].double() - o).abs() <= attn8_bound(o, pv, big, va, 200, False, False)).all())
    assert int(k[0].abs().max()) == 0 and int(k[n_pages - 2].abs().max()) == 0


def test_stream_and_graph(cuda):
    """Store, attention and reading back on a stream of their own, captured and replayed on new inputs."""
    import torch
    c = Eight(cuda, 30, 3, 10, 16, 1, 2, seed=2)
    c.place([50, 17, 100], seed=3)
    cos, sin = _angles(160)
    dc, ds = _t(cos), _t(sin)
    r = np.random.default_rng(0)
    q = torch.empty((3, 4, 128), device="cuda")
    kv = torch.empty((3, 4, 128), device="cuda")
    slot, pos = _i32([0, 1, 2]), _i32([49, 16, 99])
    qo = torch.empty((3, 4, 128), dtype=torch.float16, device="cuda")
    out = torch.empty((3, 1, 4, 128), dtype=torch.float16, device="cuda")
    ko, vo = (torch.empty((3, 2, 128), device="cuda") for _ in range(2))
    work = torch.empty(c.p.attn8_work_bytes(3, 1, 4), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()

    def calls():
        c.p.append8(0, slot, pos, q, kv[:, :2], kv[:, 2:], dc, ds, qo, status=c.status, stream=s)
        c.p.attn8(0, qo.view(3, 1, 4, 128), out, slot, work, c.status, stream=s)
        c.p.read8(0, slot, pos, ko, vo, c.status, stream=s)

    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        calls()
    for step in range(3):
        x = r.standard_normal((3, 8, 128)).astype(np.float32)
        q.copy_(_t(x[:, :4]))
        kv.copy_(_t(x[:, 4:]))
        torch.cuda.synchronize()
        g.replay() if step else (calls(), s.synchronize())
        torch.cuda.synchronize()
        c.host.append(0, c.m.tables, c.m.lens, c.m.refs, [0, 1, 2], [49, 16, 99], x[:, 4:6], x[:, 6:], cos, sin)
        assert c.take_status() == 0 and all(c.same())
        check_attn8(c, 0, qo.view(3, 1, 4, 128), out, [0, 1, 2], True)
        for b, n in enumerate((50, 17, 100)):
            assert np.array_equal(ko[b].cpu().numpy(),
                                  c.host.values(0, 0, c.m.tables[b], n)[:, -1].astype(np.float32))


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_attn8_limits(cuda, dt):
    """The most sequences, query tokens and heads that a call takes."""
    import torch
    r = np.random.default_rng(1)
    n = 4096
    lens = r.integers(0, 20, n).tolist()
    c = Eight(cuda, 2 * n, n, 2, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    q = _q(5, n, 1, 1, _dt(dt))
    out = run_attn8(c, 0, q, list(range(n)), _dt(dt))
    assert c.take_status() == 0
    check_attn8(c, 0, q, out, list(range(n)), dt == "f16")
    c = Eight(cuda, 8, 1, 3, 16, 1, 1, seed=2)
    c.place([40], seed=3)
    q = _q(6, 1, 16, 1024, _dt(dt))
    out = run_attn8(c, 0, q, [0], _dt(dt))
    assert c.take_status() == 0
    check_attn8(c, 0, q, out, [0], dt == "f16")
    wide = Eight(cuda, 8, 1, 4096, 16, 1, 1, seed=2)
    wide.place([40], seed=3)
    out = run_attn8(wide, 0, q, [0], _dt(dt))
    assert wide.take_status() == 0
    check_attn8(wide, 0, q, out, [0], dt == "f16")


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_attn8_workspace_of_the_largest_call_serves_the_smaller(cuda, dt):
    """One workspace for calls of fewer and fewer sequences and query tokens; what lies behind it stays."""
    import torch
    H, n = 24, 20
    c = Eight(cuda, 900, n, 1024, 16, 1, 1, seed=2)
    c.place(np.random.default_rng(3).integers(1, 600, n).tolist(), seed=3)
    size = c.p.attn8_work_bytes(n, 4, H)
    work = torch.full((size + 4096,), 77, dtype=torch.uint8, device="cuda")
    for m, nq in ((n, 4), (7, 4), (n, 1), (3, 2), (1, 1)):
        q = _q(m + nq, m, nq, H, _dt(dt))
        out = torch.empty_like(q)
        assert c.p.attn8_work_bytes(m, nq, H) <= size
        c.p.attn8(0, q, out, _i32(list(range(m))), work[:size], c.status)
        assert c.take_status() == 0
        check_attn8(c, 0, q, out, list(range(m)), dt == "f16")
    assert bool((work[size:] == 77).all())


@pytest.mark.parametrize("dt,nq,H", [("f32", 1, 8), ("f16", 1, 8), ("f16", 3, 8)])
def test_attn8_replayed_with_other_sequences(cuda, dt, nq, H):
    """A captured call follows the lengths and slots that stand in its arrays when it is replayed; two graphs
    share a workspace, one after the other."""
    import torch
    c = Eight(cuda, 700, 6, 8192, 16, 1, 1, seed=2)
    c.place([1000, 33, 5000, 1, 700, 64], seed=3)
    q, slots = _q(5, 3, nq, H, _dt(dt)), _i32([0, 1, 2])
    outs = [torch.empty_like(q) for _ in range(2)]
    work = torch.empty(c.p.attn8_work_bytes(3, nq, H), dtype=torch.uint8, device="cuda")
    graphs = []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            c.p.attn8(0, q, out, slots, work, c.status, stream=torch.cuda.current_stream())
        graphs.append(g)
    for names in ([0, 1, 2], [3, 4, 5], [2, 2, 0]):
        slots.copy_(_i32(names))
        for x in range(2):
            q.copy_(_q(x + 7, 3, nq, H, _dt(dt)))
            graphs[x].replay()
            torch.cuda.synchronize()
            assert c.take_status() == 0
            check_attn8(c, 0, q, outs[x], names, dt == "f16")


def test_calls_at_once(cuda):
    """Stores, reads, both forms of attention and beam selection on four streams at once, a workspace each: as one
    after the other."""
    import torch
    n, H, Hkv = 24, 16, 2
    c = Eight(cuda, 2600, 2 * n, 1024, 16, 2, Hkv, seed=2)
    c.place(np.random.default_rng(3).integers(100, 1000, 2 * n).tolist(), seed=3)
    slots = _i32(list(range(n)))
    q1, q4 = _q(5, n, 1, H, torch.float16), _q(6, n, 4, H, torch.float16)
    q32 = _q(7, n, 2, H, torch.float32)
    logits, score = _q(8, 8, 4, 100, torch.float32).view(8, 4, -1), torch.zeros((8, 4), device="cuda")
    cos, sin = _angles(1024)
    dc, ds = _t(cos), _t(sin)
    x = torch.randn((n, 2 * Hkv, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    new = _i32([n + i for i in range(n)])
    pos = _i32([c.m.lens[n + i] - 1 for i in range(n)])
    start = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]

    def calls(s, work):
        o = {"one": torch.empty_like(q1), "four": torch.empty_like(q4), "f32": torch.empty_like(q32),
             "ko": torch.empty((n, Hkv, 128), device="cuda"), "vo": torch.empty((n, Hkv, 128), device="cuda"),
             "so": torch.empty((8, 4), device="cuda"), "pa": _i32([[0] * 4] * 8), "to": _i32([[0] * 4] * 8)}
        torch.cuda.synchronize()

        def go(which):
            if which == 0:
                c.p.append8(1, new, pos, None, x[:, :Hkv], x[:, Hkv:], dc, ds, status=c.status, stream=s[0])
                c.p.read8(1, new, pos, o["ko"], o["vo"], c.status, stream=s[0])
            elif which == 1:
                c.p.attn8(0, q1, o["one"], slots, work[0], c.status, stream=s[1])
                c.p.attn8(0, q32, o["f32"], slots, work[0], c.status, stream=s[1])
            elif which == 2:
                c.p.attn8(0, q4, o["four"], slots, work[1], c.status, stream=s[2])
            else:
                cuda.beam_select(logits, score, o["so"], o["pa"], o["to"], status=c.status, stream=s[3])
        return o, go

    work = [torch.empty(c.p.attn8_work_bytes(n, 4, H), dtype=torch.uint8, device="cuda") for _ in range(2)]
    one = torch.cuda.current_stream()
    want, go = calls([one] * 4, work)
    for w in range(4):
        go(w)
    torch.cuda.synchronize()
    stored = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        for t, old in zip((c.k, c.v, c.ks, c.vs), start):
            t.copy_(old)
        got, go = calls(streams, work)
        for w in (2, 0, 3, 1):
            go(w)
        torch.cuda.synchronize()
        assert c.take_status() == 0
        for name in want:
            assert torch.equal(got[name], want[name]), name
        for t, new_ in zip((c.k, c.v, c.ks, c.vs), stored):
            assert torch.equal(t, new_)


@pytest.mark.parametrize("rows", [(4, 1), (16, 1), (24, 1), (64, 1)])
@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("width", [24, 16384])
def test_attn8_queries_of_a_large_mean(cuda, dt, rows, width):
    """Queries around 1024, keys whose codes cancel in pairs: the scores are of ordinary size. All products are
    whole numbers below 2^14 and their sums whole below 2^21, so 32-bit sums of them are exact: a score is off by its
    scaling, subtraction and exponential alone, the bound's `big` is the largest |score| and not sum |q| |k|."""
    import torch
    H, nq = rows
    lens = [300, 33]
    c = Eight(cuda, 30, 2, width, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    r = np.random.default_rng(11)
    codes = np.repeat(r.integers(-15, 16, c.host.codes[0].shape[:-1] + (64,)), 2, -1).astype(np.int8)
    codes[..., 1::2] *= -1
    c.host.codes[0][:] = codes
    c.host.scales[0][:] = 0.0625
    c.k.copy_(_t(codes))
    c.ks.fill_(0.0625)
    q = _t(1024.0 + r.integers(-3, 4, (2, nq, H, 128))).to(_dt(dt))
    out = run_attn8(c, 0, q, [0, 1], torch.float32)
    assert c.take_status() == 0
    for b, L in enumerate(lens):
        k, v = (torch.from_numpy(c.host.values(w, 0, c.m.tables[b], L)).cuda()[0] for w in range(2))
        for h in range(H):
            x = q[b, :, h].double()
            o, pv, _, va = attention(x, k, v, torch.tensor([max(0, L - nq + 1 + j) for j in range(nq)], device="cuda"))
            big = (x @ k.T / math.sqrt(128)).abs().amax(-1, keepdim=True)
            assert 1 < float(big.max()) < 30
            tol = attn8_bound(o, pv, big, va, L, dt == "f16", False)
            err = (out[b, :, h].double() - o).abs()
            assert bool((err <= tol).all()), (b, h, float((err / tol).max()))


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("low", [0.0, 2.0 ** -100])
def test_attn8_many_keys_of_no_value(cuda, split, low):
    """16384 keys whose values are zeros or the least there are, scores 7.5 powers of two above the sequence's first
    keys, and after them 128 keys of ordinary values, 12 above that: the sums count those without value too. One run
    of tiles a sequence (as many sequences as two CTAs an SM), or one sequence in many parts."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n, H, page = 1 if split else 2 * sms, 24, 128
    reps = (4 * sms if split else 1) * 128
    c = Eight(cuda, 3, 1, max(reps + 2, 4096), page, 1, 1, seed=2)
    bits = 127 * math.log2(math.e) / math.sqrt(128)          # of a key of code 127 and scale 1
    k = torch.zeros((3, page, 128))
    k[1:, :, 0] = 127
    c.k[:, 0, 0] = k.to(torch.int8).cuda()
    scales = torch.tensor([1.0, 7.5 / bits, 19.5 / bits])
    c.ks[:, 0, 0] = scales[:, None].cuda()
    c.vs[:, 0, 0] = torch.tensor([low, low, 0.03125])[:, None].cuda()
    c.tables[0, :reps + 2] = _i32([0] + [1] * reps + [2])
    c.lens[0] = L = (reps + 2) * page
    q = torch.zeros((n, 1, H, 128), dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    out = run_attn8(c, 0, q, [0] * n, torch.float32)
    assert c.take_status() == 0
    # three kinds of keys: weights by 64 bits, each kind's values summed first
    w = torch.exp2(torch.tensor([0.0, 7.5, 19.5], dtype=torch.float64)) * torch.tensor([page, reps * page, page])
    w = (w / w.sum()).cuda()
    mean = c.v[:, 0, 0].double().mean(1) * torch.tensor([low, low, 0.03125], dtype=torch.float64, device="cuda")[:, None]
    o = (w[:, None] * mean).sum(0)
    size = (w[:, None] * (c.v[:, 0, 0].double().abs().mean(1) * c.vs[:, 0, 0, :1].double())).sum(0)
    # scores up to 20 in 32 bits, f16 weights, sums of at most 2^20 terms a part in 32 bits (cut: 2 units each), which all
    # are of one sign and grow by halves: 32 lanes and warps, then tiles, 2^11 of them at most
    tol = size * (2.1 * (264 + 8) * 2.0 ** -24 * 20 + 2.0 ** -11 * 1.01 + (2.0 ** 11 + 300) * 2 * 2.0 ** -24)
    assert 0.04 < float(w[2]) and bool(((out.double() - o).abs() <= tol).all())


FORMS = [("f32", 8, 1, 40), ("f16", 8, 1, 40), ("f32", 24, 1, 40), ("f16", 24, 1, 40), ("f16", 24, 1, 16384), ("f16", 16, 3, 16384)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("unit", [1e3, 1e5, 1e6, 1e8, 1e12, 1e31])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_attn8_scores_far_from_zero(cuda, form, unit, sign):
    """Scores of `unit` times whole numbers, above and below zero. One key's is 10 units above all others', so its
    weight is 1 and the others' are 0: its values come out, off by the rounding of its weight (f16: 2^-11) and by
    some 32-bit ones. Then keys of one score, whose mean comes out: each key's weight is rounded the same way."""
    import torch
    dt, H, nq, width = form
    lens = [500, 130]
    c = Eight(cuda, 50, 2, width, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    r = np.random.default_rng(4)
    bits = math.log2(math.e) / math.sqrt(128)
    c.ks.fill_(unit / 512 / bits)
    c.host.scales[0][:] = unit / 512 / bits
    q = torch.zeros((2, nq, H, 128), dtype=_dt(dt), device="cuda")
    q[..., 0] = 512.0 * sign
    one = 2.0 ** -11 * 1.01 + 16 * 2.0 ** -24 if dt == "f16" else 2.0 ** -22 * 1.01 + 16 * 2.0 ** -24
    for same in (False, True):
        codes = np.zeros(c.host.codes[0].shape, np.int8)
        codes[..., 0] = 50 if same else r.integers(-90, 91, codes.shape[:-1])
        if same:                                             # (one scale: the wide form rounds it with the score)
            c.host.scales[1][:] = 0.03125
            c.vs.fill_(0.03125)
        win = [int(r.integers(L - nq + 1)) for L in lens]
        if not same:
            for b, x in enumerate(win):
                codes[c.m.tables[b][x // 16], 0, 0, x % 16, 0] = 100 * sign
        c.k.copy_(_t(codes))
        out = run_attn8(c, 0, q, [0, 1], torch.float32)
        assert c.take_status() == 0
        for b, L in enumerate(lens):
            v = torch.from_numpy(c.host.values(1, 0, c.m.tables[b], L)).cuda()[0]
            for j in range(nq):
                seen = L - nq + 1 + j
                want = v[:seen].mean(0) if same else v[win[b]]
                size = v[:seen].abs().mean(0) if same else want.abs()
                err = (out[b, j].double() - want).abs()
                assert bool((err <= size * (one + 2 * seen * 2.0 ** -24) + 1e-37).all()), (same, b, j, float((err / size).max()))


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_attn8_rows_that_are_no_numbers(cuda, form):
    """Query rows with a NaN or an infinity come out as NaN, where they see a key; all others as they should."""
    import torch
    dt, H, nq, width = form
    lens = [200, 33, 1]
    c = Eight(cuda, 40, 3, width, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    q = _q(5, 3, nq, H, _dt(dt))
    odd = {(0, nq - 1, 3): math.nan, (0, 0, H - 1): math.inf, (1, 0, 0): -math.inf, (1, nq - 1, 5): math.nan}
    bad = q.clone()
    for (b, j, h), x in odd.items():
        bad[b, j, h, 17 + h] = x
    out = run_attn8(c, 0, bad, [0, 1, 2], torch.float32)
    assert c.take_status() == 0
    for b, j, h in odd:
        assert bool(out[b, j, h].isnan().all())
    good = run_attn8(c, 0, q, [0, 1, 2], torch.float32)
    for b, j, h in odd:
        out[b, j, h] = good[b, j, h]
    check_attn8(c, 0, q, out, [0, 1, 2], dt == "f16")


@pytest.mark.parametrize("H,nq", [(24, 1), (8, 4), (40, 1)])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_attn8_wide_unseen_places_leave_no_trace(cuda, page, H, nq):
    """test_attn8_unseen_places_leave_no_trace over tables with room for many keys; every place that no sequence
    sees is poisoned, tiles end inside pages and blocks."""
    import torch
    lens = [100, 7, 64, 300, 0]
    width = (1 << 20) // page // 4
    c = Eight(cuda, 60, 5, width, page, 1, 1, seed=2)
    c.place(lens, seed=3)
    q = _q(5, 5, nq, H, torch.float16)
    a = run_attn8(c, 0, q, [0, 1, 2, 3, 4], torch.float32)
    seen = {(c.m.tables[s][t // page], t % page) for s in range(5) for t in range(lens[s])}
    blocks = {(p, row // BLOCK) for p, row in seen}
    for p in range(60):
        for b in range(page // BLOCK):
            if (p, b) not in blocks:
                c.ks[p, :, :, b], c.vs[p, :, :, b] = math.nan, math.inf
        for row in range(page):
            if (p, row) not in seen:
                c.k[p, :, :, row], c.v[p, :, :, row] = 127, -128
    for s in range(5):
        c.tables[s, -(-lens[s] // page):] = 1 << 30
    b = run_attn8(c, 0, q, [0, 1, 2, 3, 4], torch.float32)
    assert c.take_status() == 0 and torch.equal(a, b)
    check_attn8(c, 0, q, a, [0, 1, 2, 3, 4], True)


@pytest.mark.parametrize("H,nq", [(24, 1), (8, 4), (40, 1)])
def test_attn8_wide_peaked_rows(cuda, H, nq):
    """test_attn8_peaked_rows over tables with room for many keys, value scales of e^-3 to e^3. (A product of weight and
    scale below 2^-14 of the range is off by 2^-25 of it, as test_attn8_scales_far_apart derives.)"""
    import torch
    lens = [700, 333]
    c = Eight(cuda, 70, 2, 32768, 16, 1, 1, seed=2)
    c.place(lens, seed=3)
    r = np.random.default_rng(3)
    c.host.scales[0][:] = np.exp(r.uniform(-8, 1.5, c.host.scales[0].shape)).astype(np.float32)
    c.host.scales[1][:] = np.exp(r.uniform(-3, 3, c.host.scales[1].shape)).astype(np.float32)
    c.ks.copy_(_t(c.host.scales[0]))
    c.vs.copy_(_t(c.host.scales[1]))
    q = _q(5, 2, nq, H, torch.float16, 0.2)
    out = run_attn8(c, 0, q, [0, 1], torch.float32)
    assert c.take_status() == 0
    for b, L in enumerate(lens):
        k, v = (torch.from_numpy(c.host.values(w, 0, c.m.tables[b], L)).cuda()[0] for w in range(2))
        scale = torch.from_numpy(np.repeat(np.concatenate([c.host.scales[1][p, 0, 0] for p in c.m.tables[b][:c.m.used(L)]]),
                                           BLOCK)[:L]).cuda().double()
        for h in range(H):
            lim = torch.tensor([max(0, L - nq + 1 + j) for j in range(nq)], device="cuda")
            o, pv, big, va = attention(q[b, :, h].double(), k, v, lim)
            s = q[b, :, h].double() @ k.T / math.sqrt(128)
            s[torch.arange(L, device="cuda")[None] >= lim[:, None]] = -math.inf
            top = (torch.softmax(s, -1) * scale).amax(-1, keepdim=True)
            tol = attn8_bound(o, pv, big, va, L, True, False) + 2.0 ** -32 * 1.01 * top * (v / scale[:, None]).abs().sum(0)
            assert bool(((out[b, :, h].double() - o).abs() <= tol).all()), (b, h)


@pytest.mark.parametrize("heads", [(4, 1), (6, 3), (20, 5), (16, 16)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_append8_prompts(cuda, heads, out):
    """Tokens enough for eight heads of k and v a CTA (more than four CTAs an SM with one), some of them padded, wrong
    or repeated: codes and scales of whole pools, rotated rows, rows left alone."""
    import torch
    from kv8_ref import rope
    H, Hkv = heads
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    T = 16 * (4 * sms // (2 * Hkv) + 1) + 37
    page, S = 64, 3
    lens = [T // 2 + 9, T - T // 2 + 40, 5]
    c = Eight(cuda, T // page + 9, S, T // page + 2, page, 1, Hkv, seed=3)
    c.place(lens, seed=1)
    slot = [0] * (T // 2) + [1] * (T - T // 2)
    pos = [9 + i for i in range(T // 2)] + [40 + i for i in range(T - T // 2)]
    for i in range(20, 25):
        slot[i] = -1
    slot[103:103] = [2, S + 1, 2]                            # (between two blocks: a block's tokens stay together)
    pos[103:103] = [4, 0, 5]                                # (the first fits, the slot ends before the last)
    slot.insert(300, slot[300])
    pos.insert(300, pos[300])                               # one position twice
    n = len(slot)
    cos, sin = _angles(max(lens))
    r = np.random.default_rng(H)
    qkv = r.standard_normal((n, H + 2 * Hkv, 128)).astype(np.float32) * np.exp(r.normal(0, 1, (n, 1, 1))).astype(np.float32)
    d = _t(qkv)
    qo = torch.full((n, H, 128), 7.0, dtype=_dt(out), device="cuda")
    ko, vo = (torch.full((n, Hkv, 128), 7.0, dtype=_dt(out), device="cuda") for _ in range(2))
    c.p.append8(0, _i32(slot), _i32(pos), d[:, :H], d[:, H:H + Hkv], d[:, H + Hkv:], _t(cos), _t(sin), qo, ko, vo, c.status)
    torch.cuda.synchronize()
    bad, left = c.host.append(0, c.m.tables, c.m.lens, c.m.refs, slot, pos, qkv[:, H:H + Hkv], qkv[:, H + Hkv:], cos, sin)
    assert bad and c.take_status() == -1 and all(c.same())
    got = [x.cpu().numpy() for x in (qo, ko, vo)]
    for t in range(n):
        if slot[t] < 0:
            assert all((x[t] == 7).all() for x in got)
        elif t in left:
            assert (got[1][t] == 7).all() and (got[2][t] == 7).all()
        else:
            for x, a, b, rot in ((got[0], 0, H, True), (got[1], H, H + Hkv, True), (got[2], H + Hkv, H + 2 * Hkv, False)):
                want = rope(qkv[t, a:b], cos[pos[t]], sin[pos[t]]) if rot else qkv[t, a:b]
                assert np.array_equal(x[t], want.astype(x.dtype))


@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("out", ["f32", "f16"])
@pytest.mark.parametrize("which", ["kv", "k", "v"])
def test_read8_documents(cuda, heads, out, which):
    """Tokens enough for 32 a warp, in any order, twice, wrong and padded."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = 16 * sms * 32 // (heads * len(which)) + 45
    page = 32
    c = Eight(cuda, 90, 3, 40, page, 2, heads, seed=heads)
    c.place([1200, 1, 700], seed=2)
    r = np.random.default_rng(5)
    slot, pos = r.integers(0, 3, n), r.integers(0, 700, n)
    odd = r.random(n) < 0.05
    slot[odd], pos[odd] = r.integers(-1, 5, int(odd.sum())), r.integers(-2, 1400, int(odd.sum()))
    ok = (slot >= 0) & (slot < 3)
    ok &= (pos >= 0) & (pos < np.where(ok, np.array(c.m.lens)[np.where(ok, slot, 0)], 0))
    ko, vo = (torch.full((n, heads, 128), 7.0, dtype=_dt(out), device="cuda") if w in which else None for w in "kv")
    c.p.read8(1, _i32(slot.tolist()), _i32(pos.tolist()), ko, vo, c.status)
    torch.cuda.synchronize()
    assert c.take_status() == -1
    pg = np.array(c.m.tables)[np.where(ok, slot, 0), np.where(ok, pos, 0) // page]
    row = np.where(ok, pos, 0) % page
    for w, o in ((0, ko), (1, vo)):
        if o is not None:
            got = o.cpu().numpy()
            want = c.host.codes[w][pg, 1, :, row].astype(np.float32) * c.host.scales[w][pg, 1, :, row // BLOCK][..., None]
            assert np.array_equal(got[ok], want.astype(got.dtype)[ok]) and (got[~ok] == 7).all()


FIRST = """
import importlib, sys
sys.path.insert(0, %r)
import torch
sllm = importlib.import_module("saphira-llm_b200")
i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
z = lambda shape, dt=torch.float32: torch.zeros(shape, dtype=dt, device="cuda")
k, v = (z((9, 1, 1, 16, 128), torch.int8) for _ in range(2))
ks, vs = (z((9, 1, 1, 1)) for _ in range(2))
tables = i32([list(range(8)) + [0] * 65528])
refs, lens = i32([1] * 9), i32([100])
x = torch.randn((100, 34, 128), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
cos, sin = torch.ones((100, 64), device="cuda"), z((100, 64))
slot, pos, status = i32([0] * 100), i32(list(range(100))), i32([0])
ko, vo = z((100, 1, 128)), z((100, 1, 128))
qs = [x[:1, 2:2 + h].reshape(1, 1, h, 128).to(dt).contiguous() for h, dt in ((8, torch.float32), (16, torch.float16), (32, torch.float16))]
outs = [torch.zeros_like(q) for q in qs]
lg, sc, so = torch.randn((2, 2, 500), device="cuda"), z((2, 2)), z((2, 2))
pa, to = (z((2, 2), torch.int32) for _ in range(2))
slots = i32([0])
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
p = sllm.KvPages(k, v, refs, tables, lens, ks, vs)
with torch.cuda.graph(g, stream=s):
    works = [torch.empty(p.attn8_work_bytes(1, 1, q.shape[2]), dtype=torch.uint8, device="cuda") for q in qs]
    p.append8(0, slot, pos, None, x[:, :1], x[:, 1:2], cos, sin, status=status, stream=s)
    p.read8(0, slot, pos, ko, vo, status, stream=s)
    for q, o, w in zip(qs, outs, works):
        p.attn8(0, q, o, slots, w, status, stream=s)
    sllm.beam_select(lg, sc, so, pa, to, status=status, stream=s)
g.replay()
torch.cuda.synchronize()
assert int(status) == 0
assert float((ko - x[:, :1]).abs().max()) < 0.05 and float((vo - x[:, 1:2]).abs().max()) < 0.05
for q, o in zip(qs, outs):
    w = torch.softmax(q[0, 0].double() @ ko[:, 0].double().T / 128 ** 0.5, -1)
    assert float((o[0, 0].double() - w @ vo[:, 0].double()).abs().max()) < 0.01
lp = torch.log_softmax(lg.double(), -1).view(2, -1).topk(2).values
assert float((so - lp).abs().max()) < 1e-3
print("fine")
"""


def test_first_calls_of_a_process_are_captured(cuda):
    """Nothing of a call needs one outside a capture before it."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST % root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
