"""The attention, paged cache and verification operators on a GPU, against
plain 64-bit restatements (serving_ref.py). Float tolerances are derived
there; bookkeeping and tokens have to be equal."""
import math

import numpy as np
import pytest

from serving_ref import PageModel, attention, attention_bound, verify

pytestmark = pytest.mark.gpu

def _dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16}[name]


def _i32(a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _rand(seed, *shape, dt=None, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt or torch.float32)


# ---------------------------------------------------------------------------
# prompts
# ---------------------------------------------------------------------------
def check_prompt(q, k, v, out, lens, f16, cu0=0):
    import torch
    G = q.shape[1] // k.shape[1]
    at = cu0
    for n in lens:
        for h in range(q.shape[1]):
            lim = torch.arange(1, n + 1, device="cuda")
            o, pv, big, va = attention(q[at:at + n, h].double(), k[at:at + n, h // G].double(),
                                       v[at:at + n, h // G].double(), lim)
            tol = attention_bound(o, pv, big, va, n, f16, out.dtype == torch.float16)
            err = (out[at:at + n, h].double() - o).abs()
            assert bool((err <= tol).all()), (n, h, float((err / tol).nan_to_num(math.inf).max()))
        at += n


LENS = [[1], [2, 0, 1], [16, 17], [64], [63, 65], [128, 129, 127], [255, 256, 257], [300, 1, 0, 513], [700], [0, 0, 5]]


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 1), (20, 5), (7, 1), (6, 2)])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("types", [("f32", "f32"), ("f16", "f16"), ("f16", "f32")])
def test_prompt(cuda, heads, lens, types):
    import torch
    H, Hkv = heads
    T = sum(lens)
    dt, odt = _dt(types[0]), _dt(types[1])
    qkv = _rand(T + H, T + 3, H + 2 * Hkv, 128, dt=dt, scale=1.3)      # three rows belong to no sequence
    out = torch.full((T + 3, H, 128), 7.0, dtype=odt, device="cuda")
    cu = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    cuda.attn_prompt(q, k, v, out, cu)
    torch.cuda.synchronize()
    check_prompt(q, k, v, out, lens, types[0] == "f16")
    assert bool((out[T:] == 7.0).all())


@pytest.mark.parametrize("n_seq,base", [(32, 0), (33, 3), (65, 0), (1030, 5)])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_many_sequences(cuda, dt, n_seq, base):
    """More sequences than a warp has lanes, of which many are empty; offsets
    that start behind 0."""
    import torch
    rng = np.random.default_rng(n_seq)
    lens = [int(rng.choice([0, 1, 2, 63, 64, 65, 127, 128, 129, 300])) for _ in range(n_seq)]
    lens[n_seq // 2] = 700
    lens[-1] = 0 if base else 257
    T = base + sum(lens)
    qkv = _rand(n_seq, T + 2, 4, 128, dt=_dt(dt), scale=1.3)
    q, k, v = qkv[:, :2], qkv[:, 2:3], qkv[:, 3:]
    out = torch.full((T + 2, 2, 128), 7.0, dtype=_dt(dt), device="cuda")
    cuda.attn_prompt(q, k, v, out, _i32((base + np.concatenate([[0], np.cumsum(lens)])).tolist()))
    torch.cuda.synchronize()
    check_prompt(q, k, v, out, lens, dt == "f16", base)
    assert bool((out[:base] == 7.0).all()) and bool((out[T:] == 7.0).all())


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_large_scores(cuda, dt):
    """Peaked rows: scores up to some hundreds, growing along the keys, so
    that the running maximum moves at every tile."""
    import torch
    n, H = 600, 2
    q, k, v = (_rand(s, n, H, 128, dt=_dt(dt)) for s in (1, 2, 3))
    k *= torch.linspace(0.2, 9.0, n, device="cuda")[:, None, None].to(k.dtype)
    out = torch.empty_like(q)
    cuda.attn_prompt(q, k, v, out, _i32([0, n]))
    torch.cuda.synchronize()
    check_prompt(q, k, v, out, [n], dt == "f16")


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_masked_places_leave_no_trace(cuda, dt):
    """Infinities and NaN in keys and values that a row does not see (later
    tokens of its sequence, other sequences, rows of no sequence) do not reach
    it; rows that see them are not asked about."""
    import torch
    lens = [150, 70, 200]
    T, H, Hkv = sum(lens), 4, 2
    q, k, v = _rand(1, T + 9, H, 128, dt=_dt(dt)), _rand(2, T + 9, Hkv, 128, dt=_dt(dt)), _rand(3, T + 9, Hkv, 128, dt=_dt(dt))
    out = torch.empty_like(q)
    cu = _i32([0, 150, 220, 420])
    cuda.attn_prompt(q, k, v, out, cu)
    kb, vb = k.clone(), v.clone()
    bad = [140, 219, 300, 419, T, T + 8]           # token 140 of the first, the last of the second, 80 and 199 of the third
    for i, t in enumerate(bad):
        kb[t] = [math.inf, math.nan, -math.inf][i % 3]
        vb[t, :, ::3] = [math.nan, math.inf, -math.inf][i % 3]
    got = torch.empty_like(q)
    cuda.attn_prompt(q, kb, vb, got, cu)
    torch.cuda.synchronize()
    clean = list(range(0, 140)) + list(range(150, 219)) + list(range(220, 300))
    assert bool(torch.isfinite(got[clean].float()).all())
    check_prompt(q[:140], k[:140], v[:140], got[:140], [140], dt == "f16")
    check_prompt(q[150:219], k[150:219], v[150:219], got[150:219], [69], dt == "f16")
    check_prompt(q[220:300], k[220:300], v[220:300], got[220:300], [80], dt == "f16")
    # rows that see a NaN value hold it
    assert bool(torch.isnan(got[140, :, 0].float()).all())


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_offsets_beyond_32_bits(cuda, dt):
    """Tokens 2^26 elements apart: addresses past 2^31 elements (and 2^32 bytes)."""
    import torch
    n, stride = 36, 1 << 26
    buf = torch.zeros(stride * n, dtype=_dt(dt), device="cuda")
    q, k, v = (torch.as_strided(buf, (n, 1, 128), (stride, 128, 1), storage_offset=o) for o in (0, 128, 256))
    for i, t in enumerate((q, k, v)):
        t.copy_(_rand(i, n, 1, 128, dt=_dt(dt)))
    out = torch.empty(n, 1, 128, dtype=_dt(dt), device="cuda")
    cuda.attn_prompt(q, k, v, out, _i32([0, n]))
    torch.cuda.synchronize()
    check_prompt(q, k, v, out, [n], dt == "f16")
    del buf
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_stream_and_graph(cuda, dt):
    """On a side stream, and captured once and replayed on new inputs."""
    import torch
    lens = [90, 260]
    T, H, Hkv = sum(lens), 8, 2
    s = torch.cuda.Stream()
    q, k, v = (torch.empty(T, h, 128, dtype=_dt(dt), device="cuda") for h in (H, Hkv, Hkv))
    out = torch.empty_like(q)
    cu = _i32([0, 90, 350])

    def fill(seed):
        for i, t in enumerate((q, k, v)):
            t.copy_(_rand(seed + i, *t.shape, dt=t.dtype))

    fill(1)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cuda.attn_prompt(q, k, v, out, cu, stream=s)
    s.synchronize()
    check_prompt(q, k, v, out, lens, dt == "f16")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cuda.attn_prompt(q, k, v, out, cu, stream=torch.cuda.current_stream())
    for seed in (10, 20):
        fill(seed)
        cu.copy_(_i32([0, 350, 350] if seed == 20 else [0, 90, 350]))
        g.replay()
        torch.cuda.synchronize()
        check_prompt(q, k, v, out, [350] if seed == 20 else lens, dt == "f16")


def test_prompt_wrong_offsets_stay_inside(cuda):
    """Offsets that descend or pass the arrays are clamped to them."""
    import torch
    n, H = 100, 2
    for dt in ("f32", "f16"):
        q, k, v = (_rand(s, n, H, 128, dt=_dt(dt)) for s in (1, 2, 3))
        out = torch.zeros_like(q)
        for cu in ([0, 500], [-7, 100], [60, 20], [2 ** 31 - 1, -2 ** 31], [0, 100, 50, 100]):
            cuda.attn_prompt(q, k, v, out, _i32(cu))
        torch.cuda.synchronize()
        cuda.attn_prompt(q, k, v, out, _i32([0, 100]))
        torch.cuda.synchronize()
        check_prompt(q, k, v, out, [100], dt == "f16")


def test_no_bounded_wait_gave_up(cuda):
    import torch
    for dt in ("f16", "f32"):
        q, k, v = (_rand(s, 3000, 2, 128, dt=_dt(dt)) for s in (1, 2, 3))
        cuda.attn_prompt(q, k, v, torch.empty_like(q), _i32([0, 2000, 3000]))
        c = shared_cache(cuda, 1024, [300] * 9, 16, (20, 5), dt)
        run_prefix(cuda, c, list(range(9)), 2, (20, 5), 1024, dt)
    assert cuda.attn_error() == 0


def test_host_memory_is_refused(cuda):
    import torch
    q = torch.zeros(4, 2, 128)
    d = q.cuda()
    with pytest.raises(cuda.SllmCudaError, match="current device"):
        cuda.attn_prompt(d, d, q, d, _i32([0, 4]))
    with pytest.raises(cuda.SllmCudaError, match="current device"):
        cuda.attn_prompt(d, d, d, d, torch.tensor([0, 4], dtype=torch.int32))


# ---------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------
class Cache:
    """A cache on the device and its model on the host."""

    def __init__(self, cuda, n_pages, n_slots, width, page, layers=2, heads=2, dt="f16", seed=0, fill=0.0):
        import torch
        self.dt, self.page = dt, page
        shape = (n_pages, layers, heads, page, 128)
        self.k = _rand(seed + 1, *shape, dt=_dt(dt))
        self.v = _rand(seed + 2, *shape, dt=_dt(dt))
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        self.tables = torch.zeros(n_slots, width, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(n_slots, dtype=torch.int32, device="cuda")
        self.p = cuda.KvPages(self.k, self.v, self.refs, self.tables, self.lens)
        self.work = torch.empty(self.p.work_bytes(), dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.m = PageModel(n_pages, n_slots, width, page)

    def push(self):
        """The model's bookkeeping onto the device."""
        self.refs.copy_(_i32(self.m.refs))
        self.tables.copy_(_i32(self.m.tables))
        self.lens.copy_(_i32(self.m.lens))

    def same(self):
        import torch
        torch.cuda.synchronize()
        assert self.refs.tolist() == self.m.refs
        assert self.lens.tolist() == self.m.lens
        got = self.tables.tolist()
        for s in range(self.m.n_slots):
            u = self.m.used(self.m.lens[s])
            assert got[s][:u] == self.m.tables[s][:u], s

    def take_status(self):
        v = int(self.status.item())
        self.status.zero_()
        return v

    def rows(self, s, pool=None):
        """[len][layers][heads][128] of a slot."""
        pool = self.k if pool is None else pool
        n = self.m.lens[s]
        ids = self.m.tables[s][:self.m.used(n)]
        if not ids:
            return pool[:0, :, :, 0].clone()
        x = pool[ids].permute(0, 3, 1, 2, 4).reshape(-1, pool.shape[1], pool.shape[2], 128)
        return x[:n].clone()


@pytest.mark.parametrize("page,dt,n_pages,n_slots,width,steps", [
    (16, "f16", 60, 7, 9, 120), (32, "f32", 50, 9, 6, 80), (64, "f16", 30, 5, 4, 60), (128, "f32", 24, 6, 3, 40),
    (16, "f32", 40000, 40, 40, 30), (16, "f16", 16385, 70, 20, 30),
])
def test_page_operations_in_any_order(cuda, page, dt, n_pages, n_slots, width, steps):
    """Random forks, reservations, releases and compactions: bookkeeping as the
    model has it, each slot's tokens unchanged, rows outside the copies too."""
    import torch
    heads = 1 if n_pages > 1000 else 2
    layers = 1 if n_pages > 1000 else 3
    c = Cache(cuda, n_pages, n_slots, width, page, layers, heads, dt, seed=page)
    rng = np.random.default_rng(n_pages + page)
    seen = {0: 0}
    for step in range(steps):
        n = int(rng.integers(1, n_slots + 1))
        slots = [int(x) for x in rng.permutation(n_slots)[:n]]
        op = int(rng.integers(5))
        k0, v0 = c.k.clone(), c.v.clone()
        before = {s: (c.rows(s), c.rows(s, c.v)) for s in range(n_slots)}
        lens0 = list(c.m.lens)
        copies, moved = [], {s: s for s in range(n_slots)}
        if op == 0:
            src = [int(x) for x in rng.integers(0, n_slots, n)]
            if rng.random() < 0.15:
                slots[0] = slots[-1] if n > 1 else n_slots
            want = c.m.fork(src, slots)
            if want == 0:
                moved.update(dict(zip(slots, src)))
            c.p.fork(_i32(src), _i32(slots), c.work, c.status)
        elif op in (1, 2):
            new = [int(x) for x in rng.integers(0, 3 * page, n)]
            if rng.random() < 0.5:
                new = [min(x, 1) for x in new]
            want, copies = c.m.reserve(slots, new)
            c.p.reserve(_i32(slots), _i32(new), c.work, c.status)
        elif op == 3:
            keep = [int(rng.integers(0, c.m.lens[s] + 1)) for s in slots]
            if rng.random() < 0.15:
                keep[0] = c.m.lens[slots[0]] + 1
            want = c.m.release(slots, None if step % 2 else keep)
            c.p.release(_i32(slots), None if step % 2 else _i32(keep), c.work, c.status)
        else:
            want, copies = c.m.compact()
            c.p.compact(c.work, c.status)
        c.same()
        assert c.take_status() == want, (op, want)
        seen[want] = seen.get(want, 0) + 1
        for a, b, r in copies:
            k0[b, :, :, :r], v0[b, :, :, :r] = k0[a, :, :, :r], v0[a, :, :, :r]
        assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
        for s in range(n_slots):
            m = min(c.m.lens[s], lens0[moved[s]])
            assert torch.equal(c.rows(s)[:m], before[moved[s]][0][:m])
            assert torch.equal(c.rows(s, c.v)[:m], before[moved[s]][1][:m])
    assert seen[0] > steps // 4


def test_page_operations_on_many_slots(cuda):
    """More slots than the reserving CTA has threads and the clusters have
    warps: several rounds of each, pages shared across the rounds."""
    n_slots = 2100
    c = Cache(cuda, 9000, n_slots, 6, 16, 1, 1, "f16", seed=3)
    rng = np.random.default_rng(11)

    def step(op, *args):
        want = getattr(c.m, op)(*args)
        want = want[0] if isinstance(want, tuple) else want
        getattr(c.p, op)(*[None if a is None else _i32(a) for a in args], c.work, c.status)
        c.same()
        assert c.take_status() == want
        return want

    order = [int(x) for x in rng.permutation(n_slots)]
    assert step("reserve", order[:700], [int(x) for x in rng.integers(1, 40, 700)]) == 0
    assert step("fork", [order[i % 700] for i in range(1400)], order[700:]) == 0
    # one token each: shared last pages are copied, the last owner keeps one
    assert step("reserve", order, [1] * n_slots) == 0
    again = [int(x) for x in rng.permutation(n_slots)]
    assert step("reserve", again[:1900], [int(x) for x in rng.integers(0, 30, 1900)]) == 0
    assert step("reserve", order, [97] * n_slots) == -36
    keep = [int(rng.integers(0, c.m.lens[s] + 1)) for s in again]
    assert step("release", again, keep[:-1] + [c.m.lens[again[-1]] + 1]) == -1
    assert step("release", again, keep) == 0
    assert step("compact") == 0
    assert step("fork", order[:2000], again[:2000]) == 0
    assert step("fork", order[:2000], again[:1999] + again[:1]) == -1
    assert step("release", order[:1500], None) == 0


def test_page_errors_change_nothing(cuda):
    c = Cache(cuda, 20, 4, 4, 16)
    m = c.m
    m.reserve([0, 1], [40, 10])
    c.push()
    for call, want in [
        (lambda: c.p.fork(_i32([0, 1]), _i32([2, 2]), c.work, c.status), -1),
        (lambda: c.p.fork(_i32([4]), _i32([2]), c.work, c.status), -1),
        (lambda: c.p.fork(_i32([0]), _i32([-1]), c.work, c.status), -1),
        (lambda: c.p.reserve(_i32([0, 0]), _i32([1, 1]), c.work, c.status), -1),
        (lambda: c.p.reserve(_i32([0, 7]), _i32([1, 1]), c.work, c.status), -1),
        (lambda: c.p.reserve(_i32([0]), _i32([-1]), c.work, c.status), -1),
        (lambda: c.p.reserve(_i32([1, 0]), _i32([1, 25]), c.work, c.status), -36),
        (lambda: c.p.reserve(_i32([0]), _i32([2 ** 31 - 1]), c.work, c.status), -36),
        (lambda: c.p.release(_i32([0]), _i32([41]), c.work, c.status), -1),
        (lambda: c.p.release(_i32([0]), _i32([-1]), c.work, c.status), -1),
        (lambda: c.p.release(_i32([0, 0]), None, c.work, c.status), -1),
    ]:
        call()
        c.same()
        assert c.take_status() == want
    # too few pages: 4 slots * 4 pages fit 20 pages, 3 of 20 are kept free here
    m.refs[5:20] = [1] * 15
    c.push()
    c.p.reserve(_i32([2]), _i32([17]), c.work, c.status)
    c.same()
    assert c.take_status() == -2
    # a table that names no page
    m.refs[5:20] = [0] * 15
    c.push()
    c.tables[0, 1] = 99
    for call in (lambda: c.p.fork(_i32([0]), _i32([3]), c.work, c.status),
                 lambda: c.p.release(_i32([0]), None, c.work, c.status),
                 lambda: c.p.compact(c.work, c.status)):
        call()
        assert c.take_status() == -1
    c.tables[0, 1] = m.tables[0][1]
    c.same()


def test_page_calls_captured(cuda):
    """fork, reserve, release and compact in one graph, replayed."""
    import torch
    c = Cache(cuda, 64, 6, 6, 16)
    c.m.reserve([0], [37])
    c.push()
    src, dst = _i32([0, 0, 0]), _i32([1, 2, 3])
    slots, new = _i32([0, 1, 2, 3]), _i32([1, 1, 1, 20])
    gone = _i32([0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s = torch.cuda.current_stream()
        c.p.fork(src, dst, c.work, c.status, stream=s)
        c.p.reserve(slots, new, c.work, c.status, stream=s)
        c.p.release(gone, None, c.work, c.status, stream=s)
        c.p.compact(c.work, c.status, stream=s)
    for _ in range(3):
        c.m.fork([0, 0, 0], [1, 2, 3])
        c.m.reserve([0, 1, 2, 3], [1, 1, 1, 20])
        c.m.release([0], [0])
        c.m.compact()
        g.replay()
        c.same()
        assert c.take_status() == 0
        c.m.reserve([0], [37])
        c.push()


@pytest.mark.parametrize("dt,page,heads,layers", [("f16", 16, (20, 5), 2), ("f32", 64, (8, 1), 1), ("f16", 128, (4, 4), 3),
                                                  ("f32", 32, (6, 2), 2)])
def test_append(cuda, dt, page, heads, layers):
    """Rotation and placement: bit-exact against the same f32 operations."""
    import torch
    H, Hkv = heads
    c = Cache(cuda, 40, 3, 200 // page + 2, page, layers, Hkv, dt)
    c.m.reserve([0, 1, 2], [90, 0, 150])
    c.push()
    slot = [0] * 33 + [2] * 60 + [-1, 0, 1, 2, 3, 2, 2]
    pos = list(range(57, 90)) + list(range(0, 60)) + [5, 90, 0, 150, 0, -1, 149]
    good = list(range(93)) + [99]
    T = len(slot)
    qkv = _rand(5, T, H + 2 * Hkv, 128)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    cos, sin = (torch.from_numpy(x).cuda() for x in cuda.rope_table(150, 10000.0))
    qo, ko, vo = (torch.full((T, h, 128), 3.0, dtype=_dt(dt), device="cuda") for h in (H, Hkv, Hkv))
    k0, v0 = c.k.clone(), c.v.clone()
    layer = layers - 1
    c.p.append(layer, _i32(slot), _i32(pos), q, k, v, cos, sin, qo, ko, vo, c.status)
    torch.cuda.synchronize()
    assert c.take_status() == -1              # positions and slots above are wrong in places

    def rope(x, ps):
        cs, sn = cos[ps][:, None], sin[ps][:, None]
        a, b = x[..., :64], x[..., 64:]
        return torch.cat([a * cs - b * sn, a * sn + b * cs], -1).to(_dt(dt))

    ps = torch.tensor([pos[i] for i in good], device="cuda")
    gi = torch.tensor(good, device="cuda")
    assert torch.equal(qo[gi], rope(q[gi], ps)) and torch.equal(ko[gi], rope(k[gi], ps))
    assert torch.equal(vo[gi], v[gi].to(_dt(dt)))
    for i in range(T):
        if i in good:
            pg = c.m.tables[slot[i]][pos[i] // page]
            k0[pg, layer, :, pos[i] % page] = ko[i]
            v0[pg, layer, :, pos[i] % page] = vo[i]
        else:
            assert bool((qo[i] == 3.0).all()) and bool((ko[i] == 3.0).all())
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)
    # a shared page is not written
    c.m.fork([0], [1])
    c.push()
    c.p.append(layer, _i32([1]), _i32([89]), q[:1], k[:1], v[:1], cos, sin, status=c.status,
               q_out=qo[:1], k_out=None, v_out=None)
    torch.cuda.synchronize()
    assert c.take_status() == -1 and torch.equal(c.k, k0)
    # without q and without the contiguous outputs
    c.p.append(layer, _i32([2]), _i32([3]), None, k[:1], v[:1], cos, sin, status=c.status)
    torch.cuda.synchronize()
    pg = c.m.tables[2][0]
    k0[pg, layer, :, 3], v0[pg, layer, :, 3] = rope(k[:1], torch.tensor([3], device="cuda"))[0], v[0].to(_dt(dt))
    assert c.take_status() == 0 and torch.equal(c.k, k0) and torch.equal(c.v, v0)


def test_append_in_place(cuda):
    """f32 outputs over their inputs."""
    import torch
    c = Cache(cuda, 10, 1, 8, 16, 1, 2, "f32")
    c.m.reserve([0], [40])
    c.push()
    q, k, v = _rand(1, 40, 4, 128), _rand(2, 40, 2, 128), _rand(3, 40, 2, 128)
    cos, sin = (torch.from_numpy(x).cuda() for x in cuda.rope_table(64, 10000.0))
    outs = [torch.empty_like(t) for t in (q, k, v)]
    slot, pos = _i32([0] * 40), _i32(list(range(40)))
    c.p.append(0, slot, pos, q, k, v, cos, sin, *outs, c.status)
    c.p.append(0, slot, pos, q, k, v, cos, sin, q, k, v, c.status)
    torch.cuda.synchronize()
    assert c.take_status() == 0 and all(torch.equal(a, b) for a, b in zip(outs, (q, k, v)))


# ---------------------------------------------------------------------------
# decode attention over a shared prefix
# ---------------------------------------------------------------------------
def check_prefix(c, q, out, slots, layer, skip=()):
    import torch
    n, nq, H, _ = q.shape
    Hkv = c.k.shape[2]
    for b, s in enumerate(slots):
        if b in skip:
            continue
        L = c.m.lens[s]
        k, v = c.rows(s)[:, layer].double(), c.rows(s, c.v)[:, layer].double()
        lim = torch.tensor([max(0, L - nq + 1 + j) for j in range(nq)], device="cuda")
        for h in range(H):
            o, pv, big, va = attention(q[b, :, h].double(), k[:, h // (H // Hkv)], v[:, h // (H // Hkv)], lim)
            tol = attention_bound(o, pv, big, va, L, c.dt == "f16", out.dtype == torch.float16)
            err = (out[b, :, h].double() - o).abs()
            assert bool((err <= tol).all()), (b, h, L, float((err / tol).nan_to_num(math.inf).max()))


def shared_cache(cuda, prefix, owns, page, heads, dt, layers=2, seed=0, spare_slots=2):
    """Slots 0 .. n-1: forks of one prefix with tokens of their own, on pages in no order."""
    n = len(owns)
    width = (prefix + max(owns + [0])) // page + 2
    need = prefix // page + sum(-(-o // page) for o in owns) + 5
    c = Cache(cuda, need, n + spare_slots, width, page, layers, heads[1], dt, seed)
    m = c.m
    ids = [int(x) for x in np.random.default_rng(seed).permutation(need)]
    pre = ids[:prefix // page]
    at = len(pre)
    for s, o in enumerate(owns):
        u = -(-o // page)
        row = pre + ids[at:at + u]
        at += u
        m.tables[s][:len(row)] = row
        m.lens[s] = prefix + o
        for i in row:
            m.refs[i] += 1
    c.push()
    return c


def run_prefix(cuda, c, slots, nq, heads, prefix, odt, layer=1, seed=0, stream=None):
    import torch
    n, H = len(slots), heads[0]
    q = _rand(seed + 77, n, nq, H, 128, dt=_dt(c.dt), scale=1.3)
    out = torch.full((n, nq, H, 128), 7.0, dtype=_dt(odt), device="cuda")
    work = torch.empty(c.p.attn_prefix_work_bytes(n, nq, H, prefix), dtype=torch.uint8, device="cuda")
    work.fill_(255)                                  # what a workspace held before does not matter
    c.p.attn_prefix(layer, q, out, _i32(slots), prefix, work, c.status, stream=stream)
    torch.cuda.synchronize()
    return q, out


PREFIX = [
    # prefix, own tokens, page, heads, query tokens
    (0, [1], 16, (4, 4), 1), (0, [17, 1, 130], 16, (20, 5), 1), (16, [0], 16, (8, 1), 1), (32, [0, 5, 200], 32, (8, 1), 1),
    (128, [1, 2], 128, (20, 5), 1), (256, [64, 3, 129], 64, (64, 8), 1), (144, [33, 7, 16], 16, (7, 1), 2),
    (512, [4, 90, 5], 64, (8, 1), 4), (1024, [300] * 9, 16, (20, 5), 1), (192, [16, 17, 31], 64, (6, 2), 16),
    (2048, [1] * 33, 128, (8, 1), 1), (320, [3] * 70, 32, (4, 4), 3), (4096, [257, 1], 64, (64, 8), 2),
    (0, [1500, 700, 3], 16, (20, 5), 1), (0, [5, 3], 16, (4, 2), 4), (640, [200, 300], 128, (20, 5), 8),
    (192, [40, 9], 64, (64, 1), 8), (128, [17], 32, (128, 1), 1), (64, [30, 1], 16, (256, 1), 2), (0, [700], 16, (129, 1), 1),
    (32, [1] * 300, 16, (2, 1), 1), (1600, [20, 33], 16, (4, 1), 2),
]


@pytest.mark.parametrize("case", PREFIX)
@pytest.mark.parametrize("types", [("f32", "f32"), ("f16", "f16"), ("f16", "f32")])
def test_prefix(cuda, case, types):
    prefix, owns, page, heads, nq = case
    c = shared_cache(cuda, prefix, owns, page, heads, types[0], seed=prefix + nq)
    slots = [int(x) for x in np.random.default_rng(1).permutation(len(owns))]
    q, out = run_prefix(cuda, c, slots, nq, heads, prefix, types[1])
    assert c.take_status() == 0
    check_prefix(c, q, out, slots, 1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_rows_that_see_nothing(cuda, dt):
    """Empty slots, and query tokens before the first: zeros."""
    c = shared_cache(cuda, 0, [0, 2, 40], 16, (4, 2), dt)
    q, out = run_prefix(cuda, c, [0, 1, 2, 0], 4, (4, 2), 0, dt)
    assert c.take_status() == 0
    assert bool((out[0] == 0).all()) and bool((out[3] == 0).all()) and bool((out[1, :2] == 0).all())
    check_prefix(c, q, out, [0, 1, 2, 0], 1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_unseen_rows_leave_no_trace(cuda, dt):
    """NaN and infinities behind a slot's length in its last page, in free
    pages, and in the later drafted tokens that an earlier query does not see."""
    import torch
    owns = [5, 37, 64]
    c = shared_cache(cuda, 128, owns, 64, (8, 2), dt)
    live = sorted({i for s in range(3) for i in c.m.tables[s][:c.m.used(c.m.lens[s])]})
    free = [i for i in range(c.m.n_pages) if i not in live]
    c.k[free], c.v[free] = math.nan, math.inf
    for s in range(3):
        n = c.m.lens[s]
        if n % 64:
            pg = c.m.tables[s][n // 64]
            c.k[pg, :, :, n % 64:], c.v[pg, :, :, n % 64:] = math.inf, math.nan
    q, out = run_prefix(cuda, c, [0, 1, 2], 1, (8, 2), 128, dt)
    check_prefix(c, q, out, [0, 1, 2], 1)
    # the last token of slot 1 is unseen by all but the last of three queries
    n = c.m.lens[1] - 1
    pg = c.m.tables[1][n // 64]
    keep = c.k[pg].clone(), c.v[pg].clone()
    c.k[pg, :, :, n % 64], c.v[pg, :, :, n % 64] = math.nan, math.inf
    q, out = run_prefix(cuda, c, [0, 1, 2], 3, (8, 2), 128, dt)
    assert bool(torch.isfinite(out[1, :2].float()).all()) and bool(torch.isnan(out[1, 2].float()).any())
    c.k[pg], c.v[pg] = keep
    ref_q, ref = run_prefix(cuda, c, [0, 1, 2], 3, (8, 2), 128, dt)
    check_prefix(c, ref_q, ref, [0, 1, 2], 1)
    full = ref.clone()
    full[1, :2] = out[1, :2]
    check_prefix(c, ref_q, full, [0, 1, 2], 1)
    assert c.take_status() == 0


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_bad_sequences_are_reported(cuda, dt):
    """Wrong slots, lengths and pages: *status says so, the other sequences
    come out right, nothing faults."""
    c = shared_cache(cuda, 64, [20, 30, 40, 50], 16, (4, 2), dt)
    q, out = run_prefix(cuda, c, [0, 99, 2, -1], 1, (4, 2), 64, dt)
    assert c.take_status() == -1
    check_prefix(c, q, out, [0, 99, 2, -1], 1, skip=(1, 3))
    c.lens[1] = 10 ** 6
    q, out = run_prefix(cuda, c, [0, 1, 2], 1, (4, 2), 64, dt)
    assert c.take_status() == -1
    check_prefix(c, q, out, [0, 1, 2], 1, skip=(1,))
    c.lens[1] = 40                            # shorter than the prefix
    q, out = run_prefix(cuda, c, [0, 1, 2], 1, (4, 2), 64, dt)
    assert c.take_status() == -1
    check_prefix(c, q, out, [0, 1, 2], 1, skip=(1,))
    c.push()
    for bad in (-1, c.m.n_pages, 2 ** 31 - 1):
        c.tables[1, 5] = bad
        q, out = run_prefix(cuda, c, [0, 1, 2], 1, (4, 2), 64, dt)
        assert c.take_status() == -1
        check_prefix(c, q, out, [0, 1, 2], 1, skip=(1,))
    c.push()
    c.tables[0, 1] = -5                       # the prefix of all, read from slots[0]
    run_prefix(cuda, c, [0, 1, 2], 1, (4, 2), 64, dt)
    assert c.take_status() == -1
    c.push()
    q, out = run_prefix(cuda, c, [0, 1, 2], 1, (4, 2), 64, dt)
    assert c.take_status() == 0
    check_prefix(c, q, out, [0, 1, 2], 1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_peaked_rows(cuda, dt):
    """Scores in the hundreds, the prefix and the own part far apart."""
    c = shared_cache(cuda, 512, [100, 300], 32, (8, 2), dt)
    c.k[c.m.tables[0][:8]] *= 8.0
    c.k[c.m.tables[1][17]] *= 12.0
    q, out = run_prefix(cuda, c, [0, 1], 2, (8, 2), 512, dt)
    check_prefix(c, q, out, [0, 1], 1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_many_sequences(cuda, dt):
    """More sequences than a block has threads."""
    n = 1500
    c = shared_cache(cuda, 32, [1 + i % 3 for i in range(n)], 16, (2, 1), dt, spare_slots=0)
    slots = list(range(n))
    q, out = run_prefix(cuda, c, slots, 1, (2, 1), 32, dt)
    assert c.take_status() == 0
    check_prefix(c, q, out, slots, 1, skip=set(range(n)) - set(range(0, n, 37)))
    # and page calls that name them all
    import torch
    new = [1] * n
    want, copies = c.m.reserve(slots[:100], new[:100])
    c.p.reserve(_i32(slots[:100]), _i32(new[:100]), c.work, c.status)
    c.same()
    assert c.take_status() == want
    want = c.m.release(slots, None)
    c.p.release(_i32(slots), None, c.work, c.status)
    c.same()
    assert c.take_status() == want == 0 and not any(c.m.refs)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_rows_that_see_no_numbers_are_no_numbers(cuda, dt):
    """A NaN or an infinity in a key or value that a row does see shows in it."""
    import torch
    n = 200
    for bad in (math.nan, math.inf):
        for which in (0, 1):
            q, k, v = (_rand(s, n, 2, 128, dt=_dt(dt)) for s in (1, 2, 3))
            (k, v)[which][50] = bad
            out = torch.empty_like(q)
            cuda.attn_prompt(q, k, v, out, _i32([0, n]))
            torch.cuda.synchronize()
            assert bool(torch.isfinite(out[:50].float()).all())
            if which == 1 or math.isnan(bad):
                assert not bool(torch.isfinite(out[50:].float()).any(-1).any()), (bad, which)


def test_prefix_offsets_beyond_32_bits(cuda):
    """A pool of more than 2^32 bytes and 2^31 elements, the live pages at its ends."""
    import torch
    page, layers, heads = 128, 8, (16, 8)
    n_pages = (1 << 31) // (layers * heads[1] * page * 128) + 9
    pool = torch.zeros(n_pages, layers, heads[1], page, 128, dtype=torch.float16, device="cuda")
    c = Cache(cuda, 12, 2, 8, page, layers, heads[1], "f16")
    small_k, small_v = c.k, c.v
    pages = [0, n_pages - 1, 1, n_pages - 2, n_pages // 2, n_pages - 3]
    # one pool serves as K and as V: layer 7 for K, layer 6 for V
    c.m.n_pages = n_pages
    c.m.refs = [0] * n_pages
    c.m.tables[0][:4] = pages[:4]
    c.m.tables[1][:4] = pages[:2] + pages[4:]
    c.m.lens[:2] = [500, 400]
    for r in c.m.tables[0][:4] + c.m.tables[1][:4]:
        c.m.refs[r] += 1
    for i, pg in enumerate(pages):
        pool[pg] = _rand(i, *pool.shape[1:], dt=torch.float16)
    c.k = c.v = pool
    c.refs = _i32(c.m.refs)
    c.p = cuda.KvPages(pool, pool, c.refs, c.tables, c.lens)
    c.push()
    q, out = run_prefix(cuda, c, [0, 1], 1, heads, 256, "f16", layer=layers - 1)
    assert c.take_status() == 0
    check_prefix(c, q, out, [0, 1], layers - 1)
    del pool, c, small_k, small_v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_many_items_captured(cuda, dt):
    """Enough items for the counter that hands them out: captured, replayed."""
    import torch
    n, heads, prefix = 70, (8, 8), 640
    c = shared_cache(cuda, prefix, [3 + i % 50 for i in range(n)], 32, heads, dt)
    q = _rand(9, n, 1, 8, 128, dt=_dt(dt))
    out = torch.empty_like(q)
    slots = _i32(list(range(n)))
    work = torch.empty(c.p.attn_prefix_work_bytes(n, 1, 8, prefix), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.p.attn_prefix(1, q, out, slots, prefix, work, c.status, stream=torch.cuda.current_stream())
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        check_prefix(c, q, out, list(range(n)), 1)


def test_first_calls_inside_a_capture():
    """In a fresh process, with nothing loaded before, every operator's first
    call is captured."""
    import subprocess
    import sys
    code = """
import importlib, torch
pkg = importlib.import_module("saphira-llm_b200")
i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
k = torch.randn(8, 1, 2, 16, 128, device="cuda").half()
v = torch.randn(8, 1, 2, 16, 128, device="cuda").half()
p = pkg.KvPages(k, v, i32([1, 1] + [0] * 6), i32([[0, 1, 0], [0, 0, 0]]), i32([20, 0]))
work = torch.empty(p.work_bytes(), dtype=torch.uint8, device="cuda")
q = torch.randn(1, 1, 4, 128, device="cuda").half()
o = torch.empty_like(q)
scratch = torch.empty(p.attn_prefix_work_bytes(1, 1, 4, 0), dtype=torch.uint8, device="cuda")
x = torch.randn(9, 2, 128, device="cuda")
y = torch.empty_like(x)
h, ho = x.half(), torch.empty_like(x.half())
pr = torch.full((1, 2, 6000), 1 / 6000, device="cuda")
tok, cnt = i32([[0, 0]]), i32([0])
one, zero, cu, status = i32([1]), i32([0]), i32([0, 9]), i32([0])
ua, us = torch.rand(1, 1, device="cuda"), torch.rand(1, device="cuda")
cos = torch.ones(64, 64, device="cuda")
pos20, tok1 = i32([20]), i32([[0]])
x4, x1, q4 = torch.randn(1, 4, 128, device="cuda"), x[:1], torch.empty(1, 4, 128, device="cuda").half()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = torch.cuda.current_stream()
    pkg.attn_prompt(x, x, x, y, cu, stream=s)
    pkg.attn_prompt(h, h, h, ho, cu, stream=s)
    p.fork(zero, one, work, status, stream=s)
    p.reserve(one, one, work, status, stream=s)
    p.append(0, one, pos20, x4, x1, x1, cos, cos, q4, status=status, stream=s)
    p.attn_prefix(0, q, o, one, 0, scratch, status, stream=s)
    p.release(zero, None, work, status, stream=s)
    p.compact(work, status, stream=s)
    pkg.spec_verify(pr, None, tok1, None, ua, us, tok, cnt, status, stream=s)
g.replay()
torch.cuda.synchronize()
assert status.item() == 0 and torch.isfinite(o.float()).all() and torch.isfinite(y).all() and torch.isfinite(ho.float()).all()
assert p.c.n_pages == 8
print("ok")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_captured_and_replayed(cuda, dt):
    """One graph over changing lengths, tables and slots."""
    import torch
    c = shared_cache(cuda, 256, [40, 90, 7, 64], 16, (20, 5), dt)
    q = _rand(9, 3, 1, 20, 128, dt=_dt(dt))
    out = torch.empty_like(q)
    slots = _i32([0, 1, 2])
    work = torch.empty(c.p.attn_prefix_work_bytes(3, 1, 20, 256), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.p.attn_prefix(1, q, out, slots, 256, work, c.status, stream=torch.cuda.current_stream())
    for lens, sl in (([296, 346, 263], [0, 1, 2]), ([257, 300, 256], [2, 1, 0]), ([296, 346, 263], [3, 0, 1])):
        for s, n in enumerate(lens):
            c.m.lens[s] = n
        c.lens.copy_(_i32(c.m.lens))
        slots.copy_(_i32(sl))
        q.copy_(_rand(sum(lens), *q.shape, dt=q.dtype))
        # lengths were shortened in place: the model only looks at rows below them
        keep = [min(c.m.lens[s], 256 + [40, 90, 7, 64][s]) for s in range(4)]
        c.m.lens[:4] = keep
        c.lens.copy_(_i32(c.m.lens))
        g.replay()
        torch.cuda.synchronize()
        check_prefix(c, q, out, sl, 1)
    assert c.take_status() == 0


def test_prefix_two_streams_with_their_own_workspaces(cuda):
    import torch
    a = shared_cache(cuda, 1024, [100] * 6, 16, (20, 5), "f16", seed=1)
    b = shared_cache(cuda, 512, [300] * 3, 64, (8, 1), "f16", seed=2)
    runs = []
    for c, heads, prefix, n in ((a, (20, 5), 1024, 6), (b, (8, 1), 512, 3)):
        q = _rand(n, n, 1, heads[0], 128, dt=torch.float16)
        work = torch.empty(c.p.attn_prefix_work_bytes(n, 1, heads[0], prefix), dtype=torch.uint8, device="cuda")
        runs.append((c, q, torch.empty_like(q), _i32(list(range(n))), prefix, work, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, q, out, slots, prefix, work, s in runs:
            c.p.attn_prefix(1, q, out, slots, prefix, work, c.status, stream=s)
    torch.cuda.synchronize()
    for c, q, out, slots, prefix, work, s in runs:
        check_prefix(c, q, out, slots.tolist(), 1)
        assert c.take_status() == 0


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def _probs(rng, *shape):
    x = rng.exponential(size=shape) ** 3
    return (x / x.sum(-1, keepdims=True)).astype(np.float32)


def run_verify(cuda, p, q, draft, nd, ua, us):
    import torch
    n, k1, _ = p.shape
    d = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()
    tokens = torch.full((n, k1), 77, dtype=torch.int32, device="cuda")
    count = torch.full((n,), 77, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cuda.spec_verify(d(p), d(q), d(draft), d(nd), d(ua), d(us), tokens, count, status)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), count.cpu().numpy(), int(status.item())


@pytest.mark.parametrize("n,k,V", [(1, 1, 1), (1, 1, 2), (3, 4, 5), (7, 3, 127), (5, 8, 128), (4, 2, 4096), (4, 5, 4097),
                                   (3, 64, 1000), (2, 7, 50257), (6, 4, 128256), (2, 3, 300001), (40, 1, 33)])
@pytest.mark.parametrize("point", [False, True])
def test_verify(cuda, n, k, V, point):
    rng = np.random.default_rng(n * 1000 + k * 10 + V)
    p = _probs(rng, n, k + 1, V)
    q = (0.6 * p[:, :k] + 0.4 * _probs(rng, n, k, V)).astype(np.float32)
    draft = np.array([[rng.choice(V, p=(r / r.sum()).astype(np.float64) / (r / r.sum()).astype(np.float64).sum())
                       for r in s] for s in q.astype(np.float64)], np.int32)
    nd = rng.integers(0, k + 1, n).astype(np.int32)
    ua = rng.random((n, k), np.float32) * (0.2 if point else 1.0)
    us = rng.random(n, np.float32)
    us[0] = 0.0
    if n > 1:
        us[1] = np.float32(1) - np.float32(2.0 ** -24)
    for lens in (nd, None):
        want, cnt, gap = verify(p, None if point else q, draft, lens if lens is not None else [k] * n, ua, us)
        tok, got, status = run_verify(cuda, p, None if point else q, draft, lens, ua, us)
        assert status == 0 and (got == cnt).all()
        sure = gap > 2.0 ** -52 * (V + 64)           # a border nearer than the sums' own rounding decides nothing
        sure[0] = True                               # u = 0 takes the first index with mass, exactly
        assert (tok[sure] == want[sure]).all()


def test_verify_edges(cuda):
    """Rows without mass, entries that are no numbers, equal rows, ids out of range."""
    V, k = 9, 2
    p = np.zeros((9, k + 1, V), np.float32)
    q = np.zeros((9, k, V), np.float32)
    draft = np.full((9, k), 3, np.int32)
    ua = np.full((9, k), 0.5, np.float32)
    us = np.full(9, 0.5, np.float32)
    # 0: the target has no mass at all
    # 1: accepted twice, then a draw from one entry
    p[1, :2, 3], p[1, 2, 5] = 1.0, 1.0
    q[1, :, 3] = 1.0
    # 2: refused, p below q everywhere: the residual has no mass, p stands in
    p[2, 0, 3:5] = 0.25
    q[2, 0, 3:5] = 0.75
    # 3: NaN, infinities and negatives count as nothing
    p[3, 0] = [np.nan, np.inf, -1.0, 0.0, 0.5, -np.inf, 0.0, 0.0, 0.0]
    q[3, 0, 3] = 1.0
    # 4: a NaN where the draft's token is
    p[4, 0, 3], p[4, 0, 6] = np.nan, 0.125
    q[4, 0, 3] = 1.0
    # 5, 6: ids out of range are refused
    draft[5, 0], draft[6, 0] = V, -1
    p[5:7, 0, :] = 1.0 / V
    # 7: u just below and at the ratio: q = 1, p = 0.5, u = 0.5 is refused
    p[7, 0, 3], p[7, 0, 8] = 0.5, 0.5
    q[7, 0, 3] = 1.0
    # 8: mass only behind the last border
    p[8, 0, V - 1] = 1e-30
    q[8, 0, 3] = 1.0
    for qq in (q, None):
        want, cnt, _ = verify(p, qq, draft, [k] * 9, ua, us)
        tok, got, status = run_verify(cuda, p, qq, draft, None, ua, us)
        assert status == -1 and (got == cnt).all() and (tok == want).all(), (tok, want)
    assert tok[0, 0] == -1
    # lengths out of range are clamped
    want, cnt, _ = verify(p[:2], q[:2], draft[:2], [2, 0], ua[:2], us[:2])
    tok, got, status = run_verify(cuda, p[:2], q[:2], draft[:2], np.array([99, -4], np.int32), ua[:2], us[:2])
    assert status == -1 and (got == cnt).all() and (tok == want).all()
    # uniforms outside [0, 1) stay inside the row
    for u in (np.nan, 2.0, -1.0, np.inf):
        tok, got, _ = run_verify(cuda, p[1:2], q[1:2], draft[1:2], None, ua[1:2], np.full(1, u, np.float32))
        assert tok[0].tolist() == [3, 3, 5]


def test_verify_unaligned_rows_and_graph(cuda):
    """A view that starts 4 bytes into a buffer; a captured call on new inputs."""
    import torch
    n, k, V = 3, 2, 1028
    rng = np.random.default_rng(4)
    buf = torch.empty(n * (k + 1) * V + 1, device="cuda")
    p = buf[1:].view(n, k + 1, V)
    q = torch.empty(n, k, V, device="cuda")
    draft = torch.zeros(n, k, dtype=torch.int32, device="cuda")
    ua, us = torch.rand(n, k, device="cuda"), torch.rand(n, device="cuda")
    tokens = torch.empty(n, k + 1, dtype=torch.int32, device="cuda")
    count = torch.empty(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cuda.spec_verify(p, q, draft, None, ua, us, tokens, count, stream=torch.cuda.current_stream())
    for _ in range(3):
        ph, qh = _probs(rng, n, k + 1, V), _probs(rng, n, k, V)
        dh = rng.integers(0, V, (n, k)).astype(np.int32)
        p.copy_(torch.from_numpy(ph))
        q.copy_(torch.from_numpy(qh))
        draft.copy_(torch.from_numpy(dh))
        g.replay()
        torch.cuda.synchronize()
        want, cnt, _ = verify(ph, qh, dh, [k] * n, ua.cpu().numpy(), us.cpu().numpy())
        assert (tokens.cpu().numpy() == want).all() and (count.cpu().numpy() == cnt).all()


# ---------------------------------------------------------------------------
# a run of them together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_a_serving_loop(cuda, synth, dt):
    """A layer's Q/K/V products of a prompt, its attention and its cache; three
    samples forked from it; two steps of drafted tokens scored over the shared
    prefix, verified, and the refused ones released. Every step's attention is
    held against the 64-bit form on the tokens that the cache should hold."""
    import torch
    H, Hkv, E, page = 8, 2, 1024, 16
    rng = np.random.default_rng(8)
    w = [torch.from_numpy(synth.random_i2s(rng, r * 128, E)).cuda() for r in (H, Hkv, Hkv)]
    cos, sin = (torch.from_numpy(x).cuda() for x in cuda.rope_table(256, 500000.0))
    c = Cache(cuda, 80, 5, 14, page, 1, Hkv, dt)

    def project(x):
        m = x.shape[0]
        q8 = torch.empty(m, E, dtype=torch.int8, device="cuda")
        acts = torch.empty(m, 2, dtype=torch.int32, device="cuda")
        cuda.quant_act_rows(x, m, E, q8, acts)
        ys = []
        for t, h in zip(w, (H, Hkv, Hkv)):
            y = torch.empty(m, h, 128, device="cuda")
            cuda.gemm(t, h * 128, E, m, q8, acts, y=y)
            ys.append(y / 40.0)
        return ys

    def append(x, slot, pos):
        m = x.shape[0]
        q, k, v = project(x)
        outs = [torch.empty(m, h, 128, dtype=_dt(dt), device="cuda") for h in (H, Hkv, Hkv)]
        c.p.append(0, _i32(slot), _i32(pos), q, k, v, cos, sin, *outs, c.status)
        return outs

    n0 = 5 * page + 11
    c.m.reserve([0], [n0])
    c.p.reserve(_i32([0]), _i32([n0]), c.work, c.status)
    c.same()
    q, k, v = append(_rand(1, n0, E), [0] * n0, list(range(n0)))
    o = torch.empty(n0, H, 128, device="cuda")
    cuda.attn_prompt(q, k, v, o, _i32([0, n0]))
    torch.cuda.synchronize()
    check_prompt(q, k, v, o, [n0], dt == "f16")
    assert torch.equal(c.rows(0)[:, 0], k) and torch.equal(c.rows(0, c.v)[:, 0], v)

    kids = [1, 2, 3]
    c.m.fork([0] * 3, kids)
    c.p.fork(_i32([0] * 3), _i32(kids), c.work, c.status)
    truth = {s: (k.clone(), v.clone()) for s in kids}
    for step in range(2):
        nd = 3
        x = _rand(10 + step, 3 * nd, E)
        old = [c.m.lens[s] for s in kids]
        c.m.reserve(kids, [nd] * 3)
        c.p.reserve(_i32(kids), _i32([nd] * 3), c.work, c.status)
        qs, ks, vs = append(x, [s for s in kids for _ in range(nd)], [n + j for n in old for j in range(nd)])
        for i, s in enumerate(kids):
            truth[s] = tuple(torch.cat([a, b[i * nd:(i + 1) * nd]]) for a, b in zip(truth[s], (ks, vs)))
        prefix = n0 // page * page
        qq = qs.view(3, nd, H, 128)
        out = torch.empty(3, nd, H, 128, device="cuda")
        work = torch.empty(c.p.attn_prefix_work_bytes(3, nd, H, prefix), dtype=torch.uint8, device="cuda")
        c.p.attn_prefix(0, qq, out, _i32(kids), prefix, work, c.status)
        c.same()
        for s in kids:
            assert torch.equal(c.rows(s)[:, 0], truth[s][0]) and torch.equal(c.rows(s, c.v)[:, 0], truth[s][1])
        check_prefix(c, qq, out, kids, 0)
        V = 500
        p, qp = _probs(rng, 3, nd + 1, V), _probs(rng, 3, nd, V)
        draft = rng.integers(0, V, (3, nd)).astype(np.int32)
        ua, us = rng.random((3, nd), np.float32), rng.random(3, np.float32)
        want, cnt, _ = verify(p, qp, draft, [nd] * 3, ua, us)
        tok, got, status = run_verify(cuda, p, qp, draft, None, ua, us)
        assert status == 0 and (tok == want).all() and (got == cnt).all()
        keep = [n + min(int(g), nd) for n, g in zip(old, got)]
        c.m.release(kids, keep)
        c.p.release(_i32(kids), _i32(keep), c.work, c.status)
        for s, n in zip(kids, keep):
            truth[s] = tuple(a[:n] for a in truth[s])
    c.m.release([0], None)
    c.p.release(_i32([0]), None, c.work, c.status)
    c.m.compact()
    c.p.compact(c.work, c.status)
    c.same()
    for s in kids:
        assert torch.equal(c.rows(s)[:, 0], truth[s][0]) and torch.equal(c.rows(s, c.v)[:, 0], truth[s][1])
    assert c.take_status() == 0
