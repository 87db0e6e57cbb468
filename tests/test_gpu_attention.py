"""The attention operators where rounding, masks and limits meet: against the
64-bit forms of serving_ref.py, whose bounds are derived there."""
import math

import numpy as np
import pytest

from serving_ref import attention, attention_bound
from test_gpu_serving import Cache, _dt, _i32, _rand, check_prefix, run_prefix, shared_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# weights far below the largest one
# ---------------------------------------------------------------------------
def _beside_a_large_one(k, v):
    """Keys whose scores lie about 18 below the first one's (queries of mean 1),
    which has a value of zero: what comes out is the small weights' sum."""
    k *= 0.3
    k[0], v[0] = 1.6, 0.0


def _check_small(q, k, v, out, limit):
    # the f16 bound, with the weights' subnormal unit a 2^-7 of the one that a
    # maximum of 1 would have: 2^-32 instead of 2^-25
    o, pv, big, va = attention(q.double(), k.double(), v.double(), limit)
    tol = attention_bound(o, pv, big, va * 2.0 ** -7, k.shape[0], True, False)
    assert bool((o.abs() > tol).any())              # without the small weights, zeros would come out
    err = (out.double() - o).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("n", [100, 700])
def test_prompt_small_weights(cuda, n):
    """An attention sink: weights of 2^-26 beside one of 1, in f16."""
    import torch
    q, k, v = (_rand(s, n, 2, 128, dt=torch.float16) for s in (1, 2, 3))
    q.mul_(0.5).add_(1.0)
    _beside_a_large_one(k, v)
    out = torch.empty(n, 2, 128, device="cuda")
    cuda.attn_prompt(q, k, v, out, _i32([0, n]))
    torch.cuda.synchronize()
    for h in range(2):
        _check_small(q[:, h], k[:, h], v[:, h], out[:, h], torch.arange(1, n + 1, device="cuda"))


@pytest.mark.parametrize("prefix,own", [(0, 300), (512, 100)])
def test_prefix_small_weights(cuda, prefix, own):
    """... over a paged cache: the large weight in one part, small ones in all."""
    import torch
    c = shared_cache(cuda, prefix, [own, own + 7], 16, (4, 1), "f16")
    for s in (0, 1):
        first = c.m.tables[s][0]
        if s == 0 or prefix == 0:
            c.k[first, :, :, 0], c.v[first, :, :, 0] = 1.6, 0.0
    mask = torch.ones_like(c.k[:, :1, :1, :, :1], dtype=torch.bool)
    for s in (0, 1):
        mask[c.m.tables[s][0], :, :, 0] = False
    c.k[:] = torch.where(mask, c.k * 0.3, c.k)
    n, nq, H = 2, 1, 4
    q = _rand(5, n, nq, H, 128, dt=torch.float16).mul_(0.5).add_(1.0)
    out = torch.empty(n, nq, H, 128, device="cuda")
    work = torch.empty(c.p.attn_prefix_work_bytes(n, nq, H, prefix), dtype=torch.uint8, device="cuda")
    c.p.attn_prefix(1, q, out, _i32([0, 1]), prefix, work, c.status)
    torch.cuda.synchronize()
    assert c.take_status() == 0
    for b in range(2):
        k, v = c.rows(b)[:, 1, 0], c.rows(b, c.v)[:, 1, 0]
        _check_small(q[b, 0], k, v, out[b, 0], torch.full((H,), c.m.lens[b], device="cuda"))


# ---------------------------------------------------------------------------
# values that are no numbers
# ---------------------------------------------------------------------------
def test_prompt_unseen_value_beside_a_score_of_minus_infinity(cuda):
    """A key whose score is -inf has weight 0, whether or not a later token
    that the row does not see holds a NaN."""
    import torch
    n = 150
    q, k, v = (_rand(s, n, 2, 128, dt=torch.float16) for s in (1, 2, 3))
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    k[0, :, 5] = -math.inf
    out = [torch.empty(n, 2, 128, device="cuda") for _ in range(2)]
    cuda.attn_prompt(q, k, v, out[0], _i32([0, n]))
    v[n - 1] = math.nan
    cuda.attn_prompt(q, k, v, out[1], _i32([0, n]))
    torch.cuda.synchronize()
    rows = torch.arange(1, n - 1, device="cuda")            # row i of the keys 1 .. i
    for o in out:
        for h in range(2):
            want, pv, big, va = attention(q[rows, h].double(), k[1:n - 1, h].double(), v[1:n - 1, h].double(), rows)
            err = (o[rows, h].double() - want).abs()
            tol = attention_bound(want, pv, big, va, n, True, False)
            assert bool((err <= tol).all()), float((err / tol).nan_to_num(math.inf).max())
    assert bool(torch.isnan(out[1][n - 1]).all())


ODD = [  # token of the 300, dimension, what stands there
    (3, 7, math.inf), (70, 7, -math.inf), (70, 9, math.nan), (130, 0, -math.inf), (131, 127, math.inf), (255, 64, math.nan),
    (256, 31, math.inf), (299, 100, math.nan)]


@pytest.mark.parametrize("types", [("f32", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("heads", [(2, 1), (3, 3)])
def test_prompt_odd_values_one_by_one(cuda, types, heads):
    """Single values that are no numbers, in the tiles that a causal mask cuts
    and before them: a row that sees one has no number in that dimension, and
    everything else is bit for bit as with zeros in those places."""
    import torch
    n, (H, Hkv) = 300, heads
    q, k, v = (_rand(s, n + 5, h, 128, dt=_dt(types[0])) for s, h in ((1, H), (2, Hkv), (3, Hkv)))
    for t, d, _ in ODD:
        v[5 + t, :, d] = 0.0
    cu = _i32([0, 5, n + 5])
    out = [torch.empty(n + 5, H, 128, dtype=_dt(types[1]), device="cuda") for _ in range(2)]
    cuda.attn_prompt(q, k, v, out[0], cu)
    for t, d, x in ODD:
        v[5 + t, :, d] = x
    cuda.attn_prompt(q, k, v, out[1], cu)
    torch.cuda.synchronize()
    mask = torch.zeros(n + 5, H, 128, dtype=torch.bool, device="cuda")
    for t, d, x in ODD:
        mask[5 + t:, :, d] = True
    assert torch.equal(torch.where(mask, 0.0, out[0]), torch.where(mask, 0.0, out[1]))
    assert not bool(torch.isfinite(out[1][mask]).any())
    # the first rows that see one hold the value itself; both infinities make no number
    got = out[1][5:].float()
    for t, d, x in ODD:
        if (t, d) == (70, 7):
            assert bool((got[60:70, :, 7] == math.inf).all()) and bool(torch.isnan(got[70:128, :, 7]).all())
        elif math.isnan(x):
            assert bool(torch.isnan(got[t:, :, d]).all())
        elif t % 128 > 0:               # (a value that all rows of a tile see meets the weights' planes: inf or NaN)
            assert bool((got[t, :, d] == x).all())


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("prefix,owns,page,heads,nq", [(128, [5, 37, 64, 131], 64, (8, 2), 4), (0, [3, 130, 16], 16, (64, 1), 8),
                                                       (64, [129, 9], 32, (256, 1), 3)])
def test_prefix_odd_values_one_by_one(cuda, dt, prefix, owns, page, heads, nq):
    """... in the drafted tokens that only some of a sequence's queries see."""
    import torch
    c = shared_cache(cuda, prefix, owns, page, heads, dt)
    slots = list(range(len(owns)))
    put = []
    for s in slots:
        n = c.m.lens[s]
        for back, d in ((1, 3), (1, 90), (2, 64), (nq, 5)):
            if back <= owns[s]:
                pg = c.m.tables[s][(n - back) // page]
                put.append((s, back, d, pg, (n - back) % page))
    for s, back, d, pg, r in put:
        c.v[pg, :, :, r, d] = 0.0
    q, a = run_prefix(cuda, c, slots, nq, heads, prefix, "f32")
    check_prefix(c, q, a, slots, 1)
    for s, back, d, pg, r in put:
        c.v[pg, :, :, r, d] = math.nan if d == 90 else math.inf
    _, b = run_prefix(cuda, c, slots, nq, heads, prefix, "f32")
    assert c.take_status() == 0
    mask = torch.zeros_like(a, dtype=torch.bool)
    for s, back, d, pg, r in put:
        mask[s, nq - back:, :, d] = True
    assert torch.equal(torch.where(mask, 0.0, a), torch.where(mask, 0.0, b))
    assert not bool(torch.isfinite(b[mask]).any())
    assert bool(torch.isnan(b[:, :, :, 90][mask[:, :, :, 90]]).all())


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_odd_value_of_a_vanishing_part(cuda, dt):
    """Scores of the own tokens 250 below the prefix's, so that their part weighs
    e^-250: 0 in 32 bits, but an infinity among its values is still one."""
    import torch
    c = shared_cache(cuda, 256, [40, 70], 16, (4, 2), dt)
    c.k *= 0.1
    c.k[c.m.tables[0][0], :, :, 5] = 22.0
    q = _rand(3, 2, 2, 4, 128, dt=_dt(dt), scale=0.1).add_(1.0)
    for s in (0, 1):
        n = c.m.lens[s]
        c.v[c.m.tables[s][(n - 1) // 16], :, :, (n - 1) % 16, 9] = math.inf
        c.v[c.m.tables[s][(n - 7) // 16], :, :, (n - 7) % 16, 70] = math.nan
    out = torch.empty(2, 2, 4, 128, device="cuda")
    work = torch.empty(c.p.attn_prefix_work_bytes(2, 2, 4, 256), dtype=torch.uint8, device="cuda")
    c.p.attn_prefix(1, q, out, _i32([0, 1]), 256, work, c.status)
    torch.cuda.synchronize()
    assert c.take_status() == 0
    assert not bool(torch.isfinite(out[:, 1, :, 9]).any()) and bool(torch.isfinite(out[:, 0, :, 9]).all())
    assert bool(torch.isnan(out[:, :, :, 70]).all())
    v = c.v[c.m.tables[0][0], 1, :, 5].float().repeat_interleave(2, 0)      # the one key that counts
    rest = [d for d in range(128) if d not in (9, 70)]
    assert float((out - v)[..., rest].abs().max()) < 1e-3


def test_prompt_odd_value_at_the_end_of_a_long_sequence(cuda):
    """No work grows with the sequence where a value is no number: no bounded
    wait runs out, and the rows before it are those of the run without it."""
    import torch
    n = 1 << 18
    q, k, v = (_rand(s, n, 1, 128, dt=torch.float16) for s in (1, 2, 3))
    out = [torch.empty(n, 1, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    cuda.attn_prompt(q, k, v, out[0], _i32([0, n]))
    v[n - 2] = math.inf
    cuda.attn_prompt(q, k, v, out[1], _i32([0, n]))
    torch.cuda.synchronize()
    assert cuda.attn_error() == 0
    assert torch.equal(out[0][:n - 2], out[1][:n - 2]) and not bool(torch.isfinite(out[1][n - 2:]).any())
    rows = torch.tensor([0, 127, 128, 5000, n - 3], device="cuda")
    want, pv, big, va = attention(q[rows, 0].double(), k[:, 0].double(), torch.where(v.isinf(), 0.0, v)[:, 0].double(), rows + 1)
    assert bool(((out[1][rows, 0].double() - want).abs() <= attention_bound(want, pv, big, va, n, True, True)).all())


def test_prefix_odd_value_behind_a_long_context(cuda):
    """... and in a drafted token behind a long context that is one item a
    kv head, since the sequences fill the device."""
    import torch
    page, n, heads, L, nq = 128, 40, (8, 8), 131072, 4
    c = Cache(cuda, L // page + 1, n, L // page, page, 1, heads[1], "f16")
    c.m.tables = [list(range(L // page)) for _ in range(n)]
    c.m.lens = [L] * n
    c.m.refs = [n] * (L // page) + [0]
    c.push()
    q, a = run_prefix(cuda, c, list(range(n)), nq, heads, 0, "f16", layer=0)
    last = c.m.tables[0][-1]
    c.v[last, :, :, page - 1] = math.nan
    _, b = run_prefix(cuda, c, list(range(n)), nq, heads, 0, "f16", layer=0)
    assert c.take_status() == 0
    assert torch.equal(a[:, :3], b[:, :3]) and bool(torch.isnan(b[:, 3]).all())
    for h in (0, 7):
        k, v = c.k[:L // page, 0, h].reshape(-1, 128).double(), c.v[:L // page, 0, h].reshape(-1, 128).double()
        v[-1] = 0.0
        lim = torch.tensor([L - 3, L - 2, L - 1], device="cuda")
        want, pv, big, va = attention(q[5, :3, h].double(), k, v, lim)
        assert bool(((b[5, :3, h].double() - want).abs() <= attention_bound(want, pv, big, va, L, True, True)).all())


def test_f32_values_next_to_the_largest(cuda):
    """f32 counts as infinite from where bf16 would round it to that, 2^128 -
    2^119, on; below, all 24 bits count."""
    import torch
    q, k, v = (_rand(s, 1, 1, 128) for s in (1, 2, 3))
    big = float.fromhex("0x1.fefffep127")
    v[0, 0, ::3], v[0, 0, 1::3] = big, float.fromhex("-0x1.fe8002p127")
    out = torch.empty_like(q)
    cuda.attn_prompt(q, k, v, out, _i32([0, 1]))
    torch.cuda.synchronize()
    # one key: the value itself, its planes and the sum's last bits cut
    assert bool(((out.double() - v.double()).abs() <= v.double().abs() * 4 * 2.0 ** -24).all())


# ---------------------------------------------------------------------------
# what is reported
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prompt_reports_wrong_offsets(cuda, dt):
    """Offsets that descend or leave the arrays, in *status; right ones, empty
    sequences and a last one below the array's end among them, leave it alone."""
    import torch
    n = 100
    q, k, v = (_rand(s, n, 2, 128, dt=_dt(dt)) for s in (1, 2, 3))
    out, status = torch.empty_like(q), _i32([0])
    for cu in ([0, 100], [0, 0, 40, 40, 99], [7, 100], [0] * 700 + [100] * 700):
        cuda.attn_prompt(q, k, v, out, _i32(cu), status=status)
        assert status.item() == 0, cu
    for cu in ([0, 101], [-1, 100], [60, 20], [0, 100, 50, 100], [0] * 700 + [100] * 700 + [99], [2 ** 31 - 1, -2 ** 31]):
        status.zero_()
        cuda.attn_prompt(q, k, v, out, _i32(cu), status=status)
        assert status.item() == -1, cu
    with pytest.raises(cuda.SllmCudaError, match="status"):
        cuda.attn_prompt(q, k, v, out, _i32([0, 100]), status=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_a_wait_that_runs_out_is_reported(cuda, dt):
    """With a limit of 1 ns every real wait runs out: the kernels end, *status
    and the error word say so, and the next calls are as good as ever."""
    import torch
    n = 1500
    q, k, v = (_rand(s, n, 4, 128, dt=_dt(dt)) for s in (1, 2, 3))
    cu, status, ref, out = _i32([0, 300, n]), _i32([0]), torch.empty_like(q), torch.empty_like(q)
    c = shared_cache(cuda, 1024, [300] * 3, 16, (20, 5), dt)
    cuda.attn_prompt(q, k, v, ref, cu, status=status)
    _, a = run_prefix(cuda, c, [0, 1, 2], 2, (20, 5), 1024, dt)
    assert status.item() == 0 and c.take_status() == 0 and cuda.attn_error() == 0
    cuda.set_attn_wait(1)
    try:
        cuda.attn_prompt(q, k, v, out, cu, status=status)
        run_prefix(cuda, c, [0, 1, 2], 2, (20, 5), 1024, dt)
        cuda.attn_prompt(q, k, v, out, cu)              # nobody asks
        torch.cuda.synchronize()
    finally:
        cuda.set_attn_wait(0)
    assert status.item() == -61 and c.take_status() == -61
    assert cuda.attn_error() != 0
    cuda.attn_error()                                   # (one word per file)
    status.zero_()
    cuda.attn_prompt(q, k, v, out, cu, status=status)
    _, b = run_prefix(cuda, c, [0, 1, 2], 2, (20, 5), 1024, dt)
    assert status.item() == 0 and c.take_status() == 0 and cuda.attn_error() == 0
    assert torch.equal(out, ref) and torch.equal(a, b)


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_prefix_workspace_of_the_largest_call_serves_the_smaller(cuda, dt):
    """Sequences end one after the other, and the prefix gets shorter, in one
    workspace of the first call's size; what lies behind it stays."""
    import torch
    heads, prefix, n = (8, 1), 4096, 21
    c = shared_cache(cuda, prefix, [1 + 9 * i for i in range(n)], 16, heads, dt)
    size = c.p.attn_prefix_work_bytes(n, 2, heads[0], prefix)
    work = torch.full((size + 4096,), 77, dtype=torch.uint8, device="cuda")
    for m, nq, pre in ((21, 2, 4096), (20, 2, 4096), (20, 1, 4096), (13, 2, 2048), (7, 1, 1792), (3, 2, 16), (1, 1, 0)):
        q = _rand(m, m, nq, heads[0], 128, dt=_dt(dt), scale=1.3)
        out = torch.empty(m, nq, heads[0], 128, device="cuda")
        slots = list(range(n - m, n))
        c.p.attn_prefix(1, q, out, _i32(slots), pre, work[:size], c.status)
        torch.cuda.synchronize()
        assert c.take_status() == 0
        check_prefix(c, q, out, slots, 1, skip=range(1, m - 1))
    assert bool((work[size:] == 77).all())


# ---------------------------------------------------------------------------
# f32 inputs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 17, 64, 129, 700, 4100])
def test_prompt_f32_is_as_good_as_32_bits(cuda, n):
    import torch
    from precision_ref import as_good_as_32_bits
    q, k, v = (_rand(s, n + 3, h, 128, scale=1.3) for s, h in ((1, 4), (2, 2), (3, 2)))
    out = torch.empty_like(q)
    cuda.attn_prompt(q, k, v, out, _i32([0, 3, n + 3]))
    torch.cuda.synchronize()
    for h in range(4):
        x = q[3:, h], k[3:, h // 2], v[3:, h // 2], torch.arange(1, n + 1, device="cuda")
        if n == 1:                              # one key: the value, its bits cut at most four times
            assert bool(((out[3:, h] - x[2]).abs() <= x[2].abs() * 2.0 ** -22).all())
            continue
        big, rms = as_good_as_32_bits(out[3:, h], *x)
        assert big <= 3 and rms <= 3, (h, big, rms)


@pytest.mark.parametrize("prefix,owns,nq,heads", [(0, [64, 9], 1, (20, 5)), (0, [4100], 2, (8, 1)), (256, [40, 130], 4, (8, 2)),
                                                  (4096, [700, 33, 5], 1, (8, 1)), (64, [600], 1, (256, 1))])
def test_prefix_f32_is_as_good_as_32_bits(cuda, prefix, owns, nq, heads):
    import torch
    from precision_ref import as_good_as_32_bits
    c = shared_cache(cuda, prefix, owns, 16, heads, "f32")
    slots = list(range(len(owns)))
    q, out = run_prefix(cuda, c, slots, nq, heads, prefix, "f32")
    assert c.take_status() == 0
    group = heads[0] // heads[1]
    for b in slots:
        L = c.m.lens[b]
        for g in range(heads[1]):
            rows = slice(g * group, (g + 1) * group)
            lim = torch.tensor([L - nq + 1 + j for j in range(nq)], device="cuda")
            lim = lim[:, None].expand(nq, group).reshape(-1)
            x = (q[b, :, rows].reshape(-1, 128), c.rows(b)[:, 1, g], c.rows(b, c.v)[:, 1, g], lim)
            big, rms = as_good_as_32_bits(out[b, :, rows].reshape(-1, 128), *x)
            assert big <= 3 and rms <= 3, (b, g, big, rms)


def test_prompt_one_long_sequence_among_very_many(cuda):
    """The search for the next item passes over positions that the same
    sequences reach: the others wait behind it (7 ms; 256 ms when it walked all
    sequences once for each of the long one's tiles)."""
    import torch
    short, long = 8, 1 << 17
    lens = [short] * 60000 + [long] + [0, short] * 2767 + [1]
    T, at = sum(lens), short * 60000
    q, k, v = (_rand(s, T, 1, 128, dt=torch.float16) for s in (1, 2, 3))
    out, status = torch.empty_like(q), _i32([0])
    cu = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
    ms = []
    for _ in range(3):
        out.fill_(7.0)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        cuda.attn_prompt(q, k, v, out, cu, status=status)
        b.record()
        torch.cuda.synchronize()
        ms.append(a.elapsed_time(b))
    assert status.item() == 0 and cuda.attn_error() == 0
    # the short ones all at once, the long one's rows here and there
    n = T - long
    keep = torch.cat([torch.arange(at, device="cuda"), torch.arange(at + long, T, device="cuda")])[:n - 1].view(-1, short)
    qq, kk, vv = (t[keep, 0].double() for t in (q, k, v))
    s = (qq @ kk.transpose(1, 2) / math.sqrt(128.0)).masked_fill(torch.ones(short, short, device="cuda").triu(1).bool(), -math.inf)
    want = torch.softmax(s, -1) @ vv
    assert float((out[keep, 0].double() - want).abs().max()) < 0.01     # (another sequence's keys would be off by about 1)
    assert torch.equal(out[-1], v[-1])
    rows = torch.tensor([0, 255, 256, 70000, long - 1], device="cuda")
    x = (k[at:at + long, 0].double(), v[at:at + long, 0].double())
    want, pv, big, va = attention(q[at + rows, 0].double(), *x, rows + 1)
    assert bool(((out[at + rows, 0].double() - want).abs() <= attention_bound(want, pv, big, va, long, True, True)).all())
    assert min(ms) < 60.0, ms
