"""Beam selection on a GPU against its definition in 64 bits, and a beam search
over an 8-bit cache step by step."""
import math

import numpy as np
import pytest

from kv8_ref import Cache8, beam_select

pytestmark = pytest.mark.gpu


def _i32(a):
    import torch
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def run(cuda, logits, score, done=None, eos=-1, slots=None):
    """Returns (parents, tokens, scores, done, src, status) as numpy."""
    import torch
    n, B, _ = logits.shape
    f = lambda dt: torch.full((n, B), 77, dtype=dt, device="cuda")
    so, pa, to = f(torch.float32), f(torch.int32), f(torch.int32)
    do = f(torch.int32) if eos >= 0 else None
    src = f(torch.int32) if slots is not None else None
    st = _i32([0])
    cuda.beam_select(logits, score, so, pa, to, done=done, eos=eos, done_out=do, slots=slots, src=src, status=st)
    torch.cuda.synchronize()
    return [None if x is None else x.cpu().numpy() for x in (pa, to, so, do, src, st)]


def check(cuda, logits, score, done=None, eos=-1, status=0):
    """Whole values are equal, unless candidates of two beams lie within the 32-bit exponentials' error of the
    sums (then either order is right); scores to that error and the rounding to 32 bits."""
    import torch
    n, B, V = logits.shape
    slots = torch.arange(n * B, dtype=torch.int32, device="cuda").flip(0).contiguous()
    pa, to, so, do, src, st = run(cuda, logits, score, done, eos, slots)
    assert st[0] == status
    L, S = logits.cpu().numpy(), score.double().cpu().numpy()
    D = None if done is None else done.cpu().numpy()
    for i in range(n):
        want, near, every = beam_select(L[i], S[i], None if D is None else D[i], eos, B)
        vals = [c[0] for c in near]
        # a term's argument is rounded (2^-24 of up to 2^7), its exponential off by two units, sums by two more
        tol = 2.0 ** -16 * 1.01
        # ties inside one beam are exact (same sum); those between beams are not asked about
        clear = all(a[1] == b[1] or a[0] - b[0] > 2 * tol or (a[0] == b[0]) for a, b in zip(near, near[1:]))
        if clear:
            assert pa[i].tolist() == [c[1] for c in want] and to[i].tolist() == [c[3] for c in want], i
        else:                                                # each word once, and of the value that its place has
            assert len(set(zip(pa[i].tolist(), to[i].tolist()))) == B
            want = [next(c for c in every if (c[1], c[3]) == pt) for pt in zip(pa[i].tolist(), to[i].tolist())]
            assert all(abs(c[0] - d[0]) <= 2 * tol for c, d in zip(want, near))
        for j, c in enumerate(want):
            if c[0] == -math.inf:
                assert so[i, j] == -math.inf
            else:
                assert abs(float(so[i, j]) - c[0]) <= tol + abs(c[0]) * 2.0 ** -23
            assert src[i, j] == int(slots[i * B + c[1]])
            if eos >= 0:
                assert do[i, j] == (1 if c[3] == eos or (D is not None and D[i, c[1]]) else 0)


def _logits(seed, n, B, V, scale=2.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, B, V), generator=g, device="cuda") * scale


def _scores(seed, n, B):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    return torch.randn((n, B), generator=g, device="cuda") * 1.5 - 12


@pytest.mark.parametrize("B", [1, 2, 3, 4, 5, 8, 11, 16])
@pytest.mark.parametrize("V", [1, 2, 5, 17, 50, 255, 1000, 2047, 4096, 8193, 20001, 32000])
def test_select(cuda, B, V):
    n = 3
    check(cuda, _logits(V + B, n, B, V), _scores(B, n, B))


@pytest.mark.parametrize("n,B,V", [(1, 4, 128256), (2, 16, 128256), (33, 2, 50257), (300, 3, 700), (1, 1, 1 << 20), (5, 8, 262144)])
def test_select_sizes(cuda, n, B, V):
    check(cuda, _logits(n + V, n, B, V), _scores(n, n, B))


@pytest.mark.parametrize("n,B,V", [(65536, 1, 3), (20000, 2, 2), (4, 16, 1 << 20)])
def test_select_limits(cuda, n, B, V):
    check(cuda, _logits(n + V, n, B, V), _scores(n, n, B))


@pytest.mark.parametrize("V", [40, 3001, 40000])
def test_done_beams(cuda, V):
    """Finished beams stay with their own score; all of them; one among others; of score -inf."""
    import torch
    n, B = 6, 4
    lg, sc = _logits(V, n, B, V), _scores(3, n, B)
    sc[1] += torch.tensor([9.0, 0.0, -3.0, 0.0], device="cuda")
    sc[5, 2] = -math.inf
    done = _i32([[0, 1, 0, 0], [1, 0, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0], [1, 0, 1, 0], [1, 1, 1, 1]])
    check(cuda, lg, sc, done, eos=V // 2)
    check(cuda, lg, sc, None, eos=0)


@pytest.mark.parametrize("V", [30, 1500, 40000])
def test_first_step_and_forbidden_words(cuda, V):
    """Scores of -inf (only the first beam counts yet), words of -inf, beams without a word, and so few
    candidates that some of value -inf are chosen, lowest first."""
    import torch
    n, B = 7, 5
    lg, sc = _logits(V, n, B, V), _scores(5, n, B)
    sc[0, 1:] = -math.inf
    sc[1] = -math.inf
    lg[2, :, 3:] = -math.inf
    lg[3] = -math.inf
    lg[4, 1:] = -math.inf
    lg[4, 0, 4:] = -math.inf
    lg[5, :, ::2] = -math.inf
    lg[6, :, :V - 2] = -math.inf
    check(cuda, lg, sc)
    done = _i32([[0, 0, 1, 0, 0]] * n)
    check(cuda, lg, sc, done, eos=V - 1)


def test_equal_logits(cuda):
    """Words of equal logits come out lowest first; the lists overflow; beams of equal rows and scores tie."""
    import torch
    for V in (20, 700, 9000, 70000):
        lg = torch.zeros((2, 4, V), device="cuda")
        sc = torch.tensor([[-1.0, -1.0, -1.0, -1.0], [-3.0, -1.0, -2.0, -1.0]], device="cuda")
        check(cuda, lg, sc)
        lg[:, :, V // 2:] = 1.0
        check(cuda, lg, sc)
    lg = _logits(3, 1, 1, 30000).repeat(2, 6, 1)
    check(cuda, lg, torch.full((2, 6), -4.0, device="cuda"))


def test_values_that_are_no_numbers(cuda):
    """NaN and +inf count as -inf, and are reported."""
    import torch
    lg, sc = _logits(1, 3, 3, 5000), _scores(1, 3, 3)
    lg[0, 1, 77], lg[1, 0, 4999], lg[1, 2] = math.nan, math.inf, math.nan
    check(cuda, lg, sc, status=-1)
    lg, sc = _logits(1, 2, 3, 5000), _scores(1, 2, 3)
    sc[0, 1], sc[1, 2] = math.nan, math.inf
    check(cuda, lg, sc, status=-1)


def test_large_and_small_values(cuda):
    import torch
    lg, sc = _logits(8, 3, 4, 9000), _scores(1, 3, 4)
    lg[0] *= 40.0
    lg[1] += 3000.0
    lg[2] -= 3000.0
    check(cuda, lg, sc)


@pytest.mark.parametrize("V,stride", [(1000, 1003), (40000, 40004), (40001, 40010)])
def test_rows_apart(cuda, V, stride):
    base = _logits(4, 3, 4, stride)
    base[:, :, V:] = 1e9                                     # what lies between rows is never a word
    check(cuda, base[:, :, :V], _scores(1, 3, 4))


def test_captured(cuda):
    import torch
    lg, sc = _logits(4, 2, 4, 30000), _scores(1, 2, 4)
    so, pa, to = torch.empty((2, 4), device="cuda"), _i32([[0] * 4] * 2), _i32([[0] * 4] * 2)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        cuda.beam_select(lg, sc, so, pa, to, stream=s)
    for seed in (10, 11):
        lg.copy_(_logits(seed, 2, 4, 30000))
        g.replay()
        torch.cuda.synchronize()
        want = run(cuda, lg, sc)
        assert np.array_equal(pa.cpu().numpy(), want[0]) and np.array_equal(to.cpu().numpy(), want[1])
        assert np.array_equal(so.cpu().numpy(), want[2])


def test_beam_search_over_an_8_bit_cache(cuda):
    """A search of four beams for two requests, all operators as a server calls them: a toy model whose keys,
    values and logits come from its tokens. The host searches with lists of tokens and exact attention over
    the values that the device's cache holds; the chosen tokens, the tables' meaning and the scores agree."""
    import torch
    from test_gpu_kv8 import Eight, attn8_bound
    from serving_ref import attention
    n, B, V, Hkv, H, page, steps = 2, 4, 300, 2, 8, 16, 24
    S = n * B
    c = Eight(cuda, 64, S, 6, page, 1, Hkv)
    r = np.random.default_rng(5)
    emb = r.standard_normal((V, H + 2 * Hkv, 128)).astype(np.float32)
    head = (r.standard_normal((H * 128, V)) * 0.12).astype(np.float32)
    demb, dhead = torch.from_numpy(emb).cuda(), torch.from_numpy(head).cuda()
    ang = np.arange(96)[:, None] * (10000.0 ** (-np.arange(64) / 64))[None]
    cos, sin = (torch.tensor(f(ang), dtype=torch.float32, device="cuda") for f in (np.cos, np.sin))
    slots = _i32(list(range(S)))
    prompts = [r.integers(0, V, 21).tolist(), r.integers(0, V, 30).tolist()]
    texts = [list(p) for p in prompts for _ in range(B)]
    status = c.status
    # the prompts go into each request's first slot, the other beams share its pages
    firsts = [0, B]
    c.p.reserve(_i32(firsts), _i32([len(p) - 1 for p in prompts]), c.work, status)
    for f, p in zip(firsts, prompts):
        x = demb[torch.tensor(p[:-1], device="cuda")]
        c.p.append8(0, _i32([f] * (len(p) - 1)), _i32(list(range(len(p) - 1))), None, x[:, H:H + Hkv], x[:, H + Hkv:], cos, sin,
                    status=status)
    c.p.fork(_i32([f for f in firsts for _ in range(B - 1)]), _i32([s for s in range(S) if s not in firsts]), c.work, status)
    score = torch.full((n, B), -math.inf, device="cuda")
    score[:, 0] = 0.0
    done = torch.zeros((n, B), dtype=torch.int32, device="cuda")
    eos = 7
    work = torch.empty(c.p.attn8_work_bytes(S, 1, H), dtype=torch.uint8, device="cuda")
    one = _i32([1] * S)
    token = torch.tensor([t[-1] for t in texts], dtype=torch.int64, device="cuda")
    hscore, hdone = score.double().cpu().numpy(), np.zeros((n, B), np.int64)
    for step in range(steps):
        c.p.reserve(slots, one, c.work, status)
        pos = (c.lens - 1).to(torch.int32)
        x = demb[token]
        qo = torch.empty((S, H, 128), device="cuda")
        c.p.append8(0, slots, pos, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], cos, sin, qo, status=status)
        out = torch.empty((S, 1, H, 128), device="cuda")
        c.p.attn8(0, qo.view(S, 1, H, 128), out, slots, work, status)
        logits = (out.view(S, H * 128) @ dhead).view(n, B, V)
        torch.cuda.synchronize()
        # attention over what the tables name
        for x_, y_ in zip(c.host.codes + c.host.scales, (c.k, c.v, c.ks, c.vs)):
            x_[...] = y_.cpu().numpy()
        tab, lens = c.tables.tolist(), c.lens.tolist()
        for s in range(S):
            assert lens[s] == len(texts[s])
            k, v = (torch.from_numpy(c.host.values(w, 0, tab[s], lens[s])).cuda() for w in range(2))
            for h in range(H):
                o, pv, big, va = attention(qo[s, h:h + 1].double(), k[h * Hkv // H], v[h * Hkv // H],
                                           torch.tensor([lens[s]], device="cuda"))
                assert bool(((out[s, :, h].double() - o).abs() <= attn8_bound(o, pv, big, va, lens[s], False, False)).all())
            # what the cache holds are this beam's own tokens: within half a step for each time the scale grew
            want = torch.from_numpy(emb[texts[s]][:, H + Hkv:]).double().cuda()
            top = torch.stack([want[i // 16 * 16:i // 16 * 16 + 16].abs().amax((0, 2)) for i in range(len(texts[s]))])
            assert bool(((v.transpose(0, 1) - want).abs().amax(-1) <= 8.1 * top / 127).all())
        so, pa, to, do, src = (torch.empty((n, B), dtype=d, device="cuda") for d in
                               (torch.float32, torch.int32, torch.int32, torch.int32, torch.int32))
        cuda.beam_select(logits, score, so, pa, to, done=done, eos=eos, done_out=do, slots=slots, src=src, status=status)
        c.p.fork(src.view(-1), slots, c.work, status)
        torch.cuda.synchronize()
        L = logits.cpu().numpy()
        new, hs = [], score.double().cpu().numpy()
        for i in range(n):
            want, near, _ = beam_select(L[i], hs[i], done.cpu().numpy()[i], eos, B)
            if all(a[1] == b[1] or a[0] - b[0] > 1e-4 for a, b in zip(near, near[1:])):
                assert pa[i].tolist() == [w[1] for w in want] and to[i].tolist() == [w[3] for w in want]
            for j in range(B):
                new.append(texts[i * B + int(pa[i, j])] + [int(to[i, j])])
        texts = new
        score, done, token = so, do, to.view(-1).long()
        assert c.take_status() == 0, step
    # every page is owned as often as tables name it
    tab, lens, refs = c.tables.tolist(), c.lens.tolist(), np.zeros(64, int)
    for s in range(S):
        for j in range(-(-lens[s] // page)):
            refs[tab[s][j]] += 1
    assert refs.tolist() == c.refs.tolist()
