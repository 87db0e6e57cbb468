"""Beam selection over logits far from zero: words forbidden by a large finite value instead of -inf, and
rows whose own largest logit is far away."""
import math

import numpy as np
import pytest

from kv8_ref import beam_select
from test_gpu_beam import _logits, _scores, run

pytestmark = pytest.mark.gpu

LIMIT = 2.0 ** 100                                           # logits beyond it count as it


def check_far(cuda, logits, score):
    """As test_gpu_beam.check, and its tolerances; the definition's logits are counted from their row's largest (which
    leaves the formula as it is), so that 64 bits hold the logarithm of the sum whatever the largest is."""
    pa, to, so, _, _, st = run(cuda, logits, score)
    assert st[0] == 0
    L, S, B = logits.cpu().numpy().astype(np.float64).clip(-LIMIT, LIMIT), score.double().cpu().numpy(), logits.shape[1]
    tol = 2.0 ** -16 * 1.01
    for i in range(len(L)):
        want, near, every = beam_select(L[i] - L[i].max(-1, keepdims=True), S[i], None, -1, B)
        if all(a[1] == b[1] or a[0] - b[0] > 2 * tol or a[0] == b[0] for a, b in zip(near, near[1:])):
            assert pa[i].tolist() == [c[1] for c in want] and to[i].tolist() == [c[3] for c in want], i
        else:
            assert len(set(zip(pa[i].tolist(), to[i].tolist()))) == B
            want = [next(c for c in every if (c[1], c[3]) == pt) for pt in zip(pa[i].tolist(), to[i].tolist())]
            assert all(abs(c[0] - d[0]) <= 2 * tol + abs(d[0]) * 2.0 ** -50 for c, d in zip(want, near))
        for j, c in enumerate(want):
            assert abs(float(so[i, j]) - c[0]) <= tol + abs(c[0]) * 2.0 ** -23, (i, j, float(so[i, j]), c)


def _rows(seed, n, B, V, apart):
    """Rows next to one another or `apart` words further; (not a multiple of four: copied word by word)"""
    return _logits(seed, n, B, V + apart)[:, :, :V]


@pytest.mark.parametrize("mask", [-1e9, -5e9, -1e10, -1e20, -1e30, -3.4028234663852886e38, -2e7])
@pytest.mark.parametrize("V,apart", [(40, 0), (3001, 0), (9000, 4), (40000, 0), (40001, 2), (128256, 0)])
def test_words_forbidden_by_a_finite_value(cuda, mask, V, apart):
    """1%, half, 99% of a row and all but a few words, in places of no order, at its start, at its end; the whole row
    of one beam; all rows."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(V)
    n, B = 7, 3
    lg, sc = _rows(V, n, B, V, apart), _scores(V, n, B)
    r = torch.rand((n, B, V), generator=g, device="cuda")
    for i, part in enumerate((0.01, 0.5, 0.99)):
        lg[i][r[i] < part] = mask
    lg[3, :, 3:] = mask
    lg[4, :, :V - 4] = mask
    lg[5, 1] = mask
    lg[6] = mask
    check_far(cuda, lg, sc)


@pytest.mark.parametrize("V", [40, 3001, 9000, 40001])
@pytest.mark.parametrize("far", [1.6e7, 1.7e7, 3e8, 1.6e9, 5e9, 2e10, 1e20])
def test_rows_that_are_far_from_zero(cuda, V, far):
    """Largest logits of +-far: words of the same value, some a few steps of 32 bits lower, others much lower; next to
    beams of ordinary logits and of the other sign."""
    import torch
    n, B = 4, 3
    step = float(np.spacing(np.float32(far)))
    g = torch.Generator(device="cuda").manual_seed(V)
    lg, sc = _logits(V, n, B, V), _scores(V, n, B)
    near = torch.randint(0, 4, (n, B, V), generator=g, device="cuda").float() * step
    much = torch.randint(0, 3, (n, B, V), generator=g, device="cuda").float() * far * 0.25
    lg[0] = far - near[0]
    lg[1] = -far - near[1]
    lg[2, 0], lg[2, 1] = far - near[2, 0] - much[2, 0], -far - much[2, 1]
    lg[3, :, ::7] = -far
    lg[3, 1, V // 2] = far
    check_far(cuda, lg, sc)


def test_far_and_near_in_neighbouring_words(cuda):
    """One word of a thread ordinary, all others far below, wherever it is; and one far above."""
    import torch
    V = 9000
    for mask in (-1e10, -1e20, -1e30):
        for at in (0, 4095, 4096, 8191, 8999):
            lg = torch.full((1, 2, V), mask, device="cuda")
            lg[0, 0, at], lg[0, 1, V - 1 - at] = 2.0, -mask
            check_far(cuda, lg, _scores(1, 1, 2))


@pytest.mark.parametrize("V", [3, 300, 4096])
@pytest.mark.parametrize("B", [1, 4, 16])
def test_short_rows_over_and_over(cuda, B, V):
    """Many requests of one piece a beam, some with a NaN in their last word, 20 times: every warp's sums count and
    every report arrives. (Sums and reports once passed through words that other warps might clear.)"""
    n = 1500
    lg, sc = _logits(V, n, B, V), _scores(V, n, B)
    first = run(cuda, lg, sc)
    for i in (0, 700, n - 1):
        check_far(cuda, lg[i:i + 1], sc[i:i + 1])
    lg[n - 1, B - 1, V - 1] = math.nan
    for _ in range(20):
        got = run(cuda, lg, sc)
        assert got[5][0] == -1
        for a, b in zip(got[:3], first[:3]):
            assert np.array_equal(a[:-1], b[:-1])
