"""The attention operators where rounding, masks and limits meet: against the
64-bit forms of serving_ref.py, whose bounds are derived there."""
import math

import numpy as np
import pytest

from serving_ref import attention, attention_bound
from test_gpu_serving import _dt, _i32, _rand, run_prefix, shared_cache

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
