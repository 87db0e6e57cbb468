"""What 32-bit attention may cost: a result's errors against 64 bits, held
against those of the same computation in plain 32-bit arithmetic.

A worst-case bound grows with every sum's length and lets a core pass whose
operands carry 16 bits. Errors of sums are random, though, and alike for any
order of the additions: the plain form has one rounding per product added, the
core one cut per 16 products and plane pair (48 for 128 products), which is
one-sided but a whole unit where a rounding is half: 48 cuts of mean half a
unit against the random walk of 128 roundings of a quarter. Either is a few
units of a score, so three times the plain form's errors, by their largest and by
their root mean square, leaves room for the one against the other and none for
operands cut to 16 bits (whose errors are 2^-17 of a product, 100 units)."""
import math

import torch


def attention32(q, k, v, limit):
    """Plain 32-bit attention of rows q [R, 128]; row r sees keys < limit[r]."""
    seen = torch.arange(k.shape[0], device=q.device)[None] < limit[:, None]
    s = torch.where(seen, (q @ k.T) / math.sqrt(128.0), -math.inf)
    e = torch.exp(s - s.amax(1, keepdim=True))
    return (e @ v) / e.sum(1, keepdim=True)


def attention64(q, k, v, limit):
    return attention32(q.double(), k.double(), v.double(), limit)


def as_good_as_32_bits(out, q, k, v, limit):
    """(largest, root mean square) of out's errors over the plain form's: both
    should be at most 3."""
    want = attention64(q, k, v, limit)
    a, b = (out.double() - want).abs(), (attention32(q, k, v, limit).double() - want).abs()
    return float(a.max() / b.max()), float((a.square().mean() / b.square().mean()).sqrt())


def planes(x):
    """An f32 as three bf16: rounded, the next eight bits, the rest."""
    cut = lambda t: (t.view(torch.int32) & -65536).view(torch.float32)
    a = x.bfloat16().float()
    b = cut(x - a)
    return a.double(), b.double(), cut(x - a - b).double()


PAIRS = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]


def attention_planes(q, k, v, limit, pairs=PAIRS):
    """The core's arithmetic: partial products of the planes, summed exactly."""
    mul = lambda x, y: sum(x[i] @ y[j] for i, j in pairs)
    seen = torch.arange(k.shape[0])[None] < limit[:, None]
    s = mul(planes(q), [t.T for t in planes(k)]).float()
    s = torch.where(seen, s / math.sqrt(128.0), -math.inf)
    e = torch.exp(s - s.amax(1, keepdim=True))
    return mul(planes(e), planes(v)).float() / e.sum(1, keepdim=True)
