"""The attention and cache entry points without a device: refusals of the
checked prompt call, and what the workspace sizes promise."""
import ctypes as C
import random

import pytest

from test_serving_refusals import A, cache, prompt_args


@pytest.fixture(scope="module")
def L(pkg):
    return pkg.lib()


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(cu=None), dict(out=None), dict(type=2), dict(type=0, ot=1), dict(n_seq=-1), dict(n=(1 << 24) + 1),
    dict(h=19), dict(hkv=0), dict(qs=2552), dict(os=2552), dict(vs=644), dict(q=A + 8), dict(out=A + 2),
])
def test_checked_prompt_refusals(L, bad):
    a = prompt_args(**bad)
    a.insert(-1, A)
    assert L.sllm_cuda_attn_prompt_checked(*a) == -1
    assert b"attn_prompt" in L.sllm_cuda_last_error()


def test_checked_prompt_without_a_device(cuda_absent, L):
    for status in (None, A):
        a = prompt_args()
        a.insert(-1, status)
        assert L.sllm_cuda_attn_prompt_checked(*a) == -4


def test_binding_checks_the_status_word(pkg):
    import torch
    w = torch.zeros(4, 2, 128)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for status in (torch.zeros(1), torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="status"):
            pkg.attn_prompt(w, w, w, w, cu, status=status)


HEADS = [(8, 1), (64, 8), (20, 5), (4, 4), (7, 1), (256, 1)]


def _wide(abi, kv, f16, page=16):
    return cache(abi, n_head_kv=kv, kv_type=1 if f16 else 0, page_size=page, table_width=1 << 16, n_slots=4096)


def _bytes(L, p, n, nq, h, prefix):
    return L.sllm_cuda_attn_prefix_work_bytes(C.byref(p), n, nq, h, prefix)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("f16", [False, True])
def test_prefix_workspace_never_falls(pkg, L, heads, f16):
    """More sequences, query tokens or prefix never need less: a buffer of the
    largest call's size serves the smaller ones."""
    h, kv = heads
    p = _wide(pkg.abi, kv, f16)
    for nq in (1, 3, 16):
        for prefix in (0, 16, 1792, 2304, 16384, 262144):
            sizes = [_bytes(L, p, n, nq, h, prefix) for n in list(range(1, 70)) + [100, 128, 129, 500, 1000, 4096]]
            assert all(sizes) and sizes == sorted(sizes)
    for n, nq in ((1, 1), (16, 1), (21, 2), (300, 4)):
        sizes = [_bytes(L, p, n, nq, h, 16 * x) for x in list(range(0, 400)) + [1000, 1024, 2000, 4096, 10000, 65536]]
        assert all(sizes) and sizes == sorted(sizes)
        sizes = [_bytes(L, p, n, x, h, 4096) for x in range(1, 17)]
        assert all(sizes) and sizes == sorted(sizes)


def test_prefix_workspace_of_the_largest_call_is_taken(cuda_absent, L, pkg):
    """... by the call itself, which asks for what its own splits need. Without
    a device it stops behind that check."""
    rng = random.Random(4)
    for _ in range(4000):
        h, kv = rng.choice(HEADS)
        f16 = rng.random() < 0.7
        p = _wide(pkg.abi, kv, f16)
        most = [int(2 ** rng.uniform(0, 12)), rng.randint(1, 16), 16 * int(2 ** rng.uniform(0, 15))]
        size = _bytes(L, p, most[0], most[1], h, most[2])
        for _ in range(3):
            n, nq, prefix = rng.randint(1, most[0]), rng.randint(1, most[1]), 16 * rng.randint(0, most[2] // 16)
            rc = L.sllm_cuda_attn_prefix(C.byref(p), 0, A, A, n, nq, h, prefix, A, f16, A, size, None, None)
            assert rc == -4, (h, kv, f16, most, n, nq, prefix, L.sllm_cuda_last_error())


def test_prefix_workspace_is_no_waste(L, pkg):
    """A bound far above the need would be one too: 64 sequences of four query
    tokens behind 32768, 64 heads of 8, need ten parts a row."""
    p = _wide(pkg.abi, 8, True)
    assert _bytes(L, p, 64, 4, 64, 32768) <= 22 * 64 * 4 * 64 * 520


# ---------------------------------------------------------------------------
# the measure that the f32 attention core is held against
# ---------------------------------------------------------------------------
def _rows(n, rows, seed):
    import torch
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(m, 128, generator=g) * 1.3 for m in (rows, n, n))
    return q, k, v, torch.linspace(max(1, n - 4 * rows), n, rows).long()


@pytest.mark.parametrize("n", [64, 700, 4100])
def test_six_partial_products_are_as_good_as_32_bits(n):
    from precision_ref import PAIRS, as_good_as_32_bits, attention_planes
    x = _rows(n, 48, n)
    assert max(as_good_as_32_bits(attention_planes(*x), *x)) <= 3
    # and with any of them left out they are not
    for lost in PAIRS:
        out = attention_planes(*x, [p for p in PAIRS if p != lost])
        assert min(as_good_as_32_bits(out, *x)) > 3, lost


def test_no_slots_need_no_arrays(cuda_absent, pkg, L):
    """n = 0: NULL arrays are passed over (and the call goes on to look for a
    device); a negative n, or NULL with slots named, is refused as before."""
    r = C.byref(cache(pkg.abi))
    size = L.sllm_cuda_kv_work_bytes(r)
    for n, rc in ((0, -4), (1, -1), (-1, -1)):
        assert L.sllm_cuda_kv_fork(r, None, None, n, A, size, None, None) == rc
        assert L.sllm_cuda_kv_reserve(r, None, None, n, A, size, None, None) == rc
        assert L.sllm_cuda_kv_release(r, None, None, n, A, size, None, None) == rc
