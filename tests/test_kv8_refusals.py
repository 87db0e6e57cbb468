"""Refusals of the 8-bit cache and beam selection entry points that need no
device: sizes, types, alignment, NULLs, and caches of the other kind."""
import ctypes as C

import pytest

A = 1 << 20          # an aligned address that no call here dereferences


@pytest.fixture(scope="module")
def L(pkg):
    return pkg.lib()


@pytest.fixture(scope="module")
def abi(pkg):
    return pkg.abi


def cache(abi, **kw):
    base = dict(k=A, v=A, refs=A, tables=A, lens=A, n_pages=8, n_layer=2, n_head_kv=5, page_size=16, n_slots=4,
                table_width=6, kv_type=2, k_scale=A, v_scale=A)
    base.update(kw)
    return abi.KvPages(**base)


APPEND = dict(layer=0, n=1, slot=A, pos=A, h=20, q=A, qs=2560, k=A, ks=640, v=A, vs=640, c=A, s=A, n_ctx=64, qo=A, ko=None,
              vo=None, ot=1, status=None, stream=None)
READ = dict(layer=0, n=1, slot=A, pos=A, ko=A, vo=A, ot=1, status=None, stream=None)
ATTN = dict(layer=0, q=A, qt=1, slots=A, n=2, nq=1, h=20, out=A, ot=1, work=A, wb=1 << 40, status=None, stream=None)
BEAM = dict(lg=A, rs=100, sc=A, done=A, slots=A, n=1, b=4, V=100, eos=3, so=A, pa=A, to=A, do=A, src=A, status=None,
            stream=None)


@pytest.mark.parametrize("bad,rc", [
    (dict(k_scale=None), -1), (dict(v_scale=None), -1), (dict(k_scale=A + 4), -1), (dict(v_scale=A + 8), -1), (dict(k=None), -1),
    (dict(page_size=8), -4), (dict(n_pages=0), -1), (dict(kv_type=3), -1), (dict(k=A + 4), -1),
])
def test_bad_caches(L, abi, bad, rc):
    r = C.byref(cache(abi, **bad))
    assert L.sllm_cuda_kv_work_bytes(r) == 0 and L.sllm_cuda_attn_kv8_work_bytes(r, 1, 1, 20) == 0
    assert L.sllm_cuda_kv8_append(r, *APPEND.values()) == rc
    assert L.sllm_cuda_kv8_read(r, *READ.values()) == rc
    assert L.sllm_cuda_attn_kv8(r, *ATTN.values()) == rc
    assert L.sllm_cuda_kv_fork(r, A, A, 1, A, 1 << 30, None, None) == rc
    assert L.sllm_cuda_kv_compact(r, A, 1 << 30, None, None) == rc


@pytest.mark.parametrize("kind", [0, 1])
def test_caches_of_the_other_kind(L, abi, kind):
    """The 8-bit calls take an 8-bit cache only, kv_append and attn_prefix none; a cache of 16 or 32 bits needs no
    scales, and a struct without them is as good as it was."""
    r = C.byref(cache(abi, kv_type=kind, k_scale=None, v_scale=None))
    assert L.sllm_cuda_kv8_append(r, *APPEND.values()) == -1 and b"8-bit" in L.sllm_cuda_last_error()
    assert L.sllm_cuda_kv8_read(r, *READ.values()) == -1
    assert L.sllm_cuda_attn_kv8(r, *ATTN.values()) == -1
    assert L.sllm_cuda_attn_kv8_work_bytes(r, 1, 1, 20) == 0
    assert L.sllm_cuda_kv_work_bytes(r) > 0
    e = C.byref(cache(abi))
    assert L.sllm_cuda_kv_append(e, *[v for k, v in APPEND.items() if k != "ot"]) == -1
    assert b"8-bit" in L.sllm_cuda_last_error()
    assert L.sllm_cuda_attn_prefix(e, 0, A, A, 1, 1, 20, 0, A, 1, A, 1 << 30, None, None) == -1
    assert L.sllm_cuda_attn_prefix_work_bytes(e, 1, 1, 20, 0) == 0
    assert L.sllm_cuda_kv_work_bytes(e) > 0


def test_append_refusals(L, abi):
    r = C.byref(cache(abi))
    for bad in (dict(layer=2), dict(layer=-1), dict(n=-1), dict(n=(1 << 24) + 1), dict(slot=None), dict(pos=None), dict(h=0),
                dict(h=7), dict(k=None), dict(v=None), dict(c=None), dict(s=None), dict(qo=None), dict(q=None), dict(qs=2556),
                dict(qs=2562), dict(ks=636), dict(vs=642), dict(n_ctx=0), dict(q=A + 4), dict(ko=A + 8), dict(ot=2), dict(ot=-1)):
        assert L.sllm_cuda_kv8_append(r, *dict(APPEND, **bad).values()) == -1, bad
        assert b"kv8_append" in L.sllm_cuda_last_error()


def test_read_refusals(L, abi):
    r = C.byref(cache(abi))
    for bad in (dict(layer=2), dict(layer=-1), dict(n=-1), dict(n=(1 << 24) + 1), dict(slot=None), dict(pos=None), dict(ot=2),
                dict(ko=A + 8), dict(vo=A + 4)):
        assert L.sllm_cuda_kv8_read(r, *dict(READ, **bad).values()) == -1, bad


def test_attn_refusals(L, abi):
    r = C.byref(cache(abi))
    for bad in (dict(layer=2), dict(q=None), dict(slots=None), dict(out=None), dict(work=None), dict(n=-1), dict(n=4097),
                dict(nq=0), dict(nq=17), dict(h=21), dict(h=0), dict(h=1030), dict(ot=2), dict(qt=2), dict(qt=0), dict(q=A + 8),
                dict(out=A + 8), dict(work=A + 8), dict(wb=0)):
        assert L.sllm_cuda_attn_kv8(r, *dict(ATTN, **bad).values()) == -1, bad
    assert L.sllm_cuda_attn_kv8_work_bytes(r, 2, 1, 20) > 0
    assert L.sllm_cuda_attn_kv8_work_bytes(r, 2, 1, 21) == 0


def test_beam_refusals(L):
    for bad in (dict(lg=None), dict(sc=None), dict(so=None), dict(pa=None), dict(to=None), dict(slots=None), dict(src=None),
                dict(n=-1), dict(n=65537), dict(b=0), dict(b=17), dict(V=0), dict(V=(1 << 20) + 1, rs=1 << 21), dict(rs=99),
                dict(rs=(1 << 30) + 1), dict(eos=100), dict(eos=-1), dict(eos=-1, done=None), dict(eos=-1, do=None)):
        assert L.sllm_cuda_beam_select(*dict(BEAM, **bad).values()) == -1, bad
        assert b"beam_select" in L.sllm_cuda_last_error()
    assert L.sllm_cuda_beam_select(*dict(BEAM, lg=A + 2).values()) == -1


def test_no_device_is_unsupported(cuda_absent, L, abi):
    r = C.byref(cache(abi))
    assert L.sllm_cuda_kv8_append(r, *APPEND.values()) == -4
    assert L.sllm_cuda_kv8_read(r, *READ.values()) == -4
    assert L.sllm_cuda_attn_kv8(r, *ATTN.values()) == -4
    assert L.sllm_cuda_beam_select(*BEAM.values()) == -4
    assert L.sllm_cuda_beam_select(*dict(BEAM, done=None, do=None, eos=-1, slots=None, src=None).values()) == -4


def test_python_binding_refuses(pkg):
    import torch
    k = torch.zeros((4, 1, 2, 32, 128), dtype=torch.int8)
    sc = torch.zeros((4, 1, 2, 2))
    ints = [torch.zeros(4, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)]
    p = pkg.KvPages(k, k, *ints, sc, sc)
    with pytest.raises(ValueError):
        pkg.KvPages(k, k, *ints)
    with pytest.raises(ValueError):
        pkg.KvPages(k, k, *ints, sc, None)
    with pytest.raises(ValueError):
        pkg.KvPages(k, k, *ints, sc, torch.zeros((4, 1, 2, 3)))
    with pytest.raises(ValueError):
        pkg.KvPages(k.half(), k.half(), *ints, sc, sc)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        p.read8(0, one, one)
    with pytest.raises(ValueError):
        p.read8(0, one, one, torch.zeros((1, 2, 128)), torch.zeros((1, 2, 128), dtype=torch.float16))
    with pytest.raises(TypeError):
        p.attn8(0, torch.zeros((1, 1, 4, 128), dtype=torch.bfloat16), torch.zeros((1, 1, 4, 128)), one, torch.zeros(64))
    x = torch.zeros((1, 2, 128))
    ang = torch.zeros((8, 64))
    with pytest.raises(ValueError):
        p.append8(0, one, one, x, x, x, ang, ang, x.half(), x)
    f = torch.zeros((2, 3))
    i = torch.zeros((2, 3), dtype=torch.int32)
    for lg in (torch.zeros((2, 3, 8), dtype=torch.float16), torch.zeros((2, 3, 8)).transpose(0, 1), torch.zeros((2, 3, 16))[:, :, ::2]):
        with pytest.raises(ValueError):
            pkg.beam_select(lg, f, f, i, i)
    with pytest.raises(ValueError):
        pkg.beam_select(torch.zeros((2, 3, 8)), f, f, i.long(), i)
