"""Refusals of the attention, paged cache and verification entry points that
need no device: sizes, types, alignment and NULLs, checked before any device
call, and host memory, which is never taken for a device array."""
import ctypes as C

import numpy as np
import pytest

A = 1 << 20          # an aligned address that no call here dereferences


@pytest.fixture(scope="module")
def L(pkg):
    return pkg.lib()


def cache(abi, **kw):
    base = dict(k=A, v=A, refs=A, tables=A, lens=A, n_pages=8, n_layer=2, n_head_kv=5, page_size=16, n_slots=4,
                table_width=6, kv_type=1)
    base.update(kw)
    return abi.KvPages(**base)


@pytest.fixture(scope="module")
def abi(pkg):
    return pkg.abi


def prompt_args(**kw):
    a = dict(q=A, qs=2560, k=A, ks=640, v=A, vs=640, type=1, cu=A, n_seq=1, n=4, h=20, hkv=5, out=A, os=2560, ot=1,
             stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(cu=None), dict(out=None),
    dict(type=2), dict(ot=7), dict(type=0, ot=1), dict(n_seq=-1), dict(n=-1), dict(n=(1 << 24) + 1),
    dict(h=0), dict(h=19), dict(hkv=0), dict(h=1030, hkv=1030),
    dict(qs=2552), dict(ks=632), dict(os=2552), dict(qs=2564), dict(vs=644), dict(os=1 << 31),
    dict(q=A + 8), dict(out=A + 2),
])
def test_attn_prompt_refusals(L, bad):
    assert L.sllm_cuda_attn_prompt(*prompt_args(**bad)) == -1
    assert b"attn_prompt" in L.sllm_cuda_last_error()


@pytest.mark.parametrize("bad,rc", [
    (dict(k=None), -1), (dict(lens=None), -1), (dict(kv_type=3), -1), (dict(page_size=24), -4), (dict(page_size=0), -4),
    (dict(n_pages=0), -1), (dict(n_layer=0), -1), (dict(n_head_kv=0), -1), (dict(n_slots=0), -1),
    (dict(n_slots=(1 << 16) + 1), -1), (dict(table_width=0), -1), (dict(table_width=1 << 23, page_size=128, n_slots=1024), -1),
    (dict(k=A + 4), -1), (dict(refs=A + 4), -1),
])
def test_bad_caches(L, abi, bad, rc):
    p = cache(abi, **bad)
    assert L.sllm_cuda_kv_work_bytes(C.byref(p)) == 0
    big = 1 << 30
    assert L.sllm_cuda_kv_fork(C.byref(p), A, A, 1, A, big, None, None) == rc
    assert L.sllm_cuda_kv_reserve(C.byref(p), A, A, 1, A, big, None, None) == rc
    assert L.sllm_cuda_kv_release(C.byref(p), A, None, 1, A, big, None, None) == rc
    assert L.sllm_cuda_kv_compact(C.byref(p), A, big, None, None) == rc
    assert L.sllm_cuda_attn_prefix(C.byref(p), 0, A, A, 1, 1, 20, 0, A, 1, A, big, None, None) == rc
    assert L.sllm_cuda_kv_append(C.byref(p), 0, 1, A, A, 20, A, 2560, A, 640, A, 640, A, A, 64, A, None, None, None,
                                 None) == rc
    assert L.sllm_cuda_kv_work_bytes(None) == 0


def test_page_call_refusals(L, abi):
    p = cache(abi)
    n = L.sllm_cuda_kv_work_bytes(C.byref(p))
    assert n > 0
    r = C.byref(p)
    assert L.sllm_cuda_kv_fork(r, None, A, 1, A, n, None, None) == -1
    assert L.sllm_cuda_kv_fork(r, A, A, 5, A, n, None, None) == -1            # more slots than there are
    assert L.sllm_cuda_kv_fork(r, A, A, -1, A, n, None, None) == -1
    assert L.sllm_cuda_kv_reserve(r, A, None, 1, A, n, None, None) == -1
    assert L.sllm_cuda_kv_release(r, None, None, 1, A, n, None, None) == -1
    for args in ((A, n - 1), (A + 8, n), (None, n)):                          # the workspace
        assert L.sllm_cuda_kv_fork(r, A, A, 1, *args, None, None) == -1
        assert L.sllm_cuda_kv_compact(r, *args, None, None) == -1
        assert b"workspace" in L.sllm_cuda_last_error()


def test_append_refusals(L, abi):
    r = C.byref(cache(abi))
    good = dict(layer=0, n=1, slot=A, pos=A, h=20, q=A, qs=2560, k=A, ks=640, v=A, vs=640, c=A, s=A, n_ctx=64, qo=A,
                ko=None, vo=None, status=None, stream=None)
    for bad in (dict(layer=2), dict(layer=-1), dict(n=-1), dict(slot=None), dict(pos=None), dict(h=0), dict(h=7),
                dict(k=None), dict(v=None), dict(c=None), dict(s=None), dict(qo=None), dict(q=None), dict(qs=2556),
                dict(qs=2562), dict(ks=636), dict(vs=642), dict(n_ctx=0), dict(q=A + 4), dict(ko=A + 8)):
        a = dict(good)
        a.update(bad)
        assert L.sllm_cuda_kv_append(r, *a.values()) == -1, bad


def test_prefix_refusals(L, abi):
    p = cache(abi)
    r = C.byref(p)
    big = 1 << 40
    good = dict(layer=0, q=A, slots=A, n=2, nq=1, h=20, prefix=32, out=A, ot=1, work=A, wb=big, status=None, stream=None)
    for bad in (dict(layer=2), dict(q=None), dict(slots=None), dict(out=None), dict(work=None), dict(n=-1), dict(n=4097),
                dict(nq=0), dict(nq=17), dict(h=21), dict(h=0), dict(prefix=8), dict(prefix=-16), dict(prefix=112),
                dict(ot=2), dict(q=A + 8), dict(out=A + 8), dict(work=A + 8), dict(wb=0)):
        a = dict(good)
        a.update(bad)
        assert L.sllm_cuda_attn_prefix(r, *a.values()) == -1, bad
    assert L.sllm_cuda_attn_prefix_work_bytes(r, 2, 1, 20, 32) > 0
    assert L.sllm_cuda_attn_prefix_work_bytes(r, 2, 1, 21, 32) == 0
    f32 = cache(abi, kv_type=0)
    good["ot"] = 1
    assert L.sllm_cuda_attn_prefix(C.byref(f32), *good.values()) == -1         # f16 from an f32 cache


def test_verify_refusals(L):
    good = dict(p=A, q=A, draft=A, nd=A, ua=A, us=A, n=1, k=4, V=100, tokens=A, count=A, status=None, stream=None)
    for bad in (dict(p=None), dict(draft=None), dict(ua=None), dict(us=None), dict(tokens=None), dict(count=None),
                dict(n=-1), dict(n=65537), dict(k=0), dict(k=65), dict(V=0), dict(V=(1 << 24) + 1)):
        a = dict(good)
        a.update(bad)
        assert L.sllm_cuda_spec_verify(*a.values()) == -1, bad


def test_misaligned_arrays_are_refused(L):
    """A pointer that no float or int array has, refused on the host."""
    good = dict(p=A, q=A, draft=A, nd=A, ua=A, us=A, n=1, k=4, V=100, tokens=A, count=A, status=None, stream=None)
    a = dict(good, p=A + 2)
    assert L.sllm_cuda_spec_verify(*a.values()) == -1 and b"aligned" in L.sllm_cuda_last_error()
    assert L.sllm_cuda_attn_prompt(*prompt_args(q=A, cu=A + 1)) in (-1, -4)


def test_no_device_is_unsupported(cuda_absent, L, abi):
    """Without a device good arguments come back as SLLM_CUDA_ERR_UNSUPPORTED."""
    p = cache(abi)
    r, n = C.byref(p), L.sllm_cuda_kv_work_bytes(C.byref(p))
    assert L.sllm_cuda_attn_prompt(*prompt_args()) == -4
    assert L.sllm_cuda_kv_fork(r, A, A, 1, A, n, None, None) == -4
    assert L.sllm_cuda_kv_compact(r, A, n, None, None) == -4
    assert L.sllm_cuda_attn_prefix(r, 0, A, A, 2, 1, 20, 32, A, 1, A, 1 << 40, None, None) == -4
    assert L.sllm_cuda_spec_verify(A, A, A, A, A, A, 1, 4, 100, A, A, None, None) == -4


def test_rope_table(pkg, L):
    c, s = pkg.rope_table(5, 500000.0)
    f = np.float32(500000.0) ** np.float32(-2.0 / 128)
    ang = np.arange(5, dtype=np.float64)[:, None] * np.float64(f) ** np.arange(64)[None]
    # the recurrence multiplies in f32 (half a unit per step), then cos and sin of the f32 angle
    assert np.abs(c - np.cos(ang)).max() <= 4 * 70 * 2.0 ** -24 and np.abs(s - np.sin(ang)).max() <= 4 * 70 * 2.0 ** -24
    assert (c[0] == 1).all() and (s[0] == 0).all()
    out = np.zeros(64, np.float32)
    assert L.sllm_cuda_rope_table(0, 1e4, out.ctypes.data, out.ctypes.data) == -1
    assert L.sllm_cuda_rope_table(1, -1.0, out.ctypes.data, out.ctypes.data) == -1
    assert L.sllm_cuda_rope_table(1, 1e4, None, out.ctypes.data) == -1


def test_binding_checks(pkg):
    import torch
    w = torch.zeros(4, 2, 128)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        pkg.attn_prompt(w, w[:3], w, w, cu)                       # tokens disagree
    with pytest.raises(ValueError):
        pkg.attn_prompt(w, w.half(), w, w, cu)                    # types differ
    with pytest.raises(TypeError):
        pkg.attn_prompt(w.bfloat16(), w.bfloat16(), w.bfloat16(), w.bfloat16(), cu)
    with pytest.raises(ValueError):
        pkg.attn_prompt(w, w, w, w, cu.long())
    with pytest.raises(ValueError):
        pkg.attn_prompt(w.transpose(0, 1).contiguous().transpose(0, 1), w, w, w, cu)   # heads apart
    with pytest.raises(ValueError):
        pkg.KvPages(w, w, cu, cu, cu)
    with pytest.raises(ValueError):
        pkg.spec_verify(torch.zeros(2, 3, 7), None, torch.zeros(2, 3, dtype=torch.int32), None, torch.zeros(2, 2),
                        torch.zeros(2), cu, cu)


def test_page_model_itself():
    """The tests' own bookkeeping model keeps its invariants: counts equal the
    table entries that name a page, forked slots share, copies are private."""
    from serving_ref import PageModel
    rng = np.random.default_rng(3)
    m = PageModel(40, 6, 8, 16)
    for _ in range(300):
        op = rng.integers(4)
        slots = [int(x) for x in rng.permutation(6)[:rng.integers(1, 6)]]
        if op == 0:
            m.fork([int(x) for x in rng.integers(0, 6, len(slots))], slots)
        elif op == 1:
            m.reserve(slots, [int(x) for x in rng.integers(0, 30, len(slots))])
        elif op == 2:
            m.release(slots, [int(rng.integers(0, m.lens[s] + 1)) for s in slots])
        else:
            assert m.compact()[0] == 0
            live = sum(r > 0 for r in m.refs)
            assert all(r > 0 for r in m.refs[:live])
        count = [0] * 40
        for s in range(6):
            for i in m.tables[s][:m.used(m.lens[s])]:
                count[i] += 1
        assert count == m.refs
