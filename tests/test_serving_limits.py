"""The attention and cache entry points without a device: refusals of the
checked prompt call, and what the workspace sizes promise."""
import ctypes as C

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
