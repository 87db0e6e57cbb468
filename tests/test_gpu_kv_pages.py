"""The paged cache's bookkeeping at sizes and in states that the random runs of
test_gpu_serving.py do not reach."""
import numpy as np
import pytest

from test_gpu_serving import Cache, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_slots,groups", [(1000, 3), (2049, 40), (5000, 7)])
def test_reserve_many_owners_of_a_page(cuda, n_slots, groups):
    """Samples forked from a few prompts, which write to the shared last pages
    in any order: all owners named (the last keeps the page), or not all."""
    rng = np.random.default_rng(n_slots)
    c = Cache(cuda, 3 * n_slots + 100, n_slots, 4, 16, 1, 1, "f16")
    c.m.reserve(list(range(groups)), [int(x) for x in rng.integers(1, 32, groups)])
    rest = list(range(groups, n_slots))
    c.m.fork([int(x) for x in rng.integers(0, groups, len(rest))], rest)
    c.push()
    order = [int(x) for x in rng.permutation(n_slots)]
    some = [s for s in order if s % groups != 1 or s % 5 != 0]          # the owners of most pages, but not all
    for slots in (some, order):
        k0, v0 = c.k.clone(), c.v.clone()
        new = [int(x) for x in rng.integers(0, 3, len(slots))]
        want, copies = c.m.reserve(slots, new)
        c.p.reserve(_i32(slots), _i32(new), c.work, c.status)
        c.same()
        assert c.take_status() == want == 0 and copies
        for a, b, r in copies:
            k0[b, :, :, :r], v0[b, :, :, :r] = k0[a, :, :, :r], v0[a, :, :, :r]
        assert bool((c.k == k0).all()) and bool((c.v == v0).all())


def test_reserve_takes_linear_work(cuda):
    """As many slots as a cache may have, all forks of one prompt: the writers
    of a page are counted, not compared with one another (0.5 ms; 44 ms when
    each was)."""
    import torch
    n = (1 << 16) - 1
    c = Cache(cuda, n + 8, n + 1, 2, 16, 1, 1, "f16")
    c.m.refs[0] = n + 1
    c.m.lens = [5] * (n + 1)
    slots, new = _i32(list(range(1, n + 1))), _i32([1] * n)
    ms = []
    for _ in range(3):
        c.push()
        torch.cuda.synchronize()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        c.p.reserve(slots, new, c.work, c.status)
        b.record()
        torch.cuda.synchronize()
        ms.append(a.elapsed_time(b))
    assert c.m.reserve(list(range(1, n + 1)), [1] * n)[0] == c.take_status() == 0
    c.same()
    assert min(ms) < 8.0, ms


def test_reserve_refuses_a_count_below_the_entries(cuda):
    """Three slots write to a page that counts two owners: no slot could keep it."""
    c = Cache(cuda, 20, 4, 4, 16)
    c.m.reserve([0], [21])
    c.m.fork([0, 0], [1, 2])
    c.m.refs[c.m.tables[0][1]] = 2
    c.push()
    c.p.reserve(_i32([0, 1, 2]), _i32([1, 1, 1]), c.work, c.status)
    c.same()
    assert c.take_status() == -1


def test_calls_that_name_no_slot(cuda):
    """A step in which nobody forks, grows or ends: nothing to do, no error
    (an empty tensor has no address)."""
    c = Cache(cuda, 20, 4, 4, 16)
    c.m.reserve([0], [21])
    c.push()
    none = _i32([])
    c.p.fork(none, none, c.work, c.status)
    c.p.reserve(none, none, c.work, c.status)
    c.p.release(none, None, c.work, c.status)
    c.p.release(none, none, c.work, c.status)
    c.same()
    assert c.take_status() == 0
