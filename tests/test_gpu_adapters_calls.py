"""How a program may call the adapters: copies of plans, other streams, values that other graphs saved (GPU)."""
import copy
import pickle

import pytest
import torch

from nori_amd import AdapterPlan, low_rank_update

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _make(rows, k, n, rank, adapters, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    parts = r(rows, k), r(rows, n), r(adapters, rank, k) * k**-0.5, 0.2 * r(adapters, n, rank)
    return [t.to(DEV, dtype) for t in parts]


def test_copies_of_a_plan_outlive_it():
    plan = AdapterPlan([1, -1, 0], [20, 5, 30], device=DEV)
    x, y, a, b = _make(55, 24, 40, 4, 2)
    want = low_rank_update(x, y, a, b, plan)
    copies = [copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))]
    del plan
    taken = [torch.full((512,), 2**30, dtype=torch.int32, device=DEV) for _ in range(8)]  # where the first plan's memory was
    for other in copies:
        assert other.device == DEV and torch.equal(low_rank_update(x, y, a, b, other), want)
    assert len(taken) == 8


def test_a_plan_may_go_while_another_stream_still_reads_it():
    # made on one stream, used on another behind other work, and dropped at once: its memory is not handed out meanwhile
    x, y, a, b = _make(4000, 24, 40, 4, 2)
    ids = [1, 0, -1, 1]
    want = low_rank_update(x, y, a, b, AdapterPlan(ids, 1000, device=DEV))
    side = torch.cuda.Stream(DEV)
    busy = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    plan = AdapterPlan(ids, 1000, device=DEV)
    at, size = plan._packed.data_ptr(), plan._packed.numel()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-4
        got = low_rank_update(x, y, a, b, plan)
    del plan
    taken = [torch.zeros(size, dtype=torch.int32, device=DEV) for _ in range(4)]
    assert all(t.data_ptr() != at for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
