"""Plans of adapters as objects: what a copy, a pickle or a load on another device holds (CPU; the plan's copy to the
device is left out)."""
import copy
import io
import pickle

import numpy as np
import pytest
import torch

import nori_amd
from nori_amd import _native as nat
from nori_amd import adapters as ad


@pytest.fixture
def plan(monkeypatch):
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "to", lambda self, *a, **k: self)
        return nori_amd.AdapterPlan([2, 0, -1, 2], [3, 1, 4, 2], device="cuda:0")


def _saved(plan):
    file = io.BytesIO()
    torch.save(plan, file)
    file.seek(0)
    return torch.load(file, weights_only=False)  # written just above


@pytest.mark.parametrize("again", [copy.deepcopy, copy.copy, lambda p: pickle.loads(pickle.dumps(p)), _saved])
def test_a_copy_points_at_its_own_memory(plan, again):
    other = again(plan)
    for p in (plan, other):
        assert p.pointers == (p.order.data_ptr(), p.starts.data_ptr(), p.ids.data_ptr())
        assert p.order.tolist() == [4, 5, 6, 7, 3, 0, 1, 2, 8, 9] and p.ids.tolist() == [-1, 0, 2] and p.starts.tolist() == [0, 4, 5, 10]
    assert (other.rows, other.groups, other.longest, other.most, other.adapters) == (10, 3, 5, 2, (0, 2))


def test_a_plan_is_where_its_rows_are(plan, monkeypatch):
    # a plan unpickled without its device has its rows in host memory, which no kernel may be given
    assert plan.device.type == "cpu"
    monkeypatch.setattr(nat, "require_device", lambda *t: torch.device("cuda", 0))
    x, y, a, b = torch.randn(10, 8), torch.randn(10, 6), torch.randn(3, 4, 8), torch.randn(3, 6, 4)
    with pytest.raises(RuntimeError, match="different devices"):
        ad._check(x, y, a, b, plan, None)


@pytest.mark.parametrize("ids,rows,error,match", [
    ([0, 1], [2**62, 2**62], NotImplementedError, "rows"),  # whose sum passes 64 bits
    ([0] * 3, 2**29, NotImplementedError, "rows"),
    ([0], 2**63 - 1, NotImplementedError, "rows"),
    (np.array([2**64 - 1], dtype=np.uint64), [1], ValueError, "out of range"),  # -1 where 64 bits wrap
    ([0], np.array([2**64 - 3], dtype=np.uint64), NotImplementedError, "rows"),
    ([2**63 - 1], [1], ValueError, "out of range"),
    ([2**31 - 1], [0], ValueError, "out of range"),
])
def test_numbers_past_their_range_are_refused(ids, rows, error, match):
    with pytest.raises(error, match=match):
        nori_amd.AdapterPlan(ids, rows, device="cuda:0")


def test_a_stream_is_recorded_once(plan, monkeypatch):
    recorded = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: "stream")
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: recorded.append((self.data_ptr(), stream)))
    for stream in (7, 0, 7, 0):
        plan.used_on(stream)
    assert recorded == [(plan.starts.data_ptr(), "stream")] * 2
    other = copy.deepcopy(plan)
    other.used_on(7)
    assert recorded[2:] == [(other.starts.data_ptr(), "stream")]
