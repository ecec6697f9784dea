"""Host side of the trainable readout: how a plan sorts a batch's rows, and what is refused before any
device work (CPU)."""
import numpy as np
import pytest
import torch

import nori_amd
from nori_amd import adapters as ad
from nori_amd import _native as nat


@pytest.mark.parametrize("ids,counts", [
    ([0], [1]), ([], []), ([-1, -1], [3, 2]), ([2, 0, 2, -1, 0], [3, 1, 4, 2, 5]), ([1, 1, 1], [0, 0, 0]), ([5, 4, 5], [2, 0, 1]),
])
def test_rows_are_grouped_by_adapter_in_their_order(ids, counts):
    order, starts, groups = ad._grouped(np.asarray(ids, dtype=np.int64), np.asarray(counts, dtype=np.int64))
    whose = np.repeat(np.asarray(ids, dtype=np.int64), counts)
    assert sorted(order.tolist()) == list(range(sum(counts)))
    assert groups.tolist() == sorted(set(whose.tolist()))
    assert len(starts) == len(groups) + 1 and starts[0] == 0 and starts[-1] == sum(counts)
    for g, i in enumerate(groups):
        assert order[starts[g]:starts[g + 1]].tolist() == np.flatnonzero(whose == i).tolist()


def test_plans_refuse_what_they_cannot_mean():
    make = lambda ids, rows: nori_amd.AdapterPlan(ids, rows, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="2 adapters for 3 tables"):
        make([0, 1], [1, 2, 3])
    with pytest.raises(ValueError, match="negative"):
        make([0], [-1])
    with pytest.raises(ValueError, match="numbered from 0"):
        make([-2], 4)
    with pytest.raises(TypeError):
        make([0.5], 4)
    with pytest.raises(TypeError):
        make([0], [4.0])
    with pytest.raises(ValueError, match="sequences"):
        make([[0, 1]], 4)
    with pytest.raises(ValueError, match="sequences"):
        make(0, 4)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        nori_amd.AdapterPlan([0], 4, device="cpu")


def test_updates_refuse_mismatched_arguments():
    plan = object.__new__(nori_amd.AdapterPlan)
    x, y, a, b = torch.randn(5, 8), torch.randn(5, 6), torch.randn(2, 4, 8), torch.randn(2, 6, 4)
    call = nori_amd.low_rank_update
    with pytest.raises(ValueError, match="factors"):
        call(x, y, a, torch.randn(2, 6, 3), plan)
    with pytest.raises(ValueError, match="factors"):
        call(x, y, a, torch.randn(3, 6, 4), plan)
    with pytest.raises(ValueError, match="8 inputs"):
        call(torch.randn(5, 9), y, a, b, plan)
    with pytest.raises(ValueError, match="not the projection"):
        call(x, torch.randn(4, 6), a, b, plan)
    with pytest.raises(ValueError, match="a is torch.float16"):
        call(x, y, a.half(), b, plan)
    with pytest.raises(NotImplementedError, match="float64"):
        call(x.double(), y.double(), a.double(), b.double(), plan)
    with pytest.raises(NotImplementedError, match="ranks up to 128"):
        call(x, y, torch.randn(2, 129, 8), torch.randn(2, 6, 129), plan)
    with pytest.raises(ValueError, match="empty"):
        call(x, y, torch.randn(2, 0, 8), torch.randn(2, 6, 0), plan)
    wide = torch.zeros(1)
    with pytest.raises(NotImplementedError, match="1048576 columns"):
        call(wide.expand(5, 2**20 + 1), y, wide.expand(2, 4, 2**20 + 1), b, plan)
    with pytest.raises(NotImplementedError, match="1048576 columns"):
        call(x, wide.expand(5, 2**20 + 1), a, wide.expand(2, 2**20 + 1, 4), plan)
    with pytest.raises(NotImplementedError, match="2147483648 of 8 -> 6"):
        call(x, y, wide.expand(2**31, 4, 8), wide.expand(2**31, 6, 4), plan)
    with pytest.raises(NotImplementedError, match="1073741824 elements"):
        nori_amd.trainable_layer_norm(wide.expand(2, 2**32 + 8), None, None)
    with pytest.raises(TypeError, match="AdapterPlan"):
        call(x, y, a, b, [0])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        call(x, y, a, b, plan)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        nori_amd.trainable_layer_norm(x, None, None)
    with pytest.raises(ValueError, match="at least one element"):
        nori_amd.trainable_layer_norm(torch.randn(3, 0), None, None)


def test_overlaps_are_seen():
    buffer = torch.zeros(6, 20)
    left, right = buffer[:, :8], buffer[:, 8:]
    assert not ad._overlap(left, right) and not ad._overlap(right, left)
    assert ad._overlap(buffer[:, :9], right) and ad._overlap(left, left) and ad._overlap(right, buffer[:, 4:10])
    assert ad._overlap(buffer[:, 12:], torch.as_strided(buffer, (5, 16), (20, 1), 16))  # wraps into the next row
    assert not ad._overlap(buffer[:3], buffer[3:]) and not ad._overlap(left, torch.zeros(6, 8))
    assert not ad._overlap(buffer[:0], buffer)
    assert ad._overlaps_itself(torch.zeros(1, 4).expand(3, 4)) and ad._overlaps_itself(torch.as_strided(buffer, (3, 5), (4, 1)))
    assert not any(ad._overlaps_itself(t) for t in (buffer, right, buffer.t(), buffer[:, :1], buffer[::2], torch.zeros(())))


def test_decoders_of_another_shape_are_refused():
    from torch import nn

    good = nn.Sequential(nn.Linear(8, 12), nn.LayerNorm(12), nn.GELU(), nn.Linear(12, 5))
    bank = nori_amd.ReadoutAdapters(good, 3, 2, alpha=4.0)
    assert bank.first.a.shape == (3, 2, 8) and bank.last.b.shape == (3, 5, 2) and bank.last.scales.tolist() == [2.0] * 3
    assert not bool(bank.first.b.any())
    for bad in (nn.Sequential(nn.Linear(8, 12), nn.GELU(), nn.Linear(12, 5)), nn.Linear(8, 5)):
        with pytest.raises(ValueError, match="decoder"):
            nori_amd.ReadoutAdapters(bad, 3, 2)
    with pytest.raises(NotImplementedError, match="ranks up to 128"):
        nori_amd.LowRankAdapters(1, 8, 8, 129)


def test_library_refuses_bad_arguments_before_any_device_work():
    lib = nat.lib()
    fw = [None, nat.NORI_F16, 4, 10, 10, None, 0, None, 0, 1e-5, None, nat.NORI_F16, None, None, None]
    assert lib.nori_layer_norm_train_forward(*fw) == nat.NORI_ERR_INVALID  # null pointers
    for at, value, code in ((1, nat.NORI_I8, nat.NORI_ERR_UNSUPPORTED), (3, 0, nat.NORI_ERR_INVALID), (2, -1, nat.NORI_ERR_INVALID),
                            (9, float("nan"), nat.NORI_ERR_INVALID), (4, -10, nat.NORI_ERR_INVALID), (2, 0, nat.NORI_OK)):
        bad = list(fw)
        bad[at] = value
        assert lib.nori_layer_norm_train_forward(*bad) == code, at
    fw[3] = fw[4] = 2**30 + 1
    assert lib.nori_layer_norm_train_forward(*fw) == nat.NORI_ERR_UNSUPPORTED
    bw = [16, nat.NORI_F16, 4, 10, 10, 16, nat.NORI_F16, 10, None, 0, 0, 16, 16, None, 16, None, None, 0, None]
    assert lib.nori_layer_norm_train_backward(*bw) == nat.NORI_ERR_INVALID  # dw without a workspace
    assert b"workspace" in lib.nori_last_error()
    up = [None, nat.NORI_F16, 4, 8, 8, None, 8, None, None, None, 2, 4, 8, None, None, None, 1, None, 8, None, None, 0, None]
    assert lib.nori_low_rank_update(*up) == nat.NORI_ERR_INVALID  # null pointers
    for at, value, code in ((1, nat.NORI_I8, nat.NORI_ERR_UNSUPPORTED), (11, 129, nat.NORI_ERR_UNSUPPORTED), (11, 0, nat.NORI_ERR_INVALID),
                            (3, 0, nat.NORI_ERR_INVALID), (2, 0, nat.NORI_OK), (2, 1 << 31, nat.NORI_ERR_UNSUPPORTED),
                            (16, 65536, nat.NORI_ERR_UNSUPPORTED), (3, 2**20 + 1, nat.NORI_ERR_UNSUPPORTED),
                            (12, 2**20 + 1, nat.NORI_ERR_UNSUPPORTED)):
        bad = list(up)
        bad[at] = value
        assert lib.nori_low_rank_update(*bad) == code, at
    full = [16, nat.NORI_F16, 100000, 8, 8, 16, 8, 16, 16, None, 2, 4, 8, 16, 16, 16, 1, 16, 8, None, None, 0, None]
    assert lib.nori_low_rank_update(*full) == nat.NORI_ERR_INVALID and b"workspace" in lib.nori_last_error()
    full[18] = 7
    assert lib.nori_low_rank_update(*full) == nat.NORI_ERR_INVALID and b"overlap" in lib.nori_last_error()
    full[5], full[17], full[18] = 16, 16, 9
    assert lib.nori_low_rank_update(*full) == nat.NORI_ERR_INVALID and b"another row stride" in lib.nori_last_error()
    back = [16, nat.NORI_F16, 4, 8, 8, 16, 8, 8, None, 8, 16, 16, None, 2, 4, 16, 16, 16, 1, 4, 16, 16, 8, 16, 16, None, 0, None]
    assert lib.nori_low_rank_backward(*back) == nat.NORI_ERR_INVALID and b"workspace" in lib.nori_last_error()
    for at, value, code in ((1, nat.NORI_I8, nat.NORI_ERR_UNSUPPORTED), (14, 129, nat.NORI_ERR_UNSUPPORTED), (19, 5, nat.NORI_ERR_INVALID),
                            (0, None, nat.NORI_ERR_INVALID), (20, None, nat.NORI_ERR_INVALID), (22, 7, nat.NORI_ERR_INVALID),
                            (2, 0, nat.NORI_OK)):
        bad = list(back)
        bad[at] = value
        assert lib.nori_low_rank_backward(*bad) == code, at
    back[21] = back[23] = back[24] = None
    assert lib.nori_low_rank_backward(*back) == nat.NORI_OK  # nothing is asked for
