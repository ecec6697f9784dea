"""Derivatives that the readout's operators do not have are refused (CPU: before any device work)."""
import pytest
import torch
from torch.autograd import forward_ad

import nori_amd
from nori_amd import _native as nat


@pytest.fixture
def anywhere(monkeypatch):
    """The checks as on a GPU, up to the first launch."""
    monkeypatch.setattr(nat, "require_device", lambda *t: torch.device("cpu"))

    def lib():
        raise AssertionError("a kernel would run")

    monkeypatch.setattr(nat, "lib", lib)


def _plan(rows, device="cpu"):
    plan = object.__new__(nori_amd.AdapterPlan)
    plan._packed = torch.tensor([0, rows, 0, *range(rows)], dtype=torch.int32)
    plan.rows, plan.most, plan.groups, plan.longest, plan.adapters = rows, 0, 1, rows, (0,)
    return plan


@pytest.mark.parametrize("dual", ["x", "weight", "bias"])
def test_layer_norm_refuses_tangents(anywhere, dual):
    t = {"x": torch.randn(3, 8), "weight": torch.ones(8), "bias": torch.zeros(8)}
    with forward_ad.dual_level():
        args = {n: forward_ad.make_dual(v, torch.ones_like(v)) if n == dual else v for n, v in t.items()}
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.trainable_layer_norm(**args)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: nori_amd.trainable_layer_norm(**{**t, dual: v}), (t[dual],), (t[dual],))
    with forward_ad.dual_level(), pytest.raises(AssertionError, match="a kernel would run"):
        nori_amd.trainable_layer_norm(**t)  # none of its own


@pytest.mark.parametrize("dual", ["x", "y", "a", "b", "scales", "out"])
def test_updates_refuse_tangents(anywhere, dual):
    t = {"x": torch.randn(5, 8), "y": torch.randn(5, 6), "a": torch.randn(1, 4, 8), "b": torch.randn(1, 6, 4),
         "scales": torch.ones(1), "out": torch.empty(5, 6)}
    with forward_ad.dual_level():
        args = {n: forward_ad.make_dual(v, torch.ones_like(v)) if n == dual else v for n, v in t.items()}
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.low_rank_update(**args, plan=_plan(5))
        with pytest.raises(AssertionError, match="a kernel would run"):
            nori_amd.low_rank_update(**t, plan=_plan(5))


@pytest.mark.parametrize("dual", ["x", "weight", "bias", "a", "b"])
def test_adapted_projections_refuse_tangents(anywhere, dual):
    t = {"x": torch.randn(5, 8), "weight": torch.randn(6, 8), "bias": torch.randn(6), "a": torch.randn(1, 4, 8),
         "b": torch.randn(1, 6, 4)}
    with forward_ad.dual_level():
        args = {n: forward_ad.make_dual(v, torch.ones_like(v)) if n == dual else v for n, v in t.items()}
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.adapted_linear(**args, plan=_plan(5))
