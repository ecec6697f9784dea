"""Refusals of the projections and gates kept in 8 bits, and their definition against differences (no GPU needed)."""

import pytest
import torch

import nori_amd
from checkpoint_case import activations, kept
from nori_amd import _native as nat


def test_linear_refusals():
    x, w, b = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5)
    call = nori_amd.checkpointed_linear
    for args in ((x, w[0], b), (x, torch.zeros(0, 8), None), (x, torch.zeros(5, 0), None), (x, torch.zeros(5, 9), b), (x, w, torch.zeros(4)),
                 (torch.zeros(()), w, b), (x, w, torch.zeros(5, 1))):
        with pytest.raises(ValueError):
            call(*args)
    with pytest.raises(NotImplementedError):
        call(x.double(), w.double(), b.double())
    with pytest.raises(NotImplementedError):
        call(x, w.to(torch.int8), b)
    with pytest.raises(NotImplementedError, match="columns"):
        call(torch.empty(1, 1).expand(1, 2**20 + 1), torch.empty(1, 1).expand(1, 2**20 + 1))
    with pytest.raises(RuntimeError, match="GPU"):
        call(x, w, b)


def test_silu_mul_refusals():
    call = nori_amd.checkpointed_silu_mul
    for gu, hidden in ((torch.zeros(3, 8), 3), (torch.zeros(3, 8), 0), (torch.zeros(()), 1), (torch.zeros(3, 0), 0)):
        with pytest.raises(ValueError):
            call(gu, hidden)
    with pytest.raises(NotImplementedError):
        call(torch.zeros(3, 8).double(), 4)
    with pytest.raises(NotImplementedError, match="hidden"):
        call(torch.empty(1).expand(2**25 + 2), 2**24 + 1)
    with pytest.raises(RuntimeError, match="GPU"):
        call(torch.zeros(3, 8), 4)


def test_tangents_are_refused():
    from torch.autograd import forward_ad

    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.checkpointed_linear(dual, w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.checkpointed_silu_mul(dual, 4)


def test_the_library_refuses():
    """Aligned pointers that are never read: each call is refused, or has nothing to do."""
    lib, p = nat.lib(), 1 << 20
    bad, no, ok = nat.NORI_ERR_INVALID, nat.NORI_ERR_UNSUPPORTED, nat.NORI_OK
    q = lib.nori_checkpoint_quantize
    assert q(p, nat.NORI_I8, 2, 8, 8, p, p, None) == no
    assert q(p, nat.NORI_F16, -1, 8, 8, p, p, None) == bad
    assert q(p, nat.NORI_F16, 2, 0, 8, p, p, None) == bad
    assert q(p, nat.NORI_F16, 2, 8, -8, p, p, None) == bad
    assert q(p, nat.NORI_F16, 1 << 40, 8, 8, p, p, None) == no
    assert q(p, nat.NORI_F16, 1 << 33, 8, 8, p, p, None) == no  # more workgroups than one launch has
    assert q(None, nat.NORI_F16, 2, 8, 8, p, p, None) == bad
    assert q(p, nat.NORI_F16, 2, 8, 8, p + 8, p, None) == bad
    assert q(None, nat.NORI_F16, 0, 8, 8, None, None, None) == ok
    s = lib.nori_checkpoint_silu_mul
    assert s(p, nat.NORI_F16, 2, 8, -16, p, p, p, None) == bad
    assert s(p, nat.NORI_F16, 2, 8, 16, p, p, None, None) == bad
    assert s(p, nat.NORI_F16, 2, 8, 16, None, p, p, None) == bad
    assert s(p, nat.NORI_I8, 2, 8, 16, p, p, p, None) == no
    t = lib.nori_checkpoint_silu_mul_backward
    assert t(p, p, nat.NORI_F16, 2, 8, p, -8, p, None) == bad
    assert t(p, None, nat.NORI_F16, 2, 8, p, 8, p, None) == bad
    assert t(None, None, nat.NORI_F16, 0, 8, None, 8, None, None) == ok
    g = lib.nori_checkpoint_grad
    f16, f32 = nat.NORI_F16, nat.NORI_F32
    assert g(p, nat.NORI_I8, 2, 8, 8, p, p, 8, p, f32, p, f32, None, 0, None) == no
    assert g(p, f16, 2, 8, 8, p, p, 8, p, nat.NORI_BF16, p, f32, None, 0, None) == no
    assert g(p, f32, 2, 8, 8, p, p, 8, p, f16, p, f32, None, 0, None) == no
    assert g(p, f16, 2, 0, 8, p, p, 8, p, f32, p, f32, None, 0, None) == bad
    assert g(p, f16, 2, 8, -8, p, p, 8, p, f32, p, f32, None, 0, None) == bad
    assert g(p, f16, 2, 8, (1 << 24) + 1, p, p, 8, p, f32, p, f32, None, 0, None) == no
    assert g(p, f16, 2, 8, 8, None, p, 8, p, f32, p, f32, None, 0, None) == bad
    assert g(p, f16, 2, (1 << 20) + 1, 1 << 21, p, p, 8, p, f32, p, f32, None, 0, None) == no
    need = lib.nori_checkpoint_grad_workspace_bytes(f16, f32, 100000, 64, 64)
    assert need > 0 and lib.nori_checkpoint_grad_workspace_bytes(f16, f32, 100, 64, 64) == 0
    assert g(p, f16, 100000, 64, 64, p, p, 64, p, f32, p, f32, p, need - 1, None) == bad
    assert g(p, f16, 100000, 64, 64, p, p, 64, p, f32, p, f32, p + 8, need, None) == bad
    assert g(p, f16, 2, 8, 8, p, p, 8, None, f32, None, f32, None, 0, None) == ok


def test_what_the_codes_stand_for():
    x = activations(9, 300, torch.float32)
    codes, scales, values = kept(x)
    assert codes.abs().max() == 127 and torch.equal(codes, codes.round())
    step = scales.repeat_interleave(128, 1)[:, :300]
    assert ((values - x.double()).abs() <= step * (0.5 + 2.0**-20)).all()
    assert torch.equal(codes[2, 1:100], (torch.arange(1, 100) + 0.5).double().round())


def test_the_gate_against_differences():
    g = torch.Generator().manual_seed(0)
    a, b, d, va, vb = (torch.randn(50, generator=g).double() for _ in range(5))
    value = lambda s: ((a + s * va) * torch.sigmoid(a + s * va) * (b + s * vb) * d).sum()
    sig = torch.sigmoid(a)
    along = (d * b * sig * (1 + a * (1 - sig)) * va + d * a * sig * vb).sum()
    assert abs((value(1e-4) - value(-1e-4)) / 2e-4 - along) <= 1e-6


@pytest.mark.parametrize("shape", [(8,), (3, 8), (2, 3, 8), (2, 2, 3, 8)], ids=str)
@pytest.mark.parametrize("biased", [False, True])
def test_results_are_changed_in_place(monkeypatch, shape, biased):
    """What F.linear's result takes: sums and activations in place, of rows of any number of dimensions."""
    monkeypatch.setattr(nat, "require_device", lambda *t: None)
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(shape, generator=g).requires_grad_(True), torch.randn(5, 8, generator=g)
    b = torch.randn(5, generator=g) if biased else None
    residual = torch.randn(*shape[:-1], 5, generator=g).requires_grad_(True)
    slope = torch.randn(*shape[:-1], 5, generator=g)
    y = torch.relu(nori_amd.checkpointed_linear(x, w, b) + residual)
    expected = torch.autograd.grad(y, (x, residual), slope)
    z = nori_amd.checkpointed_linear(x, w, b)
    z += residual
    z = torch.relu_(z)
    assert torch.equal(z, y)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(z, (x, residual), slope), expected))
    with torch.no_grad():
        z = nori_amd.checkpointed_linear(x, w, b)
    z += residual
    assert torch.equal(torch.autograd.grad(z, residual, slope)[0], slope)
