"""trainable_attention's refusals, and its formulas in 64 bits against differences (no GPU needed)."""

import ctypes
import gc
import math
import weakref

import pytest
import torch

import nori_amd
from attention_train_case import inputs, reference
from nori_amd import _native as nat


def tensors(q=(2, 3, 4, 8), kv=(2, 5, 2, 2, 8), dtype=torch.float16):
    return torch.zeros(q, dtype=dtype), torch.zeros(kv, dtype=dtype)


@pytest.mark.parametrize("q, kv, error", [
    ((2, 3, 8), (2, 5, 2, 2, 8), ValueError),
    ((2, 3, 4, 8), (2, 5, 2, 8), ValueError),
    ((2, 3, 4, 8), (2, 5, 3, 2, 8), ValueError),
    ((2, 3, 4, 8), (1, 5, 2, 2, 8), ValueError),
    ((2, 3, 4, 8), (2, 5, 2, 2, 12), ValueError),
    ((2, 3, 4, 8), (2, 5, 2, 3, 8), ValueError),
    ((2, 3, 4, 8), (2, 5, 2, 0, 8), ValueError),
    ((2, 3, 0, 8), (2, 5, 2, 1, 8), ValueError),
    ((2, 3, 4, 6), (2, 5, 2, 2, 6), NotImplementedError),
    ((2, 3, 4, 132), (2, 5, 2, 2, 132), NotImplementedError),
    ((2, 3, 4, 0), (2, 5, 2, 2, 0), NotImplementedError),
])
def test_shapes(q, kv, error):
    with pytest.raises(error):
        nori_amd.trainable_attention(*tensors(q, kv))


def test_types_lengths_and_scale():
    q, kv = tensors()
    with pytest.raises(ValueError, match="float32"):
        nori_amd.trainable_attention(q, kv.float())
    with pytest.raises(NotImplementedError):
        nori_amd.trainable_attention(q.double(), kv.double())
    with pytest.raises(NotImplementedError):
        nori_amd.trainable_attention(q.to(torch.int8), kv.to(torch.int8))
    for scale in (math.nan, math.inf):
        with pytest.raises(ValueError, match="finite"):
            nori_amd.trainable_attention(q, kv, scale=scale)
    with pytest.raises(TypeError):
        nori_amd.trainable_attention(q, kv, [5, 5])
    with pytest.raises(TypeError):
        nori_amd.trainable_attention(q, kv, torch.ones(2))
    for lengths in (torch.ones(3, dtype=torch.int64), torch.ones(2, 1, dtype=torch.int64), torch.ones(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="key_lengths"):
            nori_amd.trainable_attention(q, kv, lengths)
    with pytest.raises(RuntimeError, match="GPU"):
        nori_amd.trainable_attention(q, kv)


def test_tangents_are_refused():
    from torch.autograd import forward_ad

    q, kv = tensors(dtype=torch.float32)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nori_amd.trainable_attention(forward_ad.make_dual(q, torch.ones_like(q)), kv)


def arguments(**changes):
    """Arguments of one call over pointers that are aligned and never read: each of these calls is refused, or has no rows."""
    some = 1 << 20
    args = nat.AttentionTrainArgs(bg=2, nq=3, nk=5, dtype=nat.NORI_F16, heads=4, kv_heads=2, d=8, q=some, q_bg=96, q_row=32, q_head=8,
                                  kv=some, kv_bg=160, kv_row=32, kv_half=16, kv_head=8, scale=1.0, out=some, lse=some, dout=some,
                                  do_bg=96, do_row=32, do_head=8, dq=some, dkv=some)
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes, status", [
    (dict(dtype=nat.NORI_I8), nat.NORI_ERR_UNSUPPORTED),
    (dict(bg=-1), nat.NORI_ERR_INVALID),
    (dict(heads=3), nat.NORI_ERR_INVALID),
    (dict(kv_heads=0), nat.NORI_ERR_INVALID),
    (dict(d=6), nat.NORI_ERR_UNSUPPORTED),
    (dict(d=132), nat.NORI_ERR_UNSUPPORTED),
    (dict(q_row=33), nat.NORI_ERR_UNSUPPORTED),
    (dict(kv_half=18), nat.NORI_ERR_UNSUPPORTED),
    (dict(q=(1 << 20) + 4), nat.NORI_ERR_UNSUPPORTED),
    (dict(kv=(1 << 20) + 2), nat.NORI_ERR_UNSUPPORTED),
    (dict(q=None), nat.NORI_ERR_INVALID),
    (dict(kv=None), nat.NORI_ERR_INVALID),
    (dict(out=None), nat.NORI_ERR_INVALID),
    (dict(scale=math.nan), nat.NORI_ERR_INVALID),
    (dict(lengths=1 << 20, length_group=0), nat.NORI_ERR_INVALID),
    (dict(nk=(1 << 30) + 4), nat.NORI_ERR_UNSUPPORTED),
    (dict(nq=1 << 30), nat.NORI_ERR_UNSUPPORTED),
    (dict(bg=1 << 40), nat.NORI_ERR_UNSUPPORTED),
    (dict(bg=1 << 27), nat.NORI_ERR_UNSUPPORTED),  # more workgroups than one launch has
])
def test_calls_of_the_library_are_refused(changes, status):
    lib = nat.lib()
    args = arguments(**changes)
    assert lib.nori_attention_train_forward(args, None) == status
    assert lib.nori_attention_train_backward(args, None) == status
    assert lib.nori_last_error()


def test_the_backward_call_needs_its_own():
    lib = nat.lib()
    need = lib.nori_attention_train_workspace_bytes(arguments(nq=300), True)
    assert need >= 2 * 4 * 300 * 4
    assert lib.nori_attention_train_workspace_bytes(arguments(), True) == 0  # few rows and keys
    for changes in (dict(lse=None), dict(dout=None), dict(workspace=None, workspace_bytes=need), dict(workspace=1 << 20, workspace_bytes=need - 1),
                    dict(workspace=(1 << 20) + 4, workspace_bytes=need)):
        assert lib.nori_attention_train_backward(arguments(nq=300, **changes), None) == nat.NORI_ERR_INVALID
    for changes in (dict(q_row=(1 << 24) + 4), dict(kv_row=-32), dict(do_row=1 << 25)):
        assert lib.nori_attention_train_backward(arguments(**changes), None) == nat.NORI_ERR_UNSUPPORTED
    assert lib.nori_attention_train_backward(arguments(do_row=34), None) == nat.NORI_ERR_UNSUPPORTED
    assert lib.nori_attention_train_forward(None, None) == nat.NORI_ERR_INVALID
    assert lib.nori_attention_train_backward(arguments(dq=None, dkv=None), None) == nat.NORI_OK
    for empty in (dict(bg=0), dict(nq=0)):
        assert lib.nori_attention_train_forward(arguments(**empty), None) == nat.NORI_OK


def test_workspaces_go_by_what_is_split():
    lib = nat.lib()
    assert lib.nori_attention_train_workspace_bytes(arguments(bg=1000), False) == 0
    one = arguments(bg=1, nq=1, nk=65536)
    assert lib.nori_attention_train_workspace_bytes(one, False) > 0
    assert lib.nori_attention_train_workspace_bytes(one, True) > lib.nori_attention_train_workspace_bytes(arguments(bg=1, nq=1, nk=65536, dq=None), True)


def test_the_formulas_against_differences():
    """What the kernels are held to: float64 gradients along a direction, the difference's third-order term at t^2."""
    q, kv, dout = inputs(2, 5, 7, 4, 2, 8, torch.float64, seed=1, dout_scale=1.0)
    lengths = [7, 3]
    (_, _, dq, dkv), _ = reference(q, kv, lengths, dout)
    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(q.shape, generator=g).double(), torch.randn(kv.shape, generator=g).double()
    t = 1e-4
    value = lambda s: (reference(q + s * a, kv + s * b, lengths, dout)[0][0] * dout).sum().item()
    along = ((dq * a).sum() + (dkv * b).sum()).item()
    assert abs((value(t) - value(-t)) / (2 * t) - along) <= 1e-5 * dout.abs().sum().item()


def test_copies_live_until_the_kernels_are_launched(monkeypatch):
    """Operands that are not aligned go in as copies, to whose memory the arguments point: what the call allocates for its workspace
    must not be theirs, in serving, in training or in the backward pass."""
    from nori_amd import attention

    copies, launches = [], []
    in_fours = attention._in_fours

    def copied(t):
        c = in_fours(t)
        assert c is not t
        copies.append(weakref.ref(c))
        return c

    def launch(name, args, backward, device):
        gc.collect()
        at = {c().data_ptr() for c in copies if c() is not None}
        launches.append(name)
        assert len(at) == len(copies), "a copy is gone before the launch"
        assert {args.q, args.kv} | ({args.dout} if backward else set()) <= at
        copies.clear()

    monkeypatch.setattr(attention, "_in_fours", copied)
    monkeypatch.setattr(attention, "_train_call", launch)
    monkeypatch.setattr(nat, "require_device", lambda *t: None)
    q = torch.randn(2 * 3 * 4 * 8 + 1, requires_grad=True)
    kv = torch.randn(2 * 5 * 2 * 2 * 8 + 1, requires_grad=True)
    odd = lambda: (q[1:].view(2, 3, 4, 8), kv[1:].view(2, 5, 2, 2, 8))
    with torch.no_grad():
        nori_amd.trainable_attention(*odd())
    out = nori_amd.trainable_attention(*odd())
    torch.autograd.grad(out, (q, kv), torch.randn(out.numel() + 1)[1:].view(out.shape))
    assert launches == ["nori_attention_train_forward"] * 2 + ["nori_attention_train_backward"]
