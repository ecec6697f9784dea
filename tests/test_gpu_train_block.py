"""The training operators together: a step through an encoder block -- norm, stacked projection, attention over padded tables, output
projection, residual, norm, SwiGLU -- as a program that fits one calls them."""

import pytest
import torch
import torch.nn.functional as F

import nori_amd
from checkpoint_case import kept

pytestmark = pytest.mark.gpu

TABLES, GROUPS, ROWS, WIDTH, HEADS, HIDDEN = 3, 2, 70, 88, 2, 117
LENGTHS = [70, 0, 33]


def parameters(dtype, device):
    g = torch.Generator().manual_seed(0)
    p = {"norm1": 1 + 0.1 * torch.randn(WIDTH, generator=g), "norm2": 1 + 0.1 * torch.randn(WIDTH, generator=g)}
    for name, n, k in (("qkv", 3 * WIDTH, WIDTH), ("out", WIDTH, WIDTH), ("gate_up", 2 * HIDDEN, WIDTH), ("down", WIDTH, HIDDEN)):
        p[name] = torch.randn(n, k, generator=g) * k**-0.5
        p[name + "_b"] = 0.1 * torch.randn(n, generator=g)
    x = torch.randn(TABLES * GROUPS, ROWS, WIDTH, generator=g)
    dy = torch.randn(x.shape, generator=g)
    return {k: v.to(device=device, dtype=dtype).requires_grad_(True) for k, v in p.items()}, x.to(device, dtype), dy.to(device, dtype)


def block(x, p, norm, linear, attend, gate):
    h = linear(norm(x, p["norm1"]), p["qkv"], p["qkv_b"]).view(*x.shape[:2], 3, HEADS, WIDTH // HEADS)
    a = attend(h[:, :, 0], h[:, :, 1:])
    x = x + linear(a.reshape(x.shape), p["out"], p["out_b"])
    h = linear(norm(x, p["norm2"]), p["gate_up"], p["gate_up_b"])
    return x + linear(gate(h), p["down"], p["down_b"])


def ours(x, p):
    lengths = torch.tensor(LENGTHS, device="cuda")
    return block(x, p, lambda t, w: nori_amd.trainable_layer_norm(t, w, None), nori_amd.checkpointed_linear,
                 lambda q, kv: nori_amd.trainable_attention(q, kv, lengths), lambda t: nori_amd.checkpointed_silu_mul(t, HIDDEN))


def stands_for(x):
    return kept(x.detach().float().reshape(-1, x.shape[-1]))[2].view(x.shape)


class Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        ctx.save_for_backward(stands_for(x), w)
        return F.linear(x, w, b)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        return dy @ w, dy.flatten(0, 1).t() @ x.flatten(0, 1), dy.flatten(0, 1).sum(0)


class Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        g, u = gu.split(HIDDEN, -1)
        ctx.save_for_backward(stands_for(g), stands_for(u))
        return g * torch.sigmoid(g) * u

    @staticmethod
    def backward(ctx, dy):
        g, u = ctx.saved_tensors
        s = torch.sigmoid(g)
        return torch.cat((dy * u * s * (1 + g * (1 - s)), dy * g * s), -1)


def attend(q, kv):
    there = torch.arange(ROWS)[None] < torch.tensor(LENGTHS).repeat_interleave(GROUPS)[:, None]
    s = torch.einsum("bihd,bjhd->bhij", q, kv[:, :, 0]) * (WIDTH // HEADS) ** -0.5
    p = torch.softmax(s.masked_fill(~there[:, None, None], -1e30), -1) * there[:, None, None]
    return torch.einsum("bhij,bjhd->bihd", p, kv[:, :, 1])


def test_a_block_in_fp32(cuda):
    """Against the same block in 64 bits. A kept value beside the middle of two codes may take the other one where fp32 rounds before it:
    with inputs off by 2^-18, 2^-10 of the values, by a step of amax / 127 of their 128 columns (below 2^-4 of their root
    mean square): 2^-9 of the 2-norm, and as it goes on through products that add or cancel, up to 2^-7."""
    p, x, dy = parameters(torch.float32, "cuda")
    y = ours(x, p)
    grads = torch.autograd.grad(y, list(p.values()), dy)
    p64, x64, dy64 = parameters(torch.float64, "cpu")
    norm = lambda t, w: F.layer_norm(t, (WIDTH,), w)
    y64 = block(x64, p64, norm, Linear.apply, attend, Gate.apply)
    expected = torch.autograd.grad(y64, list(p64.values()), dy64)
    assert (y.double().cpu() - y64).norm() <= 2.0**-16 * y64.norm()
    for name, a, b in zip(p, grads, expected):
        assert (a.double().cpu() - b).norm() <= 2.0**-7 * b.norm(), name


def test_a_step_under_autocast_keeps_less(cuda):
    """fp16 autocast with a loss scale: finite gradients of fp32 parameters, and a layer's input held in 8 bits."""
    p, x, dy = parameters(torch.float32, "cuda")
    with torch.autocast("cuda", dtype=torch.float16):
        y = ours(x, p)
    grads = torch.autograd.grad(y, list(p.values()), dy * 1024.0)
    assert all(g.dtype == torch.float32 and torch.isfinite(g).all() and g.any() for g in grads)
    kept_bytes = []
    x16 = torch.randn(4096, 512, device="cuda", dtype=torch.float16, requires_grad=True)
    w = torch.randn(64, 512, device="cuda", dtype=torch.float16, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept_bytes.append(t.numel() * t.element_size()) or t, lambda t: t):
        nori_amd.checkpointed_linear(x16, w)
    assert sum(kept_bytes) == 4096 * (512 + 4 * 4) + w.numel() * 2
