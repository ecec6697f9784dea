"""Training with activations kept in 8 bits: projections and SwiGLU gates whose backward pass reads int8 codes.

What a layer keeps for its backward pass is most of what a training step holds. ``checkpointed_linear`` is ``F.linear`` that
keeps its input, and ``checkpointed_silu_mul`` the SwiGLU gate that keeps its gate and up halves, as int8 codes with a float32
scale for every 128 columns of a row: 1.03 bytes an element. The results are those of the whole values; the gradients that
read what was kept (the weight's, the gate's) are those at the values that the codes stand for (csrc/checkpoint.hip,
csrc/checkpoint_grad.hip). Beside them stand ``trainable_attention`` (attention) and ``trainable_layer_norm`` (norm).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _native as nat
from .norm import _FLOATS, _first_derivative, _refuse_tangents, _rows_of, unviewed

__all__ = ["checkpointed_linear", "checkpointed_silu_mul"]

GROUP = 128  # NORI_CHECKPOINT_GROUP
MAX_COLUMNS = 2**20  # of a projection
MAX_HIDDEN = 2**24


def _storage(rows: int, cols: int, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised codes [rows, cols to the next 16] and scales [rows, groups]."""
    codes = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device=device)
    return codes, torch.empty((rows, -(-cols // GROUP)), dtype=torch.float32, device=device)


def _quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x's rows in 8 bits by ``nori_checkpoint_quantize``."""
    cols = int(x.shape[-1])
    x, rows, stride = _rows_of(x, cols)
    codes, scales = _storage(rows, cols, x.device)
    if rows:
        with nat.on(x.device):
            nat.check(
                nat.lib().nori_checkpoint_quantize(x.data_ptr(), nat.dtype_code(x.dtype), rows, cols, stride, codes.data_ptr(),
                                                   scales.data_ptr(), nat.stream_of(x.device)),
                "checkpointed_linear",
            )
    return codes, scales


def _linear(x, weight, bias):
    """(x weight^T + bias, the weight as it entered the product)."""
    w = weight if weight.dtype == x.dtype else weight.to(x.dtype)
    b = bias if bias is None or bias.dtype == x.dtype else bias.to(x.dtype)
    with torch.autocast("cuda", enabled=False):
        if x.dim() == 2:
            return F.linear(x, w, b), w
        # (one product: rows that do not fold would be a batch of them)
        return unviewed(F.linear(x.reshape(-1, x.shape[-1]), w, b), (*x.shape[:-1], w.shape[0])), w


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.grad_dtypes = weight.dtype, None if bias is None else bias.dtype
        y, w = _linear(x, weight, bias)
        kept = _quantized(x) if ctx.needs_input_grad[1] else (None, None)
        ctx.save_for_backward(w if ctx.needs_input_grad[0] else None, *kept)
        ctx.cols = int(x.shape[-1])
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        w, codes, scales = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        n, k, device = int(dy.shape[-1]), ctx.cols, dy.device
        dx = dw = db = None
        if need_x:
            with torch.autocast("cuda", enabled=False):
                dx = torch.matmul(dy.reshape(-1, n), w).view(*dy.shape[:-1], k)
        if need_w or need_b:
            w_dtype, b_dtype = ctx.grad_dtypes
            dy, rows, stride = _rows_of(dy, n)
            if stride > 2**24:
                dy, stride = dy.contiguous(), n
            make = torch.empty if rows else torch.zeros
            dw = make((n, k), dtype=w_dtype, device=device) if need_w else None
            db = make((n,), dtype=b_dtype, device=device) if need_b else None
            if rows:
                lib, dtype = nat.lib(), nat.dtype_code(dy.dtype)
                with nat.on(device):
                    size = lib.nori_checkpoint_grad_workspace_bytes(dtype, nat.dtype_code(w_dtype) if need_w else dtype, rows, n, k)
                    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
                    nat.check(
                        lib.nori_checkpoint_grad(
                            dy.data_ptr(), dtype, rows, n, stride, nat.ptr(codes), nat.ptr(scales), k, nat.ptr(dw),
                            nat.dtype_code(w_dtype), nat.ptr(db), 0 if b_dtype is None else nat.dtype_code(b_dtype), nat.ptr(workspace),
                            size, nat.stream_of(device),
                        ),
                        "checkpointed_linear backward",
                    )
        return dx, dw, db


def checkpointed_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` that keeps x in 8 bits for the weight's gradient: x [..., in] float32, float16 or bfloat16, weight
    [out, in] and bias [out] or None of x's dtype or float32 (rounded to x's for the products; their gradients, summed in fp32,
    keep their own dtype). in and out up to 2^20. Where autocast is on x, and 16-bit weights, are cast to its dtype.

    The result and the gradients of x and bias are ``F.linear``'s. The weight's is dy^T x with x the values that the codes stand
    for (``code * scale``, scale = amax times fp32(1/127) of 128 columns of a row, nearest codes, ties to even); a group of columns that
    holds an infinity or NaN stands for NaN. A weight of x's dtype has these values rounded to it for the product. A float32 weight beside
    16-bit x, as under autocast, has them whole, and each term dy * x to 2^-22 of itself and 2^-33 of the largest among 128 neighbouring
    outputs: an output whose slopes are far below its neighbours' keeps fewer bits. Such a weight is cast on each call, and the cast
    kept where x asks for a gradient.

    First derivatives, in reverse mode; sums have a fixed order, so the same inputs give the same bits. Without a gradient of the
    weight nothing is kept of x."""
    if weight.dim() != 2 or min(weight.shape) == 0:
        raise ValueError(f"weight must be [out, in], got {tuple(weight.shape)}")
    n, k = (int(s) for s in weight.shape)
    if max(n, k) > MAX_COLUMNS:
        raise NotImplementedError(f"checkpointed_linear takes up to {MAX_COLUMNS} columns, got {k} -> {n}")
    if x.dim() == 0 or int(x.shape[-1]) != k:
        raise ValueError(f"x {tuple(x.shape)} does not end in the weight's {k} inputs")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias {tuple(bias.shape)} does not match {n} outputs")
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in _FLOATS:
            raise NotImplementedError(f"checkpointed_linear takes float32/float16/bfloat16, got {name} {t.dtype}")
    _refuse_tangents("checkpointed_linear", x, weight, bias)
    nat.require_device(x, weight, bias)
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x = x.to(dtype)
        weight, bias = (t if t is None or t.dtype == torch.float32 else t.to(dtype) for t in (weight, bias))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"checkpointed_linear: {name} is {t.dtype}, x {x.dtype}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _CheckpointedLinear.apply(x, weight, bias)
    return _linear(x, weight, bias)[0]


class _CheckpointedSiluMul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu, hidden):
        y, codes, scales = _silu_mul(gu, hidden, True)
        ctx.save_for_backward(codes, scales)
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        hidden = int(dy.shape[-1])
        dgu = torch.empty((*dy.shape[:-1], 2 * hidden), dtype=dy.dtype, device=dy.device)
        dy, rows, stride = _rows_of(dy, hidden)
        if rows:
            with nat.on(dy.device):
                nat.check(
                    nat.lib().nori_checkpoint_silu_mul_backward(codes.data_ptr(), scales.data_ptr(), nat.dtype_code(dy.dtype), rows, hidden,
                                                                dy.data_ptr(), stride, dgu.data_ptr(), nat.stream_of(dy.device)),
                    "checkpointed_silu_mul backward",
                )
        return dgu, None


def _silu_mul(gu, hidden, keep):
    """(silu(g) u, codes and scales of g's rows and then u's where they are kept, None else)."""
    y = torch.empty((*gu.shape[:-1], hidden), dtype=gu.dtype, device=gu.device)
    gu, rows, stride = _rows_of(gu, 2 * hidden)
    codes, scales = _storage(2 * rows, hidden, gu.device) if keep else (None, None)
    if rows:
        with nat.on(gu.device):
            nat.check(
                nat.lib().nori_checkpoint_silu_mul(gu.data_ptr(), nat.dtype_code(gu.dtype), rows, hidden, stride, y.data_ptr(),
                                                   nat.ptr(codes), nat.ptr(scales), nat.stream_of(gu.device)),
                "checkpointed_silu_mul",
            )
    return y, codes, scales


def checkpointed_silu_mul(gu: torch.Tensor, hidden: int) -> torch.Tensor:
    """``F.silu(gu[..., :hidden]) * gu[..., hidden:]`` of a stacked [gate | up] projection that keeps both halves in 8 bits for its
    gradient: gu [..., 2 * hidden] float32, float16 or bfloat16, hidden up to 2^24; the result in gu's dtype, formed in fp32 and
    rounded once (``silu_mul``, without a gradient, rounds after silu too).

    The gradient is that of the formula at the values that the codes stand for, each half in groups of 128 columns of its own,
    as in ``checkpointed_linear``. First derivatives, in reverse mode; nothing is kept where gu asks for no gradient."""
    hidden = int(hidden)
    if hidden < 1 or gu.dim() == 0 or gu.shape[-1] != 2 * hidden:
        raise ValueError(f"checkpointed_silu_mul expects the [gate | up] width {2 * hidden}, got {tuple(gu.shape)}")
    if hidden > MAX_HIDDEN:
        raise NotImplementedError(f"checkpointed_silu_mul takes up to {MAX_HIDDEN} hidden columns, got {hidden}")
    if gu.dtype not in _FLOATS:
        raise NotImplementedError(f"checkpointed_silu_mul takes float32/float16/bfloat16, got {gu.dtype}")
    _refuse_tangents("checkpointed_silu_mul", gu)
    nat.require_device(gu)
    if torch.is_grad_enabled() and gu.requires_grad:
        return _CheckpointedSiluMul.apply(gu, hidden)
    return _silu_mul(gu, hidden, False)[0]
