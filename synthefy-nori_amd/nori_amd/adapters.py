"""Low-rank adapters of many tables beside a shared projection, and the readout that is fitted with them.

A batch of tables goes through one frozen model; each table's rows may take an adapter of its own,
``out = y + s (x A^T) B^T`` with ``y`` the shared projection's output, A [rank, in] and B [out, rank].
``low_rank_update`` is that update and its gradients for every row of the batch in one call
(csrc/low_rank.hip), ``AdapterPlan`` says which rows take which adapter, ``LowRankAdapters`` holds the
factors of one projection, and ``ReadoutAdapters`` those of a quantile decoder
(``FeaturesTransformer.reg_y_decoder``): trained on the row states of the frozen model, served for many
tables at once.
"""

from __future__ import annotations

from typing import Sequence

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules import module as _module_base

from . import _native as nat
from .layer import _hooked
from .norm import _FLOATS, _first_derivative, _refuse_tangents, _rows_of, _strided_rows, trainable_layer_norm

__all__ = ["AdapterPlan", "LowRankAdapters", "ReadoutAdapters", "adapted_linear", "low_rank_update"]

MAX_RANK = 128  # NORI_LOW_RANK_MAX
MAX_COLUMNS = 2**20  # NORI_LOW_RANK_COLUMNS


class AdapterPlan:
    """Which adapter each row of a batch takes: ``adapters[i]`` (-1: none) for the ``rows[i]`` rows of table
    i, the tables one after another along the batch's flattened rows; ``rows`` is one number where every
    table has as many. Rows of padding are tables of their own, with -1.

    Made on the host once a batch and copied to ``device``: the rows sorted by adapter, so that tables which
    share an adapter share its tiles. It can be used by any number of calls and graphs on that device."""

    def __init__(self, adapters: Sequence[int], rows: int | Sequence[int], *, device: torch.device | str):
        ids = _whole_numbers(adapters)
        counts = _whole_numbers(rows)
        if ids.ndim != 1 or counts.ndim > 1:
            raise ValueError(f"adapters and rows are sequences of numbers, got shapes {ids.shape} and {counts.shape}")
        if counts.ndim == 0:
            counts = np.full(ids.shape, counts)
        if len(counts) != len(ids):
            raise ValueError(f"{len(ids)} adapters for {len(counts)} tables")
        if (counts < 0).any():
            raise ValueError("a table cannot have a negative number of rows")
        if (ids < -1).any():
            raise ValueError("adapters are numbered from 0; -1 is none")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"nori_amd kernels run on a ROCm GPU; got a plan for {device}")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        longest = int(counts.max(initial=0))  # (a sum of longer ones may pass 64 bits)
        self.rows = longest if longest > 2**29 else int(counts.sum())
        if self.rows > 2**29:
            raise NotImplementedError(f"a plan takes up to {2**29} rows, got {self.rows}")
        self.most = int(ids.max(initial=-1))  # an adapter bank has more than this many
        if self.most > 2**31 - 2:
            raise ValueError(f"adapter {self.most} is out of range")
        order, starts, groups = _grouped(ids, counts)
        self.adapters = tuple(groups[groups >= 0].tolist())  # those with rows, ascending
        self.groups = len(groups)
        self.longest = int(np.diff(starts)[groups >= 0].max(initial=0))  # the most rows of one adapter
        self._packed = torch.from_numpy(np.concatenate([starts, groups, order], dtype=np.int32, casting="unsafe")).to(device)
        self._streams: set[int] = set()

    def used_on(self, stream: int) -> None:
        """Keeps the plan's memory, once the plan is gone, from what other streams do before ``stream``, the device's
        current one, is through with it: no caller has the tensor to tell the allocator so."""
        if stream not in self._streams:
            self._packed.record_stream(torch.cuda.current_stream(self.device))
            self._streams.add(stream)

    def __getstate__(self):
        return {**self.__dict__, "_streams": set()}  # a copy's memory is its own

    # Taken from the tensor on each call: a copy of the plan, or one loaded elsewhere, has memory of its own.
    @property
    def device(self) -> torch.device:
        return self._packed.device

    @property
    def starts(self) -> torch.Tensor:
        return self._packed[: self.groups + 1]

    @property
    def ids(self) -> torch.Tensor:
        return self._packed[self.groups + 1 : 2 * self.groups + 1]

    @property
    def order(self) -> torch.Tensor:
        return self._packed[2 * self.groups + 1 :]

    @property
    def pointers(self) -> tuple[int, int, int]:
        """Of ``order``, ``starts`` and ``ids``."""
        at = self._packed.data_ptr()
        return at + 4 * (2 * self.groups + 1), at, at + 4 * (self.groups + 1)


def _whole_numbers(values) -> np.ndarray:
    values = np.asarray(values)
    if values.size and values.dtype.kind not in "iu":
        raise TypeError(f"whole numbers are wanted, got {values.dtype}")
    if values.dtype == np.uint64:
        values = np.minimum(values, np.uint64(2**63 - 1))  # stays out of range, where a cast would wrap to -1
    return values.astype(np.int64)


def _grouped(ids: np.ndarray, counts: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(the rows by ascending adapter, where each adapter's begin and the end, the adapters), tables and
    rows of one adapter in their order, adapters without rows left out."""
    ids, first, counts = ids[counts > 0], (np.cumsum(counts) - counts)[counts > 0], counts[counts > 0]
    by = np.argsort(ids, kind="stable")
    ids, first, counts = ids[by], first[by], counts[by]
    total = int(counts.sum())
    at = np.cumsum(counts) - counts
    order = np.arange(total, dtype=np.int64) + np.repeat(first - at, counts)
    groups, where = np.unique(ids, return_index=True)
    return order, np.append(at[where], total), groups


def _update(x, y, a, b, plan, scales, out, keep):
    """``out`` = y + update by ``nori_low_rank_update``; returns h [rows, rank] for the gradients where it is to
    be kept, None else."""
    k, n, rank = int(x.shape[-1]), int(out.shape[-1]), int(a.shape[1])
    x, rows, xs = _rows_of(x, k)
    if rows == 0:
        return torch.empty((0, rank), dtype=torch.float32, device=x.device) if keep else None
    y, _, ys = _rows_of(y, n)
    layout = _strided_rows(out, n)
    if layout is None:
        raise ValueError(f"out {tuple(out.shape)} has strides {out.stride()}: its rows must be at one stride")
    device = x.device
    h = torch.empty((rows, rank), dtype=torch.float32, device=device) if keep else None
    lib, dtype = nat.lib(), nat.dtype_code(x.dtype)
    with nat.on(device):
        size = lib.nori_low_rank_workspace_bytes(dtype, rows, k, n, rank, plan.groups)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        stream = nat.stream_of(device)
        plan.used_on(stream)
        nat.check(
            lib.nori_low_rank_update(
                x.data_ptr(), dtype, rows, k, xs, y.data_ptr(), ys, a.data_ptr(), b.data_ptr(), nat.ptr(scales), int(a.shape[0]),
                rank, n, *plan.pointers, plan.groups, out.data_ptr(), layout[1], nat.ptr(h), nat.ptr(workspace), size,
                stream,
            ),
            "low_rank_update",
        )
    return h


def _gradients(dy, x, a, b, h, plan, scales, needs, base=None, grad_dtype=None):
    """(dx, da, db), None where not needed, by ``nori_low_rank_backward``, da and db of ``grad_dtype``, x's (the
    default) or float32; ``base`` [..., in] is what dx is added to, and overwritten."""
    need_x, need_a, need_b = needs
    k, n, rank = int(x.shape[-1]), int(dy.shape[-1]), int(a.shape[1])
    device = x.device
    x2, rows, xs = _rows_of(x, k)
    dy2, _, ys = _rows_of(dy, n)
    dx = (torch.empty(x.shape, dtype=x.dtype, device=device) if base is None else base) if need_x else None
    make = torch.empty_like if len(plan.adapters) == a.shape[0] else torch.zeros_like  # adapters no row takes: zeros
    da = make(a, dtype=grad_dtype) if need_a else None
    db = make(b, dtype=grad_dtype) if need_b else None
    if rows and any(needs):
        lib, dtype = nat.lib(), nat.dtype_code(x.dtype)
        call = lib.nori_low_rank_backward if grad_dtype in (None, x.dtype) else lib.nori_low_rank_backward_f32
        with nat.on(device):
            size = lib.nori_low_rank_backward_workspace_bytes(dtype, rows, k, n, rank, plan.groups, plan.longest, need_x, need_a,
                                                              need_b)
            workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
            stream = nat.stream_of(device)
            plan.used_on(stream)
            nat.check(
                call(
                    x2.data_ptr(), dtype, rows, k, xs, dy2.data_ptr(), n, ys, nat.ptr(base), k, a.data_ptr(), b.data_ptr(),
                    nat.ptr(scales), int(a.shape[0]), rank, *plan.pointers, plan.groups, plan.longest, nat.ptr(h), nat.ptr(dx), k,
                    nat.ptr(da), nat.ptr(db), nat.ptr(workspace), size, stream,
                ),
                "low_rank_update backward",
            )
    return dx, da, db


def _cast(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return t if t.dtype == dtype else t.to(dtype)


class _LowRankUpdate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, a, b, plan, scales):
        ctx.grad_dtype, a, b = a.dtype, _cast(a, x.dtype), _cast(b, x.dtype)
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        h = _update(x, y, a, b, plan, scales, out, ctx.needs_input_grad[3])  # b's gradient alone reads it
        ctx.save_for_backward(x, a, b, h, scales)
        ctx.plan = plan
        return out

    @staticmethod
    @_first_derivative
    def backward(ctx, dout):
        x, a, b, h, scales = ctx.saved_tensors
        need_x, need_y, need_a, need_b = ctx.needs_input_grad[:4]
        dx, da, db = _gradients(dout, x, a, b, h, ctx.plan, scales, (need_x, need_a, need_b), None, ctx.grad_dtype)
        return dx, (dout if need_y else None), da, db, None, None


def _projected(x, weight, bias, a, b, plan, scales, keep):
    """(F.linear(x, weight, bias), updated in place; h where it is to be kept, None else)."""
    with torch.autocast("cuda", enabled=False):
        y = F.linear(x, weight, bias)
    if _strided_rows(y, int(y.shape[-1])) is None:
        y = y.contiguous()
    return y, _update(x, y, a, b, plan, scales, y, keep)


class _AdaptedLinear(torch.autograd.Function):
    """A frozen projection and its low-rank update: the update's gradient of x is added in place to the
    projection's."""

    @staticmethod
    def forward(ctx, x, weight, bias, a, b, plan, scales):
        ctx.grad_dtype, a, b = a.dtype, _cast(a, x.dtype), _cast(b, x.dtype)
        y, h = _projected(x, weight, bias, a, b, plan, scales, ctx.needs_input_grad[4])
        ctx.save_for_backward(x, weight, a, b, h, scales)
        ctx.plan = plan
        return y

    @staticmethod
    @_first_derivative
    def backward(ctx, dy):
        x, weight, a, b, h, scales = ctx.saved_tensors
        need_x, _, _, need_a, need_b = ctx.needs_input_grad[:5]
        base = None
        if need_x:
            with torch.autocast("cuda", enabled=False):
                base = torch.matmul(dy.reshape(-1, dy.shape[-1]), weight).view(x.shape)
        dx, da, db = _gradients(dy, x, a, b, h, ctx.plan, scales, (need_x, need_a, need_b), base, ctx.grad_dtype)
        return dx, None, None, da, db, None, None


def _check(x, y, a, b, plan, scales):
    """The checks of ``low_rank_update``'s arguments; (a, b, scales) as the kernels take them."""
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError(f"factors are a [adapters, rank, in] and b [adapters, out, rank], got {tuple(a.shape)} and {tuple(b.shape)}")
    adapters, rank, k = (int(s) for s in a.shape)
    n = int(b.shape[1])
    if min(adapters, rank, k, n) == 0:
        raise ValueError(f"empty factors {tuple(a.shape)} and {tuple(b.shape)}")
    if rank > MAX_RANK:
        raise NotImplementedError(f"low_rank_update takes ranks up to {MAX_RANK}, got {rank}")
    if max(k, n) > MAX_COLUMNS or adapters >= 2**31:
        raise NotImplementedError(f"low_rank_update takes up to {MAX_COLUMNS} columns and 2^31 - 1 adapters, got {adapters} of {k} -> {n}")
    if x.dim() == 0 or int(x.shape[-1]) != k:
        raise ValueError(f"x {tuple(x.shape)} does not end in the factors' {k} inputs")
    if y is not None and tuple(y.shape) != (*x.shape[:-1], n):
        raise ValueError(f"y {tuple(y.shape)} is not the projection of x {tuple(x.shape)} to {n}")
    if x.dtype not in _FLOATS:
        raise NotImplementedError(f"low_rank_update takes float32/float16/bfloat16, got {x.dtype}")
    if y is not None and y.dtype != x.dtype:
        raise ValueError(f"low_rank_update: y is {y.dtype}, x {x.dtype}")
    if a.dtype != b.dtype or a.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"low_rank_update: a is {a.dtype}, b is {b.dtype}, x {x.dtype}")
    if not isinstance(plan, AdapterPlan):
        raise TypeError(f"plan must be an AdapterPlan, got {type(plan).__name__}")
    _refuse_tangents("low_rank_update", x, y, a, b, scales)
    device = nat.require_device(x, y, a, b, scales)
    if plan.device != device:
        raise RuntimeError(f"tensors on different devices: {device} and the plan's {plan.device}")
    if x.numel() // k != plan.rows:
        raise ValueError(f"x has {x.numel() // k} rows, the plan {plan.rows}")
    if plan.most >= adapters:
        raise ValueError(f"the plan names adapter {plan.most} of {adapters}")
    if scales is not None:
        if tuple(scales.shape) != (adapters,) or scales.dtype != torch.float32:
            raise ValueError(f"scales must be float32 [{adapters}], got {scales.dtype} {tuple(scales.shape)}")
        if scales.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("low_rank_update has no gradient for scales")
        scales = scales.contiguous()
    return a.contiguous(), b.contiguous(), scales


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The bytes from t's first element to its last."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two indices of t may be one element (expanded or overlapping dimensions)."""
    if t.numel() == 0:
        return False
    inside = 0
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda d: d[1]):
        if stride <= inside:
            return True
        inside += (size - 1) * stride
    return False


def _overlap(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether ``out`` and ``t`` may share elements. Columns side by side of one buffer's rows do not."""
    (lo, hi), (tlo, thi) = _span(out), _span(t)
    if out.numel() == 0 or t.numel() == 0 or hi <= tlo or thi <= lo:
        return False
    one, other = _strided_rows(out, int(out.shape[-1])), _strided_rows(t, int(t.shape[-1]))
    if one is None or other is None or one[1] != other[1] or one[1] == 0:
        return True
    size = out.element_size()
    row = one[1] * size
    start, at = 0, (tlo - lo) % row
    return not (at >= start + int(out.shape[-1]) * size and at + int(t.shape[-1]) * size <= row)


def low_rank_update(x: torch.Tensor, y: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: AdapterPlan,
                    scales: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y + scales[id] (x a[id]^T) b[id]^T`` with ``id`` the adapter ``plan`` gives each row; rows without
    one take ``y``. x [..., in], y [..., out], a [adapters, rank, in], b [adapters, out, rank] of one
    dtype (float32, float16 or bfloat16), ``scales`` float32 [adapters] or None for 1, rank up to 128, in and
    out up to 2^20. a and b may be float32 beside 16-bit x and y: they are rounded to x's dtype, their gradients, summed
    in fp32, are not.

    Products are summed in fp32 and the sum with y is rounded once. In float16 ``x a^T`` enters the second product to 2^-22
    of itself and 2^-38 of the largest in its row, in bfloat16 to 2^-16 of itself, in float32 whole.
    Differentiable in x, y, a and b (first derivatives, in reverse mode; adapters no row takes get zeros). ``out``, in
    inference, receives the result: a tensor of y's shape and dtype, y itself included, that shares no
    element with x, the factors or the scales."""
    _refuse_tangents("low_rank_update", out)
    a, b, scales = _check(x, y, a, b, plan, scales)
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in (x, y, a, b))
    given = out is not None
    if not given:
        if grad:
            return _LowRankUpdate.apply(x, y, a, b, plan, scales)
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    elif grad or out.requires_grad:
        raise ValueError("out is for inference: an argument asks for gradients")
    elif tuple(out.shape) != tuple(y.shape) or out.dtype != y.dtype or out.device != y.device:
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} is not y's {tuple(y.shape)} {y.dtype}")
    elif any(_overlap(out, t) for t in (x, a, b, scales) if t is not None) or (
            _overlap(out, y) and (out.data_ptr(), out.stride()) != (y.data_ptr(), y.stride())):
        raise ValueError("out shares elements with an input")
    elif _overlaps_itself(out):
        raise ValueError(f"out has strides {out.stride()}: its elements overlap")
    if plan.rows == 0:
        return out
    a, b = _cast(a, x.dtype), _cast(b, x.dtype)
    if _strided_rows(out, int(out.shape[-1])) is None:
        whole = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        _update(x, y, a, b, plan, scales, whole, False)
        return out.copy_(whole)
    _update(x, y, a, b, plan, scales, out, False)
    if given and not out.is_inference():  # (which have no versions)
        torch.autograd.graph.increment_version(out)  # for graphs that saved it: the kernel wrote behind torch's back
    return out


def _factors(a: torch.Tensor, b: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """a and b as ``low_rank_update`` takes them beside rows of ``dtype``: float32 ones as they are, so that their
    gradients are not rounded on the way back."""
    if a.dtype == b.dtype == torch.float32:
        return a, b
    return a.to(dtype), b.to(dtype)


def _watched(module: nn.Module) -> bool:
    """Whether a call of the module would run a hook, in its backward pass or forward."""
    return bool(_hooked(module) or module._backward_hooks or module._backward_pre_hooks
                or _module_base._global_backward_hooks or _module_base._global_backward_pre_hooks)


def adapted_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, a: torch.Tensor, b: torch.Tensor,
                   plan: AdapterPlan, scales: torch.Tensor | None = None) -> torch.Tensor:
    """``low_rank_update(x, F.linear(x, weight, bias), a, b, plan, scales)``, with x, the weights and the
    factors in the autocast dtype where autocast is on (the factors in x's dtype elsewhere; float32 factors keep
    float32 gradients). A frozen projection's output and x gradient are updated in place."""
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype)
    a, b = _factors(a, b, x.dtype)
    trained = torch.is_grad_enabled() and (weight.requires_grad or (bias is not None and bias.requires_grad))
    if trained:
        with torch.autocast("cuda", enabled=False):
            return low_rank_update(x, F.linear(x, weight, bias), a, b, plan, scales)
    _refuse_tangents("adapted_linear", weight, bias)
    nat.require_device(x, weight, bias)
    a, b, scales = _check(x, None, a, b, plan, scales)
    if tuple(weight.shape) != (b.shape[1], a.shape[2]):
        raise ValueError(f"the projection's weight {tuple(weight.shape)} does not match factors {tuple(a.shape)} and {tuple(b.shape)}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, a, b)):
        return _AdaptedLinear.apply(x, weight, bias, a, b, plan, scales)
    return _projected(x, weight, bias, _cast(a, x.dtype), _cast(b, x.dtype), plan, scales, False)[0]


class LowRankAdapters(nn.Module):
    """The adapters of one projection: factors ``a`` [adapters, rank, in] (normal, fan-in scale) and ``b``
    [adapters, out, rank] (zeros: a new adapter changes nothing), and ``scales`` [adapters], alpha / rank
    (alpha defaults to the rank), float32 through casts of the module."""

    def __init__(self, adapters: int, in_features: int, out_features: int, rank: int, *, alpha: float | None = None,
                 device=None, dtype=None):
        super().__init__()
        if min(adapters, in_features, out_features, rank) < 1:
            raise ValueError("adapters, in_features, out_features and rank must be positive")
        if rank > MAX_RANK:
            raise NotImplementedError(f"low_rank_update takes ranks up to {MAX_RANK}, got {rank}")
        self.a = nn.Parameter(torch.randn(adapters, rank, in_features, device=device, dtype=dtype) * in_features ** -0.5)
        self.b = nn.Parameter(torch.zeros(adapters, out_features, rank, device=device, dtype=dtype))
        self.register_buffer("scales", torch.full((adapters,), (rank if alpha is None else alpha) / rank, device=device,
                                                  dtype=torch.float32))

    def _apply(self, fn, recurse=True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:  # a cast of the module is the factors': the kernels take float32 scales
            self.scales = scales.to(self.scales.device)
        return self

    def forward(self, x: torch.Tensor, y: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
        """``low_rank_update`` of y by these adapters, their factors in x's dtype."""
        return low_rank_update(x, y, *_factors(self.a, self.b, x.dtype), plan, self.scales)

    def linear(self, x: torch.Tensor, projection: nn.Linear, plan: AdapterPlan) -> torch.Tensor:
        """``adapted_linear`` of x by ``projection`` and these adapters; a projection that is hooked or of
        another class is called."""
        if type(projection) is not nn.Linear or _watched(projection):
            y = projection(x)
            return self(x.to(y.dtype), y, plan)
        return adapted_linear(x, projection.weight, projection.bias, self.a, self.b, plan, self.scales)


class ReadoutAdapters(nn.Module):
    """Adapters of a quantile decoder, ``Linear -> LayerNorm -> GELU -> Linear``
    (``FeaturesTransformer.reg_y_decoder``): one bank beside each of its two projections.

    ``readout(decoder, states, plan)`` decodes row states [..., width] of many tables, each with its own
    adapter. The decoder itself is left as it is; freeze it (``requires_grad_(False)``) to train the adapters
    alone, and its LayerNorm's affine trains with them where it asks for gradients."""

    def __init__(self, decoder: nn.Sequential, adapters: int, rank: int, *, alpha: float | None = None):
        super().__init__()
        first, _, _, last = self._parts(decoder)
        where = dict(device=first.weight.device, dtype=torch.float32)
        self.first = LowRankAdapters(adapters, first.in_features, first.out_features, rank, alpha=alpha, **where)
        self.last = LowRankAdapters(adapters, last.in_features, last.out_features, rank, alpha=alpha, **where)

    @staticmethod
    def _parts(decoder: nn.Sequential) -> tuple[nn.Linear, nn.LayerNorm, nn.Module, nn.Linear]:
        whole = isinstance(decoder, nn.Sequential) and type(decoder).forward is nn.Sequential.forward
        parts = tuple(decoder) if whole else ()
        if len(parts) != 4 or not (isinstance(parts[0], nn.Linear) and isinstance(parts[1], nn.LayerNorm)
                                   and isinstance(parts[3], nn.Linear)) or len(parts[1].normalized_shape) != 1:
            raise ValueError("ReadoutAdapters takes a decoder of Linear, LayerNorm, activation, Linear")
        return parts

    def forward(self, decoder: nn.Sequential, states: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
        first, norm, activation, last = self._parts(decoder)
        if decoder._forward_hooks or decoder._forward_pre_hooks or decoder._backward_hooks or decoder._backward_pre_hooks:
            raise NotImplementedError("the decoder's parts are called one by one, which hooks of the whole would not see")
        h = self.first.linear(states, first, plan)
        # under autocast torch's layer norm answers in float32; outside it in its input's dtype
        wide = torch.float32 if torch.is_autocast_enabled("cuda") else h.dtype
        if type(norm) is not nn.LayerNorm or _watched(norm) or tuple(norm.normalized_shape) != (h.shape[-1],):
            h = norm(h)
        else:
            h = trainable_layer_norm(h, norm.weight, norm.bias, norm.eps, out_dtype=wide)
        h = activation(h)
        return self.last.linear(h, last, plan)
