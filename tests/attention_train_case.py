"""Attention with gradients in 64 bits from its formulas, and how far a kernel's results may be from them.

The bounds count roundings. h is half a step of the type (eps / 2), u = 2^-23 bounds one fp32 operation, with the matrix
instructions' inner sums. Per element, with A(.) the same sum over magnitudes:

* a logit is a sum of D products, scaled, and the argument of an exponential: p is off by r = u ((D + 8) L + 8) relative, L the
  largest sum of magnitudes behind a logit; so is the sum of a row, by r and its own additions (N / 32 + 24 in a row of
  registers), so a probability is off by 2 r + u (N / 32 + 24) =: R relative;
* p enters the second product rounded (h; in float16 under 2^14 forward and 2^15 backward, whose subnormals add 2^-39), its
  sum has N terms (rows: G Q terms for dv and dk), and the result is rounded: out is off by (h + R + N u) A(p v) + h |out|;
* delta = sum(dout out) takes out as it was rounded: off by A(dout e_out) + D u A(dout out); dout v by D u A(dout v);
* ds = p (dout v - delta) is off by those times p, by R |..| of each term, and by h |ds| from its rounding (in float16 under a
  power of two that keeps it to 2^-32 of the largest of its sum); dq, dk add the terms' u and the result's h.
"""

import math

import torch


def reference(q, kv, lengths, dout, scale=None):
    """(out, lse, dq, dkv) in float64 and what they may be off by, [BG, Q, H, D] and so on, for a kernel of q's dtype."""
    dtype = q.dtype
    h = torch.finfo(dtype).eps / 2
    u = 2.0**-23
    tiny = {torch.float16: 2.0**-39}.get(dtype, 0.0)
    small = {torch.float16: 2.0**-32}.get(dtype, 0.0)
    least = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps  # the type's own subnormal step
    bg, nq, heads, d = q.shape
    nk, kv_heads = kv.shape[1], kv.shape[3]
    group = heads // kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    q, do = (t.double().cpu().permute(0, 2, 1, 3) for t in (q, dout))
    kv = kv.double().cpu()
    if lengths is not None:
        per = bg // len(lengths)
        there = torch.arange(nk)[None] < torch.as_tensor(lengths).cpu().clamp(0, nk).repeat_interleave(per)[:, None]
        kv = torch.where(there[:, :, None, None, None], kv, torch.zeros(()).double())
    else:
        there = torch.ones(bg, nk, dtype=torch.bool)
    mask = there[:, None, None, :]
    k, v = (kv[:, :, i].permute(0, 2, 1, 3).repeat_interleave(group, 1) for i in (0, 1))
    t = lambda x: x.transpose(-1, -2)
    s = torch.where(mask, q @ t(k) * scale, -math.inf)
    top = s.amax(-1, keepdim=True) if nk else torch.full((bg, heads, nq, 1), -math.inf).double()
    p = torch.where(mask, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)[..., 0]
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    dp = do @ t(v)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * (ds @ k), scale * (t(ds) @ q), t(p) @ do
    # what each may be off by
    logits = (q.abs() @ t(k.abs())).amax().item() * abs(scale) if s.numel() else 0.0
    r = u * ((d + 8) * logits + 8)
    r2 = 2 * r + u * (nk / 32 + 24)
    rows = group * nq
    e_out = (h + r2 + nk * u) * (p @ v.abs()) + tiny * v.abs().sum(-2, keepdim=True) + h * out.abs() + least
    e_delta = (do.abs() * e_out).sum(-1, keepdim=True) + d * u * (do.abs() * out.abs()).sum(-1, keepdim=True)
    parts = p * (do.abs() @ t(v.abs()) + (do * out).abs().sum(-1, keepdim=True))
    e_ds = p * e_delta + (r2 + d * u + 4 * u) * parts + h * ds.abs()
    low = small * ds.abs()
    a = abs(scale)
    e_dq = a * ((e_ds + nk * u * ds.abs()) @ k.abs() + (low.amax(-1, keepdim=True) if nk else 0) * k.abs().sum(-2, keepdim=True)) + h * dq.abs() + least
    e_dk = a * (t(e_ds + rows * u * ds.abs()) @ q.abs() + (t(low).amax(-1, keepdim=True) if nq else 0) * q.abs().sum(-2, keepdim=True))
    e_dv = (h + r2 + rows * u) * (t(p) @ do.abs()) + tiny * do.abs().sum(-2, keepdim=True)

    def per_head(x):  # sums over the heads that share a key head
        return x.view(bg, kv_heads, group, nk, d).sum(2).permute(0, 2, 1, 3)

    dkv = torch.stack((per_head(dk), per_head(dv)), 2)
    e_dkv = torch.stack((per_head(e_dk), per_head(e_dv)), 2) + h * dkv.abs() + least
    e_dkv = torch.where(there[:, :, None, None, None], e_dkv, 0.0)
    back = lambda x: x.permute(0, 2, 1, 3)
    return (back(out), lse, back(dq), dkv), (back(e_out), None, back(e_dq), e_dkv)


def inputs(bg, nq, nk, heads, kv_heads, d, dtype, seed=0, q_scale=1.0, dout_scale=0.1):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(bg, nq, heads, d, generator=g) * q_scale).to(dtype)
    kv = torch.randn(bg, nk, 2, kv_heads, d, generator=g).to(dtype)
    dout = (torch.randn(bg, nq, heads, d, generator=g) * dout_scale).to(dtype)
    return q, kv, dout


def assert_near(name, got, expected, bound):
    got = got.double().cpu()
    assert got.shape == expected.shape, (name, got.shape, expected.shape)
    assert torch.isfinite(got).all(), f"{name} has values that are not finite"
    over = (got - expected).abs() - bound
    if over.numel():
        i = int(over.argmax())
        assert over.max() <= 0, (f"{name}: {got.flatten()[i].item()} for {expected.flatten()[i].item()}, "
                                 f"allowed {bound.flatten()[i].item()}")
