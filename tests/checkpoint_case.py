"""What activations kept in 8 bits stand for, exactly: codes and scales in 64 bits from their definition."""

import torch

GROUP = 128


def kept(x):
    """(codes, scales, the values in float64) of x [rows, cols] on the CPU: amax fp32(1/127), rounded, of each 128 columns, nearest codes with
    ties to even. The quotient of two fp32 values in 64 bits is exact enough to tell a half from its neighbours: one that
    is not a half is at least 2^-25 of itself away from it."""
    x = x.detach().double().cpu()
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    wide = torch.zeros(rows, groups * GROUP, dtype=torch.float64)
    wide[:, :cols] = x
    wide = wide.view(rows, groups, GROUP)
    amax = wide.abs().amax(-1, keepdim=True)
    scales = (amax.float() * torch.tensor(1 / 127, dtype=torch.float32)).double()
    codes = torch.where(scales > 0, (wide / torch.where(scales > 0, scales, 1.0)).round().clamp(-127, 127), 0.0)
    bad = ~torch.isfinite(amax)
    scales = torch.where(bad, torch.nan, scales)
    values = torch.where(bad, torch.nan, codes * torch.where(bad, 0.0, scales))
    return codes.view(rows, -1)[:, :cols], scales[..., 0], values.view(rows, -1)[:, :cols]


def activations(rows, cols, dtype, seed=0):
    """Unit scale, a few columns eight times as large, a row of zeros, one whose quotients are halves, rows of any size."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    x *= 1 + 7 * (torch.rand(cols, generator=g) < 0.05)
    if rows > 3:
        x[1] = 0
        halves = torch.arange(cols) % 127 + 0.5
        halves[::GROUP] = 127  # the scale is 1
        x[2] = halves
        x[3] *= 1e-4
    return x.to(dtype)
