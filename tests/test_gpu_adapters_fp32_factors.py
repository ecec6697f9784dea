"""Factors kept in fp32 beside 16-bit rows: what reaches them in a backward pass (GPU, against float64).

The sums over m rows are off by at most (m + 64) * 2^-24 of their terms' magnitudes in fp32, x a^T and dy b by (width + 64) *
2^-24 and, as operands, by 2^-22 (float16) or 2^-16 (bfloat16) of themselves and 2^-38 of the largest in theirs; the
factors enter rounded, which the formulas do too. Nothing is rounded to 16 bits after that.
"""
import pytest
import torch
from torch import nn

from nori_amd import AdapterPlan, LowRankAdapters, adapted_linear, low_rank_update

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _want(x, a, b, dy):
    """{name: (value, magnitude)} of one adapter's gradients in float64."""
    x, a, b, dy = (t.double().cpu() for t in (x, a, b, dy))
    h, g, hm, gm = x @ a.T, dy @ b, x.abs() @ a.abs().T, dy.abs() @ b.abs()
    return {"a": (g.T @ x, gm.T @ x.abs()), "b": (dy.T @ h, dy.abs().T @ hm)}


def _near(got, value, mag, rows, width, dtype):
    off = (rows + width + 128) * 2.0**-24 + (2.0**-16 if dtype == BF16 else 2.0**-21)
    assert got.dtype == F32
    worst = float(((got.detach().double().cpu() - value).abs() / (off * mag + 2.0**-149)).max())
    print(f"  {worst:.3f} of its tolerance", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k,n,rank", [(3, 16, 24, 4), (40, 64, 999, 16), (700, 127, 5, 33), (33000, 40, 72, 16), (9000, 5, 64, 70)])
def test_gradients_of_fp32_factors_are_not_rounded(rows, k, n, rank, dtype):
    print(f"{rows} rows {k} -> {n} rank {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + rank)
    x, dy = torch.randn(rows, k, generator=g).to(dtype), (2.0**-14 * torch.randn(rows, n, generator=g)).to(dtype)
    a, b = torch.randn(1, rank, k, generator=g) * 2.0**-8, torch.randn(1, n, rank, generator=g) * 2.0**-8
    leaves = [t.to(DEV).requires_grad_(True) for t in (a, b)]
    y = torch.zeros(rows, n, dtype=dtype, device=DEV)
    out = low_rank_update(x.to(DEV), y, *leaves, AdapterPlan([0], rows, device=DEV))
    assert out.dtype == dtype
    da, db = torch.autograd.grad(out, leaves, dy.to(DEV))
    want = _want(x, a[0].to(dtype), b[0].to(dtype), dy)
    _near(da[0], *want["a"], rows, n, dtype)
    _near(db[0], *want["b"], rows, k, dtype)
    # the same values as rounded factors give
    same = low_rank_update(x.to(DEV), y, *(t.detach().to(dtype) for t in leaves), AdapterPlan([0], rows, device=DEV))
    assert torch.equal(out.detach(), same)
    with torch.no_grad():
        assert torch.equal(low_rank_update(x.to(DEV), y, *leaves, AdapterPlan([0], rows, device=DEV)), same)


@pytest.mark.parametrize("through", ["projection", "adapters", "hooked"])
def test_slopes_below_16_bits_reach_the_adapters(through):
    # each gradient is about 2^-30: float16 has nothing there but zero
    torch.manual_seed(0)
    projection = nn.Linear(16, 24).to(DEV).requires_grad_(False)
    bank = LowRankAdapters(2, 16, 24, 4).to(DEV)
    nn.init.normal_(bank.b, std=2.0**-8)
    nn.init.normal_(bank.a, std=2.0**-8)
    x, dy = torch.randn(6, 16, device=DEV), (2.0**-22 * torch.randn(6, 24, device=DEV)).half()
    plan = AdapterPlan([1], 6, device=DEV)
    handle = projection.register_forward_hook(lambda *_: None) if through == "hooked" else None
    with torch.autocast("cuda", dtype=F16):
        if through == "projection":
            y = adapted_linear(x, projection.weight, projection.bias, bank.a, bank.b, plan, bank.scales)
        else:
            y = bank.linear(x, projection, plan)
    assert y.dtype == F16
    da, db = torch.autograd.grad(y, (bank.a, bank.b), dy)
    want = _want(x.half(), bank.a[1].half(), bank.b[1].half(), dy)
    _near(da[1], *want["a"], 6, 24, F16)
    _near(db[1], *want["b"], 6, 16, F16)
    assert not bool(da[0].any()) and not bool(db[0].any()) and bool(da[1].any()) and bool(db[1].any())
    if handle is not None:
        handle.remove()


def test_sums_past_16_bits_reach_the_adapters():
    x, dy = torch.full((4000, 8), 8.0, dtype=F16), torch.full((4000, 8), 4.0, dtype=F16)
    a, b = torch.full((1, 4, 8), 0.25, device=DEV, requires_grad=True), torch.full((1, 8, 4), 0.5, device=DEV, requires_grad=True)
    out = low_rank_update(x.to(DEV), torch.zeros(4000, 8, dtype=F16, device=DEV), a, b, AdapterPlan([0], 4000, device=DEV))
    da, db = torch.autograd.grad(out, (a, b), dy.to(DEV))
    # 4000 rows of 8 * 4 * 0.5 * 8 and of 4 * 8 * 8 * 0.25, to 2^-21 of them
    assert float((da - 512000.0).abs().max()) <= 512000.0 * 2.0**-21 and float((db - 256000.0).abs().max()) <= 256000.0 * 2.0**-21


def test_factors_of_two_types_are_refused():
    x, y = torch.zeros(4, 8, dtype=F16, device=DEV), torch.zeros(4, 6, dtype=F16, device=DEV)
    a, b = torch.zeros(1, 2, 8, device=DEV), torch.zeros(1, 6, 2, device=DEV)
    plan = AdapterPlan([0], 4, device=DEV)
    for one, other in ((a.half(), b), (a, b.half()), (a.bfloat16(), b.bfloat16()), (a.double(), b.double())):
        with pytest.raises(ValueError, match="low_rank_update: a is"):
            low_rank_update(x, y, one, other, plan)


def test_a_loss_over_many_rows_under_a_scaler():
    # the mean's slopes, 2^-26 each, are below float16: scaled, they reach every adapter that has rows
    from nori_amd import ReadoutAdapters

    torch.manual_seed(0)
    decoder = nn.Sequential(nn.Linear(32, 48), nn.LayerNorm(48), nn.GELU(), nn.Linear(48, 64)).to(DEV).requires_grad_(False)
    bank = ReadoutAdapters(decoder, 3, 8).to(DEV)
    nn.init.normal_(bank.first.b, std=0.1), nn.init.normal_(bank.last.b, std=0.1)
    states, plan = torch.randn(4, 2**18, 32, device=DEV), AdapterPlan([0, 2, -1, 0], 2**18, device=DEV)
    scaler = torch.amp.GradScaler("cuda")
    optimizer = torch.optim.SGD(bank.parameters(), lr=0.1)
    with torch.autocast("cuda", dtype=F16):
        q = bank(decoder, states, plan)
    scaler.scale(q.float().mean()).backward()
    scaler.unscale_(optimizer)
    for name, p in bank.named_parameters():
        assert bool(torch.isfinite(p.grad).all()) and not bool(p.grad[1].any()), name
        assert bool(p.grad[0].any()) and bool(p.grad[2].any()), name
    # dB of the last projection is a sum of x a^T by equal slopes: its columns' rows are alike, 1 / count each
    want = bank.last.b.grad[2][:1].expand(64, 8)
    assert float((bank.last.b.grad[2] - want).abs().max()) <= 2.0**-18 * float(want.abs().max())
    scaler.step(optimizer)
    scaler.update()


def test_a_captured_step_of_fp32_factors():
    ids, counts = [1, 0, -1, 1], [300, 40, 9, 700]
    g = torch.Generator().manual_seed(3)
    rows = sum(counts)
    x, y, dy = (torch.randn(rows, c, generator=g).to(DEV, F16) for c in (96, 130, 130))
    a, b = (torch.randn(*s, generator=g).to(DEV) * 0.1 for s in ((2, 16, 96), (2, 130, 16)))
    plan = AdapterPlan(ids, counts, device=DEV)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, a, b)]
        out = low_rank_update(leaves[0], y, leaves[1], leaves[2], plan)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    want = [t.clone() for t in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(4):
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(h, w) and torch.equal(e, w) for h, e, w in zip(outs, eager, want)), turn
    # the factors are read, and rounded, on each replay
    a.mul_(2.0)
    graph.replay()
    eager = step()
    torch.cuda.synchronize()
    assert all(torch.equal(h, e) for h, e in zip(outs, eager)) and not torch.equal(outs[0], want[0])
