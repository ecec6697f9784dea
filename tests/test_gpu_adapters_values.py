"""What the 16-bit types keep of x a^T and dy b between the two products: small values beside large ones, infinities
(GPU, against arithmetic that is exact).

In float16 a value h is kept to 2^-22 of itself and to 2^-38 of the largest finite one that it shares a power of two with (a
row of h in the update, an adapter's rows in the gradients), in bfloat16 to 2^-16 of itself. Every product below has one
term that is not zero, or equal ones, so that nothing else is rounded before the result, once, to half a step of its type.
"""
import pytest
import torch

from nori_amd import AdapterPlan, low_rank_update

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
KEPT = {F16: 2.0**-22, BF16: 2.0**-16, F32: 2.0**-24}
HALF_SUBNORMAL = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}

SIZES = [(1, 16), (40, 16), (40, 100), (33000, 5), (33000, 32), (33000, 64), (70000, 40), (33000, 128)]  # rows, rank


def _near(got, want, what, shared=0.0):
    """``shared``: the largest value whose power of two the terms of ``want`` share, times what they are multiplied by."""
    got = got.double().cpu()
    d = (got - want).abs()
    kept = want.abs() * KEPT[what] + (2.0**-38 * shared if what == F16 else 0.0)
    tol = kept + (want.abs() + kept) * torch.finfo(what).eps / 2 + HALF_SUBNORMAL[what]
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,rank", SIZES)
def test_small_beside_large_in_a_row(rows, rank, dtype):
    # h = (2^13 u, 2^-13 v, 0 ...), b sorts them: columns 0 and 1 take one each
    print(f"{rows} rows rank {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows + rank)
    x = (1 + torch.rand(rows, 2, generator=g)).to(dtype)
    a = torch.zeros(1, rank, 2, dtype=dtype)
    a[0, 0, 0], a[0, 1, 1] = 2.0**13, 2.0**-13
    b = torch.zeros(1, 70, rank, dtype=dtype)
    b[0, 0, 0], b[0, 1, 1] = 2.0**-4, 1.0
    y = torch.zeros(rows, 70, dtype=dtype)
    plan = AdapterPlan([0], rows, device=DEV)
    got = low_rank_update(*(t.to(DEV) for t in (x, y, a, b)), plan)
    _near(got[:, 0], x[:, 0].double() * 2.0**9, dtype)
    _near(got[:, 1], x[:, 1].double() * 2.0**-13, dtype, x[:, 0].double() * 2.0**13)
    assert not bool(got[:, 2:].any())
    # dx by the same two products
    d = [t.to(DEV).requires_grad_(True) for t in (torch.zeros(rows, 70, dtype=dtype), b.transpose(1, 2).contiguous(), a.transpose(1, 2).contiguous())]
    out = low_rank_update(d[0], torch.zeros(rows, 2, dtype=dtype, device=DEV), d[1], d[2], plan)
    (dx,) = torch.autograd.grad(out, d[0], x.to(DEV))
    _near(dx[:, 0], x[:, 0].double() * 2.0**9, dtype)
    _near(dx[:, 1], x[:, 1].double() * 2.0**-13, dtype, x[:, 0].double() * 2.0**13)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,rank", [(2, 4), (40, 16), (40, 100), (5000, 32), (5000, 64)])
def test_small_beside_large_in_an_adapters_rows(rows, rank, dtype):
    # rows 0, 2, ... have a large h and take column 0 of dy, rows 1, 3, ... a small one and column 1: db's entries are sums of equals
    print(f"{rows} rows rank {rank} {dtype}", flush=True)
    x = torch.zeros(rows, 2, dtype=dtype)
    x[0::2, 0], x[1::2, 1] = 1.25, 1.6181640625
    a = torch.zeros(1, rank, 2, dtype=dtype)
    a[0, 0, 0], a[0, 0, 1] = 2.0**12, 2.0**-12
    dy = torch.zeros(rows, 12, dtype=dtype)
    dy[0::2, 0], dy[1::2, 1] = 2.0**-10, 1.0
    leaf = torch.zeros(1, 12, rank, dtype=dtype).to(DEV).requires_grad_(True)
    out = low_rank_update(x.to(DEV), torch.zeros(rows, 12, dtype=dtype, device=DEV), a.to(DEV), leaf, AdapterPlan([0], rows, device=DEV))
    (db,) = torch.autograd.grad(out, leaf, dy.to(DEV))
    half = (rows + 1) // 2
    _near(db[0, 0, 0], torch.tensor(half * 1.25 * 4.0, dtype=torch.float64), dtype)
    _near(db[0, 1, 0], (rows - half) * x[1, 1].double() * 2.0**-12, dtype, (rows - half) * 1.25 * 2.0**12)
    assert not bool(db[0, 2:].any()) and not bool(db[0, :, 1:].any())


def _same_kind(got, want):
    """Infinities and NaN where ``want`` (float64) has them."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,rank", SIZES)
def test_infinities_come_out_as_the_formulas_have_them(rows, rank, dtype):
    print(f"{rows} rows rank {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows * 3 + rank)
    inf = float("inf")
    k, n = 24, 75
    # eighths of small integers: sums are exact, and half of the x a^T are what the type holds in one piece
    draw = lambda *s: torch.randint(-4, 5, s, generator=g).double() / 8  # noqa: E731
    x, a, b, dy = draw(rows, k), draw(1, rank, k), draw(1, n, rank), draw(rows, n)
    x[rows // 2, 3], x[0, 5], dy[rows // 3, 7] = inf, -inf, inf
    b[0, 11, 0], b[0, 12, rank - 1], b[0, 74, rank // 2], b[0, 13] = inf, -inf, inf, 0.0
    a[0, 1, 9] = inf
    y = draw(rows, n)
    d = [t.to(DEV, dtype) for t in (x, y, a, b)]
    for i in (0, 2, 3):
        d[i].requires_grad_(True)
    plan = AdapterPlan([0], rows, device=DEV)
    out = low_rank_update(*d, plan)
    dx, da, db = torch.autograd.grad(out, (d[0], d[2], d[3]), dy.to(DEV, dtype))
    h, gr = x @ a[0].T, dy @ b[0]
    for got, want in ((out, y + h @ b[0].T), (dx, gr @ a[0]), (da[0], gr.T @ x), (db[0], dy.T @ h)):
        _same_kind(got.detach(), want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,rank", SIZES)
def test_one_infinite_factor(rows, rank, dtype):
    # every other value finite: the infinity's column, and no other, is infinite, with the sign of x a^T and of dy b
    print(f"{rows} rows rank {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(rows * 5 + rank)
    draw = lambda *s: (torch.randint(1, 9, s, generator=g) * (2 * torch.randint(0, 2, s, generator=g) - 1)).double() / 8  # noqa: E731
    k, n = 24, 75
    x, a, b, y = draw(rows, k), torch.zeros(1, rank, k).double(), draw(1, n, rank), draw(rows, n)
    a[0, 0, 0], a[0, rank - 1, 1] = 1.0, 1.0  # x a^T: columns of x, exact in one piece
    b[0, 40, rank - 1] = float("inf")
    plan = AdapterPlan([0], rows, device=DEV)
    out = low_rank_update(*(t.to(DEV, dtype) for t in (x, y, a, b)), plan).double().cpu()
    assert torch.equal(torch.nonzero(~torch.isfinite(out)).unique(dim=0)[:, 1].unique(), torch.tensor([40]))
    want = x[:, 1 if rank > 1 else 0].sign() * float("inf")
    assert torch.equal(out[:, 40], want)
    # in the gradients, an infinite value of one row
    dy = draw(rows, n)
    x[rows // 2, 0] = float("inf")
    b[0, 40, rank - 1] = 1.0
    d = [t.to(DEV, dtype) for t in (x, y, a, b)]
    d[2].requires_grad_(True)
    (da,) = torch.autograd.grad(low_rank_update(*d, plan), d[2], dy.to(DEV, dtype))
    gr = dy[rows // 2] @ b[0]
    some = gr != 0
    assert torch.equal(da[0, some.to(DEV), 0].double().cpu(), gr[some].sign() * float("inf"))
    assert bool(torch.isnan(da[0, ~some.to(DEV), 0]).all()) and bool(torch.isfinite(da[0, :, 1:]).all())


@pytest.mark.parametrize("power", [-100, -112, -120, -125])
@pytest.mark.parametrize("rows,rank", SIZES)
def test_bfloat16_keeps_values_near_its_smallest(rows, rank, power):
    # x a^T = 2^power u with u of 8 bits, b brings it back to size: 2^-16 of it is left out at most, or 2^-133 below 2^-117
    print(f"{rows} rows rank {rank} 2^{power}", flush=True)
    g = torch.Generator().manual_seed(rows + rank)
    x = (1 + torch.randint(0, 128, (rows, 1), generator=g).double() / 128) * 2.0 ** (power // 2)
    a, b = torch.zeros(1, rank, 1).double(), torch.zeros(1, 70, rank).double()
    a[0, rank - 1], b[0, ::3, rank - 1] = 2.0 ** (power - power // 2), 2.0 ** (-power - 10)
    y = torch.zeros(rows, 70, dtype=BF16)
    d = [t.to(DEV, BF16) for t in (x, y, a, b)]
    leaf = d[3].float().requires_grad_(True)
    plan = AdapterPlan([0], rows, device=DEV)
    got = low_rank_update(*d, plan).double().cpu()
    want = (x * 2.0 ** (power - power // 2)) * b[0, :, rank - 1]
    kept = want.abs() * 2.0**-16 + 2.0**-133 * b[0, :, rank - 1]
    assert bool(((got - want).abs() <= kept + (want.abs() + kept) * 2.0**-8).all()), float(((got - want).abs() / want.abs().clamp_min(1e-30)).max())
    # and in the sums over rows: the same value in each of two rows, 2^k times it
    dy = torch.zeros(rows, 70, dtype=BF16)
    dy[0, 4] = dy[-1, 4] = 2.0 ** (-power - 10)
    (db,) = torch.autograd.grad(low_rank_update(d[0], d[1], d[2].float(), leaf, plan), leaf, dy.to(DEV))
    want = (x[0] + x[-1] if rows > 1 else x[0]) * 2.0 ** (power - power // 2) * 2.0 ** (-power - 10)
    assert float((db[0, 4, rank - 1].double().cpu() - want).abs()) <= float(want) * (2.0**-16 + 2.0**-22) + 2 * 2.0**-133 * 2.0 ** (-power - 10)
