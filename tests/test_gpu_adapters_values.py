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
