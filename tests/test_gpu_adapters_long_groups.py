"""Gradients of long groups of rows, cut into parts that are joined, against sums that are exact (GPU).

Values are whole numbers. Those that go between the products lie between 2^11 and 2^15, so that neither of float16's two
pieces, nor of bfloat16's, is idle, and both hold them whole; sums of their products with -1, 0 and 1 stay below 2^24, where fp32 has
every whole number. So dA and dB, in fp32, are whole numbers but for float16's 2^-38 of a term (at most 60,000 of 2^15: 2^-7):
less than 0.25 off is right, and one row too many or too few is off by 1 or more.
"""
import math

import pytest
import torch

from nori_amd import AdapterPlan, low_rank_update

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

CASES = [
    # ids, rows, k, n, rank, adapters
    ([0], [33001], 1, 1, 40, 1),
    ([0], [57001], 5, 3, 40, 1),
    ([0], [33000], 3, 999, 16, 1),
    ([0, -1, 1], [30000, 90, 28011], 136, 199, 64, 2),
    ([-1, 0, 1], [100, 22007, 28000], 64, 96, 12, 2),
    ([1, 0, 2, 0], [300, 9001, 1, 12000], 127, 33, 5, 3),
    ([0, 1], [16501, 4503], 97, 65, 32, 2),
    ([2, 0, -1, 1], [257, 6000, 33, 20001], 72, 264, 100, 3),
    ([0, 1], [256, 257], 40, 24, 128, 2),
    ([0], [1025], 24, 40, 1, 1),
    (list(range(40)), [37 * i + 1 for i in range(40)], 56, 72, 17, 40),
]


def _whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g).double()


def _small(terms):
    """The most that one of the factors is, so that sums of ``terms`` products with up to 127 stay between 2^11 and 2^15."""
    return max(1, int(31 / math.sqrt(terms)))


def _near(got, want, last):
    """``last``: what the last 128 rows of the longest group add, which a part left out would at least lack."""
    assert got.dtype == F32
    off = float((got.double() - want).abs().max())
    print(f"  off by {off:.2e}", flush=True)
    assert off < 0.25
    # what this can see: neither zeros nor a result without those rows would pass
    assert float(want.abs().max()) > 100 and float((last.abs() >= 1).double().mean()) > 0.5


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("ids,counts,k,n,rank,adapters", CASES)
def test_every_row_of_a_long_group_is_summed_once(ids, counts, k, n, rank, adapters, dtype):
    print(f"{counts[:4]} rows {k} -> {n} rank {rank} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(counts) + k + n + rank)
    rows = sum(counts)
    whose = torch.tensor([i for i, c in zip(ids, counts) for _ in range(c)], device=DEV)
    longest = max(range(adapters), key=lambda i: int((whose == i).sum()))
    plan = AdapterPlan(ids, counts, device=DEV)
    y = torch.zeros(rows, n, dtype=dtype, device=DEV)
    for big in ("h", "g"):
        # h = x a^T large and dy of -1, 0, 1 for dB; g = dy b large and x of -1, 0, 1 for dA
        x, dy = (_whole(g, 127 if (big == "h") == left else 1, rows, c).to(DEV) for left, c in ((True, k), (False, n)))
        a = _whole(g, _small(k) if big == "h" else 1, adapters, rank, k).to(DEV)
        b = _whole(g, _small(n) if big == "g" else 1, adapters, n, rank).to(DEV)
        leaves = [t.float().requires_grad_(True) for t in (a, b)]
        out = low_rank_update(x.to(dtype), y, *leaves, plan)
        got = torch.autograd.grad(out, leaves, dy.to(dtype))[1 if big == "h" else 0]
        want, last, size = torch.zeros_like(got, dtype=torch.float64), None, 0.0
        for i in range(adapters):
            at = torch.nonzero(whose == i).flatten()
            left, right = (dy[at], x[at] @ a[i].T) if big == "h" else (dy[at] @ b[i], x[at])
            want[i] = left.T @ right
            size = max(size, float((right if big == "h" else left).abs().max()))
            if i == longest:
                last = left[-128:].T @ right[-128:]
        assert 2**11 < size < 2**15 and float(want.abs().max()) < 2**24
        _near(got, want, last)
