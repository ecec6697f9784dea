"""Low-rank updates of many tables (``low_rank_update``), their gradients and the readout fitted with them, on
the GPU against the formulas in 64 bits.

Tolerances, elementwise. Sums of K products in fp32 are off by at most (K + rank + 64) * 2^-24 of the sum of their
terms' magnitudes (any order of adding); x a^T and dy b are held to PIECE of the largest in their row where they enter the
second product (2^-24 in fp32, 2^-21 for float16's two halves, 2^-16 for bfloat16's two), the magnitude of which is
bounded by H = max over the rank of |x| |a|^T; each result is then rounded once, eps / 2 of its type.
"""
import pytest
import torch
from torch import nn

import nori_amd
from nori_amd import AdapterPlan, LowRankAdapters, ReadoutAdapters, adapted_linear, low_rank_update

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
PIECE = {F32: 2.0**-24, F16: 2.0**-21, BF16: 2.0**-16}
HALF_SUBNORMAL = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}


def _make(rows, k, n, rank, adapters, dtype, seed=0, dy_scale=0.1):
    g = torch.Generator().manual_seed(seed * 7919 + rows + k + n + rank)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": r(rows, k).to(dtype), "y": r(rows, n).to(dtype), "a": (r(adapters, rank, k) * k**-0.5).to(dtype),
            "b": (0.2 * r(adapters, n, rank)).to(dtype), "scales": 0.5 + torch.rand(adapters, generator=g),
            "dy": (dy_scale * r(rows, n)).to(dtype)}


def _rows(ids, counts):
    counts = [counts] * len(ids) if isinstance(counts, int) else counts
    return torch.tensor([i for i, c in zip(ids, counts) for _ in range(c)], dtype=torch.long)


def _formulas(s, whose):
    """{name: (value, magnitude)} in float64; the magnitude is what an error of one unit is relative to."""
    x, y, a, b, dy = (s[t].double() for t in ("x", "y", "a", "b", "dy"))
    scales = s["scales"].double() if s["scales"] is not None else torch.ones(a.shape[0]).double()
    out = {"y": [y.clone(), torch.zeros_like(y)], "dx": [torch.zeros_like(x) for _ in range(2)],
           "da": [torch.zeros_like(a) for _ in range(2)], "db": [torch.zeros_like(b) for _ in range(2)]}
    for i in range(a.shape[0]):
        at = torch.nonzero(whose == i).flatten()
        if not at.numel():
            continue
        xs, ds, f, c = x[at], dy[at], scales[i], scales[i].abs()
        h, g = f * xs @ a[i].T, f * ds @ b[i]
        hm = (c * xs.abs() @ a[i].abs().T).amax(1, keepdim=True)
        gm = (c * ds.abs() @ b[i].abs()).amax(1, keepdim=True)
        out["y"][0][at] += h @ b[i].T
        out["y"][1][at] = hm * b[i].abs().sum(1)
        out["dx"][0][at] = g @ a[i]
        out["dx"][1][at] = gm * a[i].abs().sum(0)
        out["da"][0][i], out["da"][1][i] = g.T @ xs, (gm.max() * xs.abs().sum(0)).expand(a.shape[1], -1)
        out["db"][0][i], out["db"][1][i] = ds.T @ h, (hm.max() * ds.abs().sum(0))[:, None].expand(-1, a.shape[1])
    return out


def _check(got, s, whose, names=("y", "dx", "da", "db")):
    dtype, k, n, rank = s["x"].dtype, s["x"].shape[1], s["y"].shape[1], s["a"].shape[1]
    want = _formulas(s, whose)
    for name in names:
        value, mag = want[name]
        # the second product's terms: the rank's, or an adapter's rows
        terms = (k if name in ("y", "db") else n) + rank + 64 + (len(whose) if name in ("da", "db") else 0)
        off = (terms * 2.0**-24 + PIECE[dtype]) * mag
        if name == "y":
            off = off + 2.0**-24 * (value.abs() + s["y"].double().abs())
        assert got[name].dtype == dtype and got[name].shape == value.shape
        tol = torch.finfo(dtype).eps / 2 * (value.abs() + off) + HALF_SUBNORMAL[dtype] + off
        worst = float(((got[name].double().cpu() - value).abs() / tol).max()) if value.numel() else 0.0
        print(f"  {name}: {worst:.3f} of its tolerance", flush=True)
        assert worst <= 1.0, (name, worst)


def _train(s, plan, y=None):
    d = {n: None if t is None else t.to(DEV) for n, t in s.items()}
    leaves = [d[n].detach().requires_grad_(True) for n in ("x", "a", "b")]
    out = low_rank_update(leaves[0], d["y"], leaves[1], leaves[2], plan, d["scales"])
    dx, da, db = torch.autograd.grad(out, leaves, d["dy"])
    return {"y": out.detach(), "dx": dx, "da": da, "db": db}


CASES = [
    # ids, rows, k, n, rank, adapters
    ([0], 1, 384, 999, 16, 1),
    ([1], 1, 33, 7, 1, 3),
    ([0, 1, 2, -1, 2], [1, 1, 1, 1, 1], 64, 48, 8, 3),
    ([3, 0, -1, 3], [5, 64, 17, 63], 128, 384, 16, 4),
    ([0, 1], [129, 300], 352, 1408, 16, 2),
    ([2, 0, 1, 2], [1, 200, 33, 0], 127, 385, 6, 3),
    ([0, -1, 1], [70, 30, 31], 560, 200, 32, 2),
    ([1, 0], [40, 100], 96, 130, 64, 2),
    ([0, 1], [20, 45], 100, 72, 100, 2),
    ([0], 50, 1, 1, 3, 1),
    ([-1, -1], 20, 40, 24, 4, 2),
    ([0] * 9, 7, 256, 384, 128, 1),
    (list(range(40)), 3, 72, 88, 12, 40),
    ([0], 700, 1680, 999, 16, 1),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ids,counts,k,n,rank,adapters", CASES)
def test_against_the_formulas(ids, counts, k, n, rank, adapters, dtype):
    whose = _rows(ids, counts)
    print(f"low-rank update of {len(ids)} tables, {len(whose)} rows {k} -> {n} rank {rank} {dtype}", flush=True)
    s = _make(len(whose), k, n, rank, adapters, dtype)
    plan = AdapterPlan(ids, counts, device=DEV)
    got = _train(s, plan)
    torch.cuda.synchronize()
    _check(got, s, whose)
    idle = whose < 0
    assert torch.equal(got["y"][idle.to(DEV)].cpu(), s["y"][idle])  # rows without an adapter keep their bits
    assert not bool(got["dx"][idle.to(DEV)].any())
    # inference, new and in place, gives the training pass's bits
    d = {n: t.to(DEV) for n, t in s.items()}
    fresh = low_rank_update(d["x"], d["y"], d["a"], d["b"], plan, d["scales"])
    assert torch.equal(fresh, got["y"])
    assert low_rank_update(d["x"], d["y"], d["a"], d["b"], plan, d["scales"], out=d["y"]) is d["y"]
    assert torch.equal(d["y"], fresh)


# enough rows, or adapters, that workgroups take tiles of many rows: ends of rows, ranks and groups of every kind
MANY = [
    ([0, -1, 1], [20000, 500, 14007], 130, 77, 5, 2),
    ([1, 0], [33333, 1], 64, 128, 16, 2),
    ([0], [33000], 3, 999, 16, 1),
    ([0, 1], [16501, 16503], 97, 65, 32, 2),
    ([0, 1, -1], [30000, 3001, 90], 560, 72, 24, 2),
    ([0, 1], [16400, 16700], 136, 200, 64, 2),
    ([1, 0], [32900, 200], 71, 130, 50, 2),
    ([0, 1], [20000, 13000], 128, 63, 128, 2),
    ([0, 1], [20000, 13011], 33, 321, 77, 2),
    ([1, -1, 0], [15000, 30, 18001], 40, 5, 8, 2),
    ([0], [33001], 1, 1, 40, 1),
    ([0, -1, 1], [9000, 100, 8009], 135, 203, 128, 2),
    ([1, 0], [17, 17003], 63, 64, 65, 2),
    ([0, -1, 1], [30000, 90, 28011], 136, 199, 64, 2),
    ([1, 0], [50001, 7003], 71, 130, 50, 2),
    ([0], [57001], 5, 3, 40, 1),
    ([0, 1, -1], [20000, 13, 1007], 72, 139, 30, 2),
    ([-1, 0, 1], [100, 22007, 28000], 64, 96, 12, 2),
    ([0, -1, 1], [17000, 100, 4009], 135, 203, 128, 2),
    ([1, 0], [13, 8500], 63, 264, 90, 2),
    ([-1 if i % 99 == 0 else (7 * i) % 540 for i in range(540)], [(i * 13) % 50 for i in range(540)], 56, 100, 9, 540),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ids,counts,k,n,rank,adapters", MANY)
def test_many_rows_against_the_formulas(ids, counts, k, n, rank, adapters, dtype):
    test_against_the_formulas(ids, counts, k, n, rank, adapters, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_many_rows_in_a_shared_buffer(dtype):
    # x, y and out as columns of one buffer's rows, at no vector's alignment: nothing beside them moves
    ids, counts = [1, -1, 0], [17000, 40, 16001]
    whose = _rows(ids, counts)
    s = _make(len(whose), 72, 85, 16, 2, dtype)
    plan = AdapterPlan(ids, counts, device=DEV)
    d = {n: t.to(DEV) for n, t in s.items()}
    buffer = torch.full((len(whose), 165), float("nan"), dtype=dtype, device=DEV)
    x, y = buffer[:, 3:75], buffer[:, 77:162]
    x.copy_(d["x"])
    y.copy_(d["y"])
    _check({"y": low_rank_update(x, y, d["a"], d["b"], plan, d["scales"]).contiguous()}, s, whose, names=("y",))
    before = buffer.clone()
    low_rank_update(x, y, d["a"], d["b"], plan, d["scales"], out=y)
    _check({"y": y.contiguous()}, s, whose, names=("y",))
    mask = torch.ones(165, dtype=torch.bool, device=DEV)
    mask[77:162] = False
    assert torch.equal(buffer[:, mask].view(torch.uint8), before[:, mask].view(torch.uint8))
    # non-finite rows stay in their rows
    d["x"][5, 3], d["x"][20000, 71] = float("inf"), float("nan")
    got = low_rank_update(d["x"], d["y"], d["a"], d["b"], plan, d["scales"])
    assert torch.nonzero(~torch.isfinite(got).all(1)).flatten().tolist() == [5, 20000]


def test_without_scales_and_one_gradient_at_a_time():
    ids, counts = [1, 0, -1], [30, 80, 9]
    s = _make(119, 96, 104, 8, 3, F16)  # adapter 2 has no rows: its gradients are zeros
    s["scales"] = None
    plan = AdapterPlan(ids, counts, device=DEV)
    whole = _train(s, plan)
    _check(whole, s, _rows(ids, counts))
    assert not bool(whole["da"][2].any()) and not bool(whole["db"][2].any())
    for one in ("x", "y", "a", "b"):
        d = {n: t.to(DEV).requires_grad_(n == one) for n, t in s.items() if t is not None}
        out = low_rank_update(d["x"], d["y"], d["a"], d["b"], plan)
        (grad,) = torch.autograd.grad(out, d[one], d["dy"].detach())
        assert torch.equal(grad, d["dy"].detach() if one == "y" else whole["d" + one]), one


@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_shapes(dtype):
    ids, rows = [2, -1, 0, 1], 25
    s = _make(100, 72, 56, 8, 3, dtype)
    plan = AdapterPlan(ids, rows, device=DEV)
    want = _train(s, plan)
    d = {n: t.to(DEV) for n, t in s.items()}
    # the columns of one buffer's rows, off any vector's alignment; rows at two strides; column-major rows
    buffer = torch.full((4, 25, 135), float("nan"), dtype=dtype, device=DEV)
    x, y = buffer[..., 3:75], buffer[..., 77:133]
    x.copy_(d["x"].view(4, 25, 72))
    y.copy_(d["y"].view(4, 25, 56))
    got = low_rank_update(x, y, d["a"], d["b"], plan, d["scales"])
    assert got.shape == (4, 25, 56) and torch.equal(got.reshape(100, 56), want["y"])
    turned = d["x"].view(4, 25, 72).transpose(0, 1).contiguous().transpose(0, 1)
    columns = d["y"].t().contiguous().t()
    assert torch.equal(low_rank_update(turned, d["y"].view(4, 25, 56), d["a"], d["b"], plan, d["scales"]).reshape(100, 56), want["y"])
    assert torch.equal(low_rank_update(d["x"], columns, d["a"], d["b"], plan, d["scales"]), want["y"])
    a = d["a"].transpose(1, 2).contiguous().transpose(1, 2)
    b = d["b"].transpose(0, 2).contiguous().transpose(0, 2)
    assert torch.equal(low_rank_update(d["x"], d["y"], a, b, plan, d["scales"]), want["y"])
    # out: a slice of the buffer beside x, in place there, and rows at two strides
    before = buffer.clone()
    assert low_rank_update(x, y, d["a"], d["b"], plan, d["scales"], out=y) is y
    assert torch.equal(y.reshape(100, 56), want["y"])
    mask = torch.ones(135, dtype=torch.bool, device=DEV)
    mask[77:133] = False
    assert torch.equal(buffer[..., mask].view(torch.uint8), before[..., mask].view(torch.uint8))  # nothing beside it moved
    out = torch.empty(25, 4, 56, dtype=dtype, device=DEV).transpose(0, 1)
    low_rank_update(x, d["y"].view(4, 25, 56), d["a"], d["b"], plan, d["scales"], out=out)
    assert torch.equal(out.reshape(100, 56), want["y"])
    # gradients of strided and broadcast inputs
    leaf = buffer.detach().clone().nan_to_num_(0.0).requires_grad_(True)
    z = low_rank_update(leaf[..., 3:75], d["y"].view(4, 25, 56), d["a"], d["b"], plan, d["scales"])
    z.backward(d["dy"].view(4, 25, 56))
    assert torch.equal(leaf.grad[..., 3:75].reshape(100, 72), want["dx"]) and not bool(leaf.grad[..., 75:].any())


def test_broadcast_rows_and_a_summed_loss():
    s = _make(30, 40, 24, 4, 2, F32)
    s["x"] = s["x"][:1].expand(30, 40)
    s["dy"] = torch.ones(30, 24)
    plan = AdapterPlan([0, 1], 15, device=DEV)
    d = {n: t.to(DEV) for n, t in s.items()}
    row = s["x"][:1].to(DEV).clone().requires_grad_(True)
    a = d["a"].clone().requires_grad_(True)
    low_rank_update(row.expand(30, 40), d["y"], a, d["b"], plan, d["scales"]).sum().backward()
    want = _formulas(s, _rows([0, 1], 15))
    off = (24 + 4 + 64 + 30) * 2.0**-24
    assert bool(((row.grad.double().cpu()[0] - want["dx"][0].sum(0)).abs() <= off * 4 * want["dx"][1].sum(0)).all())
    assert bool(((a.grad.double().cpu() - want["da"][0]).abs() <= off * 4 * want["da"][1]).all())


def test_no_rows():
    s = _make(0, 16, 8, 4, 2, F16)
    for ids, counts in (([], []), ([0, 1], [0, 0])):
        got = _train(s, AdapterPlan(ids, counts, device=DEV))
        assert got["y"].shape == (0, 8) and got["dx"].shape == (0, 16)
        assert not bool(got["da"].any()) and not bool(got["db"].any()) and got["da"].shape == (2, 4, 16)


def test_tables_that_share_an_adapter_and_any_order_of_tables():
    # the same rows under another order of tables: the same outputs, row for row
    s = _make(90, 64, 80, 8, 2, F16)
    d = {n: t.to(DEV) for n, t in s.items()}
    one = low_rank_update(d["x"], d["y"], d["a"], d["b"], AdapterPlan([0, 1, 0], 30, device=DEV), d["scales"])
    _check({"y": one}, s, _rows([0, 1, 0], 30), names=("y",))
    flip = torch.arange(90).flip(0).to(DEV)
    two = low_rank_update(d["x"][flip], d["y"][flip], d["a"], d["b"], AdapterPlan([0, 1, 0], 30, device=DEV), d["scales"])
    assert torch.equal(two[flip], one)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_small_large_and_non_finite_values(dtype):
    ids, counts = [0, 1], [40, 25]
    whose = _rows(ids, counts)
    plan = AdapterPlan(ids, counts, device=DEV)
    # gradients far below float16's normal numbers inside the products, and rows of very different sizes
    s = _make(65, 64, 48, 8, 2, dtype, dy_scale=2.0**-13)
    s["b"] *= 2.0**-6
    s["a"] *= 64
    s["x"][3] *= 2.0**-10
    s["x"][9] *= 2.0**7
    _check(_train(s, plan), s, whose)
    # x a^T past float16's largest value, its product with b inside it
    s = _make(65, 64, 48, 8, 2, dtype)
    s["x"] *= 256
    s["a"] *= 128
    s["b"] *= 2.0**-13
    _check(_train(s, plan), s, whose, names=("y",))
    # a non-finite row stays in its row, and in its adapter's gradients
    s = _make(65, 64, 48, 8, 2, dtype)
    s["x"][7, 3], s["x"][11, 0] = float("inf"), float("nan")
    got = _train(s, plan)
    for name in ("y",):
        bad = ~torch.isfinite(got[name]).all(1).cpu()
        assert bad.tolist() == [i in (7, 11) for i in range(65)]
    assert bool(torch.isfinite(got["dx"]).all())
    assert bool(torch.isfinite(got["da"][1]).all()) and bool(torch.isfinite(got["db"][1]).all())
    assert bool(torch.isnan(got["da"][0, :, 0]).all()) and bool(torch.isfinite(got["da"][0, :, 1]).all())
    # NaN in a row without an adapter, and in a factor no row takes, touches nothing
    s = _make(65, 64, 48, 8, 3, dtype)
    s["x"][2], s["a"][2], s["b"][2] = float("nan"), float("nan"), float("nan")
    idle = AdapterPlan([-1, 0, 1], [5, 35, 25], device=DEV)
    got = _train(s, idle)
    assert all(bool(torch.isfinite(got[n]).all()) for n in got)


def test_against_differences():
    ids, counts = [1, 0, -1], [3, 4, 1]
    s = _make(8, 6, 5, 2, 2, F32)
    whose = _rows(ids, counts)
    got = _train(s, AdapterPlan(ids, counts, device=DEV))
    d = {n: t.double() for n, t in s.items()}
    for name in ("x", "a", "b"):
        t, diff = d[name], torch.zeros_like(d[name])
        for i in range(t.numel()):
            old, ends = t.view(-1)[i].item(), []
            for step in (1e-5, -1e-5):
                t.view(-1)[i] = old + step
                ends.append(float((_formulas(d, whose)["y"][0] * d["dy"]).sum()))
            t.view(-1)[i] = old
            diff.view(-1)[i] = (ends[0] - ends[1]) / 2e-5
        # the function is quadratic in each factor at most: the differences are off by rounding, 1e-10 / 1e-5
        assert float((got["d" + name].double().cpu() - diff).abs().max()) <= 2e-5, name


def test_the_same_bits_again_and_on_another_stream():
    ids, counts = [4, 0, 2, -1, 4, 1], [300, 1000, 17, 60, 2000, 1]
    s = _make(sum(counts), 256, 384, 16, 5, F16)
    plan = AdapterPlan(ids, counts, device=DEV)
    want = _train(s, plan)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _train(s, plan)
    torch.cuda.current_stream().wait_stream(side)
    for again in (_train(s, plan), other):
        assert all(torch.equal(again[n], want[n]) for n in want)


def test_two_graphs_replayed_in_turn():
    cases = []
    for ids, counts, seed in (([0, 2, -1], [100, 64, 9], 1), ([1, 1, 0], [700, 3, 400], 2)):
        s = {n: t.to(DEV) for n, t in _make(sum(counts), 128, 200, 16, 3, F16, seed).items()}
        cases.append((s, AdapterPlan(ids, counts, device=DEV)))
    want = [_train(*c) for c in cases]
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_train(*c))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1, 1, 0):
            for t in outs[i].values():
                t.fill_(float("nan"))
            graphs[i].replay()
            eager = _train(*cases[1 - i])
            torch.cuda.synchronize()
            assert all(torch.equal(outs[i][n], want[i][n]) for n in want[i]), (turn, i)
            assert all(torch.equal(eager[n], want[1 - i][n]) for n in want[i])


def test_refusals():
    s = {n: t.to(DEV) for n, t in _make(10, 16, 12, 4, 2, F32).items()}
    x, y, a, b, scales = (s[n] for n in ("x", "y", "a", "b", "scales"))
    plan = AdapterPlan([0, 1], 5, device=DEV)
    with pytest.raises(ValueError, match="10 rows, the plan 9"):
        low_rank_update(x, y, a, b, AdapterPlan([0], 9, device=DEV))
    with pytest.raises(ValueError, match="adapter 2 of 2"):
        low_rank_update(x, y, a, b, AdapterPlan([0, 2], 5, device=DEV))
    with pytest.raises(ValueError, match="scales"):
        low_rank_update(x, y, a, b, plan, scales.half())
    with pytest.raises(NotImplementedError, match="scales"):
        low_rank_update(x, y, a, b, plan, scales.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="shares elements"):
        low_rank_update(x, x[:, :12], a, b, plan, out=x[:, :12])
    with pytest.raises(ValueError, match="shares elements"):
        low_rank_update(x, y, a, b, plan, out=torch.as_strided(y, (10, 12), (11, 1)))
    with pytest.raises(ValueError, match="not y's"):
        low_rank_update(x, y, a, b, plan, out=y.half())
    with pytest.raises(ValueError, match="gradients"):
        low_rank_update(x, y, a.clone().requires_grad_(True), b, plan, out=y)
    with pytest.raises(ValueError, match="overlap"):
        low_rank_update(x, y, a, b, plan, out=torch.zeros(1, 12, device=DEV).expand(10, 12))
    out = low_rank_update(x, y, a.clone().requires_grad_(True), b, plan)
    assert out.requires_grad
    with pytest.raises(ValueError, match="weight"):
        adapted_linear(x, torch.zeros(13, 16, device=DEV), None, a, b, plan)


# ------------------------------------------------------------------ the projection and the readout together
def _adapted_formula(x, weight, bias, a, b, whose, scales):
    y = x @ weight.T + (0 if bias is None else bias)
    for i in range(a.shape[0]):
        at = whose == i
        y = torch.where(at[:, None], y + scales[i] * (x @ a[i].T) @ b[i].T, y)
    return y


@pytest.mark.parametrize("frozen", [True, False])
def test_adapted_linear_and_its_gradients(frozen):
    ids, counts = [0, -1, 1], [20, 6, 31]
    whose = _rows(ids, counts)
    s = _make(57, 48, 36, 4, 2, F32)
    g = torch.Generator().manual_seed(5)
    weight, bias = torch.randn(36, 48, generator=g) * 48**-0.5, torch.randn(36, generator=g)
    plan = AdapterPlan(ids, counts, device=DEV)
    names = ["x", "a", "b"] + ([] if frozen else ["weight", "bias"])
    host = {"x": s["x"], "a": s["a"], "b": s["b"], "weight": weight, "bias": bias}
    d = {n: t.to(DEV).requires_grad_(n in names) for n, t in host.items()}
    y = adapted_linear(d["x"], d["weight"], d["bias"], d["a"], d["b"], plan, s["scales"].to(DEV))
    with torch.no_grad():
        served = adapted_linear(d["x"], d["weight"], d["bias"], d["a"], d["b"], plan, s["scales"].to(DEV))
    assert not served.requires_grad and torch.equal(served, y)
    got = torch.autograd.grad(y, [d[n] for n in names], s["dy"].to(DEV))
    e = {n: t.double().requires_grad_(True) for n, t in host.items()}
    want_y = _adapted_formula(e["x"], e["weight"], e["bias"], e["a"], e["b"], whose, s["scales"].double())
    want = torch.autograd.grad(want_y, [e[n] for n in names], s["dy"].double())
    # fp32 throughout: 200 roundings of terms of about the results' size
    assert float((y.detach().double().cpu() - want_y.detach()).abs().max()) <= 200 * 2.0**-24 * 8
    for name, have, need in zip(names, got, want):
        assert float((have.double().cpu() - need).abs().max()) <= 200 * 2.0**-24 * 8 * max(1.0, float(need.abs().max())), name


def _decoder(width=64, hidden=96, levels=41, seed=0):
    torch.manual_seed(seed)
    return nn.Sequential(nn.Linear(width, hidden), nn.LayerNorm(hidden), nn.GELU(), nn.Linear(hidden, levels))


def _readout_formula(decoder, bank, states, whose):
    first, norm, _, last = (m for m in decoder)
    h = _adapted_formula(states, first.weight, first.bias, bank.first.a, bank.first.b, whose, bank.first.scales)
    h = (h - h.mean(1, keepdim=True)) / (h.var(1, unbiased=False, keepdim=True) + norm.eps).sqrt() * norm.weight + norm.bias
    h = h * 0.5 * (1 + torch.erf(h / 2**0.5))
    return _adapted_formula(h, last.weight, last.bias, bank.last.a, bank.last.b, whose, bank.last.scales)


def test_readout_trains_against_the_formula():
    import copy

    ids = [1, -1, 0, 1]
    decoder = _decoder().requires_grad_(False)
    decoder[1].requires_grad_(True)  # the norm's affine trains beside the adapters
    torch.manual_seed(1)
    bank = ReadoutAdapters(decoder, 2, 8)
    for p in (bank.first.b, bank.last.b):
        nn.init.normal_(p, std=0.1)
    states, target = torch.randn(4, 30, 64), torch.randn(4, 30, 1)
    exact, twin = copy.deepcopy(decoder).double(), copy.deepcopy(bank).double()

    def pinball(q):
        tau = torch.linspace(0.02, 0.98, 41, device=q.device, dtype=q.dtype)
        d = target.to(q) - q
        return torch.maximum(tau * d, (tau - 1) * d).mean()

    bank.to(DEV), decoder.to(DEV)
    plan = AdapterPlan(ids, 30, device=DEV)
    out = bank(decoder, states.to(DEV), plan)
    pinball(out).backward()
    whose = _rows(ids, 30)
    want = _readout_formula(exact, twin, states.double().view(120, 64), whose).view(4, 30, 41)
    pinball(want).backward()
    # fp32 products of up to 96 terms, twice, and the norm between them
    assert float((out.detach().double().cpu() - want.detach()).abs().max()) <= 2e-5
    pairs = list(zip(bank.parameters(), twin.parameters())) + list(zip(decoder[1].parameters(), exact[1].parameters()))
    for have, need in pairs:
        # the loss's slope is a step: an output within 2e-5 of its target may take the other one, none does here
        assert float((have.grad.double().cpu() - need.grad).abs().max()) <= 1e-6 + 1e-4 * float(need.grad.abs().max())
    assert all(p.grad is None for p in decoder[0].parameters())


def test_readout_under_autocast_and_without_adapters():
    decoder = _decoder().to(DEV).requires_grad_(False).eval()
    bank = ReadoutAdapters(decoder, 3, 16).to(DEV)
    states = torch.randn(5, 20, 64, device=DEV)
    none = AdapterPlan([-1] * 5, 20, device=DEV)
    some = AdapterPlan([0, 1, 2, 0, -1], 20, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=F16):
        base = decoder(states)
        # new adapters (b zero) and no adapters change nothing but the norm's order of sums
        for plan in (none, some):
            got = bank(decoder, states, plan)
            assert got.dtype == F16 and got.shape == base.shape
            assert float((got.float() - base.float()).abs().max()) <= 2 * 2.0**-10 * float(base.float().abs().max())
    with torch.autocast("cuda", dtype=F16):
        bank(decoder, states, some).float().square().mean().backward()
    assert all(p.grad is not None and p.grad.dtype == F32 and bool(torch.isfinite(p.grad).all()) for p in bank.parameters())
    assert bool(bank.last.b.grad.any())


def test_hooked_projections_are_called():
    decoder = _decoder().to(DEV).requires_grad_(False)
    bank = ReadoutAdapters(decoder, 1, 4).to(DEV)
    plan = AdapterPlan([0, 0], 8, device=DEV)
    states = torch.randn(2, 8, 64, device=DEV)
    with torch.no_grad():
        want = bank(decoder, states, plan)
        seen = []
        handles = [m.register_forward_hook(lambda m, i, o: seen.append(type(m).__name__)) for m in (decoder[0], decoder[1], decoder[3])]
        got = bank(decoder, states, plan)
        for h in handles:
            h.remove()
    assert seen == ["Linear", "LayerNorm", "Linear"]
    assert float((got - want).abs().max()) <= 1e-5
    single = LowRankAdapters(1, 64, 96, 4, device=DEV)
    y = decoder[0](states)
    assert torch.equal(single(states, y, plan), y)  # b is zero


def test_models_decode_with_adapters():
    """A nori-6m-shaped dense model: states by apply_context_cache, adapters trained on them, and the adapted
    predictions of the same tables through the cache."""
    from nori_amd.api import NORI_6M_CONFIG, build_model

    torch.manual_seed(0)
    config = dict(NORI_6M_CONFIG, nlayers=2)
    model = build_model(config).to(DEV).eval().requires_grad_(False)
    x, y = torch.randn(3, 40, 6, device=DEV), torch.randn(3, 32, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=F16):
        cache = model.build_context_cache(x[:, :32], y)
        base = model.apply_context_cache(x[:, 32:], cache)
        states = model.apply_context_cache(x[:, 32:], cache, return_embeddings=True)
        assert states.shape == (3, 8, 128) and torch.equal(model.decode(states), base)
    bank = ReadoutAdapters(model.reg_y_decoder, 2, 8).to(DEV)
    ids = [1, -1, 0]
    optimizer = torch.optim.SGD(bank.parameters(), lr=0.1)
    for _ in range(2):
        with torch.autocast("cuda", dtype=F16):
            q = model.decode(states, bank, ids)
        optimizer.zero_grad()
        q.float().square().mean().backward()
        assert all(bool(torch.isfinite(p.grad).all()) for p in bank.parameters())
        optimizer.step()
    with torch.no_grad(), torch.autocast("cuda", dtype=F16):
        whole = model.apply_context_cache(x[:, 32:], cache, readout_adapters=bank, table_adapters=ids)
        parts = model.apply_context_cache(x[:, 32:], cache, row_chunk_size=3, readout_adapters=bank, table_adapters=ids)
    moved = (whole.float() - base.float()).abs().amax((1, 2))
    limit = 2 * 2.0**-10 * float(base.float().abs().max())
    # the table without an adapter is decoded as before (the norm's sums in another order), the others moved
    assert float(moved[1]) <= limit and float(moved[0]) > 0 and float(moved[2]) > 0
    assert whole.shape == base.shape and float((whole.float() - parts.float()).abs().max()) <= 0.02 * float(base.float().abs().max())
    with pytest.raises(ValueError, match="each of the 3 tables"):
        model.decode(states, bank, [0])
    with pytest.raises(ValueError, match="without readout_adapters"):
        model.decode(states, table_adapters=[0, 0, 0])
    assert nori_amd.ReadoutAdapters is ReadoutAdapters
