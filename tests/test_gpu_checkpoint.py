"""Projections and SwiGLU gates kept in 8 bits, on the GPU against their formulas in 64 bits.

Bounds, h half a step of the type (eps / 2), least its subnormal step: a sum of K products in fp32 is off by at most K 2^-23 of
the sum of their magnitudes A (the matrix instructions' inner sums included), its result by h once more, and weights and kept
values enter the products rounded (h each where they are wider than the type).
"""

import math

import pytest
import torch
import torch.nn.functional as F

import nori_amd
from checkpoint_case import activations, kept
from nori_amd import checkpoint as cp

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
U = 2.0**-23


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps


def near(name, got, expected, bound):
    over = (got.double().cpu() - expected).abs() - bound
    assert torch.isfinite(got).all() and over.max() <= 0, f"{name}: {over.max().item()} over, at {int(over.argmax())}"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("cols", [1, 7, 8, 16, 127, 128, 129, 200, 352, 938, 2049])
def test_codes_are_the_nearest(cuda, cols, dtype):
    x = activations(37, cols, dtype, seed=cols)
    codes, scales, values = kept(x)
    got, s = cp._quantized(x.cuda())
    assert torch.equal(s.double().cpu(), scales)
    assert torch.equal(got[:, :cols].double().cpu(), codes)
    assert not got[:, cols:].any()


def test_codes_beside_halves(cuda):
    """fp32 rows of values one step from the halves between two codes, under scales of every last digit."""
    g = torch.Generator().manual_seed(0)
    amax = (1 + torch.rand(500, generator=g)) * 2.0 ** torch.randint(-60, 60, (500,), generator=g)
    s = amax * torch.tensor(1 / 127, dtype=torch.float32)
    x = ((torch.arange(128) - 63.5) * s[:, None].double()).float()
    for step in (-1, 0, 1):
        y = x if step == 0 else torch.nextafter(x, x + step * x.abs())
        y[:, 0] = amax
        codes, scales, _ = kept(y)
        got, sc = cp._quantized(y.cuda())
        assert torch.equal(sc.double().cpu(), scales) and torch.equal(got.double().cpu(), codes)


def test_codes_of_extremes(cuda):
    x = torch.zeros(8, 130)
    x[0, 3] = 2.0**-149            # a scale that rounds to 0
    x[1, :100] = 190 * 2.0**-149   # one of a single bit: quotients past 127
    x[2] = torch.finfo(torch.float32).max
    x[3, 5], x[3, 6] = math.inf, 1.0
    x[4, 5], x[4, 129] = math.nan, 1.0
    x[5] = 2.0**-126
    codes, scales, values = kept(x)
    got, s = cp._quantized(x.cuda())
    assert torch.equal(s.double().cpu().nan_to_num(nan=-1.0), scales.nan_to_num(nan=-1.0))
    fine = torch.isfinite(values)
    assert torch.equal(got[:, :130].double().cpu()[fine], codes[fine])


LINEAR = [(1, 1, 1), (5, 7, 3), (37, 128, 128), (640, 352, 385), (1000, 129, 130), (3000, 20, 33), (20011, 127, 64), (513, 560, 1120)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("rows,k,n", LINEAR)
def test_linear(cuda, rows, k, n, wide, dtype):
    g = torch.Generator().manual_seed(rows)
    wt = torch.float32 if wide else dtype
    x = activations(rows, k, dtype, seed=rows)
    w, b = (torch.randn(n, k, generator=g) * k**-0.5).to(wt), torch.randn(n, generator=g).to(wt)
    dy = (torch.randn(rows, n, generator=g) * 0.1).to(dtype)
    xd, wd, bd = (t.cuda().requires_grad_(True) for t in (x, w, b))
    y = nori_amd.checkpointed_linear(xd, wd, bd)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda())
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (dtype, dtype, wt, wt)
    assert torch.equal(y, F.linear(xd, wd.to(dtype), bd.to(dtype)))
    h = half(dtype)
    w16, _, xh = w.to(dtype).double(), None, kept(x)[2]
    near("dx", dx, dy.double() @ w16, (n * U + h) * (dy.double().abs() @ w16.abs()) + least(dtype))
    a = dy.double().t().abs() @ xh.abs()
    # kept values are rounded to the rows' type, below its normal range to its subnormal step, or held to 2^-22 (and 2^-33 of the largest
    # of any) for an fp32 gradient
    fine = wt == torch.float32 and dtype != torch.float32
    rounding = 2.0**-22 if fine else (0.0 if dtype == torch.float32 else h)
    sub = 2.0**-33 * rows * dy.double().abs().max() * xh.abs().max() if fine else dy.double().abs().sum(0)[:, None] * least(dtype)
    near("dw", dw, dy.double().t() @ xh, (rows * U + rounding + half(wt)) * a + sub + least(wt))
    near("db", db, dy.double().sum(0), (rows * U + half(wt)) * dy.double().abs().sum(0) + least(wt))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (5, 7), (33, 128), (700, 129), (64, 938), (3, 4100), (2000, 20)])
def test_silu_mul(cuda, rows, hidden, dtype):
    g = torch.Generator().manual_seed(hidden)
    gu = activations(rows, 2 * hidden, dtype, seed=hidden)
    dy = (torch.randn(rows, hidden, generator=g) * 0.1).to(dtype)
    x = gu.cuda().requires_grad_(True)
    y = nori_amd.checkpointed_silu_mul(x, hidden)
    (dgu,) = torch.autograd.grad(y, x, dy.cuda())
    h = half(dtype)
    a, b = gu[:, :hidden].double(), gu[:, hidden:].double()
    # an exponential to 2^-22, a quotient, products: 2^-20 of the result; the exponential's argument adds |g| 2^-24
    near("y", y, a * torch.sigmoid(a) * b, (h + 2.0**-20 + a.abs() * 2.0**-23) * (a * torch.sigmoid(a) * b).abs() + least(dtype))
    a, b, d = kept(gu[:, :hidden])[2], kept(gu[:, hidden:])[2], dy.double()
    sig = torch.sigmoid(a)
    dg, du = d * b * sig * (1 + a * (1 - sig)), d * a * sig
    # 1 + g (1 - sigma) cancels for g < 0: its terms' magnitudes, 1 + |g| (1 - sigma), carry the error
    u = 2.0**-20 + a.abs() * 2.0**-23
    near("dg", dgu[:, :hidden], dg, h * dg.abs() + u * (d * b * sig).abs() * (1 + a.abs() * (1 - sig)) + least(dtype))
    near("du", dgu[:, hidden:], du, (h + u) * du.abs() + least(dtype))
    with torch.no_grad():
        assert torch.equal(nori_amd.checkpointed_silu_mul(x, hidden), y)


def test_strides_and_shapes(cuda):
    g = torch.Generator().manual_seed(3)
    for dtype in DTYPES:
        buffer = torch.randn(6, 9, 700, generator=g).to(dtype).cuda()
        w = torch.randn(33, 129, generator=g).to(dtype).cuda().requires_grad_(True)
        dy = torch.randn(6, 9, 33, generator=g).to(dtype).cuda()
        views = [buffer[:, :, 1:130], buffer.transpose(0, 1)[:, :, 3:132].transpose(0, 1), buffer[:, :, ::2][:, :, :129]]
        for view in views:
            def grads(x, slope):
                return torch.autograd.grad(nori_amd.checkpointed_linear(x, w), w, slope)[0]
            expected = grads(view.contiguous(), dy)
            assert torch.equal(grads(view, dy), expected)
            assert torch.equal(grads(view, dy.transpose(0, 1).contiguous().transpose(0, 1)), expected)
        one = torch.ones((), dtype=dtype, device="cuda").expand(6, 9, 33)
        assert torch.equal(grads(view, one), grads(view, one.contiguous()))
        gu = buffer[:, :, 5:263]
        def gates(t, slope):
            t = t.detach().requires_grad_(True)
            y = nori_amd.checkpointed_silu_mul(t, 129)
            return y, torch.autograd.grad(y, t, slope)[0]
        slope = torch.randn(6, 9, 129, generator=g).to(dtype).cuda()
        for a, b in zip(gates(gu, slope), gates(gu.contiguous(), slope.transpose(0, 1).contiguous().transpose(0, 1))):
            assert torch.equal(a, b)


def test_no_rows(cuda):
    x = torch.empty(0, 3, 16, device="cuda", requires_grad=True)
    w, b = torch.randn(5, 16, device="cuda", requires_grad=True), torch.randn(5, device="cuda", requires_grad=True)
    y = nori_amd.checkpointed_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == (0, 3, 5) and dx.shape == x.shape and not dw.any() and not db.any()
    y = nori_amd.checkpointed_silu_mul(x, 8)
    assert y.shape == (0, 3, 8) and torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape


def test_gradients_asked_for_apart(cuda):
    g = torch.Generator().manual_seed(4)
    x, w, b = torch.randn(300, 40, generator=g).cuda(), torch.randn(50, 40, generator=g).cuda(), torch.randn(50, generator=g).cuda()
    dy = torch.randn(300, 50, generator=g).cuda()
    def grads(*which):
        t = [v.clone().requires_grad_(i in which) for i, v in enumerate((x, w, b))]
        return torch.autograd.grad(nori_amd.checkpointed_linear(*t), [t[i] for i in which], dy)
    whole = grads(0, 1, 2)
    for i in range(3):
        assert torch.equal(grads(i)[0], whole[i])
    with torch.no_grad():
        assert torch.equal(nori_amd.checkpointed_linear(x, w, b), F.linear(x, w, b))


def test_bad_groups_reach_the_weight(cuda):
    x = torch.randn(64, 300, device="cuda")
    x[7, 130] = math.inf
    w = torch.randn(8, 300, device="cuda", requires_grad=True)
    dw = torch.autograd.grad(nori_amd.checkpointed_linear(x, w), w, torch.ones(64, 8, device="cuda"))[0]
    assert dw[:, 128:256].isnan().all() and torch.isfinite(dw[:, :128]).all() and torch.isfinite(dw[:, 256:]).all()


def test_autocast(cuda):
    x = torch.randn(100, 64, device="cuda", requires_grad=True)
    w, b = torch.randn(32, 64, device="cuda", requires_grad=True), torch.randn(32, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.float16):
        y = nori_amd.checkpointed_linear(x, w, b)
        assert y.dtype == torch.float16 and torch.equal(y, F.linear(x, w, b))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert dx.dtype == dw.dtype == db.dtype == torch.float32


def test_the_same_bits_again_and_captured(cuda):
    g = torch.Generator().manual_seed(5)
    x, dy = torch.randn(5000, 300, generator=g).half().cuda(), torch.randn(5000, 128, generator=g).half().cuda()
    w, b = torch.randn(256, 300, generator=g).cuda().requires_grad_(True), torch.randn(256, generator=g).cuda().requires_grad_(True)
    x.requires_grad_(True)

    def step():
        y = nori_amd.checkpointed_silu_mul(nori_amd.checkpointed_linear(x, w, b), 128)
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    def eager():
        return [t.detach().clone() for t in step()]

    first = eager()
    assert all(torch.equal(a, b) for a, b in zip(first, eager()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(first, eager()))
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = [t.detach() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(5000, 300, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, eager()))


def test_overlapping_and_distant_rows(cuda):
    """Windows that share elements, and rows whose offsets pass 2^32 elements: what contiguous copies of them give."""
    g = torch.Generator().manual_seed(6)
    line = torch.randn(4000, generator=g).half().cuda()
    windows = line.unfold(0, 40, 9)[:400]
    w = torch.randn(24, 40, generator=g).half().cuda().requires_grad_(True)
    slopes = line.unfold(0, 24, 9)[:400]

    def grads(x, dy):
        return torch.autograd.grad(nori_amd.checkpointed_linear(x, w), w, dy)[0]

    assert torch.equal(grads(windows, slopes), grads(windows.contiguous(), slopes.contiguous()))
    far = torch.empty(70000 * 65536, dtype=torch.float16, device="cuda").view(70000, 65536)[:, :40]
    x = torch.randn(70000, 40, generator=g).half().cuda()
    far.copy_(x)
    dy = torch.randn(70000, 24, generator=g).half().cuda()
    assert torch.equal(grads(far, dy), grads(x, dy))


def test_second_derivatives_are_refused(cuda):
    x, w = torch.randn(5, 8, device="cuda", requires_grad=True), torch.randn(3, 8, device="cuda", requires_grad=True)
    dx = torch.autograd.grad(nori_amd.checkpointed_linear(x, w).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), w)
    gu = torch.randn(5, 8, device="cuda", requires_grad=True)
    d = torch.autograd.grad(nori_amd.checkpointed_silu_mul(gu, 4).square().sum(), gu, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), gu)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_fp32_gradients_of_slopes_of_any_size(cuda, dtype):
    """Slopes that grow by 2^24 from row to row's end, beside infinities in other columns and in the memory between rows: each weight's
    gradient to 2^-22 of its terms and 2^-33 of the largest of any."""
    g = torch.Generator().manual_seed(7)
    rows, k, n = 700, 40, 21
    x = torch.randn(rows, k, generator=g).to(dtype)
    buffer = torch.full((rows, n + 3), math.inf, dtype=dtype)
    buffer[:, :n] = torch.randn(rows, n, generator=g) * 2.0 ** torch.linspace(-12, 12, rows)[:, None]
    buffer[3, 5] = math.inf
    dy = buffer.cuda()[:, :n]
    w = torch.randn(n, k, generator=g).cuda().requires_grad_(True)
    dw = torch.autograd.grad(nori_amd.checkpointed_linear(x.cuda(), w), w, dy)[0].double().cpu()
    d, xh = buffer[:, :n].double(), kept(x)[2]
    others = [i for i in range(n) if i != 5]
    assert not torch.isfinite(dw[5]).any()
    d = d[:, others]
    bound = (rows * U + 2.0**-22) * (d.t().abs() @ xh.abs()) + 2.0**-33 * rows * d.abs().max() * xh.abs().max()
    near("dw", dw[others], d.t() @ xh, bound)


@pytest.mark.parametrize("dtype, weight", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)],
                         ids=str)
def test_values_at_the_top_of_the_range(cuda, dtype, weight):
    """Rows up to the type's largest number beside slopes down to 2^-100: 128 scales are past fp32, a scale times a power of two too."""
    x = activations(70, 130, torch.float32).to(dtype)
    x[5] *= 2.0**100
    x[40, 129] = torch.finfo(dtype).max
    dy = (torch.randn(70, 9, generator=torch.Generator().manual_seed(3)) * 2.0**-100).to(dtype)
    w = torch.zeros(9, 130, dtype=weight, device="cuda", requires_grad=True)
    dw = torch.autograd.grad(nori_amd.checkpointed_linear(x.cuda(), w), w, dy.cuda())[0].double().cpu()
    xh, d = kept(x)[2], dy.double()
    assert torch.isfinite(xh).all()
    # x to the rows' type, the result to the weight's, sums in fp32; float32 weights take two pieces of the slopes instead
    fine = weight != dtype
    each = 2.0**-22 if fine else torch.finfo(dtype).eps / 2
    bound = (71 * U + each) * (d.t().abs() @ xh.abs()) + torch.finfo(weight).eps / 2 * (d.t() @ xh).abs()
    if fine:
        bound[:, :128] += 2.0**-33 * 70 * (d.abs().amax(1) * xh[:, :128].abs().amax(1)).max()
        bound[:, 128:] += 2.0**-33 * 70 * (d.abs().amax(1) * xh[:, 128:].abs().amax(1)).max()
    near("dw", dw, d.t() @ xh, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gates_at_the_top_of_the_range(cuda, dtype):
    gu = torch.ones(3, 260, dtype=dtype)
    gu[1, 130:] = torch.finfo(dtype).max
    dy = torch.full((3, 130), 2.0**-100, dtype=dtype)
    gu = gu.cuda().requires_grad_(True)
    dgu = torch.autograd.grad(nori_amd.checkpointed_silu_mul(gu, 130), gu, dy.cuda())[0].double().cpu()
    g, u = torch.ones(3, 130).double(), kept(gu[:, 130:])[2]
    s = torch.sigmoid(g)
    expected = torch.cat([dy.double() * u * s * (1 + g * (1 - s)), dy.double() * g * s], 1)
    near("dgu", dgu, expected, expected.abs() * (torch.finfo(dtype).eps / 2 + 64 * U))


def test_nothing_is_kept_where_nothing_is_trained(cuda, monkeypatch):
    x = activations(37, 130, torch.float16).cuda()
    w = torch.randn(9, 130, device="cuda", dtype=torch.float16, requires_grad=True)
    expected = F.linear(x, w.detach())

    def kept_anyway(x):
        raise AssertionError("the input was quantised")

    monkeypatch.setattr(cp, "_quantized", kept_anyway)
    with torch.no_grad():
        assert torch.equal(nori_amd.checkpointed_linear(x, w), expected)
    assert torch.equal(nori_amd.checkpointed_linear(x, w.detach()), expected)
    leaf = x.clone().requires_grad_(True)
    y = nori_amd.checkpointed_linear(leaf, w.detach())
    assert torch.equal(y, expected)
    assert torch.equal(torch.autograd.grad(y, leaf, torch.ones_like(y))[0], torch.ones_like(y) @ w.detach())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_that_do_not_fold(cuda, dtype):
    """A batch of rows cut out of a larger one, and rows of a single dimension: what their contiguous copies give, bit for bit."""
    big = activations(6 * 11, 48, dtype).view(6, 11, 48).cuda()
    w = torch.randn(20, 32, device="cuda").to(dtype).requires_grad_(True)
    b = torch.randn(20, device="cuda").to(dtype).requires_grad_(True)
    for cut in (big[1:5, 2:9, 8:40], big[1, 2, 8:40]):
        dy = torch.randn(*cut.shape[:-1], 20, device="cuda").to(dtype)
        got = []
        for x in (cut, cut.contiguous()):
            x = x.detach().requires_grad_(True)
            y = nori_amd.checkpointed_linear(x, w, b)
            assert y.shape == dy.shape
            got.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
        for one, other in zip(*got):
            assert torch.equal(one, other)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n", [1, 3, 5, 7, 8, 9, 130])
def test_slopes_cut_out_of_a_wider_buffer(cuda, n, dtype):
    """Columns beside the slopes, finite and far larger, are not looked at: the contiguous slopes' bits, in fp32 and in the type."""
    g = torch.Generator().manual_seed(n)
    rows, k = 700, 150
    x = torch.randn(rows, k, generator=g).to(dtype).cuda()
    buffer = torch.full((rows, n + 14), torch.finfo(dtype).max, dtype=dtype)
    buffer[:, 2 : 2 + n] = (torch.randn(rows, n, generator=g) * 1e-3).to(dtype)
    dy = buffer.cuda()[:, 2 : 2 + n]
    for wt in (torch.float32, dtype):
        w, b = (torch.randn(s, generator=g).to(wt).cuda().requires_grad_(True) for s in ((n, k), (n,)))
        got = torch.autograd.grad(nori_amd.checkpointed_linear(x, w, b), (w, b), dy)
        expected = torch.autograd.grad(nori_amd.checkpointed_linear(x, w, b), (w, b), dy.contiguous())
        assert all(torch.equal(a, c) for a, c in zip(got, expected))
        assert got[0].any(1).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("biased", [False, True])
def test_results_are_changed_in_place(cuda, biased, dtype):
    """A residual is added to the result, which goes through a gate, in place: what the same out of place gives."""
    g = torch.Generator().manual_seed(8)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda().requires_grad_(True)
    for lead in ((), (3,), (3, 5), (2, 3, 5)):
        x, w, b, r = make(*lead, 24), make(20, 24), make(20) if biased else None, make(*lead, 20)
        leaves = [t for t in (x, w, b, r) if t is not None]
        slope = torch.randn(*lead, 20, generator=g).to(dtype).cuda()
        y = torch.relu(nori_amd.checkpointed_linear(x, w, b) + r)
        z = nori_amd.checkpointed_linear(x, w, b)
        z += r
        z = F.relu(z, inplace=True)
        assert torch.equal(y, z)
        pairs = zip(torch.autograd.grad(y, leaves, slope), torch.autograd.grad(z, leaves, slope))
        assert all(torch.equal(a, c) for a, c in pairs)
        gu = make(*lead, 40)
        h = nori_amd.checkpointed_silu_mul(gu, 20) + r
        v = nori_amd.checkpointed_silu_mul(gu, 20)
        v += r
        pairs = zip(torch.autograd.grad(h, (gu, r), slope), torch.autograd.grad(v, (gu, r), slope))
        assert torch.equal(h, v) and all(torch.equal(a, c) for a, c in pairs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows", [5, 300])
def test_an_infinite_slope_among_zeros(cuda, rows, dtype):
    """The fp32 gradient is what the formula gives: infinite where the row's kept value is not zero, NaN where it is."""
    x = activations(rows, 150, dtype, seed=1)
    x[4, 7] = 0
    dy = torch.zeros(rows, 9, dtype=dtype)
    dy[4, 2] = math.inf
    w = torch.zeros(9, 150, device="cuda", requires_grad=True)
    dw = torch.autograd.grad(nori_amd.checkpointed_linear(x.cuda(), w), w, dy.cuda())[0].double().cpu()
    xh = kept(x)[2]
    expected = torch.zeros(9, 150).double()
    expected[2] = math.inf * xh[4]
    assert torch.equal(dw.nan_to_num(nan=1.0), expected.nan_to_num(nan=1.0))


def test_codes_beside_halves_of_the_smallest_scales(cuda):
    """fp32 rows whose scales lie about and below the least normal number, values at and one step from the halves between two codes:
    where half a scale is no number, a quotient next to a half rounds to it."""
    g = torch.Generator().manual_seed(9)
    step = 2.0**-149
    scale = torch.cat([torch.randint(2**21, 2**25, (400,), generator=g), torch.randint(1, 2**10, (100,), generator=g),
                       torch.tensor([2**23 - 1, 2**23, 2**23 + 1, 2**24 - 1, 2**24, 2**24 + 1])]).double() * step
    amax = (scale * 127).float()
    s = (amax * torch.tensor(1 / 127, dtype=torch.float32)).double()
    middle = (torch.arange(128) - 63.5) * s[:, None]
    for way in (torch.floor, torch.ceil):
        for beside in (-1, 0, 1):
            x = ((way(middle / step) + beside) * step).float()
            x[:, 0] = amax
            codes, scales, _ = kept(x)
            got, sc = cp._quantized(x.cuda())
            assert torch.equal(sc.double().cpu(), scales) and torch.equal(got.double().cpu(), codes)
