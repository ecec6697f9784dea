"""LayerNorm with its gradients (``trainable_layer_norm``) on the GPU against the formulas in 64 bits.

Tolerances. A sum of m terms taken in fp32 as partial sums of at most p terms, joined, is off by at most
(p + joins) * 2^-24 of the sum of its terms' magnitudes; 256 steps cover every size here (a lane's share of
a row of 8192 is 128 terms, a part's share of 5000 rows under 140, plus the joins). Each result is then
rounded once: half a step of its type, eps / 2 relative (and half the smallest subnormal).
"""
import pytest
import torch

from nori_amd import trainable_layer_norm
from nori_amd.norm import layer_norm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
STEPS = 256 * 2.0**-24
HALF_SUBNORMAL = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}


def _make(rows, cols, x_dtype, y_dtype, w_dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + rows + cols)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + torch.randn(cols, generator=g)).to(x_dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(w_dtype)
    b = (0.3 * torch.randn(cols, generator=g)).to(w_dtype)
    dy = (0.1 * torch.randn(rows, cols, generator=g)).to(y_dtype)
    return x, w, b, dy


def _formulas(x, w, b, dy, eps):
    """{name: (value, the magnitude its fp32 error is relative to)} in float64."""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1]).double() if w is None else w.double()
    b = torch.zeros(x.shape[1]).double() if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    # how far xh may be off: the mean's error over the spread, and the spread's own, relative
    off = STEPS * (x.abs().mean(1, keepdim=True) * rstd * (1 + 2 * xh.abs()) + 2 * xh.abs() + 1)
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - m1 - xh * m2)
    grown = 1 + off / STEPS  # per unit of STEPS
    mag = rstd * (g.abs() + g.abs().mean(1, keepdim=True) * 2 + xh.abs() * (g.abs() * (xh.abs() + grown)).mean(1, keepdim=True)
                  + m2.abs() * grown) * 2 + dx.abs() * x.abs().mean(1, keepdim=True) * rstd
    return {
        "y": (xh * w + b, off / STEPS * w.abs() + (xh * w).abs() + b.abs()),
        "dx": (dx, mag),
        "dw": ((dy * xh).sum(0), (dy.abs() * (xh.abs() + off / STEPS)).sum(0)),
        "db": (dy.sum(0), dy.abs().sum(0)),
    }


def _near(got, want, mag, what):
    value = got.double().cpu()
    tol = torch.finfo(got.dtype).eps / 2 * (want.abs() + STEPS * mag) + HALF_SUBNORMAL[got.dtype] + STEPS * mag
    worst = float(((value - want).abs() / tol).max()) if value.numel() else 0.0
    print(f"  {what}: {worst:.3f} of its tolerance", flush=True)
    assert value.shape == want.shape and worst <= 1.0, (what, worst)


def _run(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = trainable_layer_norm(*args, eps, out_dtype=dy.dtype)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    got = {"y": y.detach()}
    for name, t in zip(("dx", "dw", "db"), args):
        if t is not None:
            got[name] = next(grads)
    return got


@pytest.mark.parametrize("x_dtype,y_dtype,w_dtype", [(F32, F32, F32), (F16, F16, F32), (F16, F32, F32), (F32, F16, F32),
                                                     (BF16, BF16, BF16), (F32, BF16, F16), (F16, F16, F16)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 384), (3, 2), (5, 7), (64, 64), (333, 100), (2049, 999), (640, 384), (17, 2048),
                                       (9, 2047), (130, 4096), (5, 8192), (3, 20001), (5000, 24)])
def test_against_the_formulas(rows, cols, x_dtype, y_dtype, w_dtype):
    print(f"layer norm {rows} x {cols} {x_dtype} -> {y_dtype}, weights {w_dtype}", flush=True)
    x, w, b, dy = _make(rows, cols, x_dtype, y_dtype, w_dtype)
    got = _run(*(t.to(DEV) for t in (x, w, b, dy)))
    torch.cuda.synchronize()
    want = _formulas(x, w, b, dy, 1e-5)
    assert got["y"].dtype == y_dtype and got["dx"].dtype == x_dtype and got["dw"].dtype == got["db"].dtype == w_dtype
    for name, (value, mag) in want.items():
        _near(got[name], value, mag, name)


@pytest.mark.parametrize("which", ["weight", "bias", "neither", "mixed"])
def test_parameters_left_out(which):
    x, w, b, dy = _make(70, 130, F32, F32, F32)
    w = None if which in ("bias", "neither") else w
    b = None if which in ("weight", "neither") else b
    if which == "mixed":
        b = b.to(BF16)
    got = _run(*(None if t is None else t.to(DEV) for t in (x, w, b, dy)))
    want = _formulas(x, w, b, dy, 1e-5)
    for name in got:
        _near(got[name], *want[name], name)
    if which == "mixed":
        assert got["db"].dtype == BF16 and got["dw"].dtype == F32


def test_gradients_asked_for_one_at_a_time():
    x, w, b, dy = (t.to(DEV) for t in _make(300, 96, F16, F16, F32))
    whole = _run(x, w, b, dy)
    for i, name in enumerate(("dx", "dw", "db")):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        (one,) = torch.autograd.grad(trainable_layer_norm(*args), args[i], dy)
        assert torch.equal(one, whole[name]), name


def test_strides_and_shapes():
    # layouts that take vectors and layouts that do not sum a row in other orders: each is held to the formula
    x, w, b, dy = _make(6 * 50, 72, F16, F16, F32)
    want = _formulas(x, w, b, dy, 1e-5)
    wide = torch.full((6, 50, 3, 75), float("nan"), dtype=F16, device=DEV)
    at = wide[:, :, 1, 3:]  # rows at one stride, off the alignment of any vector
    at.copy_(x.view(6, 50, 72))
    turned = x.view(6, 50, 72).transpose(0, 1).contiguous().to(DEV).transpose(0, 1)  # rows at two strides
    columns = x.to(DEV).t().contiguous().t()  # a column-major matrix
    for name, v in (("slice", at), ("turned", turned), ("columns", columns)):
        grad = dy.to(DEV).view(v.shape)
        got = _run(v, w.to(DEV), b.to(DEV), grad)
        for k in ("y", "dx"):
            assert got[k].shape == v.shape
            _near(got[k].reshape(-1, 72), *want[k], f"{name} {k}")
        for k in ("dw", "db"):
            _near(got[k], *want[k], f"{name} {k}")
    strided = torch.zeros(72, 2, device=DEV)
    strided[:, 1] = w.to(DEV)
    got = _run(x.to(DEV), strided[:, 1], b.to(DEV), dy.to(DEV))
    _near(got["y"], *want["y"], "y")
    _near(got["dw"], *want["dw"], "dw")


def test_broadcast_inputs():
    # one row expanded to many: its gradient is the sum over them; a scalar's expanded gradient as dy
    x, w, b, _ = _make(1, 40, F32, F32, F32)
    leaf = x.to(DEV).requires_grad_(True)
    y = trainable_layer_norm(leaf.expand(33, 40), w.to(DEV), b.to(DEV))
    y.sum().backward()
    want = _formulas(x.expand(33, 40), w, b, torch.ones(33, 40), 1e-5)
    _near(y.detach(), *want["y"], "y")
    _near(leaf.grad, want["dx"][0].sum(0, keepdim=True), want["dx"][1].sum(0, keepdim=True), "dx")


def test_no_rows():
    w = torch.ones(48, device=DEV, requires_grad=True)
    x = torch.empty(0, 48, device=DEV, requires_grad=True)
    y = trainable_layer_norm(x, w, torch.zeros(48, device=DEV))
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 48, device=DEV))
    assert y.shape == (0, 48) and dx.shape == (0, 48) and torch.equal(dw, torch.zeros_like(w))


def test_against_differences():
    # the gradient of sum(y dy) by central differences of the float64 formula, a step of 1e-5
    x, w, b, dy = (t.double() for t in _make(4, 12, F32, F32, F32))
    got = _run(*(t.float().to(DEV) for t in (x, w, b, dy)))

    def loss(x, w, b):
        return float((_formulas(x, w, b, dy, 1e-5)["y"][0] * dy).sum())

    for name, t in (("dx", x), ("dw", w), ("db", b)):
        d = torch.zeros_like(t)
        for i in range(t.numel()):
            old = t.view(-1)[i].item()
            t.view(-1)[i] = old + 1e-5
            up = loss(x, w, b)
            t.view(-1)[i] = old - 1e-5
            d.view(-1)[i] = (up - loss(x, w, b)) / 2e-5
            t.view(-1)[i] = old
        # the differences' own error, about 1e-10 / 1e-5, and the gradient's
        assert float((got[name].double().cpu() - d).abs().max()) <= 2e-5, name


def test_large_means_and_non_finite_rows():
    x = torch.randn(8, 256) + 300.0
    w, b = torch.ones(256), torch.zeros(256)
    got = _run(x.to(DEV), w.to(DEV), b.to(DEV), torch.ones(8, 256, device=DEV))
    _near(got["y"], *_formulas(x, w, b, torch.ones(8, 256), 1e-5)["y"], "y")
    x[2, 5], x[5, 0] = float("inf"), float("nan")
    dy = torch.randn(8, 256)
    got = _run(x.to(DEV), w.to(DEV), b.to(DEV), dy.to(DEV))
    for name in ("y", "dx"):
        bad = torch.isnan(got[name]).all(1).cpu()
        assert bad.tolist() == [i in (2, 5) for i in range(8)] and bool(torch.isfinite(got[name][~bad.to(DEV)]).all()), name
    assert bool(torch.isnan(got["dw"]).all())
    _near(got["db"], dy.double().sum(0), dy.double().abs().sum(0), "db")
    zero = _run(torch.zeros(4, 64, device=DEV), torch.ones(64, device=DEV), torch.ones(64, device=DEV), torch.ones(4, 64, device=DEV))
    assert torch.equal(zero["y"], torch.ones(4, 64, device=DEV)) and bool(torch.isfinite(zero["dx"]).all())


def test_the_same_bits_again_and_on_another_stream():
    x, w, b, dy = (t.to(DEV) for t in _make(4096, 384, F16, F16, F32))
    want = _run(x, w, b, dy)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    for again in (_run(x, w, b, dy), other):
        assert all(torch.equal(again[n], want[n]) for n in want)
    # inference gives the training pass's bits
    assert torch.equal(trainable_layer_norm(x, w, b), want["y"])
    # and is near the inference kernel's: both are within their tolerance of the formula
    far = (layer_norm(x, w, b, 1e-5).float() - want["y"].float()).abs().max()
    assert float(far) <= 2 * 2.0**-10 * float(want["y"].float().abs().max())


def test_two_graphs_replayed_in_turn():
    cases = [[t.to(DEV) for t in _make(rows, 384, F16, F16, F32, seed)] for rows, seed in ((700, 1), (2500, 2))]
    want = [_run(*c) for c in cases]
    graphs, outs, held = [], [], [[t.clone() for t in c] for c in cases]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in held:
            _run(*c)
    torch.cuda.current_stream().wait_stream(side)
    for c in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(*c))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1, 1, 0):
            for t in outs[i].values():
                t.fill_(float("nan"))
            graphs[i].replay()
            eager = _run(*cases[1 - i])
            torch.cuda.synchronize()
            assert all(torch.equal(outs[i][n], want[i][n]) for n in want[i]), (turn, i)
            assert all(torch.equal(eager[n], want[1 - i][n]) for n in want[i])


def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    with pytest.raises(ValueError, match="weight"):
        trainable_layer_norm(x, torch.ones(4, device=DEV), None)
    with pytest.raises(NotImplementedError, match="float64"):
        trainable_layer_norm(x.double(), None, None)
    with pytest.raises(NotImplementedError, match="int8"):
        trainable_layer_norm(x, None, None, out_dtype=torch.int8)
    with pytest.raises(ValueError, match="eps"):
        trainable_layer_norm(x, w, None, float("nan"))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        trainable_layer_norm(x, w.cpu(), None)
    y = trainable_layer_norm(x.requires_grad_(True), w, None)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()  # first derivatives only
