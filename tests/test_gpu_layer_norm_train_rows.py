"""LayerNorm with its gradients where kernels go round more than once, and at widths past their grids (GPU)."""
import pytest
import torch

from nori_amd import trainable_layer_norm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_affine_gradients_of_rows_past_one_grid():
    # 2^27 columns, 32 to a workgroup of 1024, pass what a grid may have. A row of as many 1 as -1: xh is x / sqrt(1 + eps)
    # but for the sums of squares, 2^27 ones in fp32, 2^-20 off at most
    cols = 2**27 + 40
    at = torch.arange(cols, device=DEV, dtype=torch.int32)
    x = (1 - 2 * (at // 3 % 2)).to(F16)
    assert int(x.to(torch.int32).sum()) == 0
    dy = (1 + at % 3).to(F16)[None]
    del at
    w, b = (torch.ones(cols, device=DEV, requires_grad=True) for _ in range(2))
    y = trainable_layer_norm(x[None], w, b, 0.0, out_dtype=F16)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    torch.cuda.synchronize()
    assert torch.equal(db, dy[0].float())
    assert float((dw - dy[0].float() * x.float()).abs().max()) <= 3 * 2.0**-20


# rows enough that every group of lanes goes round several times, unevenly: 4, 8, 16 and 64 lanes a row and a workgroup,
# rows of whole vectors and not, the last trip of some groups only
ROUNDS = [(600011, 24), (600011, 23), (270001, 60), (200003, 57), (150001, 100), (130003, 128), (30001, 384), (20011, 999), (20001, 1000),
          (9001, 1500), (9001, 2047), (5001, 4096), (5003, 4001), (4999, 8192), (700, 9000)]


@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,cols", ROUNDS)
def test_rows_past_the_first_round(rows, cols, x_dtype, y_dtype):
    """Rows of as many 1 as -1 (and a 0 in odd ones), times a power of two of the row's own, and dy of -1, 0 and 1. Mean 0 and the
    variance are exact but for the division: xh is off by 2^-21 of itself at most, and dw, sums of xh that fp32 adds with 2^-24 of
    the largest so far, by rows * 2^-21 < 0.3. db is a whole number below 2^24, and exact. A row too many or too few is 1
    off."""
    print(f"{rows} x {cols} {x_dtype} -> {y_dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    sign = 1.0 - 2.0 * (torch.arange(cols, device=DEV) % 2)
    if cols % 2:
        sign[-1] = 0.0
    turn = torch.randint(0, cols, (rows, 1), generator=g, device=DEV)
    at = (torch.arange(cols, device=DEV)[None] + turn) % cols  # each row's order is its own
    x = sign[at]
    del at, turn
    scale = torch.exp2(torch.randint(-4, 5, (rows, 1), generator=g, device=DEV).float())
    xh = x * (cols / (cols - cols % 2)) ** 0.5
    dy = torch.randint(-1, 2, (rows, cols), generator=g, device=DEV, dtype=torch.int8)
    w = torch.randint(1, 4, (cols,), generator=g, device=DEV).float()
    b = torch.randint(-3, 4, (cols,), generator=g, device=DEV).float()
    leaves = [t.requires_grad_(True) for t in ((x * scale).to(x_dtype), w.clone(), b.clone())]
    y = trainable_layer_norm(*leaves, 0.0, out_dtype=y_dtype)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(y_dtype))
    y = y.detach()
    half = torch.finfo(y_dtype).eps / 2 + 2.0**-20
    assert float(((y.float() - (xh * w + b)).abs() - half * (xh.abs() * w + b.abs())).max()) <= 0.0
    assert torch.equal(db, dy.sum(0, dtype=torch.int64).float())
    want = torch.zeros(cols, dtype=torch.float64, device=DEV)
    m1, m2 = [], []
    for i in range(0, rows, 50000):
        part = slice(i, i + 50000)
        want += (dy[part].double() * xh[part].double()).sum(0)
        gr = dy[part].double() * w
        m1.append(gr.mean(1)), m2.append((gr * xh[part]).mean(1))
    off = float((dw - want).abs().max())
    print(f"  dw off by {off:.2e}", flush=True)
    assert off < max(0.01, rows * 2.0**-21) and float(want.abs().max()) > 8
    # dx: the terms are at most 3, 3 and 3 in size, each off by 2^-18 of that, over the row's scale
    half = torch.finfo(x_dtype).eps / 2
    for i, one, other in zip(range(0, rows, 50000), m1, m2):
        part = slice(i, i + 50000)
        dxw = dy[part] * w - one[:, None] - xh[part] * other[:, None]
        dxw = dxw / scale[part] * (cols / (cols - cols % 2)) ** 0.5
        tol = half * dxw.abs() + 9 * 2.0**-18 / scale[part] + (2.0**-25 if x_dtype == F16 else 0.0)
        assert bool(((dx[part].double() - dxw).abs() <= tol).all()), i
