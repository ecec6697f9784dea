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
