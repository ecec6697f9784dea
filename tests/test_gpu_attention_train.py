"""Attention with gradients on the GPU against its formulas in 64 bits (the bounds: attention_train_case.py)."""

import math

import pytest
import torch

import nori_amd
from attention_train_case import assert_near, inputs, reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]

# (bg, queries, keys, heads, key heads, width, lengths of the tables or None)
SHAPES = [
    (1, 1, 1, 1, 1, 4, None),
    (2, 33, 33, 2, 2, 44, None),
    (1, 1, 300, 2, 2, 64, None),
    (6, 31, 65, 3, 1, 20, [65, 0, 7]),
    (2, 130, 64, 4, 2, 128, None),
    (2, 257, 1000, 2, 2, 56, [1, 1000]),
    (1, 5, 3001, 2, 1, 96, None),       # few rows, many keys: keys in parts
    (1, 3000, 7, 1, 1, 64, None),       # few keys, many rows: rows in parts
    (4, 129, 200, 2, 2, 64, [33, 128, 64, 0]),
    (300, 3, 5, 8, 8, 32, None),
    (2, 1, 2000, 4, 2, 48, [1999, 3]),
    (3, 64, 32, 2, 1, 112, [-4, 32, 99]),  # lengths outside 0 .. keys are taken at its ends
]


def run(q, kv, lengths, dout, scale=None):
    q, kv = q.cuda().requires_grad_(True), kv.cuda().requires_grad_(True)
    lengths = None if lengths is None else torch.tensor(lengths, device="cuda")
    out = nori_amd.trainable_attention(q, kv, lengths, scale=scale)
    dq, dkv = torch.autograd.grad(out, (q, kv), dout.cuda())
    return out.detach(), dq, dkv


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_result_and_gradients(cuda, shape, dtype):
    *sizes, lengths = shape
    q, kv, dout = inputs(*sizes, dtype)
    out, dq, dkv = run(q, kv, lengths, dout)
    expected, bounds = reference(q, kv, lengths, dout)
    assert_near("out", out, expected[0], bounds[0])
    assert_near("dq", dq, expected[2], bounds[2])
    assert_near("dkv", dkv, expected[3], bounds[3])
    with torch.no_grad():
        served = nori_amd.trainable_attention(q.cuda(), kv.cuda(), None if lengths is None else torch.tensor(lengths, device="cuda"))
    assert torch.equal(served, out)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_factors_of_the_logits(cuda, scale, dtype):
    q, kv, dout = inputs(2, 40, 70, 2, 2, 24, dtype, seed=1)
    out, dq, dkv = run(q, kv, None, dout, scale)
    expected, bounds = reference(q, kv, None, dout, scale)
    for name, got, i in (("out", out, 0), ("dq", dq, 2), ("dkv", dkv, 3)):
        assert_near(name, got, expected[i], bounds[i])


@pytest.mark.parametrize("dout_scale", [1e-6, 2e3])
def test_float16_gradients_far_from_one(cuda, dout_scale):
    """Slopes near float16's least, and ones whose products with v pass its largest."""
    q, kv, dout = inputs(1, 200, 500, 2, 2, 64, torch.float16, seed=2, dout_scale=dout_scale)
    kv[:, :, 1] *= 8
    out, dq, dkv = run(q, kv, None, dout)
    expected, bounds = reference(q, kv, None, dout)
    assert_near("dq", dq, expected[2], bounds[2])
    assert_near("dkv", dkv, expected[3], bounds[3])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_long_contexts_keep_small_probabilities(cuda, dtype):
    """One key far above many: the many carry a share that float16's subnormals would cut."""
    q, kv, dout = inputs(1, 3, 20000, 1, 1, 32, dtype, seed=3)
    kv[:, :, 0] *= 0.1
    kv[:, 17, 0] = 6 * q[:, 0] / q[:, 0].float().norm().to(dtype) * 3
    out, dq, dkv = run(q, kv, None, dout)
    expected, bounds = reference(q, kv, None, dout)
    for name, got, i in (("out", out, 0), ("dq", dq, 2), ("dkv", dkv, 3)):
        assert_near(name, got, expected[i], bounds[i])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_padding_is_not_looked_at(cuda, dtype):
    q, kv, dout = inputs(4, 70, 90, 2, 2, 44, dtype, seed=4)
    lengths = [50, 0]
    clean = run(q, kv, lengths, dout)
    for bad in (math.nan, math.inf, torch.finfo(dtype).min):
        dirty = kv.clone()
        dirty[:2, 50:] = bad
        dirty[2:] = bad
        for a, b in zip(clean, run(q, dirty, lengths, dout)):
            assert torch.equal(a, b)
    out, dq, dkv = clean
    assert not out[2:].any() and not dq[2:].any() and not dkv[2:].any() and not dkv[:2, 50:].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_a_key_at_minus_infinity_has_no_part(cuda, dtype):
    """Logits of -inf (a key of -inf under a positive query) leave the other keys' probabilities as they are."""
    q, kv, dout = inputs(1, 40, 100, 1, 1, 32, dtype, seed=5)
    q = q.abs() + 0.5
    kv[:, :33, 0] = -math.inf  # a whole first tile of the scan
    out, dq, dkv = run(q, kv, None, dout)
    expected, bounds = reference(q, kv[:, 33:], None, dout)
    assert_near("out", out, expected[0], bounds[0])
    assert_near("dv", dkv[:, 33:, 1], expected[3][:, :, 1], bounds[3][:, :, 1])
    assert not dkv[:, :33, 1].any()


def test_rows_that_are_not_finite_stay_apart(cuda):
    q, kv, dout = inputs(2, 100, 100, 2, 2, 64, torch.float16, seed=6)
    clean = run(q, kv, None, dout)
    q[0, 7, 1, 3] = math.nan
    out, dq, _ = run(q, kv, None, dout)
    assert out[0, 7, 1].isnan().all() and dq[0, 7, 1].isnan().all()
    keep = torch.ones(2, 100, 2, dtype=torch.bool)
    keep[0, 7, 1] = False
    assert torch.equal(out.cpu()[keep], clean[0].cpu()[keep]) and torch.equal(dq.cpu()[keep], clean[1].cpu()[keep])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strides(cuda, dtype):
    """Queries and keys out of one stacked projection, expanded and transposed slopes, odd offsets: the contiguous call's bits."""
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(3, 50, 3, 2, 24, generator=g).to(dtype).cuda()
    dout = torch.randn(3, 50, 2, 24, generator=g).to(dtype)
    expected = run(qkv[:, :, 0].contiguous(), qkv[:, :, 1:].contiguous(), None, dout)
    assert all(torch.equal(a, b) for a, b in zip(expected, run(qkv[:, :, 0], qkv[:, :, 1:], None, dout)))
    odd = torch.empty(qkv.numel() + 1, dtype=dtype, device="cuda")[1:].view(qkv.shape).copy_(qkv)
    assert all(torch.equal(a, b) for a, b in zip(expected, run(odd[:, :, 0], odd[:, :, 1:], None, dout)))
    across = qkv.permute(4, 0, 1, 2, 3).contiguous().permute(1, 2, 3, 4, 0)
    assert all(torch.equal(a, b) for a, b in zip(expected, run(across[:, :, 0], across[:, :, 1:], None, dout)))
    turned = dout.transpose(1, 2).contiguous().transpose(1, 2)
    assert all(torch.equal(a, b) for a, b in zip(expected, run(qkv[:, :, 0], qkv[:, :, 1:], None, turned)))
    one = torch.ones((), dtype=dtype, device="cuda").expand(3, 50, 2, 24)
    whole = run(qkv[:, :, 0], qkv[:, :, 1:], None, one.clone())
    assert all(torch.equal(a, b) for a, b in zip(whole, run(qkv[:, :, 0], qkv[:, :, 1:], None, one)))


def test_gradients_asked_for_apart(cuda):
    q, kv, dout = (t.cuda() for t in inputs(2, 70, 90, 4, 2, 44, torch.bfloat16, seed=8))
    _, dq, dkv = run(q, kv, [90, 11], dout)
    lengths = torch.tensor([90, 11], dtype=torch.int32, device="cuda")
    lone = q.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nori_amd.trainable_attention(lone, kv, lengths), lone, dout)[0], dq)
    lone = kv.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(nori_amd.trainable_attention(q, lone, lengths), lone, dout)[0], dkv)


def test_no_rows_and_no_keys(cuda):
    for shape in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)):
        bg, nq, nk = shape
        q = torch.randn(bg, nq, 2, 8, device="cuda", requires_grad=True)
        kv = torch.randn(bg, nk, 2, 1, 8, device="cuda", requires_grad=True)
        out = nori_amd.trainable_attention(q, kv)
        assert out.shape == q.shape and not out.any()
        dq, dkv = torch.autograd.grad(out, (q, kv), torch.ones_like(out))
        assert dq.shape == q.shape and dkv.shape == kv.shape and not dq.any() and not dkv.any()


def test_the_same_bits_again(cuda):
    for sizes in ((1, 3, 5000, 2, 1, 64), (2, 300, 300, 2, 2, 44), (1, 4000, 40, 2, 1, 64)):
        q, kv, dout = inputs(*sizes, torch.float16, seed=9)
        first = run(q, kv, None, dout)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, run(q, kv, None, dout)))


def test_differences(cuda):
    """The fp32 gradients along a direction against the difference of two results: with step t its third-order term is
    below t^2 times the third derivative (of order the values themselves here, all of unit scale), the results' error over t."""
    q, kv, dout = (t.cuda() for t in inputs(2, 20, 30, 2, 1, 16, torch.float32, seed=10))
    _, dq, dkv = run(q, kv, [30, 12], dout)
    lengths = torch.tensor([30, 12], device="cuda")
    g = torch.Generator().manual_seed(11)
    a, b = torch.randn(q.shape, generator=g).cuda(), torch.randn(kv.shape, generator=g).cuda()
    t = 2.0**-7
    value = lambda s: (nori_amd.trainable_attention(q + s * a, kv + s * b, lengths).double() * dout).sum()
    along = ((dq.double() * a).sum() + (dkv.double() * b).sum()).item()
    # values: 1280 results of about 0.5 times slopes of 0.1; third derivatives along unit directions of 16 columns: about 50
    # times as much at t^2 / 6; errors of the results 2^-20 of each over t
    size = (dout.abs().sum()).item()
    assert abs((value(t) - value(-t)).item() / (2 * t) - along) <= size * (50 * t * t / 6 + 2.0**-20 / t)


def test_other_stream_and_captured(cuda):
    q, kv, dout = (t.cuda() for t in inputs(2, 100, 700, 2, 2, 44, torch.float16, seed=12))
    lengths = torch.tensor([700, 31], device="cuda")
    q.requires_grad_(True), kv.requires_grad_(True)

    def step():
        out = nori_amd.trainable_attention(q, kv, lengths)
        return (out, *torch.autograd.grad(out, (q, kv), dout))

    def eager():
        return [t.detach().clone() for t in step()]

    first = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(first, eager()))
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = [t.detach() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        with torch.no_grad():
            for t, s in zip((q, kv, dout), inputs(2, 100, 700, 2, 2, 44, torch.float16, seed=20 + seed)):
                t.copy_(s)
            lengths.copy_(torch.tensor([650 - seed, seed]))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in kept]
        assert all(torch.equal(a, b) for a, b in zip(got, eager()))


def test_rows_whose_offsets_pass_32_bits(cuda):
    """A context whose rows lie 2^16 elements apart, 70,000 of them: the contiguous call's bits."""
    g = torch.Generator().manual_seed(13)
    far = torch.empty(70000 * 65536, dtype=torch.float16, device="cuda").as_strided((1, 70000, 2, 1, 16), (70000 * 65536, 65536, 16, 16, 1))
    kv = torch.randn(1, 70000, 2, 1, 16, generator=g).half()
    far.copy_(kv)
    q, dout = torch.randn(1, 3, 2, 16, generator=g).half(), torch.randn(1, 3, 2, 16, generator=g).half()

    def grads(t):
        a, b = q.cuda().requires_grad_(True), t.detach().requires_grad_(True)
        out = nori_amd.trainable_attention(a, b)
        return (out, *torch.autograd.grad(out, (a, b), dout.cuda()))

    assert all(torch.equal(x, y) for x, y in zip(grads(far), grads(kv.cuda())))


def test_few_keys_keep_small_differences(cuda):
    """Two keys: ds is a difference of nearly equal products, which delta of a rounded result would swamp."""
    for dtype in (torch.float16, torch.bfloat16):
        for nq in (5, 300):  # both backward passes
            q, kv, dout = inputs(8, nq, 2, 2, 2, 64, dtype, seed=14)
            kv[:, 1] = kv[:, 0]
            kv[:, 1, 1, :, ::7] += 0.5
            kv[:, 0, 1] += 4
            kv[:, 1, 1] += 4
            out, dq, dkv = run(q, kv, None, dout)
            expected, _ = reference(q, kv, None, dout)
            # p is 1/2 and ds exact but for its own rounding, p's, and the fp32 sums beside products of up to 64 x 4.5 x 0.5:
            # 2^-23 x 144 x 64 at most of terms that are 0.05 in the mean
            h = torch.finfo(dtype).eps / 2
            assert (dkv[:, :, 0].double().cpu() - expected[3][:, :, 0]).norm() <= 4 * h * expected[3][:, :, 0].norm()


def test_shared_and_broadcast_contexts(cuda):
    """One context expanded over the batch: its gradient is the sum over the batch."""
    q, kv, dout = (t.cuda() for t in inputs(3, 40, 50, 4, 2, 24, torch.float32, seed=15))
    one = kv[:1].clone().requires_grad_(True)
    d = torch.autograd.grad(nori_amd.trainable_attention(q, one.expand(3, -1, -1, -1, -1)), one, dout)[0]
    whole = kv[:1].repeat(3, 1, 1, 1, 1).requires_grad_(True)
    each = torch.autograd.grad(nori_amd.trainable_attention(q, whole), whole, dout)[0]
    assert torch.equal(d, each.sum(0, keepdim=True))


def test_second_derivatives_are_refused(cuda):
    q, kv, _ = (t.cuda().requires_grad_(True) for t in inputs(1, 3, 4, 1, 1, 8, torch.float32))
    dq = torch.autograd.grad(nori_amd.trainable_attention(q, kv).square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), kv)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [
    (3, 48, 48, 2, 2, 44, [48, 0, 47]),
    (3, 47, 33, 1, 1, 64, [33, 16, 32]),
    (2, 24, 41, 4, 2, 56, None),        # 48 rows of two heads that share a key head
    (2, 49, 48, 2, 2, 44, [48, 17]),
    (2, 48, 49, 2, 1, 32, [49, 48]),
    (5, 1, 48, 1, 1, 48, None),
    (5, 48, 1, 1, 1, 40, None),
    (70, 33, 33, 3, 3, 12, None),
], ids=lambda s: "x".join(map(str, s[:6])))
def test_units_of_about_48_rows_and_keys(cuda, shape, dtype):
    """Rows and keys at and beside the ends of the tiles' halves, NaN and infinities behind the lengths among them."""
    *sizes, lengths = shape
    q, kv, dout = inputs(*sizes, dtype, seed=9)
    expected, bounds = reference(q, kv, lengths, dout)
    if lengths is not None:
        for i, n in enumerate(lengths * (len(kv) // len(lengths))):
            kv[i, n:] = (math.nan, math.inf, -math.inf)[i % 3]
    out, dq, dkv = run(q, kv, lengths, dout)
    for name, got, i in (("out", out, 0), ("dq", dq, 2), ("dkv", dkv, 3)):
        assert_near(name, got, expected[i], bounds[i])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 33, 300])
def test_one_key_takes_no_gradient_of_queries(cuda, queries, dtype):
    q, kv, dout = inputs(3, queries, 5, 2, 1, 36, dtype, seed=10)
    _, dq, _ = run(q, kv[:, :1], None, dout)
    assert not dq.any()
    _, dq, _ = run(q, kv, [1, 0, 1], dout)
    assert not dq.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("queries, keys", [(1, 3001), (5, 3001), (1, 65536), (3, 20000)])
def test_copied_operands_beside_a_workspace(cuda, queries, keys, dtype):
    """Few rows over many keys, in parts whose results lie in a workspace, with q and kv at odd offsets and with their heads' elements
    apart, which go in as copies: the contiguous call's bits, served and trained."""
    q, kv, dout = (t.cuda() for t in inputs(2, queries, keys, 2, 2, 64, dtype, seed=16))
    apart = lambda t: t.movedim(-1, 0).contiguous().movedim(0, -1)
    odd = lambda t: torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t)
    lengths = torch.tensor([keys, keys - 7], device="cuda")
    with torch.no_grad():
        served = nori_amd.trainable_attention(q, kv, lengths)
    trained = run(q, kv, [keys, keys - 7], dout)
    assert torch.equal(served, trained[0])
    for change in (odd, apart):
        for x, y in ((change(q), change(kv)), (change(q), kv), (q, change(kv))):
            with torch.no_grad():
                assert torch.equal(nori_amd.trainable_attention(x, y, lengths), served)
            assert all(torch.equal(a, b) for a, b in zip(trained, run(x, y, [keys, keys - 7], change(dout))))


@pytest.mark.parametrize("queries, keys", [(1, 30000), (3, 3000), (200, 3000), (40, 64)])
def test_float16_probabilities_far_below_the_largest(cuda, queries, keys):
    """One key 2^23 to 2^30 above all others, whose values are the larger ones. The forward pass holds a probability in float16 beside
    the largest so far (of a part of the keys), under 2^8: normal down to 2^-22 of it, and off by at most half of float16's
    subnormal step, 2^-25 / 2^8 = 2^-33 of the row's largest, below. The other bounds are those of every shape."""
    g = torch.Generator().manual_seed(17)
    q, kv, dout = inputs(2, queries, keys, 2, 1, 32, torch.float16, seed=17)
    q[..., 0], q[..., 1:] = 4, q[..., 1:] * 2.0**-6
    kv[:, :, 0] *= 2.0**-6
    kv[:, :, 0, :, 0] = (22 - math.log(2) * (23 + 7 * torch.rand(2, keys, 1, generator=g))) / 4
    kv[:, :, 1] = kv[:, :, 1].abs() * 256
    at = torch.randint(keys, (2,), generator=g).tolist()
    for i in range(2):
        kv[i, at[i], 0, :, 0] = 5.5
        kv[i, at[i], 1] *= 2.0**-12
    out, dq, dkv = run(q, kv, None, dout, 1.0)
    expected, bounds = reference(q, kv, None, dout, 1.0)
    low = 2.0**-33 * kv[:, :, 1].double().abs().sum(1)[:, None]  # one key head
    assert_near("out", out, expected[0], bounds[0] + low)
    # delta of a result that is off by as much, in each ds = p (dout v - delta)
    off = (dout.double().abs() * low).sum(-1)  # [BG, Q, H]
    p = torch.softmax(torch.einsum("bqhd,bkd->bqhk", q.double(), kv[:, :, 0, 0].double()), -1) * off[..., None]
    k = kv[:, :, 0, 0].double().abs()
    assert_near("dq", dq, expected[2], bounds[2] + torch.einsum("bqhk,bkd->bqhd", p, k))
    more = torch.zeros_like(expected[3])
    more[:, :, 0, 0] = torch.einsum("bqhk,bqhd->bkd", p, q.double().abs())
    assert_near("dkv", dkv, expected[3], bounds[3] + more)
