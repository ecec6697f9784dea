"""What a call of the adapters does to torch's own records, with the kernels left out (CPU)."""
import types

import pytest
import torch

import nori_amd
from nori_amd import _native as nat


@pytest.fixture
def calls(monkeypatch):
    """Calls of the library by name and arguments; each is a success of no effect."""
    made = []

    class Library:
        def __getattr__(self, name):
            def call(*args):
                made.append((name, args))
                return 0

            return call

    monkeypatch.setattr(nat, "require_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    monkeypatch.setattr(nat, "lib", lambda: library)
    monkeypatch.setattr(nori_amd.AdapterPlan, "used_on", lambda plan, stream: made.append(("used_on", (plan, stream))), raising=False)
    library = Library()
    return made


def _plan(rows):
    plan = object.__new__(nori_amd.AdapterPlan)
    plan._packed = torch.tensor([0, rows, 0, *range(rows)], dtype=torch.int32)
    plan.rows, plan.most, plan.groups, plan.longest, plan.adapters = rows, 0, 1, rows, (0,)
    return plan


def _args(rows=5):
    return types.SimpleNamespace(x=torch.randn(rows, 8), y=torch.randn(rows, 6), a=torch.randn(1, 4, 8), b=torch.randn(1, 6, 4))


@pytest.mark.parametrize("place", ["y", "columns", "turned"])
def test_out_is_seen_to_change(calls, place):
    # another graph saved the tensor: its backward pass has to notice that the values are gone, as after torch's own calls
    t = _args()
    out = {"y": t.y, "columns": torch.randn(5, 9)[:, 2:8], "turned": torch.randn(6, 5).t()}[place]
    w = torch.randn(5, 6, requires_grad=True)
    loss = (w * out).sum()
    with torch.no_grad():
        nori_amd.low_rank_update(t.x, t.y, t.a, t.b, _plan(5), out=out)
    assert any(name == "nori_low_rank_update" for name, _ in calls)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_out_in_inference_mode(calls):
    with torch.inference_mode():
        t = _args()
        assert nori_amd.low_rank_update(t.x, t.y, t.a, t.b, _plan(5), out=t.y) is t.y


def _decoder():
    return torch.nn.Sequential(torch.nn.Linear(8, 12), torch.nn.LayerNorm(12), torch.nn.GELU(), torch.nn.Linear(12, 6))


@pytest.mark.parametrize("watch", ["register_full_backward_hook", "register_full_backward_pre_hook", "register_forward_hook"])
@pytest.mark.parametrize("part", [0, 1, 3])
def test_watched_parts_of_a_decoder_are_called(calls, watch, part):
    decoder = _decoder().requires_grad_(False)
    bank = nori_amd.ReadoutAdapters(decoder, 1, 4)
    seen = []
    getattr(decoder[part], watch)(lambda m, *rest: seen.append(m))
    bank(decoder, torch.randn(5, 8, requires_grad=True), _plan(5)).sum().backward()
    assert seen == [decoder[part]]


@pytest.mark.parametrize("watch", ["register_full_backward_hook", "register_full_backward_pre_hook", "register_forward_hook",
                                   "register_forward_pre_hook"])
def test_watched_decoders_are_refused(calls, watch):
    # the decoder's parts are called one by one: a hook of the whole would not see them
    decoder = _decoder()
    bank = nori_amd.ReadoutAdapters(decoder, 1, 4)
    handle = getattr(decoder, watch)(lambda m, *rest: None)
    with pytest.raises(NotImplementedError, match="hooks"):
        bank(decoder, torch.randn(5, 8), _plan(5))
    handle.remove()
    assert bank(decoder, torch.randn(5, 8), _plan(5)).shape == (5, 6)


def test_decoders_with_a_forward_of_their_own_are_refused(calls):
    class Doubled(torch.nn.Sequential):
        def forward(self, x):
            return 2 * super().forward(x)

    class Named(torch.nn.Sequential):
        pass

    with pytest.raises(ValueError, match="decoder"):
        nori_amd.ReadoutAdapters(Doubled(*_decoder()), 1, 4)
    decoder = _decoder()
    bank = nori_amd.ReadoutAdapters(decoder, 1, 4)
    with pytest.raises(ValueError, match="decoder"):
        bank(Doubled(*decoder), torch.randn(5, 8), _plan(5))
    assert bank(Named(*decoder), torch.randn(5, 8), _plan(5)).shape == (5, 6)


def test_out_shares_nothing_with_scales(calls):
    # the scales are read while out is written
    t = _args()
    memory = torch.randn(40)
    y, scales = memory[:30].view(5, 6), memory[3:4]
    with pytest.raises(ValueError, match="shares elements"):
        nori_amd.low_rank_update(t.x, y, t.a, t.b, _plan(5), scales, out=y)
    assert nori_amd.low_rank_update(t.x, y, t.a, t.b, _plan(5), memory[30:31], out=y) is y


def test_sizes_are_asked_for_on_the_tensors_device(calls, monkeypatch):
    # workspaces go by the compute units of the current device, as the launch does: both have to be asked in its context
    import contextlib

    inside, asked = [], []

    @contextlib.contextmanager
    def on(device):
        inside.append(device)
        yield
        inside.pop()

    class Library:
        def __getattr__(self, name):
            def call(*args):
                asked.append((name, bool(inside)))
                return 0

            return call

    monkeypatch.setattr(nat, "on", on)
    monkeypatch.setattr(nat, "lib", Library)
    t = _args()
    for leaf in (t.x, t.a, t.b):
        leaf.requires_grad_(True)
    nori_amd.low_rank_update(t.x, t.y, t.a, t.b, _plan(5)).sum().backward()
    x = torch.randn(5, 8, requires_grad=True)
    nori_amd.trainable_layer_norm(x, torch.ones(8, requires_grad=True), None).sum().backward()
    names = [n for n, _ in asked if n.startswith("nori_low_rank") or n.startswith("nori_layer_norm")]
    assert {"nori_low_rank_workspace_bytes", "nori_low_rank_backward_workspace_bytes", "nori_layer_norm_train_workspace_bytes"} <= set(names)
    assert all(ok for n, ok in asked if n in names), asked


def test_plans_are_told_of_the_streams_that_read_them(calls):
    t = _args()
    plan = _plan(5)
    x = t.x.requires_grad_(True)
    nori_amd.low_rank_update(x, t.y, t.a, t.b, plan).sum().backward()
    at = [i for i, (name, _) in enumerate(calls) if name == "used_on"]
    assert [calls[i + 1][0] for i in at] == ["nori_low_rank_update", "nori_low_rank_backward"]  # just before each launch
    assert all(calls[i][1][0] is plan for i in at)


@pytest.mark.parametrize("leaf", ["x", "y", "a", "b"])
@pytest.mark.parametrize("frozen", [True, False])
def test_x_times_a_is_kept_for_b_alone(calls, leaf, frozen):
    # no other gradient reads it
    t = _args()
    getattr(t, leaf).requires_grad_(True)
    if frozen:
        if leaf == "y":
            return
        out = nori_amd.adapted_linear(t.x, torch.randn(6, 8), None, t.a, t.b, _plan(5))
    else:
        out = nori_amd.low_rank_update(t.x, t.y, t.a, t.b, _plan(5))
    out.sum().backward()
    sent = {name: args for name, args in calls}
    assert (sent["nori_low_rank_update"][19] is not None) == (leaf == "b")
    if leaf != "y":
        assert (sent["nori_low_rank_backward"][20] is not None) == (leaf == "b")


def test_the_library_wants_x_times_a_for_db_alone():
    lib = nat.lib()
    back = [16, nat.NORI_F32, 4, 8, 8, 16, 8, 8, None, 8, 16, 16, None, 2, 4, 16, 16, 16, 1, 4, None, 16, 8, 16, 16, None, 0, None]
    assert lib.nori_low_rank_backward(*back) == nat.NORI_ERR_INVALID and b"null pointer" in lib.nori_last_error()
    back[24] = None  # dx and da: refused for the workspace, before any device work
    assert lib.nori_low_rank_backward(*back) == nat.NORI_ERR_INVALID and b"workspace" in lib.nori_last_error()
    needs = [lib.nori_low_rank_backward_workspace_bytes(nat.NORI_F32, 100000, 8, 8, 4, 1, 100000, *n) for n in ((1, 0, 0), (1, 1, 0))]
    assert needs[0] < 100000 * 4 * 4 <= needs[1]  # dy b is kept for da alone


def test_a_norm_of_another_width_is_refused(calls):
    # without an affine nothing else names the width; torch's own layer norm raises
    decoder = torch.nn.Sequential(torch.nn.Linear(8, 12), torch.nn.LayerNorm(10, elementwise_affine=False), torch.nn.GELU(),
                                  torch.nn.Linear(12, 6))
    bank = nori_amd.ReadoutAdapters(decoder, 1, 4)
    with pytest.raises(RuntimeError, match="normalized_shape"):
        bank(decoder, torch.randn(5, 8), _plan(5))


@pytest.mark.parametrize("shape", [(0,), (2, 0), (0, 3), (2, 0, 3)])
def test_batches_without_rows(calls, shape):
    # of any number of dimensions: an empty one has no stride to go by
    plan = _plan(0)
    plan.groups, plan.adapters, plan._packed = 0, (), torch.zeros(1, dtype=torch.int32)
    a, b = (t.requires_grad_(True) for t in (torch.randn(2, 4, 8), torch.randn(2, 6, 4)))
    x, weight, bias = torch.randn(*shape, 8, requires_grad=True), torch.randn(6, 8), torch.randn(6)
    for call in (lambda: nori_amd.low_rank_update(x, torch.randn(*shape, 6), a, b, plan),
                 lambda: nori_amd.adapted_linear(x, weight, bias, a, b, plan)):
        out = call()
        grads = torch.autograd.grad(out.sum(), (x, a, b))
        assert out.shape == (*shape, 6) and [g.shape for g in grads] == [x.shape, a.shape, b.shape]
        assert not any(bool(g.any()) for g in grads)
        with torch.no_grad():
            assert call().shape == (*shape, 6)
    y = nori_amd.trainable_layer_norm(x, torch.ones(8, requires_grad=True), None)
    assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    out = torch.empty(*shape, 6)
    with torch.no_grad():
        assert nori_amd.low_rank_update(x, torch.randn(*shape, 6), a, b, plan, out=out) is out
