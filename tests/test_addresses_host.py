"""Kernels are called with addresses: each is of a tensor that is still there when the call is made (no GPU needed, nothing is launched)."""

import gc

import pytest
import torch

from nori_amd import _native as nat
from nori_amd import encoders, norm


class Library:
    """Stands for the library: each call is recorded with those of its addresses at which no tensor lives."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            live = {t.data_ptr() for t in gc.get_objects() if issubclass(type(t), torch.Tensor)}
            addresses = [getattr(a, "value", a) for a in args]
            self.calls.append((name, [a for a in addresses if isinstance(a, int) and a > 1 << 32 and a not in live]))
            return nat.NORI_OK

        return call


class OnGPU(torch.Tensor):
    """A tensor that says it is on a GPU."""

    is_cuda = True


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(nat, "lib", lambda: lib)
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    return lib


def transposed(*shape):
    return torch.randn(*reversed(shape)).half().t()


def test_residual_epilogues_of_transposed_weights(library):
    x = torch.randn(64, 128).half().as_subclass(OnGPU)
    stream = torch.randn(64, 128)
    weights = transposed(512, 128), transposed(128, 256)
    assert norm.swiglu_mlp_residual(x, *weights, 256, stream, 0.5)
    assert norm.swiglu_mlp_residual_norm(x, *weights, 256, stream, 0.5, 1e-5, 128) is not None
    assert library.calls == [("nori_swiglu_mlp_residual", []), ("nori_swiglu_mlp_residual_rms_norm", [])]


def test_cell_tokens_of_double_centers(library):
    encoder = encoders.MaskEmbEncoder(
        num_features=2, emsize=128, mask_embedding_size=128, numeric_embed_type="RBF",
        RBF_config=dict(token_embed_dim=8, n_kernels=16, sigma=0.5, use_learn_sigma=False, use_learn_embeddings=False,
                        use_original_features=False),
        prompt_quantile_ple_bins=32)
    encoder.numeric_mlp.centers = encoder.numeric_mlp.centers.double()
    encoder.numeric_mlp.sigma = encoder.numeric_mlp.sigma.double()
    x = torch.randn(2, 5, 3, 2)
    key = encoders.PromptQuantilePLEEncoder.reference_key
    torch.set_autocast_enabled("cuda", True)
    try:
        with torch.no_grad():
            assert encoder._tokens_on_device(x, {key: {"edges": torch.randn(2, 3, 2, 33)}}) is not None
    finally:
        torch.set_autocast_enabled("cuda", False)
    assert [name for name, _ in library.calls] == ["nori_cell_tokens"] and not library.calls[0][1]
