"""The adapters' modules apart from their kernels: casts, moves and saved states (CPU)."""
import copy

import pytest
import torch
from torch import nn

import nori_amd


def _decoder():
    return nn.Sequential(nn.Linear(8, 12), nn.LayerNorm(12), nn.GELU(), nn.Linear(12, 5))


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                                  lambda m: nn.Sequential(m).half()])
def test_scales_stay_as_they_are_through_casts(cast):
    # low_rank_update takes float32 scales, and 1 / 3 has more digits than 16 bits hold
    bank = nori_amd.LowRankAdapters(2, 8, 12, 3, alpha=1.0)
    cast(bank)
    assert bank.a.dtype != torch.float32 and bank.scales.dtype == torch.float32
    assert bank.scales.tolist() == [torch.tensor(1.0 / 3.0).item()] * 2
    assert copy.deepcopy(bank).scales.dtype == torch.float32


def test_scales_move_and_load_with_the_bank():
    bank = nori_amd.ReadoutAdapters(_decoder(), 2, 3, alpha=1.0)
    other = nori_amd.ReadoutAdapters(_decoder(), 2, 3, alpha=6.0).half()
    other.load_state_dict(bank.state_dict())
    assert other.last.scales.dtype == torch.float32 and torch.equal(other.last.scales, bank.last.scales)
    assert bank.half().float().first.scales.tolist() == [torch.tensor(1.0 / 3.0).item()] * 2
    assert bank.to("meta").first.scales.device.type == "meta" and bank.first.scales.dtype == torch.float32
    empty = nori_amd.LowRankAdapters(2, 8, 12, 3, device="meta").to_empty(device="cpu")
    assert empty.scales.device.type == "cpu" and empty.scales.dtype == torch.float32


@pytest.fixture(scope="module")
def models():
    from nori_amd.api import NORI_6M_CONFIG, build_model

    two_phase = dict(NORI_6M_CONFIG, nlayers=1, two_phase_config=dict(target_tokens=1, row_layers=1, row_heads=2, row_hidden_dim=64))
    return build_model(dict(NORI_6M_CONFIG, nlayers=1)), build_model(two_phase)


@pytest.mark.parametrize("ids,match", [([0, 1, -1], "return_embeddings gives the row states"), (None, "each of the 3 tables"),
                                       ([0, 1], "each of the 3 tables")])
def test_adapters_are_not_left_out_of_row_states(models, ids, match):
    # row states are not decoded: adapters asked for beside them would do nothing; refused before the layers run
    dense, two_phase = models
    bank = nori_amd.ReadoutAdapters(dense.reg_y_decoder, 2, 4)
    x, y = torch.randn(3, 10, 6), torch.randn(3, 8)
    with pytest.raises(ValueError, match=match):
        dense.apply_context_cache(x, None, return_embeddings=True, readout_adapters=bank, table_adapters=ids)
    with pytest.raises(ValueError, match=match):
        two_phase(x, y, 8, task_type="reg", return_embeddings=True, readout_adapters=bank, table_adapters=ids)
    with pytest.raises(ValueError, match="without readout_adapters"):
        dense.apply_context_cache(x, None, return_embeddings=True, table_adapters=[0, 0, 0])
    with pytest.raises(ValueError, match="without readout_adapters"):
        two_phase(x, y, 8, task_type="reg", return_embeddings=True, table_adapters=[0, 0, 0])
