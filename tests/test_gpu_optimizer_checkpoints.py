"""Checkpoints of the fused optimizers that do not belong to the optimizer that loads them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _params(*shapes):
    return [torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in shapes]


def test_adam_refuses_a_muon_checkpoint_without_others():
    """One group and equal sizes on both sides."""
    import swingnn_amd as S
    muon = S.FusedMuonEMA(_params((4, 8)), lr=1e-3)
    adam = S.FusedAdamEMA(_params((4, 8)), lr=1e-3)
    with pytest.raises(ValueError):
        adam.load_state_dict(muon.state_dict())
    with pytest.raises(ValueError):
        muon.load_state_dict(adam.state_dict())
    assert set(adam.param_groups[0]) >= {"betas", "eps"} and "momentum" not in adam.param_groups[0]
    adam.load_state_dict(adam.state_dict())
    muon.load_state_dict(muon.state_dict())
