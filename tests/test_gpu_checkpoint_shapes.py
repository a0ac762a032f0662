"""A checkpoint goes back into parameters of the same shapes, not of the same sizes alone: moments and averages of an
(a, b) matrix are another matrix's when they are read as (b, a)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _make(kind, *shapes):
    import swingnn_amd as S
    g = torch.Generator(device=DEV).manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV, generator=g)) for s in shapes]
    opt = S.FusedMuonEMA(params[:1], params[1:], lr=1e-3) if kind == "muon" else S.FusedAdamEMA(params, lr=1e-3)
    for p in params:
        p.grad = torch.randn(*p.shape, device=DEV, generator=g)
    opt.step()
    return opt


@pytest.mark.parametrize("kind", ["muon", "adam"])
@pytest.mark.parametrize("shapes", [((8, 4), (6, 2)), ((4, 8), (12,)), ((2, 16), (6, 2))])
def test_other_shapes_of_the_same_sizes(kind, shapes):
    saved, other = _make(kind, (4, 8), (6, 2)), _make(kind, *shapes)
    sd, m, steps = saved.state_dict(), other.m.clone(), other.step_count
    sd["fused"]["m"].add_(1.0)
    with pytest.raises(ValueError, match="shapes"):
        other.load_state_dict(sd)
    assert torch.equal(other.m, m) and other.step_count == steps
    saved.load_state_dict(sd)
    assert torch.equal(saved.m, sd["fused"]["m"])


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_a_checkpoint_that_holds_no_shapes_still_loads(kind):
    saved, same = _make(kind, (4, 8), (6, 2)), _make(kind, (4, 8), (6, 2))
    sd = saved.state_dict()
    del sd["fused"]["shapes"]
    same.load_state_dict(sd)
    assert torch.equal(same.m, saved.m)
