"""Parameters and gradients whose layout changed under an optimizer that holds their addresses, at the SAME address: the
call is refused before anything is read or written.  Where storage moved and the layout stayed, the step goes on."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _make(kind):
    import swingnn_amd as S
    g = torch.Generator(device=DEV).manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV, generator=g)) for s in [(24, 24), (16, 40), (48,)]]
    opt = S.FusedMuonEMA(params[:2], params[2:], lr=1e-3) if kind == "muon" else S.FusedAdamEMA(params, lr=1e-3)
    for p in params:
        p.grad = torch.randn(*p.shape, device=DEV, generator=g)
    opt.step()
    return params, opt


def _refused(params, opt):
    before, steps = [p.detach().clone() for p in params], opt.step_count
    m = opt.m.clone()
    with pytest.raises(NotImplementedError):
        opt.step()
    assert opt.step_count == steps and torch.equal(opt.m, m) and all(torch.equal(p, q) for p, q in zip(params, before))


@pytest.mark.parametrize("kind", ["muon", "adam"])
@pytest.mark.parametrize("change", ["square transposed", "transposed", "other shape", "flat"])
def test_layout_changed_in_place(kind, change):
    params, opt = _make(kind)
    k = 0 if change == "square transposed" else 1
    p = params[k]
    at = p.data_ptr()
    p.grad = None
    p.data = {"square transposed": lambda t: t.t(), "transposed": lambda t: t.t(), "other shape": lambda t: t.view(40, 16),
              "flat": lambda t: t.view(-1)}[change](p.data)
    assert p.data_ptr() == at
    p.grad = torch.ones(p.shape, device=DEV)
    _refused(params, opt)


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_fewer_rows_in_place(kind):
    params, opt = _make(kind)
    p = params[1]
    p.grad = None
    p.data = p.data[:5]
    p.grad = torch.ones(5, 40, device=DEV)
    _refused(params, opt)


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_gradient_of_another_shape(kind):
    params, opt = _make(kind)
    params[1].grad.data = torch.ones(5, 40, device=DEV)
    _refused(params, opt)


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_moved_storage_and_gradients_of_other_strides_go_on(kind):
    params, opt = _make(kind)
    twins, other = _make(kind)
    params[1].data = params[1].data.clone()
    g = params[1].grad
    params[1].grad = g.t().contiguous().t()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins)) and torch.equal(opt.m, other.m)
