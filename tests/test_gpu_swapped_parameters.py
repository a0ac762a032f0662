"""Parameters of a fused optimizer that are swapped with others (torch.utils.swap_tensors, module.to() with
set_swap_module_params_on_conversion): the optimizer holds nothing that forbids it, and goes on with the new storage."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


@pytest.fixture
def swapping():
    was = torch.__future__.get_swap_module_params_on_conversion()
    torch.__future__.set_swap_module_params_on_conversion(True)
    yield
    torch.__future__.set_swap_module_params_on_conversion(was)


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_module_conversion_between_steps(kind, swapping):
    import swingnn_amd as S
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(24, 40), torch.nn.LayerNorm(40)).to(DEV)
    x = torch.randn(7, 24, device=DEV)
    opt = S.FusedMuonEMA(*S.FusedMuonEMA.split(net), lr=1e-2) if kind == "muon" else S.FusedAdamEMA(net.parameters(), lr=1e-2)

    def step():
        opt.zero_grad(set_to_none=True)
        net(x).square().sum().backward()
        before, version = [p.detach().clone() for p in net.parameters()], [p._version for p in net.parameters()]
        opt.step()
        for p, q, v in zip(net.parameters(), before, version):
            assert p._version > v and not torch.equal(p, q)

    step()
    opt.zero_grad(set_to_none=True)
    ids = [id(p) for p in net.parameters()]
    net.double()
    net.float()
    assert ids == [id(p) for p in net.parameters()]
    step()
    step()


@pytest.mark.parametrize("kind", ["muon", "adam"])
def test_swap_tensors(kind):
    import swingnn_amd as S
    p = torch.nn.Parameter(torch.randn(8, 16, device=DEV))
    opt = S.FusedMuonEMA([p], lr=1e-2) if kind == "muon" else S.FusedAdamEMA([p], lr=1e-2)
    p.grad = torch.randn_like(p)
    opt.step()
    q = torch.nn.Parameter(torch.zeros(8, 16, device=DEV))
    torch.utils.swap_tensors(p, q)
    p.grad = torch.randn_like(p)
    version = p._version
    opt.step()
    assert p._version > version and bool((p != 0).any())
