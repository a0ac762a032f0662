"""LayerNorm under autocast: what nn.LayerNorm, whose place it takes, does there -- inputs and parameters of a half type
are normalised and returned in float32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


@pytest.mark.parametrize("xt,wt", [(F32, F32), (BF16, F32), (F16, F32), (BF16, BF16), (F32, BF16), (F32, F16)])
def test_types_and_values_as_nn_layer_norm(xt, wt):
    import swingnn_amd as S
    D = 120
    g = torch.Generator(device=DEV).manual_seed(1)
    plain, own = torch.nn.LayerNorm(D, device=DEV, dtype=wt), S.LayerNorm(D, device=DEV, dtype=wt)
    with torch.no_grad():
        plain.weight.copy_(1 + 0.3 * torch.randn(D, device=DEV, generator=g))
        plain.bias.copy_(0.2 * torch.randn(D, device=DEV, generator=g))
    own.load_state_dict(plain.state_dict())
    x = torch.randn(31, D, device=DEV, generator=g).to(xt)
    dy = torch.randn(31, D, device=DEV, generator=g)
    got = []
    for mod in (plain, own):
        xs = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=BF16):
            y = mod(xs)
        y.backward(dy)
        got.append((y, xs.grad, mod.weight.grad, mod.bias.grad))
    for p, q in zip(*got):
        assert p.dtype is q.dtype and p.shape == q.shape
    # float32 inside on both sides (64 u of values up to 8 in y and dx, of sums of 31 terms up to 12 in dw and db), then
    # dx, dw and db are rounded to their leaf's type: half a step each, two halves where the sides round apart
    for k, (p, q) in enumerate(zip(*got)):
        step = 0.0 if p.dtype is F32 else torch.finfo(p.dtype).eps
        bound = 64 * 2.0 ** -24 * (16 if k < 2 else 31 * 12) + step * p.double().abs()
        assert bool(((p.double() - q.double()).abs() <= bound).all()), k


def test_without_autocast_x_keeps_its_type():
    import swingnn_amd as S
    own = S.LayerNorm(64, device=DEV)
    x = torch.randn(5, 64, device=DEV).bfloat16()
    assert own(x).dtype is BF16
    with torch.autocast("cuda", dtype=BF16):
        assert S.layer_norm(x, own.weight, own.bias).dtype is BF16   # the function takes what it is given
        with torch.autocast("cuda", enabled=False):
            assert own(x).dtype is BF16
