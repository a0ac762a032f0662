"""layer_norm on rows whose mean is large beside their spread.

The mean is a sum in 64 bits, kept as a pair of float32 numbers: x - mean has no error that grows with the mean.  u = 2^-24.
Equal values: the sum of D of them is exact in 64 bits (24 + 24 bits), so is the mean, and y is the bias to the bit, dw
zero and dx = r (g - mean(g)).  Other rows: x - hi is exact for x within a factor of two of hi, - lo rounds it once; the
variance is a sum of squares of those (chains of at most 32 additions a lane, 12 joins: 48 u), its root and the division add
3 u, so xh is off by 32 u |xh| and u |lo| r, |lo| <= half a step of the mean; two more operations for w and b."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# every register form of the forward pass, its ragged ends, and the looped form
DIMS32 = [1, 3, 7, 33, 96, 97, 191, 250, 384, 500, 766, 1001, 2047, 4099, 8191, 16384, 16385, 20001]


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


def _affine(D, t=F32):
    g = torch.Generator(device=DEV).manual_seed(D)
    return (1 + 0.3 * torch.randn(D, device=DEV, generator=g)).to(t), (0.2 * torch.randn(D, device=DEV, generator=g)).to(t)


VALUES = [0.1, 100.1, 1000.1, 4096.3, 30000.7, -1234567.0]


@pytest.mark.parametrize("D", DIMS32)
def test_equal_values_fp32(D):
    import swingnn_amd as S
    w, b = (t.requires_grad_(True) for t in _affine(D))
    x = torch.tensor(VALUES, device=DEV)[:, None].expand(-1, D).contiguous().requires_grad_(True)
    y = S.layer_norm(x, w, b)
    assert torch.equal(y, b.detach().expand(len(VALUES), D))
    dy = torch.randn(len(VALUES), D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert not dw.any()
    g = dy.double() * w.detach().double()
    want = (g - g.mean(-1, keepdim=True)) / 1e-5 ** 0.5
    # sums of g in float32 (64 u of the largest term), r and two products; eps itself is off by u in float32
    assert float((dx.double() - want).abs().max()) <= 80 * U * 2 * float(g.abs().max()) / 1e-5 ** 0.5


@pytest.mark.parametrize("D", [96, 1001, 4096, 20000, 32769])
@pytest.mark.parametrize("t", [BF16, F16])
def test_equal_values_half(D, t):
    import swingnn_amd as S
    w, b = _affine(D, t)
    x = torch.tensor([0.1, 100.1, 1000.1, 30000.7], device=DEV).to(t)[:, None].expand(-1, D)
    assert torch.equal(S.layer_norm(x, w, b), b.expand(4, D))


@pytest.mark.parametrize("D", DIMS32)
@pytest.mark.parametrize("at", [1000.1, 30000.7])
def test_values_a_few_steps_apart(D, at):
    import swingnn_amd as S
    w, b = _affine(D)
    c = torch.tensor(at, device=DEV)
    step = float(torch.nextafter(c, c + 1) - c)
    k = torch.randint(-3, 4, (33, D), device=DEV, generator=torch.Generator(device=DEV).manual_seed(D))
    x = c + step * k.float()
    xd = x.double()
    xc = xd - xd.mean(-1, keepdim=True)
    r = 1 / (xc.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    xh = xc * r
    want = xh * w.double() + b.double()
    bound = w.double().abs() * (34 * U * xh.abs() + U * step * r) + 2 * U * (want.abs() + b.double().abs())
    d = (S.layer_norm(x, w, b).double() - want).abs()
    assert float((d - bound).max()) <= 0, (float(d.max()), float((d / bound).max()))
