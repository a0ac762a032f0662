"""FusedMuonEMA where the momentum and the gradient nearly cancel: u = a m + b g is then the rounding of its own sums, and
its norm as the three sums of m and g give it (a^2 <m,m> + 2 a b <m,g> + b^2 <g,g>) is the rounding of theirs.

Held: the step stays finite and no larger than an orthogonalised matrix can be.  Singular values of the result lie below
1.2024 (the quintic maps [0, 1.2024] into itself) and the kernels' roundings add less than 0.0076 (tests/orth_ref.py gives
1.5e-3), so |O|_F <= 1.21 sqrt(min(rows, cols)); the parameter's own rounding adds one step of 2^-24 |p| at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gauss(shape, seed):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _cancelling(opt, params, mu, nesterov, scale, seed):
    """m at `scale`, and the gradients that cancel it but for rounding."""
    a, b = (mu * mu, (1 - mu) * (1 + mu)) if nesterov else (mu, 1 - mu)
    opt.m.zero_()
    for i, (p, o) in enumerate(zip(params, opt._offs)):
        m = scale * _gauss(p.shape, 100 * seed + i)
        opt.m[o:o + p.numel()].copy_(m.reshape(-1))
        p.grad = (m.double() * (-a / b)).float()


def _step_and_check(opt, params, lr):
    before = [p.detach().clone() for p in params]
    opt.step()
    for p, q in zip(params, before):
        moved, (rows, cols) = (p.detach().double() - q.double()), p.shape
        bound = lr * 0.2 * max(rows, cols) ** 0.5 * 1.21 * min(rows, cols) ** 0.5 + 2.0 ** -23 * float(q.double().norm())
        assert bool(p.isfinite().all()), tuple(p.shape)
        assert float(moved.norm()) <= bound, (tuple(p.shape), float(moved.norm()), bound)


@pytest.mark.parametrize("mu,nesterov", [(0.5, True), (0.95, True), (0.3, True), (0.9, False)])
@pytest.mark.parametrize("scale", [1.0, 1e4])
@pytest.mark.parametrize("shapes", [[(1, 1), (1, 8), (8, 1), (4, 4), (1, 1000), (300, 1), (64, 200)],   # one workgroup each
                                    [(1, 1), (300, 400), (1, 2300), (5, 5), (257, 3)]])                 # the launches
def test_bounded(shapes, scale, mu, nesterov):
    import swingnn_amd as S
    params = [torch.nn.Parameter(0.02 * _gauss(s, i)) for i, s in enumerate(shapes)]
    opt = S.FusedMuonEMA(params, lr=1e-2, momentum=mu, nesterov=nesterov, ema_betas=(0.9,))
    for seed in range(4):
        _cancelling(opt, params, mu, nesterov, scale, seed)
        _step_and_check(opt, params, 1e-2)
    assert bool(opt.ema.isfinite().all())


def test_cancels_after_the_clip():
    """The clip factor belongs to the update: gradients that cancel once they are clipped."""
    import swingnn_amd as S
    mu = 0.5
    params = [torch.nn.Parameter(0.02 * _gauss(s, i)) for i, s in enumerate([(3, 7), (1, 500), (200, 150)])]
    opt = S.FusedMuonEMA(params, lr=1e-2, momentum=mu, max_norm=2.0)
    for seed in range(4):
        _cancelling(opt, params, mu, True, 1.0, seed)
        norm = sum(float(p.grad.double().square().sum()) for p in params) ** 0.5
        clip = 2.0 / (norm + 1e-6)
        opt.m.mul_(clip)
        _step_and_check(opt, params, 1e-2)


def test_exact_zero_and_ordinary_updates():
    """m = g = 0 moves nothing; an update that does not cancel is what orthogonalise() makes of it, to the bit."""
    import swingnn_amd as S
    p = torch.nn.Parameter(0.02 * _gauss((200, 150), 1))
    opt = S.FusedMuonEMA([p], lr=1.0, momentum=0.5, nesterov=False)
    p.grad = torch.zeros_like(p)
    before = p.detach().clone()
    opt.step()
    assert torch.equal(p, before)
    p.data.zero_()
    p.grad = _gauss((200, 150), 2)
    opt.step()
    o = S.orthogonalise(0.5 * p.grad, out_dtype=torch.float16).double()
    f = 0.2 * 200 ** 0.5
    # the fp16 result is off by half a step of values up to 1.21 (2^-11), its norm by fp64 rounding alone
    assert float((p.detach().double() + f * o).abs().max()) <= f * (1.21 * 2.0 ** -11 + 2.0 ** -22)
