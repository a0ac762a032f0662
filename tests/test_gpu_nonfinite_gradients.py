"""A gradient with a NaN or an infinity and the clip of both optimizers, as clip_grad_norm_ has it: the coefficient
max_norm / (norm + 1e-6) goes to EVERY gradient, a NaN one too."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _params():
    g = torch.Generator(device=DEV).manual_seed(1)
    # 16-byte aligned and odd sizes: both forms of the Adam kernel
    return [torch.nn.Parameter(torch.randn(*s, device=DEV, generator=g)) for s in [(40, 64), (33, 7), (64,), (7,), (300, 200)]]


def _grads(params, bad, where):
    g = torch.Generator(device=DEV).manual_seed(2)
    for i, p in enumerate(params):
        p.grad = torch.randn(*p.shape, device=DEV, generator=g)
        if i == where:
            p.grad.view(-1)[3] = bad


@pytest.mark.parametrize("where", [0, 2, 3])
def test_nan_reaches_every_parameter(where):
    import swingnn_amd as S
    for make in (lambda p: S.FusedMuonEMA([p[0], p[1], p[4]], p[2:4], lr=1e-3, max_norm=1.0),
                 lambda p: S.FusedAdamEMA(p, lr=1e-3, max_norm=1.0)):
        params = _params()
        opt = make(params)
        _grads(params, float("nan"), where)
        opt.step()
        assert bool(opt.grad_norm().isnan())
        for p in params:
            assert bool(p.isnan().all()), tuple(p.shape)


def test_infinite_norm_as_clip_grad_norm_has_it():
    """coef = max_norm / inf = 0: the infinity itself becomes NaN, every other gradient 0."""
    import swingnn_amd as S
    params, plain = _params(), _params()
    opt, ref = S.FusedAdamEMA(params, lr=1e-3, max_norm=1.0), torch.optim.Adam(plain, lr=1e-3)
    for ps in (params, plain):
        _grads(ps, float("inf"), 2)
    opt.step()
    torch.nn.utils.clip_grad_norm_(plain, 1.0)
    ref.step()
    for p, q in zip(params, plain):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.nan_to_num(), q.nan_to_num())


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_finite_gradients_as_before(max_norm):
    """The comparison form of the clip gives what min() gave: torch's clip and Adam within their roundings."""
    import swingnn_amd as S
    params, plain = _params(), _params()
    opt, ref = S.FusedAdamEMA(params, lr=1e-3, max_norm=max_norm), torch.optim.Adam(plain, lr=1e-3)
    for ps in (params, plain):
        _grads(ps, 1.0, 0)
    opt.step()
    torch.nn.utils.clip_grad_norm_(plain, max_norm)
    ref.step()
    for p, q in zip(params, plain):
        # first step: lr g / (|g| + eps), a quotient of values that are off by 2^-20 at most (the norm's sum and the clip)
        assert float((p - q).detach().abs().max()) <= 1e-3 * 2.0 ** -18 + 2.0 ** -22 * 5
