"""Inputs whose sign is a flag of the tensor (the imaginary part of a conjugate view): what they stand for counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


def _flagged(*shape):
    t = torch.randn(*shape, dtype=torch.cfloat, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).conj().imag
    assert t.is_neg()
    return t


@pytest.mark.parametrize("shape", [(50, 1), (1, 50), (1, 1), (40, 60), (3, 7, 1)])
def test_orthogonalise(shape):
    import swingnn_amd as S
    g = _flagged(*shape)
    assert torch.equal(S.orthogonalise(g), S.orthogonalise(g.resolve_neg().clone()))


@pytest.mark.parametrize("D", [1, 2, 33])
def test_layer_norm(D):
    import swingnn_amd as S
    got = []
    for plain in (False, True):
        x, w, b, dy = _flagged(9, D), _flagged(D), _flagged(D), _flagged(9, D)
        if plain:
            x, w, b, dy = (t.resolve_neg().clone() for t in (x, w, b, dy))
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = S.layer_norm(x, w, b)
        got.append([y] + list(torch.autograd.grad(y, leaves, dy)))
    for p, q in zip(*got):
        assert torch.equal(p, q)
