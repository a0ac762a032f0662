"""Forward-mode tangents and traces do not see work that is queued through raw pointers: the training operators refuse
them instead of dropping the tangent or recording uninitialised memory.  The checks come before any GPU call."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(autouse=True)
def _grad_mode():
    """Other modules of the suite switch gradients off for the process."""
    with torch.enable_grad():
        yield


@pytest.fixture(scope="module")
def S():
    import swingnn_amd
    return swingnn_amd


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_layer_norm_refuses_tangents(S, which):
    t = {"x": torch.randn(4, 8), "weight": torch.ones(8), "bias": torch.zeros(8)}
    with fwd.dual_level():
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward"):
            S.layer_norm(**t)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            S.layer_norm(**t)


def test_module_refuses_tangents(S):
    with fwd.dual_level():
        x = fwd.make_dual(torch.randn(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward"):
            S.LayerNorm(8)(x)


def test_tensors_without_a_tangent_pass_inside_a_level(S):
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            S.layer_norm(torch.randn(4, 8))
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            S.orthogonalise(torch.randn(4, 8))


def test_orthogonalise_refuses_tangents(S):
    with fwd.dual_level():
        g = fwd.make_dual(torch.randn(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="forward"):
            S.orthogonalise([torch.zeros(2, 2), g])


CALLS = {"layer_norm": lambda S: lambda x: S.layer_norm(x), "LayerNorm": lambda S: S.LayerNorm(8),
         "orthogonalise": lambda S: lambda x: S.orthogonalise(x), "list": lambda S: lambda x: S.orthogonalise([x])[0]}


@pytest.mark.parametrize("call", list(CALLS))
def test_jit_trace_is_refused(S, call):
    with torch.no_grad(), pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(CALLS[call](S), torch.randn(4, 8))


@pytest.mark.parametrize("kw", [{}, {"tracing_mode": "fake"}, {"tracing_mode": "symbolic"}, {"pre_dispatch": True}])
@pytest.mark.parametrize("call", list(CALLS))
def test_make_fx_is_refused(S, call, kw):
    with torch.no_grad(), pytest.raises(NotImplementedError, match="trace"):
        make_fx(CALLS[call](S), **kw)(torch.randn(4, 8))
