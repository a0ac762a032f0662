"""Refusals of the training operators: argument checks come before any GPU call, so they run on the CPU."""
import pytest
import torch


@pytest.fixture(scope="module")
def S():
    import swingnn_amd
    return swingnn_amd


def test_layer_norm_refusals(S):
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.layer_norm(x, w, w)
    with pytest.raises(ValueError):
        S.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        S.layer_norm(x, w, torch.ones(4, 8))
    with pytest.raises(ValueError):
        S.layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        S.layer_norm(torch.zeros(()))
    with pytest.raises(NotImplementedError):
        S.layer_norm(x.double(), w)
    with pytest.raises(NotImplementedError):
        S.layer_norm(x, w.bfloat16())
    with pytest.raises(NotImplementedError):
        S.layer_norm(x.bfloat16(), w, w.bfloat16())
    with pytest.raises(NotImplementedError):
        S.LayerNorm((4, 8))
    with pytest.raises(ValueError):
        S.LayerNorm(8)(torch.zeros(2, 9))
    with pytest.raises(NotImplementedError):
        S.SwinGNN(img_size=24, patch_size=3, in_chans=1, embed_dim=60, depths=[1], drop_path_rate=0., norm_layer=torch.nn.Identity)


def test_layer_norm_entry_points_refuse(S):
    """C entries: no GPU call is reached (pointers are not read on the host)."""
    from swingnn_amd import _lib as L
    f, b, w = L.lib.swg_layer_norm_fwd, L.lib.swg_layer_norm_bwd, L.lib.swg_layer_norm_bwd_workspace_bytes
    p = 4096  # any non-null address
    assert f(4, 0, p, 8, 0, p, p, 0, 1e-5, p, 8, None, None, None) == -1
    assert f(-1, 8, p, 8, 0, p, p, 0, 1e-5, p, 8, None, None, None) == -1
    assert f(1 << 31, 8, p, 8, 0, p, p, 0, 1e-5, p, 8, None, None, None) == -1
    assert f(4, 8, p, 8, 3, p, p, 0, 1e-5, p, 8, None, None, None) == -2
    assert f(4, 8, p, 8, 0, p, p, 1, 1e-5, p, 8, None, None, None) == -2
    assert f(4, 8, p, 8, 1, p, p, 2, 1e-5, p, 8, None, None, None) == -2
    assert f(4, 8, None, 8, 0, p, p, 0, 1e-5, p, 8, None, None, None) == -4
    assert f(4, 8, p, 8, 0, p, p, 0, 1e-5, p, 8, p, None, None) == -4
    assert f(4, 8, p, 8, 0, p, p, 0, 1e-5, p, 7, None, None, None) == -1
    assert f(0, 8, None, 8, 0, None, None, 0, 1e-5, None, 8, None, None, None) == 0
    assert b(4, 8, p, 8, p, 8, 0, p, 0, None, p, p, 8, p, p, p, 1 << 20, None) == -4
    assert b(4, 8, p, 8, p, 8, 0, p, 0, p, p, p, 8, p, p, None, 0, None) == -4
    assert b(4, 8, p, 8, p, 8, 0, p, 0, p, p, p, 8, p, p, p, 16, None) == -3
    assert b(4, 8, p, -1, p, 8, 0, p, 0, p, p, p, 8, p, p, p, 1 << 20, None) == -1
    assert w(4, 0, 0) == 0 and w(4, 8, 5) == 0
    # one partial row of 2 D sums per workgroup, at most 1024 of them
    assert w(10 ** 6, 96, 0) <= 1025 * 2 * 96 * 4 + 256
