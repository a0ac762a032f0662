"""Refusals of the training operators: argument checks come before any GPU call, so they run on the CPU."""
import pytest
import torch


@pytest.fixture(autouse=True)
def _grad_mode():
    """Other modules of the suite switch gradients off for the process."""
    with torch.enable_grad():
        yield


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


def test_orthogonalise_refusals(S):
    g = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.orthogonalise(g)
    with pytest.raises(ValueError):
        S.orthogonalise(torch.zeros(8))
    with pytest.raises(ValueError):
        S.orthogonalise(torch.zeros(1, 2, 3, 4))
    with pytest.raises(NotImplementedError):
        S.orthogonalise(g.double())
    with pytest.raises(NotImplementedError):
        S.orthogonalise(g, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        S.orthogonalise(g, steps=0)
    with pytest.raises(ValueError):
        S.orthogonalise(g, eps=-1.0)
    with pytest.raises((ValueError, RuntimeError)):
        S.orthogonalise([g, g.half()])
    with pytest.raises(NotImplementedError, match="no gradient"):
        S.orthogonalise(g.clone().requires_grad_(True))
    assert S.orthogonalise([]) == []


def test_orthogonalise_entry_points_refuse(S):
    from swingnn_amd import _lib as L
    f, w = L.lib.swg_orthogonalise, L.lib.swg_orthogonalise_workspace_bytes
    p = 4096

    def items(rows=8, cols=8, batch=1, g=p, out=p, ld=8, ldo=8):
        return (L.SwgOrthItem * 1)(L.SwgOrthItem(g, out, ld, 64, ldo, 64, rows, cols, batch))

    big = 1 << 30
    assert f(1, items(), 0, 1, 0, 1e-7, p, big, None) == -1
    assert f(1, items(), 0, 1, 65, 1e-7, p, big, None) == -1
    assert f(1, items(), 0, 1, 5, -1.0, p, big, None) == -1
    assert f(1, items(), 0, 1, 5, float("nan"), p, big, None) == -1
    assert f(-1, items(), 0, 1, 5, 1e-7, p, big, None) == -1
    assert f(1, None, 0, 1, 5, 1e-7, p, big, None) == -4
    assert f(1, items(), 3, 1, 5, 1e-7, p, big, None) == -2
    assert f(1, items(), 0, 0, 5, 1e-7, p, big, None) == -2
    assert f(1, items(rows=-1), 0, 1, 5, 1e-7, p, big, None) == -1
    assert f(1, items(rows=(1 << 20) + 1), 0, 1, 5, 1e-7, p, big, None) == -1
    assert f(1, items(ld=7), 0, 1, 5, 1e-7, p, big, None) == -1
    assert f(1, items(ldo=7), 0, 1, 5, 1e-7, p, big, None) == -1
    assert f(1, items(g=None), 0, 1, 5, 1e-7, p, big, None) == -4
    assert f(1, items(), 0, 1, 5, 1e-7, None, big, None) == -4
    assert f(1, items(), 0, 1, 5, 1e-7, p, 64, None) == -3
    assert f(1, items(rows=0), 0, 1, 5, 1e-7, None, 0, None) == 0
    assert f(0, None, 0, 1, 5, 1e-7, None, 0, None) == 0
    assert w(0, items()) == 0 and w(1, None) == 0 and w(1, items(rows=-1)) == 0
    # 6 bytes an element of X and 4 an element of A and B, padded to 32, beside the tables
    assert w(1, items(rows=384, cols=1536)) <= 6 * 384 * 1536 + 4 * 384 * 384 + 8 * 384 + 8192
    # sizes past 2^31 bytes keep all their terms
    assert w(1, items(rows=40000, cols=50000)) >= 6 * 40000 * 50000 + 4 * 40000 * 40000


def test_muon_refusals(S):
    from swingnn_amd import _lib as L
    P = lambda *s: torch.nn.Parameter(torch.zeros(*s))
    a, b = P(4, 8), P(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        S.FusedMuonEMA([a], [b])
    with pytest.raises(ValueError):
        S.FusedMuonEMA([], [b])
    with pytest.raises(ValueError):
        S.FusedMuonEMA([b])
    with pytest.raises(ValueError):
        S.FusedMuonEMA([a, a])
    with pytest.raises(ValueError):
        S.FusedMuonEMA([a], [a])
    with pytest.raises(ValueError):
        S.FusedMuonEMA([a], [b], ns_steps=0)
    with pytest.raises(ValueError):
        S.FusedMuonEMA([a], [b], momentum=1.0)
    lin = torch.nn.Linear(3, 3)
    tied = torch.nn.ModuleList([lin, lin, torch.nn.LayerNorm(3), torch.nn.Conv2d(1, 2, 3), torch.nn.Embedding(4, 3)])
    mats, others = S.FusedMuonEMA.split(tied)
    assert len(mats) == 1 and mats[0] is lin.weight and len(others) == 6
    items = (L.SwgMuonItem * 1)(L.SwgMuonItem(0, 8, 8, 0, 1.0))
    p, st = 4096, L.lib.swg_muon_ema_step
    ok = [1, items, p, p, p, p, p, 64, 0, None, p, p, p, 1, p, 0.0, 1e-3, 0.9, 1, 0.0, 5, 1e-7, p, 1 << 20, None]
    for at, bad, code in ((0, 0, -1), (7, 0, -1), (8, 9, -1), (13, -1, -1), (20, 0, -1), (20, 65, -1), (21, -1.0, -1), (1, None, -4), (2, None, -4),
                          (3, None, -4), (4, None, -4), (5, None, -4), (10, None, -4), (11, None, -4), (12, None, -4), (22, None, -4),
                          (23, 64, -3), (8, 1, -4), (22, p + 16, -3), (2, p + 8, -3)):
        args = list(ok)
        args[at] = bad
        assert st(*args) == code, at
    assert L.lib.swg_muon_table(0, items, p, 1 << 20, None) == -1
    assert L.lib.swg_muon_table(1, items, p, 8, None) == -3
    assert L.lib.swg_muon_table(1, items, None, 1 << 20, None) == -4
    zero = (L.SwgMuonItem * 1)(L.SwgMuonItem(0, 0, 8, 0, 1.0))
    assert L.lib.swg_muon_table(1, zero, p, 1 << 20, None) == -1
