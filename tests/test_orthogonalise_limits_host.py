"""A launch holds fewer than 2^32 threads: calls that would need more are refused before any GPU call."""
import pytest


@pytest.fixture(scope="module")
def L():
    from swingnn_amd import _lib
    return _lib


def _call(L, *items):
    arr = (L.SwgOrthItem * len(items))(*(L.SwgOrthItem(4096, 4096, c, r * c, c, r * c, r, c, b) for r, c, b in items))
    nbytes = L.lib.swg_orthogonalise_workspace_bytes(len(items), arr)
    # a workspace that is too small: an accepted call ends at that check, before it touches the GPU
    return nbytes, L.lib.swg_orthogonalise(len(items), arr, 0, 1, 5, 1e-7, 4096, 8, None)


@pytest.mark.parametrize("batch,ok", [(8_000_000, True), (8_388_608, False), (2 ** 31 - 1, False)])
def test_batches_of_small_matrices(L, batch, ok):
    nbytes, code = _call(L, (2, 2, batch))   # one workgroup of 512 threads a matrix
    assert (nbytes > 0) == ok and code == (-3 if ok else -1)


@pytest.mark.parametrize("batch,ok", [(16_000_000, True), (16_777_216, False)])
def test_small_ones_beside_a_larger_one(L, batch, ok):
    nbytes, code = _call(L, (200, 200, 1), (2, 2, batch))   # launches of 256 threads a tile
    assert (nbytes > 0) == ok and code == (-3 if ok else -1)


def test_the_sum_over_a_list_counts(L):
    nbytes, code = _call(L, (2, 2, 5_000_000), (3, 3, 5_000_000))
    assert nbytes == 0 and code == -1


def test_optimizer_step(L):
    n = 1 << 10
    big = (L.SwgMuonItem * n)(*(L.SwgMuonItem(0, 1 << 20, 1 << 14, 0, 1.0) for _ in range(n)))
    assert L.lib.swg_muon_workspace_bytes(n, big) == 0
    few = (L.SwgMuonItem * 8)(*(L.SwgMuonItem(0, 4096, 4096, 0, 1.0) for _ in range(8)))
    assert L.lib.swg_muon_workspace_bytes(8, few) > 0
