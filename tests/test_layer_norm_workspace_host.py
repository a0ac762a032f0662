"""The workspace of the layer norm's backward pass: one row of 2 D partial sums for each workgroup, 512 of them at most (64
slabs of rows where a row is wider than the register forms), and one row more."""
import pytest


def _bytes(rows, D, elem):
    from swingnn_amd import _lib as L
    return L.lib.swg_layer_norm_bwd_workspace_bytes(rows, D, {4: L.SWG_F32, 2: L.SWG_BF16}[elem])


def _align(n):
    return (n + 255) // 256 * 256


@pytest.mark.parametrize("rows,D,elem,workgroups", [(10 ** 6, 96, 4, 512), (2 ** 31 - 1, 8, 4, 512), (10 ** 6, 4096, 2, 512), (100, 4096, 2, 100),
                                                    (33, 96, 4, 2), (1, 96, 4, 1), (0, 96, 4, 0), (10 ** 6, 16385, 4, 64),
                                                    (10 ** 6, 16392, 2, 64), (10, 40000, 4, 10)])
def test_rows_of_partial_sums(rows, D, elem, workgroups):
    assert _bytes(rows, D, elem) == _align((workgroups + 1) * 2 * D * 4)
