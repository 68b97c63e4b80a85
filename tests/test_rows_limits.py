"""Checks of the row operators (``featgraph_b200.module.rows``) and of their C entry points that happen on the host."""
import pytest
import torch


@pytest.mark.skipif(torch.cuda.is_available(), reason="CUDA present")
def test_waits_are_a_device_s():
    from featgraph.module import check_waits
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        check_waits()


def test_waits_are_not_those_of_a_cpu():
    from featgraph.module import check_waits
    with pytest.raises(RuntimeError, match="CUDA"):
        check_waits("cpu")


def test_workspaces_off_the_16_byte_grid_are_refused():
    """The kernels store 16 bytes at a time there.  The addresses are never used: the check comes before any CUDA call."""
    from featgraph_b200 import _native
    L = _native.lib()
    here = 1 << 20

    def refused(name, *args):
        assert getattr(L, name)(*args) == 1
        assert b"16-byte boundary" in L.fg_last_error(), L.fg_last_error()

    for off in (4, 8, 12):
        refused("fg_grouped_matmul", here, 0, None, here, 40, 8, 1, None, here, None, 1, 200, here, 200, 2, 8, 200, 0, 0, here + off, 1 << 30, None)
        refused("fg_grouped_matmul_backward", here, 0, here, 40, 8, 1, here, None, None, 1, 200, here, 0, here, here, 200, 2, 8, 5, 0, here + off, 1 << 30, None)
        refused("fg_group_rows", here, 1 << 20, 8, here, here, here, here + off, 1 << 30, None)
        refused("fg_route", here, 0, here, here, here, here, here, 1 << 20, 8, 2, 0, 0, 0, here + off, 1 << 30, None)
