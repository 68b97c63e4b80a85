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


def test_widths_beyond_32_bits_are_refused():
    """They would be cut to their low bits on the way into the library.  Tensors without storage: nothing is computed."""
    from featgraph.module import RowGroups, combine_rows, grouped_matmul
    from featgraph_b200 import _native
    groups = RowGroups(*(torch.zeros(s, dtype=torch.int32) for s in ((3,), (4,), (2, 2))))
    empty = lambda *shape: torch.empty(shape, device="meta", dtype=torch.float16)  # noqa: E731
    for wide in (2 ** 31 - 1023, 2 ** 31 + 8, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="weight has shape"):
            grouped_matmul(empty(4, wide), empty(2, 8, wide), groups)
        with pytest.raises(ValueError, match="weight has shape"):
            grouped_matmul(empty(4, 8), empty(2, wide, 8), groups)
        with pytest.raises(ValueError, match="row for each"):
            combine_rows(empty(4, wide), groups)
    L, wide = _native.lib(), 2 ** 31 - 1023
    assert L.fg_combine_rows(16, 0, None, 16, 16, 4, 2, wide, 1, None) == 1 and b"bad sizes" in L.fg_last_error()
    for inner, outer in ((wide, 8), (8, wide)):
        assert L.fg_grouped_matmul(16, 0, None, 16, 40, 8, 1, None, 16, None, 1, 4, 16, 4, 2, inner, outer, 1, 1, None, 0, None) == 1
        assert b"bad sizes" in L.fg_last_error()
