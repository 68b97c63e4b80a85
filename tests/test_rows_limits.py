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
