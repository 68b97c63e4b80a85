"""Argument checks of the row operators (``featgraph_b200.module.rows``) and of their C entry points: all of them happen
on the host before any CUDA call, so they run without a device."""
import pytest
import torch

from featgraph.module import (QuantizedRows, RowGroups, combine_rows, group_rows, grouped_matmul, quantize_rows,
                              rms_norm, route)


def _groups(n=3, k=2, g=4):
    return RowGroups(torch.zeros(g + 1, dtype=torch.int32), torch.zeros(n * k, dtype=torch.int32), torch.zeros(n, k, dtype=torch.int32))


X = torch.zeros(3, 8)
BAD = [
    (TypeError, "torch.Tensor", lambda: rms_norm([1.0])),
    (TypeError, "float32 or float16 or bfloat16", lambda: rms_norm(X.double())),
    (ValueError, "rows of 1 to 16384", lambda: rms_norm(torch.zeros(3, 0))),
    (ValueError, "rows of 1 to 16384", lambda: rms_norm(torch.zeros(1, 16385))),
    (ValueError, "rows of 1 to 16384", lambda: rms_norm(torch.tensor(1.0))),
    (ValueError, "weight has 7", lambda: rms_norm(X, torch.ones(7))),
    (TypeError, "weight must be", lambda: rms_norm(X, torch.ones(8).half())),
    (ValueError, "residual has shape", lambda: rms_norm(X, residual=torch.zeros(4, 8))),
    (TypeError, "residual must be", lambda: rms_norm(X, residual=X.half())),
    (ValueError, "eps", lambda: rms_norm(X, eps=-1.0)),
    (ValueError, "eps", lambda: rms_norm(X, eps=float("nan"))),
    (TypeError, "float32 or float16", lambda: quantize_rows(X.int())),
    (TypeError, "int32 or int64", lambda: group_rows(X, 3)),
    (ValueError, "keys must be", lambda: group_rows(torch.zeros(2, 33, dtype=torch.int32), 3)),
    (ValueError, "keys must be", lambda: group_rows(torch.zeros(2, 2, 2, dtype=torch.int32), 3)),
    (ValueError, "num_groups", lambda: group_rows(torch.zeros(2, dtype=torch.int32), 0)),
    (ValueError, "num_groups", lambda: group_rows(torch.zeros(2, dtype=torch.int32), 1025)),
    (ValueError, "2 dimensions", lambda: route(torch.zeros(8), 1)),
    (ValueError, "k must be 1 to 8", lambda: route(X, 9)),
    (ValueError, "k must be 1 to 8", lambda: route(X, 0)),
    (ValueError, "k must be 1 to 32", lambda: route(torch.zeros(2, 64), 33)),
    (ValueError, "experts", lambda: route(torch.zeros(2, 1025), 1)),
    (ValueError, "scoring", lambda: route(X, 1, scoring="relu")),
    (TypeError, "RowGroups", lambda: grouped_matmul(X, torch.zeros(4, 5, 8), None)),
    (ValueError, "weight has 5 groups", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(5, 5, 8), _groups())),
    (ValueError, "weight takes 7", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 5, 7), _groups())),
    (ValueError, "x has 3 rows, the groups 6 slots", lambda: grouped_matmul(X, torch.zeros(4, 5, 8), _groups())),
    (ValueError, "x has 6 rows, the groups 3", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 5, 8), _groups(), gather=True)),
    (TypeError, "weight must be float32", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 5, 8).half(), _groups())),
    (TypeError, "out_dtype", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 5, 8), _groups(), out_dtype=torch.float16)),
    (ValueError, "weight has shape", lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 0, 8), _groups())),
    (TypeError, "both be QuantizedRows", lambda: grouped_matmul(QuantizedRows(X, X[:, 0]), torch.zeros(4, 5, 8), _groups())),
    (TypeError, "float8_e4m3fn", lambda: grouped_matmul(QuantizedRows(X, X[:, 0]), QuantizedRows(X, X[:, 0]), _groups())),
    (ValueError, "a scale for each row", lambda: grouped_matmul(
        QuantizedRows(torch.zeros(6, 8).to(torch.float8_e4m3fn), torch.ones(5)),
        QuantizedRows(torch.zeros(4, 5, 8).to(torch.float8_e4m3fn), torch.ones(4, 5)), _groups())),
    (ValueError, "row for each of 6 slots", lambda: combine_rows(X, _groups())),
    (ValueError, "weights have shape", lambda: combine_rows(torch.zeros(6, 8), _groups(), torch.zeros(2, 3))),
    (TypeError, "weights must be float32", lambda: combine_rows(torch.zeros(6, 8), _groups(), torch.zeros(3, 2).half())),
    (TypeError, "RowGroups", lambda: combine_rows(X, (1, 2, 3))),
    (ValueError, "int32", lambda: RowGroups(torch.zeros(3), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int32))),
    (ValueError, "offsets must have", lambda: RowGroups(*(torch.zeros(s, dtype=torch.int32) for s in ((1,), (2,), (2, 1))))),
    (ValueError, "same entries", lambda: RowGroups(*(torch.zeros(s, dtype=torch.int32) for s in ((3,), (3,), (2, 1))))),
]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_bad_arguments_are_refused(i):
    kind, text, call = BAD[i]
    with pytest.raises(kind, match=text):
        call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="CUDA present")
@pytest.mark.parametrize("call", [
    lambda: rms_norm(X), lambda: quantize_rows(X), lambda: group_rows(torch.zeros(2, dtype=torch.int32), 3), lambda: route(X, 2),
    lambda: grouped_matmul(torch.zeros(6, 8), torch.zeros(4, 5, 8), _groups()), lambda: combine_rows(torch.zeros(6, 8), _groups())])
def test_there_is_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()


def test_c_entries_report_bad_arguments():
    from featgraph_b200 import _native
    L = _native.lib()

    def refused(name, *args, text):
        assert getattr(L, name)(*args) == 1
        assert text in L.fg_last_error(), L.fg_last_error()

    refused("fg_rms_norm", 1, 0, None, 0, None, None, 1, None, 4, 0, 1e-6, 0, 0, 0, None, text=b"bad sizes")
    refused("fg_rms_norm", 1, 0, None, 0, None, None, 1, None, 4, 16385, 1e-6, 0, 0, 0, None, text=b"bad sizes")
    refused("fg_rms_norm", 1, 7, None, 0, None, None, 1, None, 4, 8, 1e-6, 0, 0, 0, None, text=b"row strides")
    refused("fg_rms_norm", 1, 0, None, 0, None, None, 1, None, 4, 8, 1e-6, 7, 7, 7, None, text=b"value type")
    refused("fg_rms_norm", 1, 0, None, 0, None, None, 1, None, 4, 8, 1e-6, 0, 0, 3, None, text=b"NULL")
    refused("fg_rms_norm", 1, 0, None, 0, None, None, 1, None, 4, 8, 1e-6, 0, 0, 1, None, text=b"rows' type")
    refused("fg_quantize_rows", None, 0, 1, 1, 4, 8, 0, None, text=b"NULL")
    refused("fg_rms_norm_backward", 1, 0, None, 1, 0, None, 0, 1, None, None, 0, 4, 8, 1e-6, 0, 0, None, text=b"blocks")
    refused("fg_route", 1, 0, 1, 1, None, None, None, 4, 8, 9, 0, 0, 0, None, 0, None, text=b"bad sizes")
    refused("fg_route", 1, 0, 1, 1, None, None, None, 4, 8, 2, 0, 5, 0, None, 0, None, text=b"scoring")
    refused("fg_route", 1, 0, 1, 1, 1, 1, 1, 1 << 20, 8, 2, 0, 0, 0, None, 0, None, text=b"workspace")
    refused("fg_route", 1, 0, 1, 1, 1, None, 1, 4, 8, 2, 0, 0, 0, None, 0, None, text=b"NULL")
    refused("fg_route_backward", 1, 0, 1, 1, None, 1, 4, 8, 2, 0, 0, 0, None, text=b"NULL")
    refused("fg_group_rows", 1, 4, 1025, 1, 1, 1, None, 0, None, text=b"bad sizes")
    refused("fg_group_rows", 1, 1 << 20, 8, 1, 1, 1, None, 0, None, text=b"workspace")
    refused("fg_grouped_matmul", 1, 0, None, 1, 40, 8, 1, None, 1, None, 0, 4, 1, 4, 2, 8, 5, 0, 0, None, 0, None, text=b"bad sizes")
    refused("fg_grouped_matmul", 1, 0, None, 1, 40, 8, 1, None, 1, None, 1, 4, 1, 4, 2, 8, 5, 3, 2, None, 0, None, text=b"NULL")
    refused("fg_grouped_matmul", 1, 0, None, 1, 40, 8, 1, None, 1, None, 1, 4, 1, 4, 2, 8, 5, 0, 2, None, 0, None, text=b"inputs' type")
    refused("fg_grouped_matmul_backward", 1, 0, 1, 40, 8, 1, 1, None, None, 1, 4, 1, 4, 1, 1, 4, 2, 8, 5, 0, None, 0, None, text=b"row strides")
    refused("fg_grouped_matmul_backward", 1, 0, 1, 40, 8, 1, 1, 1, None, 1, 4, 1, 0, 1, 1, 4, 2, 8, 5, 2, None, 0, None, text=b"NULL")
    refused("fg_grouped_matmul_backward", 1, 0, 1, 40, 8, 1, 1, 1, 1, 2, 4, 1, 0, 1, 1, 4, 2, 8, 5, 2, None, 0, None, text=b"choices")
    refused("fg_grouped_matmul_backward", 1, 0, 1, 40, 8, 1, 1, None, None, 1, 4, 1, 0, 1, 1, 4, 2, 8, 5, 0, None, 0, None, text=b"workspace")
    refused("fg_grouped_matmul_backward", 1, 0, 1, 40, 8, 1, 1, None, None, 1, 4, 1, 0, 1, 1, 4, 2, 8, 5, 3, None, 0, None, text=b"value type")
    refused("fg_combine_rows", 1, 0, None, 1, 1, 4, 33, 8, 0, None, text=b"bad sizes")
    refused("fg_combine_rows_backward", 1, 0, None, None, 1, 2, 1, 0, 1, None, 4, 2, 8, 0, None, text=b"NULL")
    # nothing to do is no error
    assert L.fg_rms_norm(None, 0, None, 0, None, None, None, None, 0, 8, 1e-6, 0, 0, 0, None) == 0
    assert L.fg_combine_rows(None, 0, None, None, None, 0, 2, 8, 0, None) == 0
