from .sddmm import SDDMMbase, VanillaSDDMMx86, VanillaSDDMMcuda
from .spmm import SpMMbase, VanillaSpMMx86, VanillaSpMMcuda

# the names the hot path is usually referred to by
VanillaSpMM = VanillaSpMMcuda
VanillaSDDMM = VanillaSDDMMcuda

# SpMM followed by SDDMM on its output, in one pass (no counterpart class in the reference: it runs the two
# modules above back to back)
from .fused import AggregateThenScore

# what a layer with several experts, node types or relations computes densely around them (module/rows.py)
from .rows import (QuantizedRows, Routing, RowGroups, check_waits, combine_rows, group_rows, grouped_matmul, quantize_rows,
                   rms_norm, route)
