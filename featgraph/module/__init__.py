from featgraph_b200.module import (SDDMMbase, SpMMbase, VanillaSDDMM, VanillaSDDMMcuda,  # noqa: F401
                                   VanillaSDDMMx86, VanillaSpMM, VanillaSpMMcuda, VanillaSpMMx86)
from featgraph_b200.module import (QuantizedRows, Routing, RowGroups, check_waits, combine_rows, group_rows,  # noqa: F401
                                   grouped_matmul, quantize_rows, rms_norm, route)
