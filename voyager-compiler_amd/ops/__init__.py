"""``torch.ops.quantized_ops`` on MI355X kernels (see ``quantized.py``, ``kv4.py``)."""

from .quantized import (  # noqa: F401
    calculate_mx_qparam,
    dequantize,
    linear_mx,
    matmul_mx,
    mx_fake_quantize,
    quantize,
    quantize_mx,
    quantized_ops_lib,
    register_table,
    vmap,
)
from .kv4 import kv4_accumulate, kv4_append, kv4_attention, kv4_evict, kv4_read  # noqa: F401
