"""galactus_b200: the routed-expert FFN of a quantized MoE layer on B200 (sm_100a).

The product is the C-ABI library libgalactus_b200.so (include/galactus_b200.h);
this package is its Python binding plus the model shapes used by the tests and
the benchmark. Importing it loads the library and fails loudly if it is absent.
"""
from ._lib import (  # noqa: F401
    ACT_SWIGLU, ACT_SWIGLU_OAI, BLOCK_BYTES, BLOCK_ELEMS, GX_OK, GxError,
    GX_ERR_ALIGN, GX_ERR_BATCH, GX_ERR_COMM, GX_ERR_COPY, GX_ERR_CUDA, GX_ERR_DEVICE, GX_ERR_DOMAIN, GX_ERR_INVALID,
    GX_ERR_NOMEM, GX_ERR_SLOTS, GX_ERR_STATE, GX_ERR_TIMEOUT, GX_ERR_TYPE,
    POLICY_AUTO, POLICY_FREQUENCY, POLICY_LRU, POLICY_PLAN, POLICY_UNIFORM,
    TYPE_BF16, TYPE_F16, TYPE_F32, TYPE_IQ1_S, TYPE_MXFP4, TYPE_NAMES, TYPE_Q4_0, TYPE_Q4_1, TYPE_Q4_K, TYPE_Q6_K, TYPE_Q8_0, TYPE_Q8_K,
    check, declared_symbols, lib, row_bytes, vec_dot_type,
)
from .moe import Arena, LayerShape, SlotPolicy, mul_mat_id, record_layout  # noqa: F401
from .models import MODELS, ModelShape  # noqa: F401

__all__ = [
    "Arena", "LayerShape", "SlotPolicy", "mul_mat_id", "record_layout", "MODELS", "ModelShape", "lib", "check",
    "GxError", "group_rows", "lora_mul_mat", "mul_mat_grouped", "mul_mat_grouped_glu", "round_rows",
    "block_out", "mul_mat_q4", "mul_mat_q4_glu", "rms_norm",
]


# the operators on torch tensors: torch is imported with the first of them
_GROUPED = ("group_rows", "lora_mul_mat", "mul_mat_grouped", "mul_mat_grouped_glu", "round_rows")
_BLOCK = ("block_out", "mul_mat_q4", "mul_mat_q4_glu", "rms_norm")


def __getattr__(name):
    if name in _GROUPED:
        from . import grouped as module
        names = _GROUPED
    elif name in _BLOCK:
        from . import block as module
        names = _BLOCK
    else:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    for n in names:
        globals()[n] = getattr(module, n)
    return globals()[name]
