"""ghostflow_hip -- Python bindings of the gfx950 backend for GhostFlow's dense
hot path (fp32 GEMM / Linear, int8 quantized linear, decode GEMV, SDPA), the
layers built on it (MultiHeadAttention with a KV cache, SwiGLU), and a decode
step of many sequences (caches in pages, 4-bit weights, sampling).

All compute goes through the C ABI of libghostflow_hip.so
(include/ghostflow_hip.h); see ops.py.  The package lives in the
`ghost-flow_amd/` directory; put that directory on sys.path to import it.
"""
from . import _lib  # noqa: F401
from .ops import (  # noqa: F401
    GhostFlowError,
    StateDict,
    dequantize,
    dequantize_grouped_i4,
    flash_attention_blockwise,
    gemv_f32,
    gemv_w8,
    init,
    kv_attention,
    lib,
    linear,
    linear_w4,
    linear_w4_workspace_size,
    load_state_dict,
    matmul,
    matmul_backward,
    mha_forward_cached,
    mha_forward_with_cache,
    mha_workspace_size,
    paged_append,
    paged_attention,
    paged_attention_workspace_size,
    paged_read,
    qlinear,
    qlinear_dynamic,
    qswiglu,
    quantize_grouped_i4,
    quantize_per_channel,
    quantize_per_tensor,
    quantize_per_tensor_workspace_size,
    qweight_rowsum,
    sample,
    sample_workspace_size,
    save_state_dict,
    sdpa,
    set_pointer_checks,
    silu_mul,
    sgemm,
    softmax_lastdim,
    swiglu,
)
from .nn import (  # noqa: F401
    FlashAttention,
    FlashAttentionConfig,
    GroupQuantizedSwiGLU,
    KVCache,
    MultiHeadAttention,
    PagedBatch,
    PagedKVCache,
    QuantizedSwiGLU,
    SwiGLU,
)
from .quantization import (  # noqa: F401
    DynamicQuantization,
    GroupQuantizedLinear,
    QuantizationAwareTraining,
    QuantizationConfig,
    QuantizationScheme,
    QuantizedTensor,
)
from .synth import normal, uniform  # noqa: F401
