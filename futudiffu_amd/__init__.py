"""MI355X-native (gfx950) SageAttention forward and backward for sqcu/futudiffu.

Importing this package registers the ``futudiffu_ii::sage_attn_masked``,
``futudiffu_ii::sage_attn``, ``futudiffu_ii::sage_attn_ext``,
``futudiffu_ii::sage_attn_masked_merged_heads`` and
``futudiffu_ii::sage_attn_qkv_masked`` custom ops, and the backward ops
``futudiffu_ii::sage_bwd_masked``, ``futudiffu_ii::sage_bwd`` and
``futudiffu_ii::sage_bwd_ext`` their autograd formulas call.  ``futudiffu_amd.fused_kernels``
(imported separately) registers ``futudiffu::fused_qkv_postprocess``.  ``block_ops`` holds
what surrounds the attention in a transformer block: RMS norms with modulation, gate and
residual, and linear layers with bias, activation and residual; ``mxfp4`` the linear layers over
weights in 4-bit floating point, and the norms that feed them.
The compute lives in ``libsage_mi355x.so`` (HIP, built by ``build.py``).
"""

from . import attention_srcii  # noqa: F401  (registers the custom ops)
from .attention_srcii import (  # noqa: F401
    sage_attn_ext_op,
    sage_attn_masked_merged_heads_op,
    sage_attn_masked_op,
    sage_attn_qkv_masked_op,
    sage_attn_op,
    sage_bwd_ext_op,
    sage_bwd_masked_op,
    sage_bwd_op,
)
from .block_ops import (  # noqa: F401  (registers the ops around the attention)
    fused_linear,
    rms_norm_gate_residual,
    rms_norm_gate_residual_modulate,
    rms_norm_modulate,
)
from .mxfp4 import (  # noqa: F401  (registers the ops in 4-bit floating point)
    MXFP4,
    mxfp4_dequantize,
    mxfp4_linear,
    mxfp4_quantize,
    rms_norm_gate_residual_modulate_mxfp4,
    rms_norm_modulate_mxfp4,
)
from .block_mask import build_block_mask, build_doc_ids  # noqa: F401
from .sage_attention import (  # noqa: F401
    configure_sage,
    sage_attn_backward,
    sage_attn_backward_masked,
    sage_backward,
    qkv_postprocess,
    quantize_from_qkv,
    quantize_qkv,
    sage_attn_forward,
    sage_attn_forward_masked,
    sage_attn_forward_masked_merged_heads,
    sage_attn_forward_masked_with_lse,
    sage_attn_forward_with_lse,
    sage_forward,
    sage_forward_from_qkv,
)
