"""inferflux_amd: MI355X (gfx950) quantized GEMV/GEMM path for InferFlux.

The kernels and the C ABI live in libifx_qgemm.so (include/ifx_qgemm.h);
`ops` wraps them for torch device tensors, `attention` (include/ifx_attention.h)
the paged cache and the attention between the projections, `fused_quant_gemm` mirrors the
reference's FusedQuantGemm host interface.
"""
from . import attention, ops  # noqa: F401
