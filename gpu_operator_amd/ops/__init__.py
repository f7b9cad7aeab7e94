"""GPU compute ops of the validator workloads (hand-written HIP kernels for gfx950)."""

from .gemm import gemm_bf16, fill_uniform_, verify, tflops  # noqa: F401
from .smoke import vector_add  # noqa: F401
from .blockscale import gemm_fp8_block, gemm_grouped_fp8_block, quantize_fp8_block  # noqa: F401
from .grouped import gemm_grouped, gemm_grouped_dgrad, gemm_grouped_wgrad, grouped_linear  # noqa: F401
