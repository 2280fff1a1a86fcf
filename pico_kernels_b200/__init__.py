"""B200 (sm_100a) quantized-matmul path: a drop-in for pico-kernels'
``gemm_int4``, ``gemm_fp8``, ``gemm_splitk``, ``gemm`` and ``quantize``
(round-to-nearest, and a GPTQ producer of packed int4 weights), and a W8A8
path beside it (``gemm_w8a8``, ``norm``: 8-bit weights and activations with a
scale per row).

The kernels live in ``libpico_b200.so`` (hand-written CUDA, C ABI in
``include/pico_b200.h``); these modules are thin PyTorch-facing wrappers.
"""

from . import (gemm, gemm_fp8, gemm_int4, gemm_splitk, gemm_w8a8, gptq, linear,  # noqa: F401
               norm, quantize)
from ._lib import (DtypeError, KernelError, ShapeError, device_status, load,  # noqa: F401
                   reset_workspaces, set_wait_limit)
from .gemm_fp8 import fp8_gemm, fp8_gemm_precast  # noqa: F401
from .gemm_splitk import triton_gemm, triton_gemm_splitk  # noqa: F401
from .gemm_int4 import (int4_gemm, int4_gemm_host, pack_int4_n, quantize_int4,  # noqa: F401
                        quantize_int4_grouped, unpack_int4_n)
from .gemm_w8a8 import (dequantize_rows, quantize_rows, w8a8_gated_gemm,  # noqa: F401
                        w8a8_gemm)
from .gptq import gptq_quantize_int4  # noqa: F401
from .linear import (W4A16Linear, W8A8GatedMLP, W8A8Linear,  # noqa: F401
                     quantize_linear_layers)
from .norm import rms_norm_quant  # noqa: F401

__version__ = "0.1.0"
