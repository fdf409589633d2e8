"""MI355X-native GEMM engine behind the portBLAS `_gemm` interface.

`from sycl_blas_amd import SB_Handle, _gemm, _gemm_batched, _gemm_strided_batched`
gives the reference's call signatures over hand-written gfx950 HIP kernels
(loaded from sycl_blas_amd/lib/libsbamd.so through the C ABI of
include/sbamd_gemm.h).  The feed-forward layers on top of it (`_quantize`, `_gemm_scaled`,
`_gated_gemm`, `_gated_gemm_scaled`, `_gated_gemm_grad`) are those of include/sbamd_ffn.h.
"""
from . import _lib
from .interface import (DeviceBuffer, Event, SB_Handle, SbamdError, _gated_gemm, _gated_gemm_grad,
                        _gated_gemm_scaled, _gemm, _gemm_batched, _gemm_scaled, _gemm_strided_batched, _quantize,
                        _symm, _trsm, activation_t, gemm_batch_type_t, helper, uniform_reference)

__all__ = [
    "DeviceBuffer", "Event", "SB_Handle", "SbamdError", "_gated_gemm", "_gated_gemm_grad", "_gated_gemm_scaled",
    "_gemm", "_gemm_batched", "_gemm_scaled", "_gemm_strided_batched", "_quantize", "_symm", "_trsm",
    "activation_t", "gemm_batch_type_t", "helper", "uniform_reference", "_lib",
]
