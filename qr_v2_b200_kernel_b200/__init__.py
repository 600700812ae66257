"""qr_v2_b200_kernel_b200 -- batched Householder QR on B200 (sm_100a).

Public API (the reference's drop-in operator, ``submission.py:560-596``)::

    from qr_v2_b200_kernel_b200 import custom_kernel
    H, tau = custom_kernel(A)          # A: (batch, n, n) float32 CUDA tensor
    H, tau = custom_kernel_host(A)     # A on the host: copies overlapped with the factorisation
    Q = householder_product(H, tau)    # explicit Q (sorgqr), on the tensor cores
    X = ormqr(H, tau, B, transpose=True)   # Q^T B (sormqr)

Operators on data in 8 and 4 bits, which an orthogonal ``Q`` makes fit for them (``quant``):
``rms_norm_int8``, ``quantize_int8``, ``dequantize_int8``, ``int8_linear``, ``kv4_cache``,
``kv4_write``, ``kv4_read``, ``kv4_attention``, and their 8-bit kin ``kv8_cache``, ``kv8_write``,
``kv8_read``, ``kv8_attention``; in 8-bit floating point ``quantize_fp8``, ``dequantize_fp8``, ``fp8_linear``.

Helpers: ``gen`` (seeded inputs), ``checker`` (the FP64 correctness gate),
``sharding`` (host-side batch split over several GPUs).
"""

from .api import custom_kernel, custom_kernel_host, geqrf, householder_product, ormqr, workspace_bytes  # noqa: F401
from .quant import (KV4Cache, KV8Cache, dequantize_fp8, dequantize_int8, fp8_linear, int8_linear,  # noqa: F401
                    kv4_attention, kv4_cache, kv4_read, kv4_write, kv8_attention, kv8_cache, kv8_read, kv8_write,
                    quantize_fp8, quantize_int8, rms_norm_int8)

__version__ = "0.1.0"
