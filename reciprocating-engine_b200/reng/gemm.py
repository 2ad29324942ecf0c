"""The packed tcgen05 GEMM on its own: y = x @ w.T in f32 from bf16 bit
patterns (the projection kernel of steps with more than 8 rows).

    y, ms = gemm_bf16(w_bits, x_bits, splits=0, iters=0)

w_bits: uint16 [rows][K] bf16 bits, x_bits: uint16 [M][K] (1 <= M <= 1024,
N-tiles of 256 rows beyond 256; K % 8 == 0).  iters > 0 also times the kernel alone (mean ms per launch).

And the block-scaled FP8 product on torch CUDA tensors:

    y = gemm_fp8_blocks(x, x_scales, w, w_scales)

with x from fp8.quantize_blocks(.., 1) / fp8.swiglu_quantize /
norm.block_norm_fp8 and w from fp8.quantize_blocks(.., 128).
gemm_fp8_blocks_status() tells whether all products so far came to their end.
"""
import ctypes as C

import numpy as np

from . import _lib

_impl = None  # ._tensors, bound on first use (it needs torch; an import statement costs 0.6 us a call)


def _tensors():
    global _impl
    if _impl is None:
        from . import _tensors as m
        _impl = m
    return _impl


def gemm_bf16(w_bits, x_bits, splits=0, iters=0):
    w = np.ascontiguousarray(w_bits, dtype=np.uint16)
    x = np.ascontiguousarray(x_bits, dtype=np.uint16)
    if w.ndim != 2 or x.ndim != 2 or w.shape[1] != x.shape[1]:
        raise ValueError("w [rows][K] and x [M][K] must share K")
    rows, K = w.shape
    M = x.shape[0]
    y = np.empty((M, rows), np.float32)
    ms = C.c_float(0.0)
    _lib.call("reng_gemm_bf16", w.ctypes.data, rows, K, x.ctypes.data, M, y.ctypes.data, splits, iters,
              C.byref(ms), _lib.RENG_MEM_HOST)
    return y, float(ms.value)


def gemm_fp8_blocks(x, x_scales, w, w_scales, out=None, dtype=None, x_fmt=_lib.RENG_FP8_E4M3,
                    w_fmt=_lib.RENG_FP8_E4M3, stream=None):
    """y[m][n] = sum_b x_scales[m][b] w_scales[n / 128][b] sum_{k in b} x[m][k] w[n][k].

    x uint8 codes [M, K] with scales [M, ceil(K / 128)], w uint8 codes [N, K]
    with scales [ceil(N / 128), ceil(K / 128)]; rows start on 16 bytes
    (fp8.quantize_blocks lays them out so).  y [M, N] is `out`, or a new
    tensor of `dtype` (bf16 by default, or f32).  Should a device wait of the
    product run out (a fault of the device or of this library), y is invalid
    and gemm_fp8_blocks_status raises.  `stream` as for fp8.quantize_blocks."""
    t = _impl or _tensors()
    if stream is not None:
        return t.on_stream(stream, x, t.gemm_fp8_blocks, x, x_scales, w, w_scales, out, dtype, x_fmt, w_fmt)
    return t.gemm_fp8_blocks(x, x_scales, w, w_scales, out, dtype, x_fmt, w_fmt)


def gemm_fp8_blocks_status(device=None):
    """Raise RengError (code RENG_E_TIMEOUT) if a product on the device (the
    current one by default) gave up on a bounded wait since the last call: its
    results are invalid.  Waits for all work of the device."""
    if device is None:
        _lib.call("reng_gemm_fp8_blocks_status")
    else:
        import torch
        with torch.cuda.device(device):
            _lib.call("reng_gemm_fp8_blocks_status")
