"""The step between two decoder blocks on torch CUDA tensors
(libreng_cuda's reng_block_norm): the norm after a block, its gate and
residual scale, the residual add and the norm before the next block, in one
pass over the rows.

    u = branch
    u = u * r(u) * post_gain              with post_gain
    u = u * gate                          with gate
    y = round(residual + scale * u)       the residual stream, in its own type
    h = y * r(y) * pre_gain               r(v) = 1 / sqrt(mean(v^2) + eps), from y as rounded

`block_norm` returns (y, h) with h in bf16 or f32; `block_norm_fp8` returns
(y, codes, scales), h as FP8 codes with one f32 scale per 1 x 128 group, the
operand of gemm.gemm_fp8_blocks.  Sums and norms are f32.  `out` may be
`residual` itself (in place); without a branch y is `residual`, unwritten.
"""
import ctypes as C

import torch

from . import _lib
from ._tensors import TYPES, blocks_out, call, index, matrix, on_stream, vector

_FP8_OUT = {_lib.RENG_FP8_E4M3: _lib.RENG_NORM_E4M3, _lib.RENG_FP8_E5M2: _lib.RENG_NORM_E5M2}


def _desc(residual, branch, post_gain, gate, scale, pre_gain, eps, out):
    dev = index(residual)
    d = _lib.BlockNormDesc()
    d.ld_residual = matrix(residual, "residual", TYPES, dev)
    rows, cols = residual.shape
    d.rows, d.cols = rows, cols
    d.residual = residual.data_ptr()
    d.residual_type = TYPES[residual.dtype]
    d.scale, d.eps = scale, eps
    d.post_gain = vector(post_gain, "post_gain", cols, dev)
    d.pre_gain = vector(pre_gain, "pre_gain", cols, dev)
    if branch is None:
        if gate is not None or post_gain is not None or out is not None:
            raise ValueError("a gate, a post norm or an output residual without a branch")
        return d, residual
    d.ld_branch = matrix(branch, "branch", TYPES, dev, rows, cols)
    d.branch = branch.data_ptr()
    d.branch_type = TYPES[branch.dtype]
    if gate is not None:
        if gate.dim() == 1:
            gate = gate.unsqueeze(0)
            matrix(gate, "gate", TYPES, dev, 1, cols)
            d.ld_gate = 0
        else:
            d.ld_gate = matrix(gate, "gate", TYPES, dev, rows, cols)
        d.gate = gate.data_ptr()
        d.gate_type = TYPES[gate.dtype]
    if out is None:
        out = torch.empty((rows, cols), dtype=residual.dtype, device=residual.device)
        d.ld_y = cols
    else:
        d.ld_y = matrix(out, "out", (residual.dtype,), dev, rows, cols)
    d.y = out.data_ptr()
    return d, out


def _norm(residual, branch, post_gain, gate, scale, pre_gain, eps, norm, out, h, dtype):
    d, y = _desc(residual, branch, post_gain, gate, scale, pre_gain, eps, out)
    dev = residual.get_device()
    if norm:
        if h is None:
            h = torch.empty((d.rows, d.cols), dtype=dtype, device=residual.device)
        d.ld_h = matrix(h, "h", TYPES, dev, d.rows, d.cols)
        d.h = h.data_ptr()
        d.out = _lib.RENG_NORM_BF16 if h.dtype == torch.bfloat16 else _lib.RENG_NORM_F32
    elif h is not None or pre_gain is not None:
        raise ValueError("norm=False takes no h and no pre_gain")
    call(dev, "reng_block_norm", C.byref(d))
    return y, h


def _norm_fp8(residual, branch, post_gain, gate, scale, pre_gain, eps, fmt, out, codes, scales):
    d, y = _desc(residual, branch, post_gain, gate, scale, pre_gain, eps, out)
    dev = residual.get_device()
    codes, d.ld_h, scales, d.ld_scales = blocks_out(residual, dev, d.rows, d.cols, d.rows, codes, scales)
    d.h, d.h_scales = codes.data_ptr(), scales.data_ptr()
    d.out = _FP8_OUT.get(fmt, -1)
    call(dev, "reng_block_norm", C.byref(d))
    return y, codes, scales


def block_norm(residual, branch=None, post_gain=None, gate=None, scale=1.0, pre_gain=None, eps=1e-5, norm=True,
               out=None, h=None, dtype=torch.bfloat16, stream=None):
    """(y, h); with norm=False no h is formed and (y, None) returned."""
    args = (residual, branch, post_gain, gate, scale, pre_gain, eps, norm, out, h, dtype)
    return _norm(*args) if stream is None else on_stream(stream, residual, _norm, *args)


def block_norm_fp8(residual, branch=None, post_gain=None, gate=None, scale=1.0, pre_gain=None, eps=1e-5,
                   fmt=_lib.RENG_FP8_E4M3, out=None, codes=None, scales=None, stream=None):
    """(y, codes, scales): h quantized in 1 x 128 groups of `fmt`."""
    args = (residual, branch, post_gain, gate, scale, pre_gain, eps, fmt, out, codes, scales)
    return _norm_fp8(*args) if stream is None else on_stream(stream, residual, _norm_fp8, *args)
