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
`stream` as for fp8.quantize_blocks.
"""
import struct

import torch

from . import _lib
from ._tensors import TYPES, blocks_out, call, index, matrix, on_stream, vector

_FP8_OUT = {_lib.RENG_FP8_E4M3: _lib.RENG_NORM_E4M3, _lib.RENG_FP8_E5M2: _lib.RENG_NORM_E5M2}
# reng_block_norm_desc, field for field (packed at once: filling the ctypes
# struct costs a call as much as its checks do)
_DESC = struct.Struct("8P8q4i2f")


def _run(residual, branch, post_gain, gate, scale, pre_gain, eps, out, h_out, h, ld_h, scales, ld_scales):
    """The checks of what is common and the call; returns y.  h, scales: tensors or None."""
    dev = index(residual)
    ldr = matrix(residual, "residual", TYPES, dev)
    rows, cols = residual.shape
    post, pre = vector(post_gain, "post_gain", cols, dev), vector(pre_gain, "pre_gain", cols, dev)
    rtype = TYPES[residual.dtype]
    pb = pg = py = ldb = ldg = ldy = tb = tg = 0
    if branch is None:
        if gate is not None or post_gain is not None or out is not None:
            raise ValueError("a gate, a post norm or an output residual without a branch")
        out = residual
    else:
        ldb = matrix(branch, "branch", TYPES, dev, rows, cols)
        pb, tb = branch.data_ptr(), TYPES[branch.dtype]
        if gate is not None:
            if gate.dim() == 1:
                matrix(gate.unsqueeze(0), "gate", TYPES, dev, 1, cols)
            else:
                ldg = matrix(gate, "gate", TYPES, dev, rows, cols)
            pg, tg = gate.data_ptr(), TYPES[gate.dtype]
        if out is None:
            out = torch.empty(rows, cols, dtype=residual.dtype, device=residual.device)
            ldy = cols
        else:
            ldy = matrix(out, "out", (residual.dtype,), dev, rows, cols)
        py = out.data_ptr()
    call(dev, "reng_block_norm", _DESC.pack(
        pb, residual.data_ptr(), pg, post or 0, pre or 0, py, 0 if h is None else h.data_ptr(),
        0 if scales is None else scales.data_ptr(), rows, cols, ldb, ldr, ldg, ldy, ld_h, ld_scales,
        tb, rtype, tg, h_out, scale, eps))
    return out


def _norm(residual, branch, post_gain, gate, scale, pre_gain, eps, norm, out, h, dtype):
    ldh, kind = 0, _lib.RENG_NORM_NONE
    if norm:
        dev = index(residual)
        if h is None:
            h = torch.empty(residual.shape, dtype=dtype, device=residual.device)
        ldh = matrix(h, "h", TYPES, dev, *residual.shape)
        kind = _lib.RENG_NORM_BF16 if h.dtype == torch.bfloat16 else _lib.RENG_NORM_F32
    elif h is not None or pre_gain is not None:
        raise ValueError("norm=False takes no h and no pre_gain")
    y = _run(residual, branch, post_gain, gate, scale, pre_gain, eps, out, kind, h, ldh, None, 0)
    return y, h


def _norm_fp8(residual, branch, post_gain, gate, scale, pre_gain, eps, fmt, out, codes, scales):
    dev = index(residual)
    if residual.dim() != 2:
        raise ValueError("residual has shape %s" % (tuple(residual.shape),))
    rows, cols = residual.shape
    codes, ldh, scales, lds = blocks_out(residual, dev, rows, cols, rows, codes, scales)
    y = _run(residual, branch, post_gain, gate, scale, pre_gain, eps, out, _FP8_OUT.get(fmt, -1), codes, ldh, scales, lds)
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
