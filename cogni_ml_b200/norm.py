"""The norms around a block, with its gate and the addition to the residual stream, in one launch
(cogni_qmm_norm_residual): what stands between the products of a layer when many rows run together."""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Optional

import torch

from ._lib import lib
from .quant_matmul import _ROW_TYPE, _call, _output, _record, _row_type, _rows, _vector

_KINDS = {"rms": 0, "layer": 1}
_NORM_ARGS = struct.Struct("5Q5q2Qfi2Qfi5if2i")  # cogni_qmm_norm_args
_NO_NORM = (0, 0, 0.0, 0)


@dataclass
class Norm:
    """An RMS or layer norm: weight and bias f32 [n] on the device (Qwen35CPU#rms_norm, qwen35_cpu.cr:484-490)."""

    weight: torch.Tensor
    eps: float = 1.0e-6
    kind: str = "rms"
    bias: Optional[torch.Tensor] = None

    def _fields(self, n: int, dev: int):
        kind = _KINDS.get(self.kind)
        if kind is None:
            raise ValueError(f"kind must be one of {tuple(_KINDS)}, got {self.kind!r}")
        return _vector(self.weight, n, dev, "weight"), _vector(self.bias, n, dev, "bias"), self.eps, kind


def _side(t: torch.Tensor, m: int, n: int, dev: int, name: str):
    """(address, stride, type) of an [m, n] argument."""
    rows, stride = _rows(t, n, dev, name)
    if rows != m:
        raise ValueError(f"{name} must have a row for every row of residual")
    return t.data_ptr(), stride, _row_type(t, name)


def norm_residual(residual: torch.Tensor, block: Optional[torch.Tensor] = None, *, post_norm: Optional[Norm] = None,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0, norm: Optional[Norm] = None,
                  out_dtype=torch.bfloat16, hidden: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, stream=None):
    """h = residual + scale * gate * post_norm(block), y = norm(h); returns (h, y).

    residual, block [M, n], f32 or bf16.  gate: [n] for all rows or [M, n].  Without a block h is the
    residual itself, returned as it is (and not written unless `hidden` is given); without `norm` y is
    None.  hidden / out: where h and y go; each may be residual or block, other overlaps are refused.  h has the
    residual's type unless `hidden` says otherwise, y is out_dtype."""
    n = residual.shape[-1]
    dev = residual.get_device()
    if dev < 0 or not n:
        raise ValueError("residual must be on a CUDA device and have columns")
    m, res_stride = _rows(residual, n, dev, "residual")
    res_type = _row_type(residual, "residual")
    block_ptr = block_stride = block_type = gate_ptr = gate_stride = gate_type = 0
    if block is not None:
        block_ptr, block_stride, block_type = _side(block, m, n, dev, "block")
        if gate is not None:
            if gate.numel() == n:  # one row for all
                if gate.shape[-1] != n or not gate.is_contiguous() or gate.get_device() != dev:
                    raise ValueError(f"gate must have {n} contiguous elements, or a row for every row of residual")
                gate_ptr, gate_type = gate.data_ptr(), _row_type(gate, "gate")
            else:
                gate_ptr, gate_stride, gate_type = _side(gate, m, n, dev, "gate")
    elif post_norm is not None or gate is not None:
        raise ValueError("post_norm and gate belong to a block")
    elif norm is None:
        raise ValueError("nothing to compute: neither block nor norm")
    h_ptr = h_stride = h_type = 0
    if hidden is not None:
        h_ptr, h_stride, h_type = _side(hidden, m, n, dev, "hidden")
    elif block is not None:
        hidden = _output(residual, n, residual.dtype, stream) if stream or res_stride != n else torch.empty_like(residual)
        h_ptr, h_stride, h_type = hidden.data_ptr(), n, res_type
    y_ptr = y_stride = y_type = 0
    if norm is not None:
        if out is None:
            out = _output(residual, n, out_dtype, stream)
            y_ptr, y_stride, y_type = out.data_ptr(), n, _ROW_TYPE[out_dtype]
        else:
            y_ptr, y_stride, y_type = _side(out, m, n, dev, "out")
    elif out is not None:
        raise ValueError("out is the result of norm")
    post = _NO_NORM if post_norm is None else post_norm._fields(n, dev)
    pre = _NO_NORM if norm is None else norm._fields(n, dev)
    args = _NORM_ARGS.pack(residual.data_ptr(), block_ptr, gate_ptr, h_ptr, y_ptr,
                           res_stride, block_stride, gate_stride, h_stride, y_stride, *post, *pre,
                           res_type, block_type, gate_type, h_type, y_type, scale, m, n)
    if m:
        _call(lib.cogni_qmm_norm_residual, "cogni_qmm_norm_residual", args, dev, stream)
        if stream:
            _record(stream, residual, block, gate, hidden, out)
            for side in (post_norm, norm):
                if side is not None:
                    _record(stream, side.weight, side.bias)
    return hidden if hidden is not None else residual, out
