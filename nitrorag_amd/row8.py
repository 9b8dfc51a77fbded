"""Rows held in 8 bits (binding of nitro_rms_norm_row8, nitro_row8_* and nitro_q8_weights_*).

A row of n fp32 numbers is held as int8 codes and one fp32 scale: scale = max|y| / 127,
code = rint(y * (127 / max|y|)).  codes is an int8 tensor [rows][n], scales an fp32
tensor [rows], both of the caller's.  Q8Weights lays a Q8_0 matrix out once and
multiplies such rows with it; bias, activation and residual are part of the launch.
"""
from __future__ import annotations

import ctypes

from . import _native as N
from .attention import _dev, _stream_ptr, _torch_module
from .q8 import BLOCK, BLOCK_BYTES

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _refuse(func: str, message: str):
    raise N.NitroError(N.INVALID_ARGUMENT, func, message)


def _here(func: str, t, dev: int):
    if t.get_device() != dev:
        _refuse(func, f"every tensor must be on the current device, cuda:{dev}")


def _rows(func: str, codes, scales):
    """(rows, n, current device) of rows held in 8 bits."""
    torch = _torch_module()
    dev = torch._C._cuda_getDevice()
    for t, dtype, name in ((codes, torch.int8, "codes"), (scales, torch.float32, "scales")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError(f"{name} must be a GPU tensor")
        if t.dtype is not dtype or not t.is_contiguous():
            raise TypeError(f"{name} must be contiguous {str(dtype)[6:]}")
        _here(func, t, dev)
    if codes.dim() != 2 or scales.shape != codes.shape[:1]:
        _refuse(func, "codes must be [rows][n] and scales [rows]")
    rows, n = codes.shape
    return rows, n, dev


def _f32(func: str, t, shape, name: str, dev: int):
    if t is None:
        return None
    p = _dev(t, name)
    if t.shape != shape:
        _refuse(func, f"{name} must be {'x'.join(map(str, shape))}")
    _here(func, t, dev)
    return p


def rms_norm_row8(x, weight, codes, scales, residual=None, sum=None, eps: float = 1e-5, stream=None) -> None:
    """codes, scales = rms_norm(x + residual) * weight, held; sum receives x + residual
    (it may be x or residual)."""
    f = "rms_norm_row8"
    rows, n, dev = _rows(f, codes, scales)
    shape = (rows, n)
    if x is None or weight is None:
        _refuse(f, "x and weight are required")
    N.call("nitro_rms_norm_row8", _f32(f, x, shape, "x", dev), _f32(f, residual, shape, "residual", dev),
           _f32(f, weight, (n,), "weight", dev), eps, _f32(f, sum, shape, "sum", dev), codes.data_ptr(), scales.data_ptr(),
           rows, n, _stream_ptr(stream))


def row8_quantize(x, codes, scales, stream=None) -> None:
    """codes, scales = the rows of x, held."""
    rows, n, dev = _rows("row8_quantize", codes, scales)
    N.call("nitro_row8_quantize", _f32("row8_quantize", x, (rows, n), "x", dev), codes.data_ptr(), scales.data_ptr(), rows, n,
           _stream_ptr(stream))


def row8_read(codes, scales, x, stream=None) -> None:
    """x = the values that the rows hold."""
    rows, n, dev = _rows("row8_read", codes, scales)
    N.call("nitro_row8_read", codes.data_ptr(), scales.data_ptr(), _f32("row8_read", x, (rows, n), "x", dev), rows, n,
           _stream_ptr(stream))


class Q8Weights:
    """A Q8_0 matrix w (uint8 GPU tensor, d rows of n / 32 BlockQ8) laid out for products
    with 8-bit rows, or with two matrices the gated pair: Q8Weights(gate, up) computes
    act(gate . x) * (up . x).  The tensors may go afterwards."""

    def __init__(self, w, up=None):
        import torch

        for t in (w, up):
            if t is None and t is not w:
                continue
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise TypeError("weights must be GPU tensors")
            if t.dtype is not torch.uint8 or not t.is_contiguous():
                raise TypeError("weights must be contiguous uint8")
            if t.dim() < 2 or t.numel() == 0 or t.numel() // t.shape[0] % BLOCK_BYTES:
                _refuse("Q8Weights", f"weights must be rows of whole {BLOCK_BYTES}-byte blocks")
            if t.shape[0] != w.shape[0] or t.numel() != w.numel():
                _refuse("Q8Weights", "the two matrices must have one shape")
            _here("Q8Weights", t, torch.cuda.current_device())
        self.d = w.shape[0]
        self.n = w.numel() // self.d // BLOCK_BYTES * BLOCK
        self.gated = up is not None
        h = ctypes.c_void_p()
        N.call("nitro_q8_weights_create", (up if self.gated else w).data_ptr(), w.data_ptr() if self.gated else None,
               self.n, self.d, ctypes.byref(h))
        self._h = h

    def matmul(self, codes, scales, out, bias=None, residual=None, activation: str = "none", stream=None) -> None:
        """out[rows][d] = act(rows . w^T + bias) + residual; of a pair act(rows . gate^T +
        bias[:d]) * (rows . up^T + bias[d:]) + residual.  residual may be out."""
        f = "Q8Weights.matmul"
        rows, n, dev = _rows(f, codes, scales)
        if n != self.n:
            _refuse(f, f"the rows have {n} entries, the weights {self.n}")
        if activation not in ACTIVATIONS:
            _refuse(f, f"activation must be one of {', '.join(ACTIVATIONS)}")
        if out is None:
            _refuse(f, "out is required")
        shape = (rows, self.d)
        N.call("nitro_row8_matmul", self._h, codes.data_ptr(), scales.data_ptr(),
               _f32(f, bias, (self.d * (1 + self.gated),), "bias", dev), _f32(f, residual, shape, "residual", dev),
               _f32(f, out, shape, "out", dev), rows, ACTIVATIONS[activation], _stream_ptr(stream))

    def close(self):
        if getattr(self, "_h", None):
            N.call("nitro_q8_weights_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
