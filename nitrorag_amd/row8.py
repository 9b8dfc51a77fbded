"""Rows held in 8 bits (binding of nitro_rms_norm_row8, nitro_row8_* and nitro_q8_weights_*).

A row of n fp32 numbers is held as int8 codes and one fp32 scale: scale = max|y| / 127,
code = rint(y * (127 / max|y|)).  codes is an int8 tensor [rows][n], scales an fp32
tensor [rows], both of the caller's.  Q8Weights lays a Q8_0 matrix out once and
multiplies such rows with it; bias, activation and residual are part of the launch.
"""
from __future__ import annotations

import ctypes

from . import _native as N
from .attention import _torch_module
from .q8 import BLOCK, BLOCK_BYTES

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _refuse(func: str, message: str):
    raise N.NitroError(N.INVALID_ARGUMENT, func, message)


def _ptr(func: str, t, dtype, shape, name: str, dev: int):
    """The address of a contiguous tensor of that type and shape on the current device."""
    try:
        if t.dtype is dtype and t.get_device() == dev and t.is_contiguous() and t.shape == shape:
            return t.data_ptr()
    except AttributeError:
        pass
    if not isinstance(t, _torch_module().Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a GPU tensor")
    if t.dtype is not dtype or not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous {str(dtype)[6:]}")
    if t.shape != shape:
        _refuse(func, f"{name} must be [{']['.join(map(str, shape))}]")
    _refuse(func, f"{name} must be on the current device, cuda:{dev}")


def _rows(func: str, codes, scales, stream):
    """Of rows held in 8 bits: rows, n, the addresses of codes and scales; the current
    device, the stream's address, and torch.float32."""
    torch = _torch_module()
    dev = torch._C._cuda_getDevice()
    f32 = torch.float32
    shape = getattr(codes, "shape", (0, 0))
    if len(shape) != 2:
        _refuse(func, "codes must be [rows][n]")
    rows, n = shape
    pc = _ptr(func, codes, torch.int8, shape, "codes", dev)
    ps = _ptr(func, scales, f32, (rows,), "scales", dev)
    return rows, n, pc, ps, dev, torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream, f32


def rms_norm_row8(x, weight, codes, scales, residual=None, sum=None, eps: float = 1e-5, stream=None) -> None:
    """codes, scales = rms_norm(x + residual) * weight, held; sum receives x + residual
    (it may be x or residual)."""
    f = "rms_norm_row8"
    rows, n, pc, ps, dev, s, f32 = _rows(f, codes, scales, stream)
    shape = (rows, n)
    N.call("nitro_rms_norm_row8", _ptr(f, x, f32, shape, "x", dev),
           None if residual is None else _ptr(f, residual, f32, shape, "residual", dev),
           _ptr(f, weight, f32, (n,), "weight", dev), eps,
           None if sum is None else _ptr(f, sum, f32, shape, "sum", dev), pc, ps, rows, n, s)


def row8_quantize(x, codes, scales, stream=None) -> None:
    """codes, scales = the rows of x, held."""
    f = "row8_quantize"
    rows, n, pc, ps, dev, s, f32 = _rows(f, codes, scales, stream)
    N.call("nitro_row8_quantize", _ptr(f, x, f32, (rows, n), "x", dev), pc, ps, rows, n, s)


def row8_read(codes, scales, x, stream=None) -> None:
    """x = the values that the rows hold."""
    f = "row8_read"
    rows, n, pc, ps, dev, s, f32 = _rows(f, codes, scales, stream)
    N.call("nitro_row8_read", pc, ps, _ptr(f, x, f32, (rows, n), "x", dev), rows, n, s)


class Q8Weights:
    """A Q8_0 matrix w (uint8 GPU tensor, d rows of n / 32 BlockQ8) laid out for products
    with 8-bit rows, or with two matrices the gated pair: Q8Weights(gate, up) computes
    act(gate . x) * (up . x).  The tensors may go afterwards."""

    def __init__(self, w, up=None):
        torch = _torch_module()
        dev = torch.cuda.current_device()
        for t in (w,) if up is None else (w, up):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise TypeError("weights must be GPU tensors")
            if t.dim() < 2 or t.numel() == 0 or t.numel() // t.shape[0] % BLOCK_BYTES:
                _refuse("Q8Weights", f"weights must be rows of whole {BLOCK_BYTES}-byte blocks")
            _ptr("Q8Weights", t, torch.uint8, w.shape, "weights", dev)
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
        rows, n, pc, ps, dev, s, f32 = _rows(f, codes, scales, stream)
        if n != self.n:
            _refuse(f, f"the rows have {n} entries, the weights {self.n}")
        act = ACTIVATIONS.get(activation)
        if act is None:
            _refuse(f, f"activation must be one of {', '.join(ACTIVATIONS)}")
        d = self.d
        shape = (rows, d)
        N.call("nitro_row8_matmul", self._h, pc, ps,
               None if bias is None else _ptr(f, bias, f32, (2 * d if self.gated else d,), "bias", dev),
               None if residual is None else _ptr(f, residual, f32, shape, "residual", dev),
               _ptr(f, out, f32, shape, "out", dev), rows, act, s)

    def close(self):
        if getattr(self, "_h", None):
            N.call("nitro_q8_weights_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
