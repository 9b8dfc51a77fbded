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
_INT32 = (1 << 31) - 1  # (ctypes takes a larger number's low 32 bits without a word)


def _refuse(func: str, message: str):
    raise N.NitroError(N.INVALID_ARGUMENT, func, message)


def _refuse_sizes(func: str, rows: int, n: int):
    raise N.NitroError(N.UNSUPPORTED, func,
                       "rows of more than 2^30 entries" if n > _INT32 else "more than 2^31 - 1 rows")


_bound = None


def _torch():
    """torch.int8, torch.float32 and what gives the current device and its stream's address."""
    global _bound
    if _bound is None:
        t = _torch_module()
        _bound = t.int8, t.float32, t._C._cuda_getDevice, t._C._cuda_getCurrentRawStream
    return _bound


def _check(func: str, t, dtype, shape, name: str, dev: int) -> None:
    """Refuses t unless it is a contiguous tensor of that type and shape on the current device."""
    if not isinstance(t, _torch_module().Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a GPU tensor")
    if t.dtype is not dtype or not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous {str(dtype)[6:]}")
    if t.shape != shape:
        _refuse(func, f"{name} must be [{']['.join(map(str, shape))}]")
    if t.get_device() != dev:
        _refuse(func, f"{name} must be on the current device, cuda:{dev}")


def _check_call(func: str, codes, scales, dev: int, others) -> None:
    """Says what is wrong with a call's tensors.  others(rows, n): (name, tensor or None, shape)
    of the fp32 ones.  (A call looks at them all in one expression first, which costs it 0.7 us
    of 5 less than a function for each.)"""
    i8, f32, *_ = _torch()
    shape = getattr(codes, "shape", (0, 0))
    if len(shape) != 2:
        _refuse(func, "codes must be [rows][n]")
    _check(func, codes, i8, shape, "codes", dev)
    _check(func, scales, f32, shape[:1], "scales", dev)
    for name, t, want in others(*shape):
        if t is not None:
            _check(func, t, f32, want, name, dev)


def _missing(t):
    """What stands for a tensor that is not optional: None is no tensor either."""
    return False if t is None else t


def rms_norm_row8(x, weight, codes, scales, residual=None, sum=None, eps: float = 1e-5, stream=None) -> None:
    """codes, scales = rms_norm(x + residual) * weight, held; sum receives x + residual
    (it may be x or residual)."""
    i8, f32, device, raw_stream = _bound or _torch()
    dev = device()
    try:
        shape = rows, n = codes.shape
        good = (codes.dtype is i8 and codes.get_device() == dev and codes.is_contiguous()
                and scales.dtype is f32 and scales.get_device() == dev and scales.is_contiguous() and scales.shape == (rows,)
                and x.dtype is f32 and x.get_device() == dev and x.is_contiguous() and x.shape == shape
                and weight.dtype is f32 and weight.get_device() == dev and weight.is_contiguous() and weight.shape == (n,)
                and (residual is None or residual.dtype is f32 and residual.get_device() == dev and residual.is_contiguous()
                     and residual.shape == shape)
                and (sum is None or sum.dtype is f32 and sum.get_device() == dev and sum.is_contiguous() and sum.shape == shape))
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        _check_call("rms_norm_row8", codes, scales, dev, lambda rows, n: (
            ("x", _missing(x), (rows, n)), ("residual", residual, (rows, n)), ("weight", _missing(weight), (n,)), ("sum", sum, (rows, n))))
    if rows | n > _INT32:
        _refuse_sizes("rms_norm_row8", rows, n)
    N.call("nitro_rms_norm_row8", x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(), eps,
           None if sum is None else sum.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, n,
           raw_stream(dev) if stream is None else stream.cuda_stream)


def _rows_and_values(func: str, x, codes, scales, stream):
    """Of rows held in 8 bits and their values: x, codes and scales as addresses, rows, n, the stream's address."""
    i8, f32, device, raw_stream = _bound or _torch()
    dev = device()
    try:
        shape = rows, n = codes.shape
        good = (codes.dtype is i8 and codes.get_device() == dev and codes.is_contiguous()
                and scales.dtype is f32 and scales.get_device() == dev and scales.is_contiguous() and scales.shape == (rows,)
                and x.dtype is f32 and x.get_device() == dev and x.is_contiguous() and x.shape == shape)
    except (AttributeError, TypeError, ValueError):
        good = False
    if not good:
        _check_call(func, codes, scales, dev, lambda rows, n: (("x", _missing(x), (rows, n)),))
    if rows | n > _INT32:
        _refuse_sizes(func, rows, n)
    return (x.data_ptr(), codes.data_ptr(), scales.data_ptr(), rows, n,
            raw_stream(dev) if stream is None else stream.cuda_stream)


def row8_quantize(x, codes, scales, stream=None) -> None:
    """codes, scales = the rows of x, held."""
    N.call("nitro_row8_quantize", *_rows_and_values("row8_quantize", x, codes, scales, stream))


def row8_read(codes, scales, x, stream=None) -> None:
    """x = the values that the rows hold."""
    px, pc, ps, rows, n, s = _rows_and_values("row8_read", x, codes, scales, stream)
    N.call("nitro_row8_read", pc, ps, px, rows, n, s)


def product_tile(rows: int, n: int, d: int, d_kv: int = 0, gated: bool = False) -> tuple:
    """(rows, weight rows, waves that split the blocks) of the kernel that takes a product of
    8-bit rows, a gated pair's or a model's wq, wk and wv (nitro_row8_tile)."""
    if max(rows, n, d, d_kv) > _INT32:
        raise N.NitroError(N.UNSUPPORTED, "product_tile", "sizes past 2^31 - 1")
    tile = (ctypes.c_int32 * 3)()
    N.call("nitro_row8_tile", rows, n, d, d_kv, gated, tile)
    return tuple(tile)


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
            _check("Q8Weights", t, torch.uint8, w.shape, "weights", dev)
        self.d = w.shape[0]
        self.n = w.numel() // self.d // BLOCK_BYTES * BLOCK
        self.gated = up is not None
        if self.n > 1 << 30 or self.d > 1 << 29:
            raise N.NitroError(N.UNSUPPORTED, "Q8Weights", "more than 2^30 columns or 2^29 rows")
        h = ctypes.c_void_p()
        N.call("nitro_q8_weights_create", (up if self.gated else w).data_ptr(), w.data_ptr() if self.gated else None,
               self.n, self.d, ctypes.byref(h))
        self._h = h

    def matmul(self, codes, scales, out, bias=None, residual=None, activation: str = "none", stream=None) -> None:
        """out[rows][d] = act(rows . w^T + bias) + residual; of a pair act(rows . gate^T +
        bias[:d]) * (rows . up^T + bias[d:]) + residual.  residual may be out."""
        i8, f32, device, raw_stream = _bound or _torch()
        dev, d = device(), self.d
        wide = 2 * d if self.gated else d
        try:
            rows, n = codes.shape
            shape = (rows, d)
            good = (codes.dtype is i8 and codes.get_device() == dev and codes.is_contiguous()
                    and scales.dtype is f32 and scales.get_device() == dev and scales.is_contiguous() and scales.shape == (rows,)
                    and out.dtype is f32 and out.get_device() == dev and out.is_contiguous() and out.shape == shape
                    and (bias is None or bias.dtype is f32 and bias.get_device() == dev and bias.is_contiguous() and bias.shape == (wide,))
                    and (residual is None or residual.dtype is f32 and residual.get_device() == dev and residual.is_contiguous()
                         and residual.shape == shape))
        except (AttributeError, TypeError, ValueError):
            good = False
        if not good:
            _check_call("Q8Weights.matmul", codes, scales, dev, lambda rows, n: (
                ("bias", bias, (wide,)), ("residual", residual, (rows, d)), ("out", _missing(out), (rows, d))))
        if n != self.n:
            _refuse("Q8Weights.matmul", f"the rows have {n} entries, the weights {self.n}")
        if rows > _INT32:
            _refuse_sizes("Q8Weights.matmul", rows, n)
        act = ACTIVATIONS.get(activation)
        if act is None:
            _refuse("Q8Weights.matmul", f"activation must be one of {', '.join(ACTIVATIONS)}")
        N.call("nitro_row8_matmul", self._h, codes.data_ptr(), scales.data_ptr(), None if bias is None else bias.data_ptr(),
               None if residual is None else residual.data_ptr(), out.data_ptr(), rows, act,
               raw_stream(dev) if stream is None else stream.cuda_stream)

    def close(self):
        if getattr(self, "_h", None):
            N.call("nitro_q8_weights_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
