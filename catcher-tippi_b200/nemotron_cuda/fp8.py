"""Python bindings of the 8-bit floating-point linear (include/cqfp8.h).

``Fp8Linear`` holds e4m3 weights with an f32 scale for each 128 x 128 block;
``forward`` brings the rows of x to e4m3 (a power-of-two scale for each 128
values), multiplies and applies bias and activation in f32.  There is no backward
pass: rows that require a gradient are refused outside torch.no_grad().
"""
from __future__ import annotations

import contextlib
import ctypes

import numpy as np
import torch

from . import ACTS, CQ_INVALID_ARGUMENT, DTYPES, CQError, _check, _ptr, lib

BLOCK = 128
TYPES = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
# dtype -> the library's code, for the calls
CODES = {t: DTYPES[name] for t, name in TYPES.items()}
SIZE_MAX = ctypes.c_size_t(-1).value
# the stream as a number, without building torch's Stream object (2 us a call); a
# private name, which a torch may lack
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _refuse(message: str):
    raise CQError(CQ_INVALID_ARGUMENT, message)


def _stream_of(stream, device) -> int:
    if stream is None:
        return _raw_stream(device.index) if _raw_stream else torch.cuda.current_stream(device).cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


_HERE = contextlib.nullcontext()


def _allocating(stream, device):
    """The context in which a call's tensors are allocated: torch's memory pool goes by the stream that uses it."""
    if stream is None:
        return _HERE
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream)


def _contiguous(a):
    """The array without gaps: numpy or torch, on the host or the device."""
    return np.ascontiguousarray(a) if isinstance(a, np.ndarray) else a.contiguous()


def _fits32(shape, what: str):
    """Refuses sizes that the library's 32-bit arguments would cut."""
    if any(n > 0x7FFFFFFF for n in shape):
        _refuse(f"{what} of shape {tuple(shape)}: sizes must fit 32 bits")


def _packed(a, *shape):
    """An array argument of a layer: its shape checked, without gaps."""
    if tuple(a.shape) != shape:
        _refuse(f"array has shape {tuple(a.shape)}, expected {shape}")
    _fits32(shape, "an array")
    return _contiguous(a)


def _typed(a, name: str, what: str):
    """Refuses an array argument of a layer whose type is not `name`: its bits would be read as another's."""
    kind = a.dtype.name if isinstance(a, np.ndarray) else str(a.dtype).removeprefix("torch.")
    if name == "codes":
        fits = kind in ("uint8", "float8_e4m3fn")
    elif isinstance(a, np.ndarray) and name in ("float16", "bfloat16"):
        # numpy holds bf16, which it lacks, as raw 16-bit values
        fits = a.itemsize == 2 and kind in (name, "uint16", "int16")
    else:
        fits = kind == name
    if not fits:
        _refuse(f"{what} has type {kind}, expected {'uint8 or float8_e4m3fn' if name == 'codes' else name}")


T_NAMES = {"f16": "float16", "bf16": "bfloat16"}


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def _no_gradient(x, what: str):
    """Refuses what autograd follows: these operators have no backward pass, and the result would silently have none."""
    if x.requires_grad and torch.is_grad_enabled():
        _refuse(f"{what} requires a gradient, and there is no backward pass: call under torch.no_grad() or detach it")


def _rows_of(x, dims: int, what: str = "input") -> tuple[int, int]:
    """(rows, row stride) of device rows for the library, which asks for a stride of at least the width; that of a
    single row may be anything in torch (a transposed column has 1)."""
    if not x.is_cuda:
        _refuse(f"{what} must be on the device, got {x.device}")
    shape, strides = x.shape, x.stride()
    if len(shape) != 2 or shape[1] != dims or (dims > 1 and strides[1] != 1):
        _refuse(f"{what} must be rows of {dims} values next to each other, got shape {tuple(shape)} "
                f"with strides {tuple(strides)}")
    if x.requires_grad:
        _no_gradient(x, what)
    rows = shape[0]
    if rows > 0x7FFFFFFF:
        _fits32(shape, what)
    return rows, strides[0] if rows > 1 else max(strides[0], dims)


def _check_output(y, dtype, rows: int, dims: int, device) -> int:
    """The row stride of a caller's output, which is refused where the call could not write it."""
    if y.dtype != dtype or y.shape[0] != rows:
        _refuse(f"output must be {dtype} with {rows} rows")
    if y.device != device:
        _refuse(f"output is on {y.device}, the input on {device}")
    return _rows_of(y, dims, "output")[1]


class _Layer:
    """A handle of the library and what its calls need to know."""

    _destroy = ""

    def __init__(self, handle: ctypes.c_void_p, experts: int, output_dims: int, input_dims: int, dtype: str,
                 device: int):
        self._h = handle
        self.experts, self.output_dims, self.input_dims = experts, output_dims, input_dims
        self.dtype, self.device = dtype, device
        self._type = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        self._device = torch.device("cuda", device)
        self._sizes: dict[int, int] = {}

    def _output(self, x, rows: int, y):
        """(the call's output, its row stride), made where the caller gave none."""
        if x.device != self._device:
            _refuse(f"input is on {x.device}, the layer on {self._device}")
        if x.dtype != self._type:
            _refuse(f"input has type {x.dtype}, expected {self._type}")
        if y is None:
            return x.new_empty((rows, self.output_dims)), self.output_dims
        return y, _check_output(y, self._type, rows, self.output_dims, x.device)

    def _workspace(self, entry, rows: int):
        """(tensor that keeps the memory, pointer, bytes) for a call on `rows` rows."""
        n = self._sizes.get(rows)
        if n is None:
            n = entry(self._h, rows)
            if n == SIZE_MAX:
                _check(-1)
            if len(self._sizes) > 256:
                self._sizes.clear()
            self._sizes[rows] = n
        if n == 0:
            return None, None, 0
        w = torch.empty(n, dtype=torch.uint8, device=self._device)
        return w, w.data_ptr(), n

    def close(self) -> None:
        if getattr(self, "_h", None):
            try:
                getattr(lib(), self._destroy)(self._h)
            except TypeError:  # interpreter shutdown
                pass
            self._h = None

    def __del__(self):
        self.close()


class Fp8Linear(_Layer):
    """y = act(x^ . w^T + b) with e4m3 weights in blocks of 128 x 128."""

    _destroy = "cq_fp8_linear_destroy"

    @classmethod
    def from_codes(cls, codes, scales, bias=None, dtype: str = "bf16", device: int = 0) -> "Fp8Linear":
        """codes [N, K] of one byte (torch float8_e4m3fn or uint8, or numpy uint8), scales f32
        [ceil(N / 128), ceil(K / 128)], bias T [N] or None; host or device arrays."""
        n, k = codes.shape
        _typed(codes, "codes", "an array of codes")
        _typed(scales, "float32", "an array of scales")
        if bias is not None:
            _typed(bias, T_NAMES.get(dtype, dtype), "the bias")
        c, s = _packed(codes, n, k), _packed(scales, blocks(n), blocks(k))
        b = None if bias is None else _packed(bias, n)
        h = ctypes.c_void_p()
        _check(lib().cq_fp8_linear_create(_ptr(c), _ptr(s), _ptr(b), n, k, DTYPES[dtype], device, ctypes.byref(h)))
        return cls(h, 1, n, k, dtype, device)

    @classmethod
    def from_f32(cls, weight, bias=None, dtype: str = "bf16", device: int = 0) -> "Fp8Linear":
        """An f32 weight [N, K] and bias [N] (numpy or torch, host or device), brought to e4m3 on the device."""
        n, k = weight.shape
        _typed(weight, "float32", "the weight")
        if bias is not None:
            _typed(bias, "float32", "the bias")
        w, b = _packed(weight, n, k), None if bias is None else _packed(bias, n)
        h = ctypes.c_void_p()
        _check(lib().cq_fp8_linear_create_from_f32(_ptr(w), _ptr(b), n, k, DTYPES[dtype], device, ctypes.byref(h)))
        return cls(h, 1, n, k, dtype, device)

    def forward(self, x, y=None, act: str = "none", stream=None):
        """x torch [rows, K] of T on the layer's device -> y [rows, N]."""
        rows, ldx = _rows_of(x, self.input_dims)
        L = lib()
        with _allocating(stream, x.device):
            y, ldy = self._output(x, rows, y)
            keep, ws, n = self._workspace(L.cq_fp8_linear_workspace, rows)
            _check(L.cq_fp8_linear_forward(self._h, x.data_ptr(), ldx, rows, y.data_ptr(), ldy, ACTS[act], ws, n,
                                           _stream_of(stream, x.device)))
        return y

    def forward_codes(self, codes, scales, y=None, act: str = "none", stream=None):
        """forward on rows that quantize_rows made: codes [rows, >= K], scales [ceil(K / 128), rows]."""
        if codes.device != self._device or scales.device != self._device:
            _refuse(f"codes and scales must be on {self._device}")
        if codes.dtype is not torch.float8_e4m3fn and codes.dtype is not torch.uint8:
            _refuse(f"codes have type {codes.dtype}, expected uint8 or float8_e4m3fn")
        if codes.dim() != 2 or codes.shape[1] < self.input_dims or codes.stride(1) != 1:
            _refuse(f"codes must be rows of at least {self.input_dims} bytes, got shape {tuple(codes.shape)}")
        rows, ldc = _rows_of(codes, codes.shape[1], "codes")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (blocks(self.input_dims), rows) or \
                not scales.is_contiguous():
            _refuse(f"scales must be f32 [{blocks(self.input_dims)}, {rows}] without gaps")
        _no_gradient(scales, "an array of scales")
        if y is None:
            with _allocating(stream, codes.device):
                y, ldy = torch.empty((rows, self.output_dims), dtype=self._type, device=codes.device), self.output_dims
        else:
            ldy = _check_output(y, self._type, rows, self.output_dims, codes.device)
        _check(lib().cq_fp8_linear_forward_codes(self._h, codes.data_ptr(), ldc, scales.data_ptr(), rows,
                                                 y.data_ptr(), ldy, ACTS[act], _stream_of(stream, codes.device)))
        return y


def quantize_rows(x, stream=None):
    """x torch [rows, K] (f16, bf16 or f32) -> (e4m3 codes [rows, 128 ceil(K / 128)], scales f32 [ceil(K / 128), rows])."""
    if x.dim() != 2:
        _refuse(f"input must be rows, got shape {tuple(x.shape)}")
    k = x.shape[1]
    rows, ldx = _rows_of(x, k)
    kind = TYPES.get(x.dtype)
    if kind is None:
        _refuse(f"input has type {x.dtype}, expected f16, bf16 or f32")
    with _allocating(stream, x.device):
        codes = torch.empty((rows, BLOCK * blocks(k)), dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty((blocks(k), rows), dtype=torch.float32, device=x.device)
    _check(lib().cq_fp8_quantize_rows(x.data_ptr(), ldx, rows, k, DTYPES[kind], codes.data_ptr(),
                                      codes.stride(0), scales.data_ptr(), _stream_of(stream, x.device)))
    return codes, scales


def quantize_weight(w, stream=None):
    """w torch f32 [N, K] on the device -> (e4m3 codes [N, K], scales f32 [ceil(N / 128), ceil(K / 128)])."""
    if not w.is_cuda or w.dim() != 2 or w.dtype != torch.float32 or not w.is_contiguous():
        _refuse("weight must be f32 [N, K] without gaps on the device")
    n, k = w.shape
    _fits32(w.shape, "a weight")
    with _allocating(stream, w.device):
        codes = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=w.device)
        scales = torch.empty((blocks(n), blocks(k)), dtype=torch.float32, device=w.device)
    _check(lib().cq_fp8_quantize_weight(w.data_ptr(), n, k, codes.data_ptr(), scales.data_ptr(),
                                        _stream_of(stream, w.device)))
    return codes, scales
