"""Python bindings of the linears of experts (include/cqexperts.h).

``route`` chooses each token's experts and orders the (token, expert) pairs by
expert, ``ExpertLinear`` multiplies rows so ordered by the weights of their
expert, ``combine`` sums what each token's experts made, and
``ExpertFeedForward`` is the feed-forward module of the four steps.  There is no
backward pass: tensors that require a gradient are refused outside
torch.no_grad().
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import ACTS, DTYPES, _check, _ptr, lib
from .fp8 import (CODES, SIZE_MAX, T_NAMES, TYPES, _allocating, _check_output, _Layer, _no_gradient, _packed, _refuse, _rows_of, _stream_of, _typed,
                  blocks)

FORMATS = {"16bit": 0, "e4m3": 1}


class Route(NamedTuple):
    """What cq_route says of tokens: see include/cqexperts.h."""
    expert: object    # int32 [tokens, top]
    weight: object    # f32 [tokens, top]
    offsets: object   # int32 [experts + 1]
    token: object     # int32 [tokens * top]
    position: object  # int32 [tokens, top]


@functools.lru_cache(maxsize=256)
def _route_workspace(tokens: int, experts: int, top: int) -> int:
    n = lib().cq_route_workspace(tokens, experts, top)
    if n == SIZE_MAX:
        _check(-1)
    return n


def route(logits, top: int, renormalize: bool = True, stream=None) -> Route:
    """Router logits torch [tokens, experts] (f32, f16 or bf16) -> each token's `top` best experts and the order of pairs."""
    if logits.dim() != 2:
        _refuse(f"logits must be [tokens, experts], got shape {tuple(logits.shape)}")
    experts = logits.shape[1]
    tokens, ld = _rows_of(logits, experts, "logits")
    kind = CODES.get(logits.dtype)
    if kind is None:
        _refuse(f"logits have type {logits.dtype}, expected f32, f16 or bf16")
    L, device = lib(), logits.device
    n = _route_workspace(tokens, experts, top)
    # one allocation: expert, weight, position and token, each from a 256-byte
    # boundary on, then the offsets and the call's workspace
    step = (tokens * top + 63) & ~63
    end = 4 * step + ((experts + 64) & ~63)
    with _allocating(stream, device):
        ints = logits.new_empty(end + n // 4, dtype=torch.int32)
        at = ints.data_ptr()
        _check(L.cq_route(logits.data_ptr(), ld, kind, tokens, experts, top, int(renormalize), at, at + 4 * step,
                          at + 16 * step, at + 12 * step, at + 8 * step, at + 4 * end if n else None, n,
                          _stream_of(stream, device)))
    pairs, across = (tokens, top), (top, 1)
    expert, weight = ints.as_strided(pairs, across, 0), ints.as_strided(pairs, across, step).view(torch.float32)
    position, token = ints.as_strided(pairs, across, 2 * step), ints.as_strided((tokens * top,), (1,), 3 * step)
    offsets = ints.as_strided((experts + 1,), (1,), 4 * step)
    return Route(expert, weight, offsets, token, position)


def combine(z, position, weight, y=None, stream=None):
    """y[t] = sum_j weight[t, j] z[position[t, j]]: z torch [rows, dims] f16 or bf16, position int32 and weight f32 [tokens, top]."""
    if z.dim() != 2 or position.dim() != 2 or tuple(weight.shape) != tuple(position.shape):
        _refuse(f"expected rows, and positions and weights [tokens, top]; got shapes {tuple(z.shape)}, "
                f"{tuple(position.shape)} and {tuple(weight.shape)}")
    dims = z.shape[1]
    tokens, top = position.shape
    rows, ldz = _rows_of(z, dims, "rows")
    kind = CODES.get(z.dtype)
    if kind is None or z.dtype is torch.float32:
        _refuse(f"rows have type {z.dtype}, expected f16 or bf16")
    if position.dtype != torch.int32 or weight.dtype != torch.float32 or not position.is_contiguous() or \
            not weight.is_contiguous() or position.device != z.device or weight.device != z.device:
        _refuse("positions must be int32 and weights f32, without gaps, on the device of the rows")
    if weight.requires_grad:
        _no_gradient(weight, "an array of weights")
    if y is None:
        with _allocating(stream, z.device):
            y, ldy = z.new_empty((tokens, dims)), dims
    else:
        ldy = _check_output(y, z.dtype, tokens, dims, z.device)
    _check(lib().cq_expert_combine(z.data_ptr(), ldz, rows, position.data_ptr(), weight.data_ptr(), tokens,
                                   top, dims, kind, y.data_ptr(), ldy, _stream_of(stream, z.device)))
    return y


class ExpertLinear(_Layer):
    """Rows sorted by expert, each by its expert's weights: y[r] = act(W[e] x[r] + b[e])."""

    _destroy = "cq_expert_linear_destroy"

    def __init__(self, *args, format: str):
        super().__init__(*args)
        self.format = format

    @classmethod
    def _create(cls, weight, scales, bias, format: str, dtype: str, device: int) -> "ExpertLinear":
        e, n, k = weight.shape
        if bias is not None:
            _typed(bias, T_NAMES.get(dtype, dtype), "the bias")
        w, b = _packed(weight, e, n, k), None if bias is None else _packed(bias, e, n)
        s = None if scales is None else _packed(scales, e, blocks(n), blocks(k))
        h = ctypes.c_void_p()
        _check(lib().cq_expert_linear_create(_ptr(w), _ptr(s), _ptr(b), e, n, k, FORMATS[format], DTYPES[dtype],
                                             device, ctypes.byref(h)))
        return cls(h, e, n, k, dtype, device, format=format)

    @classmethod
    def from_weight(cls, weight, bias=None, device: int = 0) -> "ExpertLinear":
        """torch f16 or bf16 weights [experts, N, K] and bias [experts, N] or None, host or device."""
        kind = TYPES.get(weight.dtype)
        if kind not in ("f16", "bf16"):
            _refuse(f"weight has type {weight.dtype}, expected f16 or bf16")
        return cls._create(weight, None, bias, "16bit", kind, device)

    @classmethod
    def from_codes(cls, codes, scales, bias=None, dtype: str = "bf16", device: int = 0) -> "ExpertLinear":
        """e4m3 codes [experts, N, K], scales f32 [experts, ceil(N / 128), ceil(K / 128)], bias T [experts, N] or None."""
        _typed(codes, "codes", "an array of codes")
        _typed(scales, "float32", "an array of scales")
        return cls._create(codes, scales, bias, "e4m3", dtype, device)

    def forward(self, x, offsets, y=None, act: str = "none", stream=None):
        """x torch [rows, K] of T, offsets int32 [experts + 1] on the device -> y [rows, N], zeros from offsets[-1] on."""
        rows, ldx = _rows_of(x, self.input_dims)
        if offsets.dtype != torch.int32 or tuple(offsets.shape) != (self.experts + 1,) or \
                not offsets.is_contiguous() or offsets.device != self._device:
            _refuse(f"offsets must be int32 [{self.experts + 1}] on {self._device}, got {offsets.dtype} "
                    f"{tuple(offsets.shape)} on {offsets.device}")
        L = lib()
        with _allocating(stream, x.device):
            y, ldy = self._output(x, rows, y)
            keep, ws, n = self._workspace(L.cq_expert_linear_workspace, rows)
            _check(L.cq_expert_linear_forward(self._h, x.data_ptr(), ldx, rows, offsets.data_ptr(), y.data_ptr(), ldy,
                                              ACTS[act], ws, n, _stream_of(stream, x.device)))
        return y


class ExpertFeedForward:
    """y = combine(down(act(up(x)))) over the `top` experts that the logits choose for each token."""

    def __init__(self, up: ExpertLinear, down: ExpertLinear, top: int, act: str = "silu", renormalize: bool = True):
        self.up, self.down, self.top, self.act, self.renormalize = up, down, top, act, renormalize
        self._sizes: dict[tuple[int, int], int] = {}
        self._workspace_bytes(0)  # the library's checks of the pair

    def _workspace_bytes(self, tokens: int) -> int:
        n = self._sizes.get((tokens, self.top))
        if n is None:
            n = lib().cq_expert_ffn_workspace(self.up._h, self.down._h, tokens, self.top)
            if n == SIZE_MAX:
                _check(-1)
            if len(self._sizes) > 256:
                self._sizes.clear()
            self._sizes[tokens, self.top] = n
        return n

    def forward(self, x, logits, y=None, stream=None):
        """x torch [tokens, K] of T, logits [tokens, experts] (f32, f16 or bf16) -> y [tokens, N]."""
        up, down = self.up, self.down
        tokens, ldx = _rows_of(x, up.input_dims)
        logit_rows, ld = _rows_of(logits, up.experts, "logits")
        kind = CODES.get(logits.dtype)
        if kind is None or logit_rows != tokens:
            _refuse(f"logits must be f32, f16 or bf16 with {tokens} rows, got {logits.dtype} {tuple(logits.shape)}")
        if tokens * self.top > 0x7FFFFFFF:
            _refuse("tokens * top does not fit 32 bits")
        if logits.device != x.device:
            _refuse(f"logits are on {logits.device}, the input on {x.device}")
        n = self._workspace_bytes(tokens)
        with _allocating(stream, x.device):
            y, ldy = down._output(x, tokens, y)
            ws = torch.empty(n, dtype=torch.uint8, device=x.device)
            _check(lib().cq_expert_ffn_forward(up._h, down._h, x.data_ptr(), ldx, tokens, logits.data_ptr(), ld,
                                               kind, self.top, int(self.renormalize), ACTS[self.act], y.data_ptr(), ldy,
                                               ws.data_ptr(), n, _stream_of(stream, x.device)))
        return y
