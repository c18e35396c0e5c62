"""What the Python bindings of the fp8 linear and the linears of experts refuse or pass on, without a GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nemotron_cuda import CQError, experts, fp8

CODES, SCALES, BIAS = torch.zeros(4, 8, dtype=torch.uint8), torch.ones(1, 1), torch.zeros(4, dtype=torch.bfloat16)


# ------------------------------------------------------------------ types of a layer's arrays

@pytest.mark.parametrize("kw", [
    dict(bias=BIAS.half()), dict(bias=BIAS.view(torch.int16)), dict(bias=np.zeros(4, np.float16)), dict(bias=BIAS.float()),
    dict(scales=SCALES.to(torch.int32)), dict(scales=np.ones((1, 1), np.int32)), dict(scales=SCALES.double()),
    dict(codes=CODES.to(torch.int8)), dict(codes=CODES.bool()), dict(codes=CODES.view(torch.float8_e5m2)),
    dict(codes=np.zeros((4, 8), np.int8)),
], ids=lambda kw: "%s %s" % next((k, v.dtype) for k, v in kw.items()))
def test_layers_refuse_arrays_of_another_type(kw):
    """Bits of another type of the same size would be read as the layer's own."""
    a = dict(codes=CODES, scales=SCALES, bias=BIAS) | kw
    with pytest.raises(CQError, match="has type"):
        fp8.Fp8Linear.from_codes(a["codes"], a["scales"], a["bias"], dtype="bf16")
    with pytest.raises(CQError, match="has type"):
        experts.ExpertLinear.from_codes(*(a[k][None] for k in ("codes", "scales", "bias")), dtype="bf16")


def test_other_constructors_refuse_arrays_of_another_type():
    with pytest.raises(CQError, match="the bias has type float16, expected bfloat16"):
        experts.ExpertLinear.from_weight(torch.zeros(1, 4, 8, dtype=torch.bfloat16), torch.zeros(1, 4, dtype=torch.float16))
    with pytest.raises(CQError, match="the weight has type int32"):
        fp8.Fp8Linear.from_f32(torch.zeros(4, 8, dtype=torch.int32))
    with pytest.raises(CQError, match="the bias has type int32"):
        fp8.Fp8Linear.from_f32(np.zeros((4, 8), np.float32), np.zeros(4, np.int32))


@pytest.mark.parametrize("bias", [BIAS, np.zeros(4, np.uint16), np.zeros(4, np.int16), None])
def test_arrays_of_the_layer_s_types_reach_the_library(bias, monkeypatch):
    reached = []

    class Library:
        def cq_fp8_linear_create(self, *args):
            reached.append(args)
            return -1

        def cq_last_error(self):
            return b"reached"

    monkeypatch.setattr(fp8, "lib", Library)
    monkeypatch.setattr(fp8, "_check", lambda status: fp8._refuse("reached"))
    for codes in (CODES, CODES.view(torch.float8_e4m3fn), CODES.numpy()):
        with pytest.raises(CQError, match="reached"):
            fp8.Fp8Linear.from_codes(codes, SCALES, bias, dtype="bf16")
    assert len(reached) == 3


# ------------------------------------------------------------------ calls, on stand-ins for device tensors

EMPTY = torch.empty


class Rows:
    """What the bindings ask of a device tensor."""

    def __init__(self, *shape, dtype=torch.bfloat16, device=0, strides=None, requires_grad=False):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", device)
        self.strides = strides or EMPTY(shape, device="meta").stride()
        self.is_cuda, self.requires_grad = True, requires_grad

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def is_contiguous(self):
        return EMPTY(self.shape, device="meta").as_strided(self.shape, self.strides).is_contiguous()

    def element_size(self):
        return self.dtype.itemsize

    def data_ptr(self):
        return 1 << 20

    def new_empty(self, shape, dtype=None):
        return Rows(*([shape] if isinstance(shape, int) else shape), dtype=dtype or self.dtype, device=self.device.index)

    def as_strided(self, shape, strides, offset):
        return Rows(*shape, dtype=self.dtype, strides=strides)

    def view(self, dtype):
        return Rows(*self.shape, dtype=dtype, strides=self.strides)


@pytest.fixture
def calls(monkeypatch):
    """The library as a list of the calls that reach it, each of which succeeds."""
    seen = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args)) or 0

    for module in (fp8, experts):
        monkeypatch.setattr(module, "lib", Library)
    monkeypatch.setattr(fp8, "_raw_stream", lambda index: 77)
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: Rows(*([shape] if isinstance(shape, int) else shape), dtype=dtype))
    experts._route_workspace.cache_clear()
    yield seen
    experts._route_workspace.cache_clear()


def layer():
    return fp8.Fp8Linear(None, 1, 8, 16, "bf16", 0)


def expert_layer(n=8, k=16):
    return experts.ExpertLinear(None, 2, n, k, "bf16", 0, format="e4m3")


OFFSETS = Rows(3, dtype=torch.int32)
PAIRS = dict(position=Rows(4, 2, dtype=torch.int32), weight=Rows(4, 2, dtype=torch.float32))


def every_call(x=None, y=None, stream=None):
    """Each call that takes rows, of 16 values and (combine's) of 8, with an output of 8."""
    up, down = expert_layer(32, 16), expert_layer(8, 32)
    x = x or Rows(4, 16)
    yield lambda: layer().forward(x, y=y, stream=stream)
    yield lambda: expert_layer().forward(x, OFFSETS, y=y, stream=stream)
    yield lambda: experts.ExpertFeedForward(up, down, 2).forward(x, Rows(x.shape[0], 2, dtype=torch.float32), y=y, stream=stream)


def codes_call(y=None, stream=None):
    return layer().forward_codes(Rows(4, 128, dtype=torch.uint8), Rows(1, 4, dtype=torch.float32), y=y, stream=stream)


def combine_call(y=None, stream=None):
    return experts.combine(Rows(8, 8), **PAIRS, y=y, stream=stream)


def test_calls_reach_the_library(calls):
    y = Rows(4, 8)
    for call in (*every_call(y=y), lambda: codes_call(y), lambda: combine_call(y)):
        calls.clear()
        assert call() is y
        assert calls[-1][0].startswith("cq_")


def test_an_output_on_another_device_is_refused(calls):
    """It would be written as if it were local."""
    y = Rows(4, 8, device=1)
    for call in (*every_call(y=y), lambda: codes_call(y), lambda: combine_call(y)):
        calls.clear()
        with pytest.raises(CQError, match="output is on cuda:1, the input on cuda:0"):
            call()
        assert not any("forward" in name or "combine" in name for name, _ in calls)


# ------------------------------------------------------------------ streams

class OnStream:
    cuda_stream = 99


def test_the_current_stream_without_torch_s_short_way_to_it(calls, monkeypatch):
    monkeypatch.setattr(fp8, "_raw_stream", None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: OnStream)
    for call in (*every_call(), codes_call, combine_call, lambda: experts.route(Rows(4, 8), 2), lambda: fp8.quantize_rows(Rows(4, 8))):
        call()
        assert calls[-1][1][-1] == 99


# ------------------------------------------------------------------ strides

def test_a_single_row_may_have_any_row_stride(calls):
    """A transposed column is one row of neighbours with a row stride of 1; the library wants at least the width."""
    x, y = Rows(1, 16, strides=(1, 1)), Rows(1, 8, strides=(1, 1))
    for call, (of_x, of_y) in zip(every_call(x, y), ((2, 5), (2, 6), (3, 12))):
        call()
        assert calls[-1][1][of_x] == 16 and calls[-1][1][of_y] == 8
    layer().forward_codes(Rows(1, 128, dtype=torch.uint8, strides=(1, 1)), Rows(1, 1, dtype=torch.float32), y=y)
    assert calls[-1][1][2] == 128 and calls[-1][1][6] == 8
    experts.combine(Rows(1, 8, strides=(1, 1)), Rows(1, 2, dtype=torch.int32), Rows(1, 2, dtype=torch.float32), y=y)
    assert calls[-1][1][1] == 8 and calls[-1][1][10] == 8
    experts.route(Rows(1, 8, strides=(1, 1)), 2)
    assert calls[-1][1][1] == 8
    fp8.quantize_rows(Rows(1, 8, strides=(1, 1)))
    assert calls[-1][1][1] == 8
    # wider strides stay, as do those of more rows
    layer().forward(Rows(1, 16, strides=(24, 1)), y=Rows(1, 8, strides=(32, 1)))
    assert calls[-1][1][2] == 24 and calls[-1][1][5] == 32
    layer().forward(Rows(3, 16, strides=(20, 1)), y=Rows(3, 8, strides=(9, 1)))
    assert calls[-1][1][2] == 20 and calls[-1][1][5] == 9


# ------------------------------------------------------------------ gradients

def test_rows_that_require_a_gradient_are_refused(calls):
    """There is no backward pass, and the result would not say so."""
    def rows(*shape, dtype=torch.bfloat16):
        return Rows(*shape, dtype=dtype, requires_grad=True)
    made = list(every_call(rows(4, 16))) + [
        lambda: experts.route(rows(4, 8, dtype=torch.float32), 2),
        lambda: experts.combine(rows(8, 8), **PAIRS),
        lambda: experts.combine(Rows(8, 8), PAIRS["position"], rows(4, 2, dtype=torch.float32)),
        lambda: experts.ExpertFeedForward(expert_layer(32, 16), expert_layer(8, 32), 2).forward(
            Rows(4, 16), rows(4, 2, dtype=torch.float32)),
        lambda: layer().forward_codes(Rows(4, 128, dtype=torch.uint8), rows(1, 4, dtype=torch.float32)),
        lambda: fp8.quantize_rows(rows(4, 8)),
    ]
    for call in made:
        with pytest.raises(CQError, match="no backward pass"):
            call()
        with torch.no_grad():
            call()


def test_parameters_may_become_a_layer(calls):
    """A layer copies its arrays, so a module's parameters are taken as they are."""
    experts.ExpertLinear.from_weight(torch.nn.Parameter(torch.zeros(1, 4, 8, dtype=torch.bfloat16)))
    assert calls[-1][0] == "cq_expert_linear_create"


# ------------------------------------------------------------------ sizes

def test_sizes_past_32_bits_are_refused(calls):
    """The library takes 32-bit sizes, and ctypes would cut larger ones without a word."""
    many = (1 << 32) + 4
    made = list(every_call(Rows(many, 16))) + [
        lambda: experts.route(Rows(many, 8, dtype=torch.float32), 2),
        lambda: experts.combine(Rows(many, 8), **PAIRS),
        lambda: layer().forward_codes(Rows(many, 128, dtype=torch.uint8), Rows(1, many, dtype=torch.float32)),
        lambda: fp8.quantize_rows(Rows(many, 8)),
        lambda: fp8.quantize_weight(Rows(many, 1, dtype=torch.float32)),
    ]
    made += [lambda: fp8.Fp8Linear.from_codes(torch.zeros(1, 1, dtype=torch.uint8).expand(many, 1), SCALES),
             lambda: fp8.Fp8Linear.from_f32(torch.zeros(1, 1).expand(many, 1))]
    for call in made:
        calls.clear()
        with pytest.raises(CQError, match="32 bits"):
            call()
        assert not any("workspace" not in name for name, _ in calls)


# ------------------------------------------------------------------ layers that are closed

def test_a_closed_layer_is_refused(calls, monkeypatch):
    """By the library's own message, not by an allocation of the size that it answers for a refusal."""
    import nemotron_cuda
    for module in (fp8, experts):
        monkeypatch.setattr(module, "lib", nemotron_cuda.lib)
    for closed in (layer(), expert_layer()):
        closed.close()
        args = () if closed.experts == 1 else (OFFSETS,)
        for _ in range(2):
            with pytest.raises(CQError, match="layer must not be null"):
                closed.forward(Rows(4, 16), *args)


# ------------------------------------------------------------------ the module's attributes

def test_top_may_be_changed_between_calls(calls, monkeypatch):
    """The workspace is the one of the call's own `top`."""
    sizes = []

    class Library:
        def cq_expert_ffn_workspace(self, up, down, tokens, top):
            return 1000 * top + tokens

        def cq_expert_ffn_forward(self, *args):
            sizes.append((args[8], args[-2]))
            return 0

        def __getattr__(self, name):
            return lambda *args: 0

    monkeypatch.setattr(experts, "lib", Library)
    module = experts.ExpertFeedForward(expert_layer(32, 16), expert_layer(8, 32), 1)
    for top in (1, 2, 1):
        module.top = top
        module.forward(Rows(4, 16), Rows(4, 2, dtype=torch.float32))
    assert sizes == [(1, 1004), (2, 2004), (1, 1004)]
