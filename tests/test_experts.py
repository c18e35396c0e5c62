"""The fp8 linear and the linears of experts without a GPU: the oracle's own rules, and every refusal that the
library makes before it touches a device."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import experts_oracle as eo

SIZE_MAX = ctypes.c_size_t(-1).value


def test_oracle_e4m3_is_the_format():
    """All 256 codes decode to values that round to themselves, and midpoints go to the even neighbour."""
    values = np.sort(np.unique(eo.decode(np.arange(0x7F, dtype=np.uint8))))
    assert values[0] == 0.0 and values[-1] == 448.0 and len(values) == 127 and values[1] == 2.0 ** -9
    assert np.array_equal(eo.e4m3(values), values) and np.array_equal(eo.e4m3(-values), -values)
    middle = (values[:-1] + values[1:]) / 2
    even = np.where(np.arange(126) % 2 == 0, values[:-1], values[1:])  # code i is even where i is
    assert np.array_equal(eo.e4m3(middle), even)
    assert np.isnan(eo.decode(np.array([0x7F, 0xFF], np.uint8))).all()


@pytest.mark.parametrize("top,scale", [(448.0, 1.0), (448.1, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8), (1.75, 2.0 ** -8),
                                       (1.76, 2.0 ** -7), (0.0, 1.0), (2.0 ** -140, 2.0 ** -126)])
def test_oracle_scale_is_the_least_power_of_two(top, scale):
    assert eo.scale_of(np.array([0.0, -top, top / 2])) == scale


def test_oracle_scale_leaves_infinities_and_nan_out():
    assert eo.scale_of(np.array([1.0, np.inf, np.nan])) == 2.0 ** -8


def test_oracle_route_by_hand():
    z = np.array([[1.0, 3.0, 3.0, 0.0], [-np.inf] * 4, [np.nan, -np.inf, 0.0, -np.inf], [5.0, 1.0, 0.0, 2.0]])
    expert, weight, offsets, token, position = eo.route(z, 2)
    assert expert.tolist() == [[1, 2], [-1, -1], [2, -1], [0, 3]]
    assert weight[0].tolist() == [0.5, 0.5] and weight[1].tolist() == [0.0, 0.0] and weight[2].tolist() == [1.0, 0.0]
    assert offsets.tolist() == [0, 1, 2, 4, 5]
    assert token.tolist() == [3, 0, 0, 2, 3, -1, -1, -1]
    assert position.tolist() == [[1, 2], [-1, -1], [3, -1], [0, 4]]


def _refused(cq, status, needle):
    assert status == cq.CQ_INVALID_ARGUMENT
    assert needle in cq.last_error(), cq.last_error()


def _fp8_create(cq, n=4, k=128, dtype=1, codes=True, scales=True, device=0):
    h = ctypes.c_void_p()
    c, s = np.zeros((4, 128), np.uint8), np.ones((1, 1), np.float32)
    return cq.lib().cq_fp8_linear_create(c.ctypes.data if codes else None, s.ctypes.data if scales else None, None, n, k,
                                         dtype, device, ctypes.byref(h))


@pytest.mark.parametrize("kw,needle", [
    (dict(codes=False), "weight must not be null"),
    (dict(scales=False), "scales must not be null"),
    (dict(n=0), "invalid linear shape"),
    (dict(k=0), "invalid linear shape"),
    (dict(n=-3), "invalid linear shape"),
    (dict(k=1 << 21), "invalid linear shape"),
    (dict(dtype=2), "dtype must be f16 or bf16"),
])
def test_fp8_create_refusals(cq, kw, needle):
    _refused(cq, _fp8_create(cq, **kw), needle)


@pytest.mark.parametrize("experts,n,k,form,dtype,needle", [
    (0, 4, 128, 0, 1, "experts must be 1 to 1024"),
    (1025, 4, 128, 0, 1, "experts must be 1 to 1024"),
    (2, 4, 128, 2, 1, "unknown weight format"),
    (2, 4, 128, 0, 2, "dtype must be f16 or bf16"),
    (2, 0, 128, 0, 1, "invalid linear shape"),
    (2, 4, 128, 1, 1, "scales must not be null"),
])
def test_expert_create_refusals(cq, experts, n, k, form, dtype, needle):
    w, h = np.zeros(8 * 128, np.uint16), ctypes.c_void_p()
    _refused(cq, cq.lib().cq_expert_linear_create(w.ctypes.data, None, None, experts, n, k, form, dtype, 0,
                                                  ctypes.byref(h)), needle)


def test_null_handles_and_outputs(cq):
    L = cq.lib()
    _refused(cq, L.cq_fp8_linear_create(None, None, None, 1, 1, 1, 0, None), "out must not be null")
    _refused(cq, L.cq_expert_linear_create(None, None, None, 1, 1, 1, 0, 1, 0, None), "out must not be null")
    _refused(cq, L.cq_fp8_linear_forward(None, None, 1, 1, None, 1, 0, None, 0, None), "layer must not be null")
    _refused(cq, L.cq_fp8_linear_forward_codes(None, None, 1, None, 1, None, 1, 0, None), "layer must not be null")
    _refused(cq, L.cq_expert_linear_forward(None, None, 1, 1, None, None, 1, 0, None, 0, None), "layer must not be null")
    _refused(cq, L.cq_expert_ffn_forward(None, None, None, 1, 1, None, 1, 2, 1, 1, 0, None, 1, None, 0, None),
             "up must not be null")
    assert L.cq_fp8_linear_workspace(None, 1) == SIZE_MAX
    assert L.cq_expert_linear_workspace(None, 1) == SIZE_MAX
    assert L.cq_expert_ffn_workspace(None, None, 1, 1) == SIZE_MAX
    assert L.cq_fp8_linear_input_dims(None) == -1 and L.cq_fp8_linear_output_dims(None) == -1
    assert L.cq_expert_linear_experts(None) == -1
    L.cq_fp8_linear_destroy(None)
    L.cq_expert_linear_destroy(None)


@pytest.mark.parametrize("rows,cols,ldx,ld,dtype,needle", [
    (4, 0, 128, 128, 1, "invalid shape"),
    (-1, 128, 128, 128, 1, "invalid shape"),
    (4, 128, 127, 128, 1, "input row stride 127 is smaller than 128"),
    (4, 100, 100, 100, 1, "must be a multiple of 16"),
    (4, 128, 128, 112, 1, "at least 128"),
    (4, 128, 128, 128, 9, "unknown dtype 9"),
    (4, 128, 128, 128, 1, "must not be null"),
])
def test_quantize_rows_refusals(cq, rows, cols, ldx, ld, dtype, needle):
    _refused(cq, cq.lib().cq_fp8_quantize_rows(None, ldx, rows, cols, dtype, None, ld, None, None), needle)
    assert cq.lib().cq_fp8_quantize_rows(None, 128, 0, 128, 1, None, 128, None, None) == cq.CQ_OK  # no rows, no work


def test_quantize_weight_refusals(cq):
    _refused(cq, cq.lib().cq_fp8_quantize_weight(None, 4, 0, None, None, None), "invalid shape")
    _refused(cq, cq.lib().cq_fp8_quantize_weight(None, 4, 4, None, None, None), "must not be null")


@pytest.mark.parametrize("tokens,experts,top,dtype,ld,needle", [
    (-1, 8, 2, 2, 8, "negative token count"),
    (4, 0, 1, 2, 8, "experts must be 1 to 1024"),
    (4, 8, 0, 2, 8, "top must be 1 to"),
    (4, 8, 9, 2, 8, "top must be 1 to"),
    (4, 64, 33, 2, 64, "top must be 1 to"),
    (1 << 30, 8, 4, 2, 8, "does not fit 32 bits"),
    (4, 8, 2, 3, 8, "unknown dtype 3"),
    (4, 8, 2, 2, 7, "logits row stride 7 is smaller than 8"),
    (4, 8, 2, 2, 8, "logits and outputs must not be null"),
])
def test_route_refusals(cq, tokens, experts, top, dtype, ld, needle):
    off = np.zeros(1026, np.int32)
    _refused(cq, cq.lib().cq_route(None, ld, dtype, tokens, experts, top, 1, None, None, off.ctypes.data, None, None,
                                   None, 0, None), needle)
    _refused(cq, cq.lib().cq_route(None, 8, 2, 0, 8, 2, 1, None, None, None, None, None, None, 0, None),
             "offsets must not be null")


@pytest.mark.parametrize("rows,tokens,top,dims,dtype,ld,needle", [
    (4, 2, 2, 8, 2, 8, "dtype must be f16 or bf16"),
    (-1, 2, 2, 8, 1, 8, "negative row count"),
    (4, 2, 0, 8, 1, 8, "top must be positive"),
    (4, 2, 2, 0, 1, 8, "invalid dims"),
    (4, 2, 2, 8, 1, 7, "row strides must be at least 8"),
    (4, 2, 2, 8, 1, 8, "must not be null"),
])
def test_combine_refusals(cq, rows, tokens, top, dims, dtype, ld, needle):
    _refused(cq, cq.lib().cq_expert_combine(None, ld, rows, None, None, tokens, top, dims, dtype, None, ld, None), needle)


def test_bindings_refuse_host_tensors(cq):
    import torch
    from nemotron_cuda import experts, fp8
    with pytest.raises(cq.CQError, match="on the device"):
        experts.route(torch.zeros(4, 8), 2)
    with pytest.raises(cq.CQError, match="on the device"):
        experts.combine(torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2))
    with pytest.raises(cq.CQError, match="on the device"):
        fp8.quantize_rows(torch.zeros(4, 8))
    with pytest.raises(cq.CQError, match="expected f16 or bf16"):
        experts.ExpertLinear.from_weight(torch.zeros(2, 4, 8))
    with pytest.raises(cq.CQError, match="expected \\(1, 1\\)"):
        fp8.Fp8Linear.from_codes(np.zeros((4, 8), np.uint8), np.zeros((2, 1), np.float32))
