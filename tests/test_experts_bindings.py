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
