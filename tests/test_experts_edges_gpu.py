"""The fp8 linear and the linears of experts on a B200 where their values leave the ordinary range."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import experts_oracle as eo
from test_experts_gpu import HALF_STEP, TYPES, codes_of, f64, offsets_of, rng_of, scales_of, values

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ SiLU

# around 0, past every cut of an exponent, and masks: the types' lowest values, infinities and NaN
SILU_AT = [0.0, 1.0, -1.0, 30.0, -30.0, -43.0, -44.0, -60.0, -80.0, -87.0, -89.0, -100.0, -1e3, -6e4, 6e4, float("nan"),
           float("inf"), -float("inf")]
SILU_AT_BF16 = SILU_AT + [-1e15, -1e20, -1e30, torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max]


def silu_bound(want, dtype):
    """The evaluation's error, derived: v log2 e is a rounded product of a rounded constant, off by 2^-23 of itself, so the
    power is off by 128 ln 2 2^-23 < 2^-16 of the value at most; flushed powers are under 2^-126, values under 2^-119.  Then
    half a step of T."""
    off = 2.0 ** -16 * np.abs(want) + 2.0 ** -119
    return off + HALF_STEP[dtype] * (np.abs(want) + off) + (2.0 ** -25 if dtype == "f16" else 0.0)


def check_silu(got, v, dtype):
    with np.errstate(over="ignore", invalid="ignore"):
        want = v / (1.0 + np.exp(-v))
    assert np.array_equal(np.isnan(got), np.isnan(want)), (v, got)
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= silu_bound(want[fine], dtype)).all(), list(zip(v, got, want))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 8, 24, 25, 130])
def test_silu_over_the_whole_range(cq, dtype, rows):
    """act(bias) where the products are zero, by few rows and by tiles, plain and grouped: a bound on SiLU itself."""
    from nemotron_cuda import experts, fp8
    at = torch.tensor(SILU_AT if dtype == "f16" else SILU_AT_BF16, dtype=TYPES[dtype], device="cuda")
    n = at.numel()
    x = torch.ones(rows, 128, dtype=TYPES[dtype], device="cuda")
    codes, scales = torch.zeros(1, n, 128, dtype=torch.uint8, device="cuda"), torch.ones(1, 1, 1, device="cuda")
    off = offsets_of([rows])
    for y in (fp8.Fp8Linear.from_codes(codes[0], scales[0], at, dtype=dtype).forward(x, act="silu"),
              experts.ExpertLinear.from_codes(codes, scales, at[None], dtype=dtype).forward(x, off, act="silu"),
              experts.ExpertLinear.from_weight(codes.to(TYPES[dtype]), at[None]).forward(x, off, act="silu")):
        assert y.shape == (rows, n)
        for r in (0, rows - 1):
            check_silu(f64(y[r]), f64(at), dtype)


@pytest.mark.parametrize("total", [-1e3, -1e20, -1e30])
@pytest.mark.parametrize("rows", [4, 40])
def test_silu_of_large_negative_sums(cq, rows, total):
    from nemotron_cuda import fp8
    x = torch.full((rows, 128), total / 128, dtype=torch.bfloat16, device="cuda")
    codes = torch.full((16, 128), 0x38, dtype=torch.uint8, device="cuda")  # 1.0
    y = fp8.Fp8Linear.from_codes(codes, torch.ones(1, 1, device="cuda")).forward(x, act="silu")
    assert (y == 0).all()


@pytest.mark.parametrize("tokens", [3, 200])
def test_a_masked_value_of_h_leaves_its_block(cq, tokens):
    """A bias at the type's lowest value inside the feed-forward module: that value of h is 0, and the other 127 of its
    e4m3 block keep their codes."""
    from nemotron_cuda import experts
    gen = rng_of("masked", tokens)
    E, n = 2, 256
    bias = values(gen, E, n, spread=0.2)
    bias[0, 3] = bias[1, 200] = torch.finfo(torch.bfloat16).min
    bias[0, 130] = -1e4
    up = experts.ExpertLinear.from_codes(torch.zeros(E, n, 128, dtype=torch.uint8, device="cuda"),
                                         torch.ones(E, 2, 1, device="cuda"), bias)
    eye = (torch.eye(n, device="cuda") * 0x38).to(torch.uint8).expand(E, n, n)
    down = experts.ExpertLinear.from_codes(eye, torch.ones(E, 2, 2, device="cuda"))
    x = torch.zeros(tokens, 128, dtype=torch.bfloat16, device="cuda")
    z = torch.zeros(tokens, E, device="cuda")
    z[torch.arange(tokens), torch.arange(tokens) % E] = 9.0
    y = f64(experts.ExpertFeedForward(up, down, top=1, act="silu").forward(x, z))
    b = f64(bias)
    with np.errstate(over="ignore"):
        h = b / (1.0 + np.exp(-b))
    # half a step of e4m3, and half of its smallest steps times the block's scale
    scale = np.repeat(np.stack([[eo.scale_of(r[:128]), eo.scale_of(r[128:])] for r in h]), 128, axis=1)
    bound = (2.0 ** -4 + 2.0 ** -10) * np.abs(h) + scale * 2.0 ** -10 * (1 + 2.0 ** -10)
    for t in range(tokens):
        assert (np.abs(y[t] - h[t % E]) <= bound[t % E]).all()
