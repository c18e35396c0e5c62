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


# ------------------------------------------------------------------ the 16-bit feed-forward module

def module16(gen, dtype, E, d, ff, out, bias=True):
    from nemotron_cuda import experts
    w1, w2 = (values(gen, E, n, k, dtype=dtype, spread=0.2) / k ** 0.5 for n, k in ((ff, d), (out, ff)))
    b1, b2 = (values(gen, E, n, dtype=dtype, spread=0.2) if bias else None for n in (ff, out))
    return (experts.ExpertLinear.from_weight(w1, b1), experts.ExpertLinear.from_weight(w2, b2)), (w1, w2, b1, b2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,E,top,d,ff,out,act", [
    (1, 8, 2, 792, 1567, 792, "silu"), (14, 4, 2, 128, 64, 72, "relu"), (60, 3, 3, 200, 333, 104, "none"),
    (300, 5, 2, 256, 1024, 256, "silu"), (900, 4, 2, 384, 2048, 512, "silu"), (3000, 3, 1, 136, 200, 1000, "relu")])
def test_h_keeps_more_than_its_type(cq, dtype, tokens, E, top, d, ff, out, act):
    """y is the definition's value rounded once.  h is held to 2^-17 (bf16) or 2^-22 (f16) of each value and the sums in f32
    lose less, so y before its rounding is off by a small part of a step and few of its values come out at the
    neighbour: their share is about twice that part, under 2^-6.  Bound: 2^-4.  With h rounded to T it would be near a half."""
    from nemotron_cuda import experts
    gen = rng_of("h", tokens, ff)
    (up, down), (w1, w2, b1, b2) = module16(gen, dtype, E, d, ff, out)
    x, z = values(gen, tokens, d, dtype=dtype, spread=0.3), torch.randn(tokens, E, device="cuda", generator=gen)
    y = experts.ExpertFeedForward(up, down, top=top, act=act).forward(x, z)
    expert, weight, offsets, token, position = eo.route(f64(z), top)
    h, _ = eo.experts(f64(x)[token], f64(w1), offsets, f64(b1), act)
    rows, _ = eo.experts(h, f64(w2), offsets, f64(b2))
    want, _ = eo.combine(rows, position, weight)
    want = torch.from_numpy(want).to(TYPES[dtype]).to("cuda")
    assert y.isfinite().all()
    assert (y != want).float().mean().item() <= 2.0 ** -4


def test_h_past_the_range_of_its_type(cq):
    """A value of h past f16's range is infinite, as a rounded one would be; the other tokens keep theirs."""
    from nemotron_cuda import experts
    up = experts.ExpertLinear.from_weight(torch.full((1, 1, 1), 300.0, dtype=torch.float16, device="cuda"))
    down = experts.ExpertLinear.from_weight(torch.full((1, 1, 1), 0.25, dtype=torch.float16, device="cuda"))
    x = torch.tensor([[2.0], [300.0], [-300.0], [1.5]], dtype=torch.float16, device="cuda")
    y = experts.ExpertFeedForward(up, down, top=1, act="none").forward(x, torch.zeros(4, 1, device="cuda"))
    assert y.flatten().tolist() == [150.0, float("inf"), -float("inf"), 112.5]


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("tokens", [6, 300])
def test_tokens_that_are_not_finite_stay_apart(cq, weights, tokens):
    """Infinities and NaN in one token reach no other: of the module, and of its first linear alone."""
    from nemotron_cuda import experts
    gen = rng_of("apart", tokens)
    E, d, ff = 4, 200, 328
    if weights == "16bit":
        (up, down), _ = module16(gen, "bf16", E, d, ff, d)
    else:
        up, down = (experts.ExpertLinear.from_codes(codes_of(gen, E, n, k), scales_of(gen, E, -(-n // 128), -(-k // 128)) / k ** 0.5)
                    for n, k in ((ff, d), (d, ff)))
    module = experts.ExpertFeedForward(up, down, top=2)
    x, z = values(gen, tokens, d, spread=0.3), torch.randn(tokens, E, device="cuda", generator=gen)
    r = experts.route(z, 2)
    clean, rows = module.forward(x, z), up.forward(x[r.token.long()], r.offsets, act="silu")
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    bad[1] = bad[4] = True
    x[1, 7], x[4, 3], x[4, 150] = float("inf"), float("nan"), -float("inf")
    y, y_rows = module.forward(x, z), up.forward(x[r.token.long()], r.offsets, act="silu")
    assert torch.equal(y[~bad], clean[~bad]) and not y[bad].isfinite().any(1).all()
    assert torch.equal(y_rows[~bad[r.token.long()]], rows[~bad[r.token.long()]])
    assert y_rows[r.token == 4].isnan().all()


# ------------------------------------------------------------------ refusals, each by its own message

def test_refusals_of_a_forward_call(cq):
    from nemotron_cuda import fp8
    f = fp8.Fp8Linear.from_codes(torch.zeros(8, 16, dtype=torch.uint8, device="cuda"), torch.ones(1, 1, device="cuda"))
    x, y = torch.zeros(40, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(40, 8, dtype=torch.bfloat16, device="cuda")
    L = cq.lib()
    need = L.cq_fp8_linear_workspace(f._h, 40)
    ws = torch.zeros(need + 512, dtype=torch.uint8, device="cuda")
    good = dict(x=x.data_ptr(), ldx=16, rows=40, y=y.data_ptr(), ldy=8, act=0, ws=ws.data_ptr(), n=need)
    for change, needle in ((dict(ws=None), "workspace has 0 bytes, expected"), (dict(n=need - 1), f"workspace has {need - 1} bytes, expected"),
                           (dict(ws=ws.data_ptr() + 16), "256-byte aligned"), (dict(act=3), "unknown activation 3"),
                           (dict(ldx=15), "input row stride 15"), (dict(ldy=7), "output row stride 7"),
                           (dict(rows=-1), "negative row count"), (dict(x=None), "must not be null"), (dict(y=None), "must not be null"),
                           (dict(x=x.data_ptr() + 1), "input must be aligned"), (dict(y=y.data_ptr() + 1), "output must be aligned")):
        a = good | change
        status = L.cq_fp8_linear_forward(f._h, a["x"], a["ldx"], a["rows"], a["y"], a["ldy"], a["act"], a["ws"], a["n"], None)
        assert status == cq.CQ_INVALID_ARGUMENT and needle in cq.last_error(), (change, cq.last_error())
    torch.cuda.synchronize()


def test_no_wait_ran_out(cq):
    assert cq.device_status(0) == 0
