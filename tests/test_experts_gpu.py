"""The fp8 linear, the linears of experts, the router and their feed-forward module on a B200 against the 64-bit
oracle, over the sizes, strides and masks where they can go wrong.

Tolerance of a product, element by element, derived: the kernels sum K products in f32.  Whatever the order, and even
where each addition drops bits instead of rounding, K additions and a few scalings lose at most (K + 8) 2^-23 of the
sum of magnitudes; an activation's slope is at most 1.1; its evaluation loses 2^-18 of the value; the rounding to T
half a step of T.  Codes are exact: they are compared bit for bit.
"""
from __future__ import annotations

import zlib

import numpy as np
import pytest
import torch

import experts_oracle as eo

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"bf16": 2.0 ** -126, "f16": 2.0 ** -24}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def close(got, want, mags, k, dtype, what=""):
    got = got.double().cpu().numpy()
    bound = 1.1 * (k + 8) * 2.0 ** -23 * mags + 2.0 ** -18 * np.abs(want)
    bound = bound + HALF_STEP[dtype] * (np.abs(want) + bound) + TINY[dtype]
    off = np.abs(got - want) / bound
    assert np.isfinite(got).all(), what
    assert off.max(initial=0.0) <= 1.0, f"{what}: {off.max():.3g} of the bound at {np.unravel_index(off.argmax(), off.shape)}"


def rng_of(*seed):
    return torch.Generator("cuda").manual_seed(zlib.crc32(repr(seed).encode()))


def values(gen, *shape, dtype="bf16", spread=1.0):
    v = torch.randn(*shape, device="cuda", generator=gen) * torch.exp(spread * torch.randn(shape[-1], device="cuda", generator=gen))
    return v.to(TYPES[dtype])


def codes_of(gen, *shape):
    """Random finite e4m3 codes."""
    c = torch.randint(0, 256, shape, device="cuda", generator=gen, dtype=torch.uint8)
    return torch.where((c & 0x7F) == 0x7F, c & 0x87, c)


def scales_of(gen, *shape):
    return torch.exp(torch.randn(*shape, device="cuda", generator=gen)) / 400.0


def f64(t):
    return t.double().cpu().numpy()


def row_values(x):
    """What the rows' e4m3 codes stand for, by the oracle."""
    return eo.spread_rows(*eo.quantize_rows(f64(x)))


def weight_values(codes, scales):
    return eo.spread_weight(eo.decode(codes.cpu().numpy()), f64(scales))


def strided(t, extra):
    """The same rows with `extra` unused values behind each, and the first shifted by as many."""
    if not extra:
        return t
    big = torch.full((t.shape[0] + 1, t.shape[1] + extra), float("nan"), dtype=t.dtype, device=t.device).flatten()
    view = big[extra:].as_strided(t.shape, (t.shape[1] + extra, 1))
    view.copy_(t)
    return view


# ------------------------------------------------------------------ rows and weights to e4m3

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,extra", [(1, 1, 0), (1, 128, 0), (3, 127, 0), (5, 129, 3), (14, 1024, 0), (33, 520, 8),
                                          (300, 4096, 0), (2, 16, 1)])
def test_quantize_rows_bit_for_bit(cq, dtype, rows, k, extra):
    from nemotron_cuda import fp8
    gen = rng_of(rows, k)
    x = values(gen, rows, k, dtype=dtype, spread=2.0)
    x[torch.rand(rows, k, device="cuda", generator=gen) < 0.1] = 0.0
    if rows > 2:
        x[1] = 0.0                      # a row of zeros
        x[2, : min(k, 7)] *= 2.0 ** -10   # next to the format's smallest steps
    codes, scales = fp8.quantize_rows(strided(x, extra))
    want, want_scales = eo.quantize_rows(f64(x))
    raw = codes.view(torch.uint8).cpu().numpy()
    assert np.array_equal(f64(scales), want_scales)
    assert np.array_equal(eo.decode(raw[:, :k]), want)
    assert not raw[:, k:].any()


def test_quantize_rows_of_every_bf16_value(cq):
    """All finite bf16 values next to 448 (scale 1), 2^120 and the smallest normal: ties, subnormal codes, underflow."""
    from nemotron_cuda import fp8
    every = torch.arange(0, 0x7F80, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    for top in (448.0, 2.0 ** 120, 2.0 ** -120, 3.0e38):
        low = every[every.float() <= top]
        x = torch.zeros(-(-low.numel() // 127), 128, dtype=torch.bfloat16, device="cuda")
        x[:, 0] = top
        x[:, 1:].flatten()[: low.numel()] = 0  # shape check only
        flat = torch.zeros(x.shape[0] * 127, dtype=torch.bfloat16, device="cuda")
        flat[: low.numel()] = low
        x[:, 1:] = flat.view(-1, 127)
        x[1::2] *= -1
        codes, scales = fp8.quantize_rows(x)
        want, want_scales = eo.quantize_rows(f64(x))
        assert np.array_equal(f64(scales), want_scales)
        assert np.array_equal(eo.decode(codes.view(torch.uint8).cpu().numpy()), want)


def test_quantize_rows_marks_what_is_not_finite(cq):
    from nemotron_cuda import fp8
    x = torch.ones(3, 256, dtype=torch.bfloat16, device="cuda")
    x[0, 5], x[1, 130], x[2, 0] = float("inf"), float("nan"), -float("inf")
    codes, scales = fp8.quantize_rows(x)
    v = eo.decode(codes.view(torch.uint8).cpu().numpy())
    bad = np.zeros((3, 256), bool)
    bad[0, 5] = bad[1, 130] = bad[2, 0] = True
    assert np.array_equal(np.isnan(v), bad)
    assert (v[~bad] == 256.0).all() and (f64(scales) == 2.0 ** -8).all()


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (1025, 640), (7, 300)])
def test_quantize_weight_bit_for_bit(cq, n, k):
    from nemotron_cuda import fp8
    w = values(rng_of(n, k), n, k, dtype="f32")
    codes, scales = fp8.quantize_weight(w)
    want, want_scales = eo.quantize_weight(f64(w))
    assert np.array_equal(f64(scales), want_scales)
    assert np.array_equal(eo.decode(codes.view(torch.uint8).cpu().numpy()), want)


# ------------------------------------------------------------------ fp8 linear

FP8_SIZES = [(1, 1, 1), (1, 4096, 1024), (2, 130, 127), (7, 64, 128), (8, 1024, 4096), (9, 16, 129), (14, 4096, 1024),
             (16, 1025, 640), (17, 1000, 1000), (31, 256, 2048), (33, 257, 520), (64, 512, 1024), (65, 1024, 4096),
             (128, 128, 256), (129, 640, 384), (200, 2048, 1024), (333, 1025, 640), (600, 1024, 1024), (896, 1024, 512)]


@pytest.mark.parametrize("rows,n,k", FP8_SIZES)
def test_fp8_linear(cq, rows, n, k):
    from nemotron_cuda import fp8
    gen = rng_of(rows, n, k)
    dtype = "bf16" if (rows + n) % 2 else "f16"
    act = ("none", "silu", "relu")[(rows + n + k) % 3]
    x = values(gen, rows, k, dtype=dtype, spread=0.5)
    codes, scales = codes_of(gen, n, k), scales_of(gen, -(-n // 128), -(-k // 128)) / k ** 0.5
    bias = values(gen, n, dtype=dtype) if k % 2 == 0 else None
    layer = fp8.Fp8Linear.from_codes(codes, scales, bias, dtype=dtype)
    y = layer.forward(x, act=act)
    want, mags = eo.linear(row_values(x), weight_values(codes, scales), None if bias is None else f64(bias), act)
    close(y, want, mags, k, dtype)
    # the same from rows brought to e4m3 beforehand, bit for bit
    assert torch.equal(layer.forward_codes(*fp8.quantize_rows(x), act=act), y)
    # again, and on strided rows of any alignment: the same bits
    assert torch.equal(layer.forward(x, act=act), y)
    for extra in (1, 8):
        out = strided(torch.zeros_like(y), extra)
        layer.forward(strided(x, extra), y=out, act=act)
        assert torch.equal(out, y)


def test_fp8_linear_from_f32(cq):
    from nemotron_cuda import fp8
    gen = rng_of(3)
    w, b, x = values(gen, 300, 200, dtype="f32", spread=0.3), values(gen, 300, dtype="f32"), values(gen, 20, 200)
    layer = fp8.Fp8Linear.from_f32(w, b, dtype="bf16")
    host = fp8.Fp8Linear.from_f32(w.cpu().numpy(), b.cpu().numpy(), dtype="bf16")
    y = layer.forward(x)
    want, mags = eo.linear(row_values(x), eo.spread_weight(*eo.quantize_weight(f64(w))), f64(b.to(torch.bfloat16)))
    close(y, want, mags, 200, "bf16")
    assert torch.equal(host.forward(x), y)


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_fp8_linear_keeps_rows_apart(cq, rows):
    """A row with an infinity, a NaN or nothing but zeros changes no other row; zero rows give act(bias)."""
    from nemotron_cuda import fp8
    gen = rng_of(rows, 5)
    codes, scales, bias = codes_of(gen, 384, 640), scales_of(gen, 3, 5), values(gen, 384)
    layer = fp8.Fp8Linear.from_codes(codes, scales, bias)
    x = values(gen, rows, 640)
    clean = layer.forward(x)
    x[0, 3], x[rows - 1] = float("inf"), 0.0
    y = layer.forward(x)
    assert y[0].isnan().all()
    assert torch.equal(y[1:-1], clean[1:-1])
    assert torch.equal(y[-1], bias)


def test_fp8_linear_large_sums_and_scales(cq):
    """Long sums of one sign: every partial sum is held in f32."""
    from nemotron_cuda import fp8
    for rows in (4, 200):
        x = torch.full((rows, 8192), 1.0, dtype=torch.bfloat16, device="cuda")
        codes = torch.full((64, 8192), 0x38, dtype=torch.uint8, device="cuda")  # 1.0
        scales = torch.full((1, 64), 2.0 ** -20, device="cuda")
        scales[0, 0] = 2.0 ** 6
        y = fp8.Fp8Linear.from_codes(codes, scales).forward(x)
        want = 128 * 2.0 ** 6 + 8064 * 2.0 ** -20
        assert (y.float() == torch.tensor(want).to(torch.bfloat16).float()).all()


# ------------------------------------------------------------------ linears of experts

def offsets_of(counts, device="cuda"):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=device)


GROUPS = {
    "one row": [0, 0, 1, 0],
    "single expert": [37],
    "first empty": [0, 3, 0, 2],
    "last empty": [5, 1, 0, 0],
    "none": [0, 0, 0],
    "even": [8] * 6,
    "one has most": [1, 250, 0, 2, 9],
    "tile edges": [128, 1, 127, 129, 0, 64, 256],
    "many": [(7 * i) % 11 for i in range(70)],
    "sixteen or less": [16, 15, 0, 1, 9, 8, 7],
    "large": [300, 517, 3, 200],
}


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("n,k", [(256, 128), (200, 520), (1025, 333)])
def test_expert_linear(cq, weights, name, n, k):
    from nemotron_cuda import experts
    counts = GROUPS[name]
    gen = rng_of(name, n, k)
    dtype = "bf16" if n % 2 == 0 else "f16"
    act = ("none", "silu", "relu")[len(counts) % 3]
    E, tail = len(counts), 5 if n == 200 else 0
    rows = sum(counts) + tail
    x, off = values(gen, rows, k, dtype=dtype, spread=0.5), offsets_of(counts)
    bias = values(gen, E, n, dtype=dtype) if n != 256 else None
    b64 = None if bias is None else f64(bias)
    if weights == "e4m3":
        codes, scales = codes_of(gen, E, n, k), scales_of(gen, E, -(-n // 128), -(-k // 128)) / k ** 0.5
        layer = experts.ExpertLinear.from_codes(codes, scales, bias, dtype=dtype)
        w = np.stack([weight_values(codes[e], scales[e]) for e in range(E)])
        x64 = row_values(x) if rows else f64(x)
    else:
        weight = values(gen, E, n, k, dtype=dtype, spread=0.2) / k ** 0.5
        layer = experts.ExpertLinear.from_weight(weight, bias)
        w, x64 = f64(weight), f64(x)
    x[rows - tail:] = float("nan")  # rows of no expert are not looked at
    y = torch.full((rows, n), float("nan"), dtype=TYPES[dtype], device="cuda")
    layer.forward(x, off, y=y, act=act)
    want, mags = eo.experts(x64, w, off.cpu().numpy(), b64, act)
    close(y, want, mags, k, dtype, name)
    assert not y[rows - tail:].any()
    for extra in (1, 8):
        out = strided(torch.zeros_like(y), extra)
        layer.forward(strided(x, extra), off, y=out, act=act)
        assert torch.equal(out, y)


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("experts,counts,n,k", [(40, 3, 2048, 1024), (40, 3, 1024, 1400), (24, 70, 1024, 640), (30, 40, 512, 2048),
                                               (4, 700, 1024, 384), (6, 400, 2048, 512)])
def test_expert_linear_many_tiles(cq, weights, experts, counts, n, k):
    """Several tiles a CTA, of every width: the rings of copies, sums and scales go on from tile to tile."""
    from nemotron_cuda import experts as ex
    gen = rng_of(experts, counts, n, k)
    sizes = [counts + (i * 7) % 5 - 2 for i in range(experts)]
    x, off = values(gen, sum(sizes), k, spread=0.3), offsets_of(sizes)
    if weights == "e4m3":
        codes, scales = codes_of(gen, experts, n, k), scales_of(gen, experts, -(-n // 128), -(-k // 128)) / k ** 0.5
        layer = ex.ExpertLinear.from_codes(codes, scales)
        w, x64 = np.stack([weight_values(codes[e], scales[e]) for e in range(experts)]), row_values(x)
    else:
        weight = values(gen, experts, n, k, spread=0.2) / k ** 0.5
        layer = ex.ExpertLinear.from_weight(weight)
        w, x64 = f64(weight), f64(x)
    y = layer.forward(x, off, act="silu")
    want, mags = eo.experts(x64, w, off.cpu().numpy(), None, "silu")
    close(y, want, mags, k, "bf16")
    assert torch.equal(layer.forward(x, off, act="silu"), y)


@pytest.mark.parametrize("rows,n,k", [(300, 8192, 512), (2500, 2048, 640), (700, 4096, 1152)])
def test_fp8_linear_many_tiles(cq, rows, n, k):
    from nemotron_cuda import fp8
    gen = rng_of(rows, n, k)
    x, codes, scales = values(gen, rows, k, spread=0.3), codes_of(gen, n, k), scales_of(gen, -(-n // 128), -(-k // 128)) / k ** 0.5
    layer = fp8.Fp8Linear.from_codes(codes, scales)
    y = layer.forward(x)
    want, mags = eo.linear(row_values(x), weight_values(codes, scales))
    close(y, want, mags, k, "bf16")
    assert torch.equal(layer.forward(x), y)


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("rows", [6, 200])
def test_expert_linear_survives_wrong_offsets(cq, weights, rows):
    """Offsets outside the rows, or falling, are cut to the rows: no access out of range, good groups keep their values."""
    from nemotron_cuda import experts
    gen = rng_of(rows)
    x = values(gen, rows, 128)
    if weights == "e4m3":
        layer = experts.ExpertLinear.from_codes(codes_of(gen, 4, 128, 128), scales_of(gen, 4, 1, 1))
    else:
        layer = experts.ExpertLinear.from_weight(values(gen, 4, 128, 128))
    good = layer.forward(x, offsets_of([2, 1, rows - 3, 0]))
    bad = layer.forward(x, torch.tensor([0, 2, 3, 1 << 30, -5], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(bad, good)
    fall = layer.forward(x, torch.tensor([0, 2, 1, -1, 2], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(fall[:2], good[:2]) and not fall[2:].any()


def test_expert_linear_refusals(cq):
    from nemotron_cuda import experts, fp8
    layer = experts.ExpertLinear.from_weight(torch.zeros(2, 8, 16, dtype=torch.bfloat16, device="cuda"))
    x, off = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda"), offsets_of([2, 2])
    for bad, needle in ((lambda: layer.forward(x.half(), off), "expected torch.bfloat16"),
                        (lambda: layer.forward(x[:, :8], off), "rows of 16 values"),
                        (lambda: layer.forward(x.t().contiguous().t(), off), "rows of 16 values"),
                        (lambda: layer.forward(x, off.long()), "offsets must be int32"),
                        (lambda: layer.forward(x, off[:2]), "offsets must be int32"),
                        (lambda: layer.forward(x, off.cpu()), "offsets must be int32"),
                        (lambda: layer.forward(x, off, y=torch.zeros(4, 7, dtype=torch.bfloat16, device="cuda")), "rows of 8")):
        with pytest.raises(cq.CQError, match=needle):
            bad()
    f = fp8.Fp8Linear.from_codes(torch.zeros(8, 16, dtype=torch.uint8, device="cuda"), torch.ones(1, 1, device="cuda"))
    x, y = torch.zeros(40, 16, dtype=torch.bfloat16, device="cuda"), torch.zeros(40, 8, dtype=torch.bfloat16, device="cuda")
    L = cq.lib()
    need = L.cq_fp8_linear_workspace(f._h, 40)
    assert L.cq_fp8_linear_workspace(f._h, 0) == 0 and need > 0
    ws = torch.zeros(need + 512, dtype=torch.uint8, device="cuda")

    def call(ptr, n, act=0, ldx=16, ldy=8):
        return L.cq_fp8_linear_forward(f._h, x.data_ptr(), ldx, 40, y.data_ptr(), ldy, act, ptr, n, None)
    for status, needle in ((call(None, need), "workspace has 0 bytes"), (call(ws.data_ptr(), need - 1), "expected"),
                           (call(ws.data_ptr() + 16, need), "256-byte aligned"), (call(ws.data_ptr(), need, act=3), "unknown activation"),
                           (call(ws.data_ptr(), need, ldx=15), "input row stride"), (call(ws.data_ptr(), need, ldy=7), "output row stride")):
        assert status == cq.CQ_INVALID_ARGUMENT
    assert call(ws.data_ptr(), need) == cq.CQ_OK
    assert L.cq_fp8_linear_forward(f._h, None, 16, 0, None, 8, 0, None, 0, None) == cq.CQ_OK  # no rows


# ------------------------------------------------------------------ router and combine

def check_route(r, logits, top, renormalize):
    expert, weight, offsets, token, position = eo.route(f64(logits), top, renormalize)
    assert np.array_equal(r.expert.cpu().numpy(), expert)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets)
    assert np.array_equal(r.token.cpu().numpy(), token)
    assert np.array_equal(r.position.cpu().numpy(), position)
    # exp and a sum of up to `experts` terms in f32, one division: 2^-23 for each of log2-many or sequential roundings
    assert np.abs(f64(r.weight) - weight).max(initial=0.0) <= (logits.shape[1] + 16) * 2.0 ** -23


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,n,top", [(1, 1, 1), (1, 8, 2), (14, 8, 2), (127, 33, 4), (128, 32, 8), (129, 5, 5),
                                          (300, 128, 8), (1000, 200, 3), (40, 600, 32), (300, 1024, 6)])
def test_route(cq, dtype, tokens, n, top):
    from nemotron_cuda import experts
    gen = rng_of(tokens, n)
    z = (torch.randn(tokens, n, device="cuda", generator=gen) * 2).to(TYPES[dtype])
    for renormalize in (True, False):
        check_route(experts.route(z, top, renormalize=renormalize), z, top, renormalize)
    wide = torch.full((tokens, n + 3), 99.0, dtype=z.dtype, device="cuda")
    wide[:, 1:n + 1] = z
    check_route(experts.route(wide[:, 1:n + 1], top), z, top, True)


@pytest.mark.parametrize("tokens", [9, 400])
def test_route_masks_and_ties(cq, tokens):
    from nemotron_cuda import experts
    z = torch.randint(0, 3, (tokens, 40), device="cuda", generator=rng_of(1)).float()  # many ties
    inf = float("inf")
    z[0] = -inf
    z[1, 4:] = -inf
    z[2] = torch.finfo(torch.float32).min
    z[3, ::2] = float("nan")
    z[4, 7], z[4, 9] = inf, inf
    z[5] = -0.0
    z[5, ::3] = 0.0
    z[6, 1:] = -inf
    for renormalize in (True, False):
        check_route(experts.route(z, 6, renormalize=renormalize), z, 6, renormalize)
    none = torch.full((tokens, 7), -inf, device="cuda")
    check_route(experts.route(none, 3), none, 3, True)


def test_route_of_no_tokens(cq):
    from nemotron_cuda import experts
    r = experts.route(torch.zeros(0, 8, device="cuda"), 2)
    assert r.offsets.tolist() == [0] * 9 and r.token.numel() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,top,dims,extra", [(1, 1, 1, 0), (14, 2, 1024, 0), (33, 3, 1001, 0), (300, 8, 520, 4), (65, 4, 64, 8)])
def test_combine(cq, dtype, tokens, top, dims, extra):
    from nemotron_cuda import experts
    gen = rng_of(tokens, dims)
    z = values(gen, tokens * top, dims, dtype=dtype)
    position = torch.randperm(tokens * top, device="cuda", generator=gen).to(torch.int32).view(tokens, top)
    if tokens > 2:
        position[1], position[2, 0] = -1, tokens * top  # a token without experts; a position past the rows
    weight = torch.rand(tokens, top, device="cuda", generator=gen)
    y = experts.combine(strided(z, extra), position, weight)
    want, mags = eo.combine(f64(z), position.cpu().numpy(), f64(weight))
    close(y, want, mags, top, dtype)
    out = strided(torch.zeros_like(y), extra)
    assert torch.equal(experts.combine(z, position, weight, y=out), y)


# ------------------------------------------------------------------ the feed-forward module

def ffn_case(gen, weights, dtype, E, d, ff, tokens):
    from nemotron_cuda import experts
    x = values(gen, tokens, d, dtype=dtype, spread=0.3)
    layers, dense = [], []
    for n, k in ((ff, d), (d, ff)):
        if weights == "e4m3":
            codes, scales = codes_of(gen, E, n, k), scales_of(gen, E, -(-n // 128), -(-k // 128)) / k ** 0.5 / 20
            layers.append(experts.ExpertLinear.from_codes(codes, scales, dtype=dtype))
            dense.append(np.stack([weight_values(codes[e], scales[e]) for e in range(E)]))
        else:
            w = values(gen, E, n, k, dtype=dtype, spread=0.2) / k ** 0.5
            layers.append(experts.ExpertLinear.from_weight(w))
            dense.append(f64(w))
    return x, layers, dense


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,E,top,d,ff", [(1, 4, 2, 128, 256), (14, 8, 2, 256, 1024), (33, 3, 3, 200, 333),
                                               (130, 8, 2, 256, 520), (700, 5, 2, 384, 640), (900, 40, 2, 512, 1024)])
def test_expert_feed_forward(cq, weights, dtype, tokens, E, top, d, ff):
    """Against the definition, by the 2-norm.  Beyond the roundings of z and y to T (and of h with 16-bit weights), each
    2^-9 (bf16) or 2^-12 (f16) in the mean, an f32 difference may bring a value of h to the next e4m3 code: a share of
    at most 3e-4 of the values, by 2^-3 of the value each, 2.2e-3 of the norm."""
    from nemotron_cuda import experts
    gen = rng_of(tokens, E, d)
    x, (up, down), (w1, w2) = ffn_case(gen, weights, dtype, E, d, ff, tokens)
    z = torch.randn(tokens, E, device="cuda", generator=gen)
    if tokens > 5:
        z[3] = -float("inf")
    y = experts.ExpertFeedForward(up, down, top=top, act="silu").forward(x, z)
    expert, weight, offsets, token, position = eo.route(f64(z), top)
    live = offsets[-1]
    rows = np.zeros((tokens * top, d))
    rows[:live] = f64(x)[token[:live]]
    through = (lambda v: eo.spread_rows(*eo.quantize_rows(v))) if weights == "e4m3" else (lambda v: v)
    h, _ = eo.experts(through(rows), w1, offsets, act="silu")
    if weights == "16bit":
        h = f64(torch.from_numpy(h).to(TYPES[dtype]))
    out, _ = eo.experts(through(h), w2, offsets)
    want, _ = eo.combine(out, position, weight)
    got = f64(y)
    assert np.isfinite(got).all()
    if tokens > 5:
        assert not got[3].any()
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= {"bf16": 4e-3, "f16": 3e-3 if weights == "e4m3" else 1e-3}[dtype], rel


def test_feed_forward_refuses_a_pair_that_does_not_fit(cq):
    from nemotron_cuda import experts
    def layer(e, n, k, dtype=torch.bfloat16):
        return experts.ExpertLinear.from_weight(torch.zeros(e, n, k, dtype=dtype, device="cuda"))
    up = layer(4, 32, 16)
    for down, needle in ((layer(3, 16, 32), "must agree"), (layer(4, 16, 24), "takes 24 values"),
                         (layer(4, 16, 32, torch.float16), "must agree")):
        with pytest.raises(cq.CQError, match=needle):
            experts.ExpertFeedForward(up, down, top=2)
    with pytest.raises(cq.CQError, match="top must be"):
        experts.ExpertFeedForward(up, layer(4, 16, 32), top=5)


# ------------------------------------------------------------------ streams and graphs

def test_calls_on_other_streams_and_in_a_graph(cq):
    from nemotron_cuda import experts
    gen = rng_of(11)
    results = {}
    for tokens in (14, 300):
        x, (up, down), _ = ffn_case(gen, "e4m3", "bf16", 8, 256, 512, tokens)
        z = torch.randn(tokens, 8, device="cuda", generator=gen)
        ffn = experts.ExpertFeedForward(up, down, top=2)
        want = ffn.forward(x, z)
        torch.cuda.synchronize()
        # one layer on several streams at once, each call with its own workspace
        streams = [torch.cuda.Stream() for _ in range(3)]
        got = [ffn.forward(x, z, stream=s) for s in streams for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
        results[tokens] = want
        # captured, replayed on new inputs in place
        out, s = torch.empty_like(want), torch.cuda.Stream()
        with torch.cuda.stream(s):
            ffn.forward(x, z, y=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            ffn.forward(x, z, y=out)
        out.zero_()
        x2, z2 = x.clone().mul_(0.5), z.flip(0)
        want2 = ffn.forward(x2, z2)
        x.copy_(x2)
        z.copy_(z2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want2)


def test_no_wait_ran_out(cq):
    assert cq.device_status(0) == 0


@pytest.mark.parametrize("weights", ["16bit", "e4m3"])
@pytest.mark.parametrize("rows", [1, 7, 32, 33])
def test_expert_linear_of_one_expert(cq, weights, rows):
    """One expert and few rows: the call says what workspace it needs, and refuses less."""
    from nemotron_cuda import experts
    gen = rng_of("one", weights, rows)
    n, k = 200, 136
    x, off = values(gen, rows, k), offsets_of([rows])
    if weights == "e4m3":
        codes, scales = codes_of(gen, 1, n, k), scales_of(gen, 1, 2, 2)
        layer = experts.ExpertLinear.from_codes(codes, scales)
        w, x64 = weight_values(codes[0], scales[0])[None], row_values(x)
    else:
        weight = values(gen, 1, n, k)
        layer = experts.ExpertLinear.from_weight(weight)
        w, x64 = f64(weight), f64(x)
    need = cq.lib().cq_expert_linear_workspace(layer._h, rows)
    assert need >= rows * k
    y = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
    assert cq.lib().cq_expert_linear_forward(layer._h, x.data_ptr(), k, rows, off.data_ptr(), y.data_ptr(), n, 0, None, 0,
                                             None) == cq.CQ_INVALID_ARGUMENT
    layer.forward(x, off, y=y)
    want, mags = eo.experts(x64, w, off.cpu().numpy(), None, "none")
    close(y, want, mags, k, "bf16")
