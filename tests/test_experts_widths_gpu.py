"""The grouped product and the feed-forward module on a B200 in every tile width, at the sizes of expert_plan.py, against the
definitions in 64 bits (torch, on the device).  Tolerances are those of test_experts_gpu.py, derived there."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import expert_plan as ep
import experts_oracle as eo
from test_experts_gpu import HALF_STEP, TINY, TYPES, codes_of, f64, rng_of, scales_of, values

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def e4m3_rows(x):
    """What rows' e4m3 codes stand for, [rows, k] in 64 bits."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 128)).view(rows, -1, 128)
    top = b.abs().amax(2, keepdim=True)
    fraction, exponent = torch.frexp(top)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), (exponent - 9 + (fraction > 0.875).int()).clamp(min=-126)), 1.0)
    v = b / scale
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 4).clamp(min=-9))
    return (torch.round(v / step) * step * scale).view(rows, -1)[:, :k], scale.expand_as(b).reshape(rows, -1)[:, :k]


def activate(v, act):
    return v / (1.0 + torch.exp(-v)) if act == "silu" else v.clamp(min=0.0) if act == "relu" else v


class Layer:
    """An expert linear and its weights in 64 bits."""

    def __init__(self, gen, weights, E, n, k, bias, dtype, identity=False):
        from nemotron_cuda import experts
        b = values(gen, E, n, dtype=dtype, spread=0.2) if bias else None
        if identity:
            one = torch.eye(n, device="cuda").expand(E, n, n).contiguous()
        if weights == "e4m3":
            codes = (one * 0x38).to(torch.uint8) if identity else codes_of(gen, E, n, k)
            blocks = (E, -(-n // 128), -(-k // 128))
            scales = torch.ones(blocks, device="cuda") if identity else scales_of(gen, *blocks) / k ** 0.5
            self.own = experts.ExpertLinear.from_codes(codes, scales, b, dtype=dtype)
            full = scales.repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
            self.w = codes.view(torch.float8_e4m3fn).double() * full
        else:
            w = one.to(TYPES[dtype]) if identity else values(gen, E, n, k, dtype=dtype, spread=0.2) / k ** 0.5
            self.own = experts.ExpertLinear.from_weight(w, b)
            self.w = w.double()
        self.bias, self.weights = b, weights

    def exact(self, x, offsets, act):
        """(act(W x + b), sums of magnitudes) for rows of no rounding; x as the values that it stands for."""
        y = torch.zeros(x.shape[0], self.w.shape[1], dtype=torch.float64, device="cuda")
        mags = torch.zeros_like(y)
        for e, (i, j) in enumerate(zip(offsets[:-1], offsets[1:])):
            v, m = x[i:j] @ self.w[e].T, x[i:j].abs() @ self.w[e].T.abs()
            if self.bias is not None:
                v, m = v + self.bias[e].double(), m + self.bias[e].double().abs()
            y[i:j], mags[i:j] = activate(v, act), m
        return y, mags


def assert_close(got, want, mags, k, dtype):
    """Element by element: (k + 8) 2^-23 of the sum of magnitudes, 2^-16 of the value for the activation, half a step of T."""
    bound = 1.1 * (k + 8) * 2.0 ** -23 * mags + 2.0 ** -16 * want.abs()
    bound = bound + HALF_STEP[dtype] * (want.abs() + bound) + TINY[dtype]
    off = ((got.double() - want).abs() / bound).max().item()
    assert got.isfinite().all() and off <= 1.0, f"{off:.3g} of the bound"


@pytest.mark.parametrize("weights,rows,E,n,k,act,bias,dtype,width", ep.PRODUCTS)
def test_products(cq, weights, rows, E, n, k, act, bias, dtype, width):
    assert ep.product_width(weights, rows, E, n, k, act, sms()) == width
    gen = rng_of(rows, E, n, k)
    layer = Layer(gen, weights, E, n, k, bias, dtype)
    x = values(gen, rows, k, dtype=dtype, spread=0.5)
    off = np.concatenate([[0], np.cumsum(ep.ragged(rows, E))])
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    y = layer.own.forward(x, offsets, act=act)
    want, mags = layer.exact(e4m3_rows(x)[0] if weights == "e4m3" else x.double(), off.tolist(), act)
    assert_close(y, want, mags, k, dtype)
    # rows of y that no tile store takes, and again: the same bits
    out = torch.full((rows, n + 1), float("nan"), dtype=TYPES[dtype], device="cuda")[:, :n]
    assert torch.equal(layer.own.forward(x, offsets, y=out, act=act), y)


@pytest.mark.parametrize("weights,tokens,E,top,d,ff,out,act,bias,renormalize,logits,dtype,up_width,down_width", ep.MODULES)
def test_modules(cq, weights, tokens, E, top, d, ff, out, act, bias, renormalize, logits, dtype, up_width, down_width):
    """16-bit: at most one value in sixteen differs from the definition's rounded once (an f32 difference next to a
    boundary).  e4m3: by the 2-norm, where a value of h next to a boundary may come to the neighbouring code: a share of at most
    3e-4 of the values by 2^-3 each, 2.2e-3 of the norm, next to 1.7e-3 (bf16) or 2.1e-4 (f16) of rounding y."""
    from nemotron_cuda import experts
    assert ep.module_widths(weights, tokens * top, E, d, ff, out, act, sms()) == (up_width, down_width)
    gen = rng_of(tokens, E, ff, out)
    up, down = Layer(gen, weights, E, ff, d, bias, dtype), Layer(gen, weights, E, out, ff, bias, dtype)
    x = values(gen, tokens, d, dtype=dtype, spread=0.3)
    z = (torch.randn(tokens, E, device="cuda", generator=gen) * 2).to(TYPES[logits])
    z[5], z[7, 1:] = -float("inf"), -float("inf")
    # rows wider than the module's, of x, logits and y
    wide = torch.cat([x, torch.full((tokens, 3), float("nan"), dtype=x.dtype, device="cuda")], 1)[:, :d]
    wide_z = torch.cat([z, torch.full((tokens, 1), 99.0, dtype=z.dtype, device="cuda")], 1)[:, :E]
    y = torch.full((tokens, out + 5), float("nan"), dtype=x.dtype, device="cuda")[:, :out]
    module = experts.ExpertFeedForward(up.own, down.own, top, act=act, renormalize=renormalize)
    module.forward(wide, wide_z, y=y)
    expert, weight, offsets, token, position = eo.route(f64(z), top, renormalize)
    live = int(offsets[-1])
    rows = x.double()[torch.from_numpy(token[:live]).to("cuda")]
    through = (lambda v: e4m3_rows(v)[0]) if weights == "e4m3" else (lambda v: v)
    h, _ = up.exact(through(rows), offsets.tolist(), act)
    r, _ = down.exact(through(h), offsets.tolist(), "none")
    r = torch.cat([r, r.new_zeros(1, out)])
    at = torch.from_numpy(np.where(position < 0, live, position)).to("cuda")
    want = (r[at] * torch.from_numpy(weight).to("cuda")[:, :, None]).sum(1)
    # (a softmax over all experts may add them up in another order where logits can be loaded at once)
    for got in (y, module.forward(x, z)):
        assert got.isfinite().all() and not got[5].any()
        if weights == "16bit":
            assert (got != want.to(got.dtype)).float().mean().item() <= 2.0 ** -4
        else:
            rel = ((got.double() - want).norm() / want.norm()).item()
            assert rel <= {"bf16": 4e-3, "f16": 3e-3}[dtype], rel


@pytest.mark.parametrize("weights,tokens,E,d,ff,act,up_width,down_width", ep.KEPT)
def test_h_as_it_is_kept(cq, weights, tokens, E, d, ff, act, up_width, down_width):
    """The second linear is the identity, so that y is h as the module kept it, element by element: e4m3 within half a step of
    a code (and half of the smallest step, of a scale that a difference of f32 may have doubled), 16-bit within the bound of
    a product.  Beyond that y's own rounding, which loses nothing of a code."""
    from nemotron_cuda import experts
    assert ep.module_widths(weights, tokens, E, d, ff, ff, act, sms()) == (up_width, down_width)
    gen = rng_of("kept", tokens, E, ff)
    up, down = Layer(gen, weights, E, ff, d, True, "bf16"), Layer(gen, weights, E, ff, ff, False, "bf16", identity=True)
    x, z = values(gen, tokens, d, spread=0.3), torch.randn(tokens, E, device="cuda", generator=gen)
    y = experts.ExpertFeedForward(up.own, down.own, 1, act=act).forward(x, z)
    expert, _, offsets, token, position = eo.route(f64(z), 1)
    rows = x.double()[torch.from_numpy(token).to("cuda")]
    h, mags = up.exact(e4m3_rows(rows)[0] if weights == "e4m3" else rows, offsets.tolist(), act)
    at = torch.from_numpy(position[:, 0]).to("cuda")
    if weights == "16bit":
        assert_close(y, h[at], mags[at], d, "bf16")
        return
    scale = e4m3_rows(h)[1]
    bound = 1.1 * (d + 8) * 2.0 ** -23 * mags + 2.0 ** -16 * h.abs()
    bound = bound + 2.0 ** -4 * (h.abs() + bound) + 2 * scale * 2.0 ** -10
    off = ((y.double() - h[at]).abs() / bound[at]).max().item()
    assert y.isfinite().all() and off <= 1.0, off


def test_no_wait_ran_out(cq):
    assert cq.device_status(0) == 0
