"""The sizes of the grouped product's tests take every tile width that a call can: without a GPU, so that constants of the
choice which are fitted anew cannot leave a kernel untested."""
from __future__ import annotations

import expert_plan as ep


def test_sizes_take_the_widths_that_they_are_there_for():
    for weights, rows, experts, n, k, act, _, _, want in ep.PRODUCTS:
        assert ep.product_width(weights, rows, experts, n, k, act) == want, (weights, rows, experts, n, k)
    for weights, tokens, experts, top, d, ff, out, act, _, _, _, _, *want in ep.MODULES:
        assert ep.module_widths(weights, tokens * top, experts, d, ff, out, act) == tuple(want), (weights, tokens, experts, ff)
    for weights, tokens, experts, d, ff, act, *want in ep.KEPT:
        assert ep.module_widths(weights, tokens, experts, d, ff, ff, act) == tuple(want), (weights, tokens, experts, ff)


def test_every_kernel_is_reached():
    """Weights, width and output: each that a call can take, T with a bias, of one group (16-bit: from 128 wide on) and of several."""
    plain = {(c[0], c[-1], c[2] > 1) for c in ep.PRODUCTS if c[6]}
    assert plain == {(w, b, g) for w in ("e4m3", "16bit") for b in (64, 128, 256) for g in (False, True)} - {("16bit", 64, False)}
    ups, downs = {(c[0], c[-2]) for c in ep.MODULES}, {(c[0], c[-1]) for c in ep.MODULES}
    assert ups == {("e4m3", 128), ("e4m3", 256)} | {("16bit", b) for b in (64, 128, 256)}
    assert downs == {(w, b) for w in ("e4m3", "16bit") for b in (64, 128, 256)}
    assert {(c[0], c[6]) for c in ep.KEPT} == ups
    # with and without each option of the module
    for at, values in ((7, {"none", "relu", "silu"}), (8, {True, False}), (9, {True, False}), (10, {"f32", "f16", "bf16"}), (11, {"f16", "bf16"})):
        assert {c[at] for c in ep.MODULES} == values


def test_ragged_groups():
    for rows in (40, 130, 4000, 16384):
        for experts in (2, 3, 20, 32):
            sizes = ep.ragged(rows, experts)
            assert sum(sizes) == rows and len(sizes) == experts and min(sizes) >= 0 and sizes[1 % experts] >= 0
