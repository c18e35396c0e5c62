"""The grouped product's choice of a tile width, compiled for the host from the kernel's own source, so that tests can say
which width a size takes.  (No GPU.)"""
from __future__ import annotations

import ctypes
import functools
import os
import re
import subprocess
import tempfile

from conftest import ROOT

OUTS = {"T": 0, "f32": 1, "codes": 2, "parts": 3}
ACTS = {"none": 0, "silu": 1, "relu": 2}
HEAD = """
#include <math.h>
#include <stdint.h>
#include <algorithm>
#include <cmath>
enum { kOutT, kOutF32, kOutCodes, kOutParts };
constexpr int kGemmRows = 128, kRowBytes = 128, kFp8Block = 128, kActSilu = 1;
constexpr int epi_sets(int bn) { return bn < 256 ? 2 : 1; }
extern "C" {
"""


@functools.cache
def _library():
    csrc = os.path.join(ROOT, "catcher-tippi_b200", "csrc")
    text = open(os.path.join(csrc, "expert_gemm.cu")).read()
    assert "constexpr int epi_sets(int bn) { return bn < 256 ? 2 : 1; }" in text and "kRowBytes = 128;" in text
    assert re.search(r"enum ExpertOut : int { kOutT = 0, kOutF32 = 1, kOutCodes = 2, kOutParts = 3 };",
                     open(os.path.join(csrc, "expert_gemm.hpp")).read())
    assert re.search(r"kActSilu = 1\b", open(os.path.join(csrc, "common.cuh")).read())
    function = re.search(r"^int plan_expert_gemm\(.*?^}\n", text, flags=re.S | re.M).group(0)
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "plan.cpp"), os.path.join(d, "plan.so")
        open(src, "w").write(HEAD + function + "}\n")
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", src, "-o", out], check=True)
        lib = ctypes.CDLL(out)
    lib.plan_expert_gemm.argtypes = [ctypes.c_bool] + [ctypes.c_int] * 8
    return lib


def width(weights: str, rows: int, experts: int, n: int, k: int, act: str = "none", out: str = "T", parts: int = 1,
          sms: int = 148) -> int:
    """Weight rows of a tile: 64, 128 or 256.  `parts`: 2 where the rows are the module's 16-bit h."""
    return _library().plan_expert_gemm(weights == "e4m3", rows, experts, n, k, parts, ACTS[act], OUTS[out], sms)


# ------------------------------------------------------------------ sizes that take each width

def ragged(rows: int, experts: int):
    """Group sizes that add up to `rows`: an empty one, one that ends on a tile's edge where there is room, uneven ones."""
    if experts == 1:
        return [rows]
    share = [(7 * e) % 5 + 1 for e in range(experts)]
    share[1] = 0
    sizes = [rows * s // sum(share) for s in share]
    if sizes[0] > 128:
        sizes[0] -= sizes[0] % 128
    sizes[-1] += rows - sum(sizes)
    return sizes


# weights, rows, experts, n, k, activation, bias, type, width
PRODUCTS = [
    ("e4m3", 333, 1, 333, 2500, "silu", True, "f16", 64), ("e4m3", 400, 3, 333, 2100, "none", True, "bf16", 64),
    ("e4m3", 1000, 1, 2048, 4096, "none", False, "bf16", 128), ("e4m3", 4000, 1, 1025, 1000, "none", True, "f16", 128),
    ("e4m3", 1200, 1, 1025, 2100, "none", True, "bf16", 128), ("e4m3", 130, 32, 264, 2100, "none", True, "f16", 128),
    ("e4m3", 4000, 2, 1025, 1000, "none", False, "bf16", 128), ("e4m3", 1792, 32, 2048, 1024, "relu", True, "bf16", 64),
    ("e4m3", 700, 1, 4096, 4096, "none", True, "f16", 256), ("e4m3", 900, 1, 2500, 2100, "silu", True, "bf16", 256),
    ("e4m3", 1200, 4, 2048, 2048, "silu", False, "bf16", 256), ("e4m3", 40, 20, 1025, 2100, "silu", True, "f16", 256),
    ("e4m3", 16384, 3, 512, 1300, "none", True, "bf16", 256),
    ("16bit", 400, 2, 333, 2100, "silu", True, "f16", 64), ("16bit", 4000, 1, 264, 1000, "silu", True, "bf16", 128),
    ("16bit", 1200, 1, 1025, 2100, "silu", True, "f16", 128), ("16bit", 130, 32, 264, 2100, "silu", True, "bf16", 128),
    ("16bit", 900, 1, 2500, 2100, "silu", False, "bf16", 256), ("16bit", 3000, 1, 1025, 1000, "none", True, "f16", 256),
    ("16bit", 70, 20, 1000, 1000, "silu", True, "bf16", 256), ("16bit", 16384, 3, 520, 264, "relu", True, "f16", 256),
]

# weights, tokens, experts, top, d, ff, out, activation, bias, renormalize, logits' type, type, widths of the two products
MODULES = [
    ("e4m3", 40, 1, 1, 136, 200, 136, "relu", True, True, "bf16", "bf16", 128, 64),
    ("e4m3", 1500, 2, 2, 136, 200, 2048, "relu", True, False, "f16", "f16", 128, 128),
    ("e4m3", 70, 32, 1, 136, 200, 1000, "silu", True, False, "f32", "bf16", 128, 256),
    ("e4m3", 40, 32, 3, 136, 520, 136, "none", True, False, "f32", "bf16", 256, 64),
    ("e4m3", 2100, 3, 3, 136, 333, 1000, "none", False, True, "bf16", "f16", 256, 128),
    ("e4m3", 2100, 2, 2, 136, 520, 1000, "relu", True, True, "f16", "bf16", 256, 256),
    ("16bit", 40, 1, 1, 136, 200, 136, "none", True, True, "bf16", "f16", 64, 64),
    ("16bit", 40, 32, 3, 136, 200, 264, "none", True, False, "f32", "bf16", 64, 128),
    ("16bit", 70, 20, 1, 136, 200, 1000, "relu", False, True, "f16", "bf16", 64, 256),
    ("16bit", 1500, 4, 3, 136, 200, 136, "relu", True, False, "bf16", "f16", 128, 64),
    ("16bit", 2100, 3, 3, 136, 200, 333, "silu", True, False, "f16", "bf16", 128, 256),
    ("16bit", 2100, 3, 3, 136, 333, 136, "none", True, True, "f32", "bf16", 256, 128),
    ("16bit", 2100, 3, 3, 136, 333, 333, "relu", True, False, "f32", "f16", 256, 256),
]

# weights, tokens, experts, d, ff, activation, widths: the second linear is the identity, so that y is h as it was kept
KEPT = [
    ("e4m3", 40, 1, 128, 200, "none", 128, 64), ("e4m3", 2100, 20, 128, 1300, "none", 128, 128),
    ("e4m3", 130, 32, 128, 520, "relu", 256, 64), ("e4m3", 40, 32, 128, 1300, "silu", 256, 128),
    ("e4m3", 4000, 32, 128, 640, "none", 256, 256), ("16bit", 40, 1, 128, 200, "silu", 64, 64),
    ("16bit", 4000, 12, 128, 200, "relu", 128, 128), ("16bit", 4000, 4, 128, 520, "none", 256, 256),
]


def product_width(weights, rows, experts, n, k, act, sms=148):
    return width(weights, rows, experts, n, k, act, sms=sms)


def module_widths(weights, pairs, experts, d, ff, out, act, sms=148):
    up = width(weights, pairs, experts, ff, d, act, "codes" if weights == "e4m3" else "parts", sms=sms)
    return up, width(weights, pairs, experts, out, ff, "none", "f32", 1 if weights == "e4m3" else 2, sms=sms)
