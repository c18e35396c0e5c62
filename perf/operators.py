"""What the 8-bit floating-point linear, the linears of experts, the router and their feed-forward module are
measured on.

Every case is one call of one operator:

  fp8_linear     y = act(x^ . w^T + b): weights held as e4m3 codes with a scale for each 128 x 128 block, rows
                 of x brought to e4m3 with a power-of-two scale for each 128 values (x^ is what the codes stand for)
  expert_linear  the same product grouped by expert: rows [offsets[e], offsets[e + 1]) of x meet the weights of
                 expert e, 16-bit or e4m3; rows from offsets[experts] on belong to no expert and come back as zeros
  route          the k best experts of each token, their weights, and the order of (token, expert) pairs by expert
  combine        each token's weighted sum of the rows that its experts made
  expert_ffn     route, first linear, activation, second linear, combine, for tokens and their router logits

`run` computes them in elementary torch operations, or with this repository's library where `own` is true.
"""
from __future__ import annotations

import math
import random
import sys

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the first feed-forward linear of one stream's chunk: 14 frames, launch latency and the weights' bytes count
        dict(name="fp8_linear_chunk", op="fp8_linear", rows=14, n=4096, k=1024, dtype="bf16", act="silu", bias=False),
        # a joint head's odd width (a vocabulary of 1025) over the frames of some tens of streams
        dict(name="fp8_linear_vocab", op="fp8_linear", rows=333, n=1025, k=640, dtype="f16", act="none", bias=True),
        # an offline batch: the tensor cores are the bound
        dict(name="fp8_linear_bulk", op="fp8_linear", rows=16384, n=4096, k=4096, dtype="bf16", act="none", bias=False),
        # one stream's chunk over two of sixteen experts each: most experts have one or two rows
        dict(name="expert_linear_chunk", op="expert_linear", rows=28, experts=16, n=4096, k=1024, weights="fp8", dtype="bf16",
             act="silu", bias=False, skew=0.5, tail=0),
        # few rows for each expert in 16-bit weights, ragged, odd widths
        dict(name="expert_linear_ragged", op="expert_linear", rows=777, experts=12, n=1000, k=520, weights="16bit", dtype="f16",
             act="relu", bias=True, skew=1.0, tail=40),
        # an offline batch over many experts in 16-bit weights
        dict(name="expert_linear_bulk", op="expert_linear", rows=16384, experts=64, n=2048, k=2048, weights="16bit", dtype="bf16",
             act="none", bias=False, skew=0.5, tail=0),
        # the router's choice for one chunk
        dict(name="route_chunk", op="route", tokens=14, experts=8, top=2, dtype="f32", renormalize=True, padded=0.0),
        # the router's choice for an offline batch, a tenth of whose tokens are padding and go nowhere
        dict(name="route_bulk", op="route", tokens=16384, experts=128, top=8, dtype="bf16", renormalize=True, padded=0.1),
        # the sum for the frames of 64 streams
        dict(name="combine_streams", op="combine", tokens=896, dims=1024, top=2, dtype="bf16", padded=0.0),
        # the sum for an offline batch with many experts a token
        dict(name="combine_bulk", op="combine", tokens=16384, dims=2048, top=8, dtype="bf16", padded=0.1),
        # the whole feed-forward module for one chunk, and for the frames of 64 streams
        dict(name="expert_ffn_chunk", op="expert_ffn", tokens=14, experts=8, top=2, hidden=1024, ff=4096, weights="fp8",
             dtype="bf16", act="silu", padded=0.0),
        dict(name="expert_ffn_streams", op="expert_ffn", tokens=896, experts=32, top=2, hidden=1024, ff=4096, weights="fp8",
             dtype="bf16", act="silu", padded=0.0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm; one in three is as it comes, the others end on 8."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    v = round(v) if v < 32 or rng.random() < 0.34 else round(v / 8) * 8
    return min(high, max(low, v))


def draw(rng):
    op = rng.choice(["fp8_linear", "expert_linear", "route", "combine", "expert_ffn"])
    dtype = rng.choice(["bf16", "f16"])
    act = rng.choice(["none", "silu", "relu"])
    if op == "fp8_linear":
        return dict(op=op, rows=_spread(rng, 1, 16384), n=_spread(rng, 256, 4096), k=_spread(rng, 256, 4096), dtype=dtype,
                    act=act, bias=rng.random() < 0.5)
    if op == "expert_linear":
        rows = _spread(rng, 1, 16384)
        return dict(op=op, rows=rows, experts=_spread(rng, 2, 64), n=_spread(rng, 256, 2048), k=_spread(rng, 256, 2048),
                    weights=rng.choice(["fp8", "16bit"]), dtype=dtype, act=act, bias=rng.random() < 0.5,
                    skew=rng.choice([0.0, 0.5, 1.0]), tail=rng.choice([0, rows // 8]))
    if op == "route":
        experts = _spread(rng, 2, 256)
        return dict(op=op, tokens=_spread(rng, 1, 16384), experts=experts, top=min(experts, rng.choice([1, 2, 4, 8])),
                    dtype=rng.choice(["f32", "bf16", "f16"]), renormalize=rng.random() < 0.5, padded=rng.choice([0.0, 0.1]))
    if op == "combine":
        return dict(op=op, tokens=_spread(rng, 1, 16384), dims=_spread(rng, 256, 2048), top=rng.choice([1, 2, 4, 8]), dtype=dtype,
                    padded=rng.choice([0.0, 0.1]))
    experts = _spread(rng, 2, 32)
    return dict(op=op, tokens=_spread(rng, 1, 4096), experts=experts, top=min(experts, rng.choice([1, 2, 4])),
                hidden=_spread(rng, 256, 1024), ff=_spread(rng, 256, 4096), weights=rng.choice(["fp8", "16bit"]), dtype=dtype, act=act,
                padded=rng.choice([0.0, 0.1]))


# ------------------------------------------------------------------ inputs

def _noise(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _activations(gen, rows, k, dtype):
    """Normalised activations: unit rows with a spread of channel gains and a few channels that stand out."""
    gain = torch.exp(0.5 * _noise(gen, k))
    gain[:: 97] *= 8.0
    return (_noise(gen, rows, k) * gain).to(TYPES[dtype])


def _scale_of_blocks(experts, n, k, top):
    return top.reshape(experts, -(-n // BLOCK), BLOCK, -(-k // BLOCK), BLOCK).amax((2, 4))


def _weights(gen, experts, n, k, kind, dtype):
    """[experts, n, k] weights of a checkpoint: 16-bit values, or e4m3 codes with the scale max / 448 of each block."""
    w = _noise(gen, experts, n, k) / math.sqrt(k)
    w *= torch.exp(0.3 * _noise(gen, experts, n, 1))
    if kind == "16bit":
        return dict(weight=w.to(TYPES[dtype]))
    pad = torch.nn.functional.pad(w.abs(), (0, -k % BLOCK, 0, -n % BLOCK))
    scale = _scale_of_blocks(experts, n, k, pad) / E4M3_MAX
    full = scale.repeat_interleave(BLOCK, 1)[:, :n].repeat_interleave(BLOCK, 2)[:, :, :k]
    return dict(codes=(w / full).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale=scale)


def _logits(gen, tokens, experts, padded, dtype="f32", skew=0.5):
    """Router logits with favoured experts; a share of the tokens is padding, masked with minus infinity."""
    z = _noise(gen, tokens, experts) * 1.5 + skew * _noise(gen, 1, experts)
    if padded:
        z[torch.rand(tokens, device="cuda", generator=gen) < padded] = -math.inf
    return z.to(TYPES[dtype])


def _offsets(gen, rows, experts, skew, tail):
    """Ragged groups: rows that favour some experts, the last `tail` rows with none."""
    chosen = _logits(gen, rows - tail, experts, 0.0, skew=skew).argmax(1)
    counts = torch.bincount(chosen, minlength=experts)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def _library():
    if "catcher-tippi_b200" not in sys.path:
        sys.path.insert(0, "catcher-tippi_b200")
    import nemotron_cuda.experts as experts
    import nemotron_cuda.fp8 as fp8
    return fp8, experts


def _expert_layer(s, dtype, bias):
    fp8, experts = _library()
    if "weight" in s:
        return experts.ExpertLinear.from_weight(s["weight"], bias)
    return experts.ExpertLinear.from_codes(s["codes"], s["scale"], bias, dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    op, dtype = case["op"], case["dtype"]
    s = dict(case=case)
    if op == "fp8_linear":
        w = _weights(gen, 1, case["n"], case["k"], "fp8", dtype)
        s |= dict(codes=w["codes"][0], scale=w["scale"][0], x=_activations(gen, case["rows"], case["k"], dtype))
        s["bias"] = (0.1 * _noise(gen, case["n"])).to(TYPES[dtype]) if case["bias"] else None
        if own:
            fp8, _ = _library()
            s["layer"] = fp8.Fp8Linear.from_codes(s["codes"], s["scale"], s["bias"], dtype=dtype)
    elif op == "expert_linear":
        s |= _weights(gen, case["experts"], case["n"], case["k"], case["weights"], dtype)
        s["bias"] = (0.1 * _noise(gen, case["experts"], case["n"])).to(TYPES[dtype]) if case["bias"] else None
        s["x"] = _activations(gen, case["rows"], case["k"], dtype)
        s["offsets"] = _offsets(gen, case["rows"], case["experts"], case["skew"], case["tail"])
        if own:
            s["layer"] = _expert_layer(s, dtype, s["bias"])
    elif op == "route":
        s["logits"] = _logits(gen, case["tokens"], case["experts"], case["padded"], dtype)
        if own:
            s["route"] = _library()[1].route
    elif op == "combine":
        tokens, top = case["tokens"], case["top"]
        s["z"] = _noise(gen, tokens * top, case["dims"]).to(TYPES[dtype])
        s["position"] = torch.randperm(tokens * top, device="cuda", generator=gen).to(torch.int32).reshape(tokens, top)
        weight = torch.softmax(_noise(gen, tokens, top), 1)
        gone = torch.rand(tokens, device="cuda", generator=gen) < case["padded"]
        s["position"][gone] = -1
        s["weight"] = torch.where(gone[:, None], 0.0, weight)
        if own:
            s["combine"] = _library()[1].combine
    else:
        s["up"] = _weights(gen, case["experts"], case["ff"], case["hidden"], case["weights"], dtype)
        s["down"] = _weights(gen, case["experts"], case["hidden"], case["ff"], case["weights"], dtype)
        s["x"] = _activations(gen, case["tokens"], case["hidden"], dtype)
        s["logits"] = _logits(gen, case["tokens"], case["experts"], case["padded"])
        if own:
            _, experts = _library()
            s["ffn"] = experts.ExpertFeedForward(_expert_layer(s["up"], dtype, None), _expert_layer(s["down"], dtype, None),
                                                 top=case["top"], act=case["act"])
    return s


# ------------------------------------------------------------------ the plain forms

def _through_e4m3(x):
    """x in 32 bits -> what its e4m3 codes stand for: the scale of 128 values is the least power of two that brings
    their largest finite magnitude to 448 or less (1 where all are zero)."""
    rows, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    top = torch.where(torch.isfinite(blocks), blocks.abs(), 0.0).amax(2, keepdim=True)
    fraction, exponent = torch.frexp(top)
    exponent = (exponent - 9 + (fraction > 0.875).int()).clamp(min=-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), exponent), 1.0)
    return ((blocks / scale).to(torch.float8_e4m3fn).float() * scale).reshape(rows, -1)[:, :k]


def _from_codes(codes, scale):
    """[..., n, k] codes and the scales of their blocks -> 32-bit weights."""
    n, k = codes.shape[-2:]
    return codes.float() * scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _activate(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return torch.clamp(v, min=0.0) if act == "relu" else v


def _grouped(x, w, offsets):
    """Rows of x by the weights of their expert, as one batched product over groups padded to the longest."""
    row = torch.arange(x.shape[0], device=x.device)
    live = row < offsets[-1]
    expert = torch.where(live, torch.searchsorted(offsets[1:], row, right=True), 0)
    most = int((offsets[1:] - offsets[:-1]).max())
    slot = torch.where(live, row - offsets[expert], most)
    padded = x.new_zeros(w.shape[0], most + 1, x.shape[1])
    padded[expert, slot] = x
    return torch.bmm(padded, w.transpose(1, 2))[expert, slot], expert, live


def _expert_rows(x, layer, offsets, act, bias=None):
    """The first or second linear of the experts in 32 bits; rows of no expert are zeros."""
    if "codes" in layer:
        y, expert, live = _grouped(_through_e4m3(x), _from_codes(layer["codes"], layer["scale"]), offsets)
    else:
        y, expert, live = _grouped(x, layer["weight"].float(), offsets)
    if bias is not None:
        y = y + bias.float()[expert]
    return torch.where(live[:, None], _activate(y, act), 0.0)


def _routed(logits, top, renormalize):
    z = logits.float()
    tokens, experts = z.shape
    best, order = torch.sort(z, dim=1, descending=True, stable=True)
    best, chosen = best[:, :top], order[:, :top]
    taken = best > -math.inf
    largest = torch.where(taken[:, :1], best[:, :1], 0.0)
    share = torch.where(taken, torch.exp(best - largest), 0.0)
    total = share.sum(1, keepdim=True) if renormalize else torch.exp(z - largest).sum(1, keepdim=True)
    weight = torch.where(taken, share / torch.where(total > 0, total, 1.0), 0.0)
    expert = torch.where(taken, chosen, -1).to(torch.int32)
    flat = torch.where(taken, chosen, experts).reshape(-1)
    by_expert = torch.argsort(flat, stable=True)
    ends = torch.searchsorted(flat[by_expert], torch.arange(experts, device=z.device), right=True)
    offsets = torch.nn.functional.pad(ends, (1, 0)).to(torch.int32)
    live = flat[by_expert] < experts
    token = torch.where(live, by_expert // top, -1).to(torch.int32)
    position = torch.empty_like(by_expert).scatter_(0, by_expert, torch.arange(flat.numel(), device=z.device))
    position = torch.where(taken, position.reshape(tokens, top), -1).to(torch.int32)
    return dict(expert=expert, weight=weight, offsets=offsets, token=token, position=position)


def _combined(z, position, weight):
    rows = torch.where((position >= 0)[:, :, None], z[position.clamp(min=0).long()], 0.0)
    return (rows * weight[:, :, None]).sum(1)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        if op == "fp8_linear":
            return state["layer"].forward(state["x"], act=case["act"])
        if op == "expert_linear":
            return state["layer"].forward(state["x"], state["offsets"], act=case["act"])
        if op == "route":
            r = state["route"](state["logits"], case["top"], renormalize=case["renormalize"])
            return dict(expert=r.expert, weight=r.weight, offsets=r.offsets, token=r.token, position=r.position)
        if op == "combine":
            return state["combine"](state["z"], state["position"], state["weight"])
        return state["ffn"].forward(state["x"], state["logits"])
    dtype = TYPES[case["dtype"]]
    if op == "fp8_linear":
        y = _through_e4m3(state["x"].float()) @ _from_codes(state["codes"], state["scale"]).T
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return _activate(y, case["act"]).to(dtype)
    if op == "expert_linear":
        return _expert_rows(state["x"].float(), state, state["offsets"], case["act"], state["bias"]).to(dtype)
    if op == "route":
        return _routed(state["logits"], case["top"], case["renormalize"])
    if op == "combine":
        return _combined(state["z"].float(), state["position"], state["weight"]).to(dtype)
    r = _routed(state["logits"], case["top"], True)
    rows = torch.where((r["token"] >= 0)[:, None], state["x"].float()[r["token"].clamp(min=0).long()], 0.0)
    rows = _expert_rows(rows, state["up"], r["offsets"], case["act"])
    rows = _expert_rows(rows, state["down"], r["offsets"], "none")
    return _combined(rows, r["position"], r["weight"]).to(dtype)


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_e4m3(v):
    """The nearest e4m3 value of each |v| <= 448, halves to even: 4 significant bits, down to steps of 2^-9."""
    _, exponent = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (exponent - 4).clamp(min=-9))
    return torch.round(v / step) * step


def _exact_activations(x):
    out = torch.zeros_like(x)
    for k0 in range(0, x.shape[1], BLOCK):
        part = x[:, k0:k0 + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        power = torch.ceil(torch.log2(torch.where(top > 0, top, E4M3_MAX) / E4M3_MAX))
        for wrong in (-1, 1):  # a logarithm next to a whole number may round across it
            other = power + wrong
            fits = top <= E4M3_MAX * torch.exp2(other)
            power = torch.where(fits & (other < power), other, power)
            power = torch.where(top > E4M3_MAX * torch.exp2(power), power + 1, power)
        scale = torch.exp2(power.clamp(min=-126))
        out[:, k0:k0 + BLOCK] = _exact_e4m3(part / scale) * scale
    return out


def _exact_weights(layer, e=None):
    pick = (lambda t: t) if e is None else (lambda t: t[e])
    if "weight" in layer:
        return pick(layer["weight"]).double()
    codes, scale = pick(layer["codes"]).double(), pick(layer["scale"]).double()
    n, k = codes.shape
    at_n, at_k = torch.arange(n, device=codes.device) // BLOCK, torch.arange(k, device=codes.device) // BLOCK
    return codes * scale[at_n][:, at_k]


def _exact_act(v, act):
    return v * torch.sigmoid(v) if act == "silu" else torch.relu(v) if act == "relu" else v


def _exact_experts(x, layer, offsets, act, bias=None):
    n = (layer["weight"] if "weight" in layer else layer["codes"]).shape[1]
    y = x.new_zeros(x.shape[0], n)
    for e, (a, b) in enumerate(zip(offsets[:-1].tolist(), offsets[1:].tolist())):
        if a < b:
            rows = _exact_activations(x[a:b]) if "codes" in layer else x[a:b]
            v = rows @ _exact_weights(layer, e).T
            y[a:b] = _exact_act(v if bias is None else v + bias[e].double(), act)
    return y


def _exact_route(logits, top, renormalize):
    z = logits.double().cpu()
    tokens, experts = z.shape
    expert, weight = torch.full((tokens, top), -1), torch.zeros(tokens, top, dtype=torch.float64)
    left, number = z.clone(), torch.arange(tokens)
    for j in range(top):
        best = left.max(1).values
        first = torch.where(left == best[:, None], torch.arange(experts), experts).min(1).values
        ok = best > -math.inf
        expert[ok, j], weight[ok, j] = first[ok], best[ok]
        left[number[ok], first[ok]] = -math.inf
    ok = expert >= 0
    logs = torch.logsumexp(torch.where(ok, weight, -math.inf) if renormalize else z, 1, keepdim=True)
    weight = torch.where(ok, torch.exp(weight - logs), 0.0)
    token, offsets = torch.full((tokens * top,), -1), [0]
    position, at = torch.full((tokens, top), -1), 0
    for e in range(experts):
        t, j = torch.nonzero(expert == e, as_tuple=True)
        token[at:at + len(t)] = t
        position[t, j] = torch.arange(at, at + len(t))
        at += len(t)
        offsets.append(at)
    as_int = lambda v: v.to(torch.int32)  # noqa: E731
    return dict(expert=as_int(expert), weight=weight, offsets=torch.tensor(offsets, dtype=torch.int32), token=as_int(token),
                position=as_int(position))


def _exact_combine(z, position, weight):
    y = z.new_zeros(position.shape[0], z.shape[1])
    for j in range(position.shape[1]):
        t = torch.nonzero(position[:, j] >= 0)[:, 0]
        y[t] += weight[t, j, None].double() * z[position[t, j].long()]
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "fp8_linear":
        y = _exact_activations(s["x"].double()) @ _exact_weights(s).T
        return _exact_act(y if s["bias"] is None else y + s["bias"].double(), case["act"])
    if op == "expert_linear":
        return _exact_experts(s["x"].double(), s, s["offsets"], case["act"], s["bias"])
    if op == "route":
        return _exact_route(s["logits"], case["top"], case["renormalize"])
    if op == "combine":
        return _exact_combine(s["z"].double(), s["position"], s["weight"])
    r = _exact_route(s["logits"], case["top"], True)
    token, live = r["token"].to(s["x"].device).long(), int(r["offsets"][-1])
    rows = s["x"].new_zeros(token.numel(), case["hidden"], dtype=torch.float64)
    rows[:live] = s["x"].double()[token[:live]]
    rows = _exact_experts(rows, s["up"], r["offsets"], case["act"])
    rows = _exact_experts(rows, s["down"], r["offsets"], "none")
    return _exact_combine(rows, r["position"].to(rows.device), r["weight"].to(rows.device))


# ------------------------------------------------------------------ what a pass cannot do without

def _weight_bytes(experts, n, k, kind):
    if kind == "16bit":
        return 2 * experts * n * k
    return experts * (n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK))


def _met(experts, rows):
    """Experts that have a row, on average over even choices."""
    return experts * (1.0 - (1.0 - 1.0 / experts) ** rows)


def work(case):
    op = case["op"]
    if op == "route":
        pairs = case["tokens"] * case["top"]
        size = 4 if case["dtype"] == "f32" else 2
        return dict(bytes=case["tokens"] * case["experts"] * size + 16 * pairs + 4 * (case["experts"] + 1),
                    flops=4 * case["tokens"] * case["experts"])
    if op == "combine":
        pairs = case["tokens"] * case["top"] * (1.0 - case["padded"])
        return dict(bytes=2 * case["dims"] * (pairs + case["tokens"]) + 8 * case["tokens"] * case["top"],
                    flops=2 * pairs * case["dims"])
    if op == "expert_ffn":
        d, f, live = case["hidden"], case["ff"], case["tokens"] * (1.0 - case["padded"])
        met = _met(case["experts"], live * case["top"])
        return dict(bytes=_weight_bytes(met, f, d, case["weights"]) + _weight_bytes(met, d, f, case["weights"])
                    + 4 * case["tokens"] * (d + case["experts"]),
                    flops=4 * live * case["top"] * d * f)
    rows, n, k = case["rows"], case["n"], case["k"]
    if op == "fp8_linear":
        return dict(bytes=_weight_bytes(1, n, k, "fp8") + 2 * rows * (n + k) + (2 * n if case["bias"] else 0), flops=2 * rows * n * k)
    live = rows - case["tail"]
    met = _met(case["experts"], live)
    return dict(bytes=_weight_bytes(met, n, k, case["weights"]) + 2 * live * k + 2 * rows * n + (2 * met * n if case["bias"] else 0)
                + 4 * (case["experts"] + 1), flops=2 * live * n * k)


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
