"""The operators of token rows around microscaled 4-bit floating point (MXFP4) and the root-mean-square norm, as cases to time: the
norm with the residual's addition, to its own type, to int8 tokens and to MXFP4 rows, the quantization of rows to MXFP4 and the
product of such rows with MXFP4 weights.

listed() and draw() describe cases as plain dicts; prepare() makes what a program holds before the call, run() is one pass,
in plain torch operations or (`own`) by the calls of tennis_amd.capi, work() the bytes and operations that a pass cannot do
without, exact() the operators' definition in 64 bits.

MXFP4: blocks of 32 consecutive values of a row share a scale 2^(s - 127), s a byte; a value is four bits, a sign and one of 0, 0.5, 1,
1.5, 2, 3, 4 and 6, the value at an even place of its row in the lower half of a byte.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One token of a serving step, between two layers: the call itself is most of the time.
        {"name": "norm one token", "kind": "rms_norm", "m": 1, "k": 4096, "type": "bf16", "residual": True, "extra": 0},
        # The tokens of a batch of prompts, with the residual stream read and written.
        {"name": "norm 8192 tokens", "kind": "rms_norm", "m": 8192, "k": 4096, "type": "bf16", "residual": True, "extra": 0},
        # A decoding batch whose projections are int8: the norm in front of them ...
        {"name": "norm to int8 64 tokens", "kind": "norm_tokens", "m": 64, "k": 4096, "type": "bf16", "residual": True, "extra": 0},
        # ... and a prompt of it, rows of no whole number of pieces in a wider buffer.
        {"name": "norm to int8 ragged", "kind": "norm_tokens", "m": 5000, "k": 2050, "type": "f16", "residual": False, "extra": 14},
        # Activations of a decoding batch to four bits and back ...
        {"name": "quantize 32 tokens", "kind": "quantize", "m": 32, "k": 4096, "type": "bf16", "extra": 0},
        # ... and a large layer's weights, as a program quantizes them once and looks at what it lost.
        {"name": "quantize 8192 rows", "kind": "quantize", "m": 8192, "k": 8192, "type": "bf16", "extra": 0},
        # One token through a square projection: the weights are all there is to read.
        {"name": "product one token", "kind": "product", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False, "act": "none", "extra": 0},
        # Sizes that are no multiple of any tile or block, fp32 in and out, rows at odd addresses.
        {"name": "product ragged", "kind": "product", "m": 777, "n": 1111, "k": 1500, "type": "f32", "bias": True, "act": "relu", "extra": 3},
        # A prompt through a square projection.
        {"name": "product 4096", "kind": "product", "m": 4096, "n": 4096, "k": 4096, "type": "bf16", "bias": True, "act": "silu", "extra": 0},
        # A large batch of prompts through a large layer: the largest pass.
        {"name": "product 8192", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False, "act": "none", "extra": 0},
        # The norm and the projection behind it, on a decoding batch ...
        {"name": "norm and product 16", "kind": "norm_product", "m": 16, "n": 4096, "k": 4096, "type": "bf16", "residual": True, "extra": 0},
        # ... and on a prompt.
        {"name": "norm and product 2048", "kind": "norm_product", "m": 2048, "n": 4096, "k": 2048, "type": "f16", "residual": True, "extra": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rms_norm", "rms_norm", "norm_tokens", "quantize", "quantize", "product", "product", "product", "norm_product"])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16", "bf16"]), "extra": rng.choice([0, 0, 1, 8, 64])}
    if kind in ("product", "norm_product"):
        case["m"], case["n"] = _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)
        case["k"] = _log_int(rng, 1 if kind == "product" else 64, 8192)
    else:
        case["k"] = _log_int(rng, 1, 16384)
        case["m"] = _log_int(rng, 1, max(2, 33554432 // case["k"]))
    if kind == "product":
        case["bias"], case["act"] = rng.choice([True, False]), rng.choice(["none", "relu", "leaky_relu", "silu", "mish_fast"])
    elif kind != "quantize":
        case["residual"] = rng.choice([True, True, False])
        if kind != "rms_norm":
            case["type"] = rng.choice(["f16", "bf16"])      # of a norm in fp32, values next to a rounding border go either way
    return case


# ---------------------------------------------------------------------------------------------- what a program holds

SLOPE = 0.1
EPSILON = 1e-6
BLOCK = 32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    t, m, k = _TYPES[case["type"]], case["m"], case["k"]
    # activations: tokens of different size, a few channels far larger than the others
    x = normal(m, k + case["extra"]) * torch.exp(0.5 * normal(m, 1))
    x *= torch.where(torch.rand(k + case["extra"], generator=g, device="cuda") < 0.01, 8.0, 1.0)
    state = {"case": case, "x": x.to(t)[:, :k]}
    if "residual" in case:
        state["weight"] = 1.0 + 0.2 * normal(k)
        state["residual"] = normal(m, k).to(t) if case["residual"] else None
    if "n" in case:
        # weights as a quantized layer stores them: two values a byte [n][ceil(k / 2)], and their blocks' scales [n][ceil(k / 32)]
        w = normal(case["n"], k) / math.sqrt(k)
        values, scale_bytes = _mxfp4(w)
        state["w"], state["w_scales"] = _packed(values, k), scale_bytes
        state["bias"] = normal(case["n"]) if case.get("bias") else None
    return state


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from tennis_amd import capi
    case, x = state["case"], state["x"]
    if "w" in state and "layer" not in state:      # a program makes the layer once and keeps it: its weights packed
        state["layer"] = capi.TokenGemmMxfp4(state["w"], state["w_scales"], bias=state["bias"], k=case["k"])
    if case["kind"] == "quantize":
        return capi.dequantize_mxfp4(*capi.quantize_mxfp4(x), k=case["k"], dtype=x.dtype)
    if case["kind"] == "product":
        return state["layer"](x, act=case["act"], slope=SLOPE)
    if case["kind"] == "rms_norm":
        return capi.rms_norm(x, state["weight"], EPSILON, residual=state["residual"])
    if case["kind"] == "norm_tokens":
        q, scales, *total = capi.rms_norm_tokens(x, state["weight"], EPSILON, residual=state["residual"])
        return [capi.dequantize_tokens(q, scales, dtype=x.dtype)] + total
    codes, scales, *total = capi.rms_norm_mxfp4(x, state["weight"], EPSILON, residual=state["residual"])
    return [state["layer"](codes, x_scales=scales, out_dtype=x.dtype)] + total


def _run_plain(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "quantize":
        return _values(x.float()).to(x.dtype)
    if case["kind"] == "product":
        return _product(state, x.float(), case["act"]).to(x.dtype)
    total = []
    if state["residual"] is not None:
        x = (x.float() + state["residual"].float()).to(x.dtype)      # the norm is that of the sum as it is kept
        total = [x]
    h = x.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPSILON) * state["weight"]
    if case["kind"] == "rms_norm":
        return [y.to(x.dtype)] + total if total else y.to(x.dtype)
    if case["kind"] == "norm_tokens":
        top = y.abs().amax(-1, keepdim=True)
        q = torch.round(y * torch.where(top > 0, 127.0 / top, 0.0))
        return [(q * (top / 127.0)).to(x.dtype)] + total
    return [_product(state, y, "none").to(x.dtype)] + total


def _mxfp4(x):
    """x [m][k] as multiples [m][blocks][32] of their blocks' scales, and the scales' bytes [m][blocks]."""
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(m, -1, BLOCK)
    # the scale: the power of two of the largest magnitude over that of 6, the largest value; an fp32 number's exponent is its bits 23 .. 30
    top = x.abs().amax(-1, keepdim=True)
    scale_bytes = torch.clamp((top.view(torch.int32) >> 23) - 2, min=0)
    v = x.double() * _power(127 - scale_bytes)            # 64 bits: exact, so that ties are ties
    size = v.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    v = torch.copysign(torch.clamp(torch.round(size / step) * step, max=6.0), v)
    return v.float(), scale_bytes.squeeze(-1).to(torch.uint8)


def _power(e):
    """2^e in 64 bits, by its exponent's bits: exp2 may be off in the last place."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _packed(values, k):
    """Four bits a value, two a byte."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=values.device)
    codes = torch.bucketize(values.abs(), grid) + 8 * torch.signbit(values)
    codes = codes.view(codes.shape[0], -1)[:, :k + k % 2].to(torch.uint8)
    return codes[:, 0::2] | codes[:, 1::2] << 4


def _values(x):
    values, scale_bytes = _mxfp4(x)
    scaled = values.double() * _power(scale_bytes.int() - 127).unsqueeze(-1)
    return scaled.view(x.shape[0], -1)[:, :x.shape[1]].float()


def _product(state, x, act):
    k, codes = x.shape[1], state["w"]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    table = torch.cat((table, -table))
    w = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).view(codes.shape[0], -1)[:, :k]
    scales = _power(state["w_scales"].int() - 127).float()
    w = w * scales.repeat_interleave(BLOCK, 1)[:, :k]
    y = torch.matmul(_values(x), w.t())
    if state["bias"] is not None:
        y = y + state["bias"]
    return _activated(y, act)


def _activated(y, act):
    if act == "relu":
        return torch.where(y > 0, y, 0.0)
    if act == "leaky_relu":
        return torch.where(y > 0, y, SLOPE * y)
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "mish_fast":
        w = torch.exp(torch.clamp(y, max=20.0))
        w = w * (w + 2.0)
        return y * (w / (w + 2.0))
    return y


# ---------------------------------------------------------------------------------------------- work and values

def work(case):
    size, m, k = 4 if case["type"] == "f32" else 2, case["m"], case["k"]
    row, blocks = (k + 1) // 2 + (k + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK      # bytes of a row of four bits a value
    if case["kind"] == "quantize":
        return {"bytes": m * k * 2 * size + m * row, "flops": 2 * m * k}
    if case["kind"] == "product":
        n = case["n"]
        return {"bytes": m * k * size + n * row + (4 * n if case["bias"] else 0) + m * n * size, "flops": 2 * m * n * k}
    read_and_kept = m * k * size * (3 if case["residual"] else 1) + 4 * k      # x, the residual and their sum, the weight
    if case["kind"] == "rms_norm":
        return {"bytes": read_and_kept + m * k * size, "flops": 5 * m * k}
    if case["kind"] == "norm_tokens":
        return {"bytes": read_and_kept + m * k * (1 + size) + 4 * m, "flops": 7 * m * k}
    n = case["n"]
    return {"bytes": read_and_kept + n * row + m * n * size, "flops": 2 * m * n * k + 7 * m * k}


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].double()
    if case["kind"] == "quantize":
        return _rounded64(x)
    if case["kind"] == "product":
        y = _rounded64(x) @ _weights64(state, case["k"])
        if state["bias"] is not None:
            y += state["bias"].double()
        return _activated64(y, case["act"])
    total = []
    if state["residual"] is not None:
        x = x + state["residual"].double()
        total = [x]
        x = x.to(state["x"].dtype).double()
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["k"] + EPSILON) * state["weight"].double()
    if case["kind"] == "rms_norm":
        return [y] + total if total else y
    if case["kind"] == "norm_tokens":
        step = y.abs().max(-1, keepdim=True).values / 127.0
        return [torch.where(step > 0, (y / step.clamp(min=1e-300)).round() * step, 0.0)] + total
    return [_rounded64(y) @ _weights64(state, case["k"])] + total


_BORDERS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]      # between the magnitudes; one that lies on a border has the magnitude of an even place


def _powers64(device):
    return torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float64, device=device)


def _rounded64(x):
    m, k = x.shape
    out = torch.zeros((m, (k + BLOCK - 1) // BLOCK * BLOCK), dtype=torch.float64, device=x.device)
    out[:, :k] = x
    out = out.view(-1, BLOCK)
    scale = _powers64(x.device)[(torch.frexp(out.abs().max(1, keepdim=True).values).exponent + 124).clamp(min=0).long()]
    size = out.abs() / scale
    place = torch.zeros_like(size)
    for i, border in enumerate(_BORDERS):
        place += (size > border if i % 2 == 0 else size >= border).double()
    value = torch.where(place < 5, place / 2, torch.where(place < 7, place - 2, 6.0))
    return (torch.sign(out) * value * scale).view(m, -1)[:, :k].contiguous()


def _weights64(state, k):
    codes = state["w"].to(torch.int64)
    codes = torch.cat(((codes % 16)[..., None], (codes // 16)[..., None]), -1).flatten(1)[:, :k]
    place = (codes % 8).double()
    value = torch.where(place < 5, place / 2, torch.where(place < 7, place - 2, 6.0)) * (1 - 2 * (codes // 8)).double()
    scales = _powers64(codes.device)[state["w_scales"].long()]
    return (value * scales[:, torch.arange(k, device=codes.device) // BLOCK]).t().contiguous()


def _activated64(y, act):
    if act == "relu":
        return y.clamp(min=0.0)
    if act == "leaky_relu":
        return torch.maximum(y, y * SLOPE)
    if act == "silu":
        return y * torch.special.expit(y)
    if act == "mish_fast":
        return y * torch.tanh(torch.logaddexp(y, torch.zeros_like(y)))
    return y
