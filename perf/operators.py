"""The operators on tokens and on channels-last tensors, as cases to time: per-token int8 quantization, the int8 product
with scales for each token and channel, group norm with an activation, and a norm whose int8 tokens a product reads.

listed() and draw() describe cases as plain dicts; prepare() makes what a program holds before the call, run() is one pass,
in plain torch operations or (`own`) by the calls of tennis_amd.capi, work() the bytes and operations that a pass cannot do
without, exact() the operators' definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One token of a serving step: the call itself is most of the time.
        {"name": "quantize one token", "kind": "quantize_tokens", "m": 1, "k": 4096, "type": "bf16", "extra": 0},
        # The tokens of a long prompt, a column range of a wider buffer, as a projection's output is handed on.
        {"name": "quantize 8192 tokens", "kind": "quantize_tokens", "m": 8192, "k": 4096, "type": "bf16", "extra": 128},
        # One token through a square projection: the weights are all there is to read.
        {"name": "product one token", "kind": "token_product", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False, "act": "none", "extra": 0},
        # The classifier of a ResNet-50 on its serving batch.
        {"name": "product classifier", "kind": "token_product", "m": 32, "n": 1000, "k": 2048, "type": "f16", "bias": True, "act": "none", "extra": 0},
        # Sizes that are no multiple of any tile, fp32 in and out, rows at odd addresses.
        {"name": "product ragged", "kind": "token_product", "m": 777, "n": 1111, "k": 1500, "type": "f32", "bias": True, "act": "relu", "extra": 3},
        # A prompt through a square projection.
        {"name": "product 4096", "kind": "token_product", "m": 4096, "n": 4096, "k": 4096, "type": "bf16", "bias": True, "act": "silu", "extra": 0},
        # A large batch of prompts through a large layer: the largest pass.
        {"name": "product 8192", "kind": "token_product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False, "act": "none", "extra": 0},
        # The innermost map of a denoising network on two images.
        {"name": "norm 8x8x1280", "kind": "group_norm", "batch": 2, "h": 8, "w": 8, "c": 1280, "groups": 32, "type": "bf16", "act": "silu"},
        # Its outermost map on a serving batch: groups of ten channels.
        {"name": "norm 64x64x320", "kind": "group_norm", "batch": 8, "h": 64, "w": 64, "c": 320, "groups": 32, "type": "f16", "act": "silu"},
        # An image decoder's last maps, larger than the caches.
        {"name": "norm 512x512x128", "kind": "group_norm", "batch": 4, "h": 512, "w": 512, "c": 128, "groups": 32, "type": "bf16", "act": "silu"},
        # A norm and the projection of its pixels to queries, keys and values, on few pixels ...
        {"name": "norm and product 16x16", "kind": "norm_product", "batch": 2, "h": 16, "w": 16, "c": 1280, "groups": 32, "n": 3840, "type": "bf16", "act": "none"},
        # ... and on a serving batch of larger maps.
        {"name": "norm and product 64x64", "kind": "norm_product", "batch": 8, "h": 64, "w": 64, "c": 320, "groups": 32, "n": 960, "type": "bf16", "act": "none"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize_tokens", "token_product", "token_product", "token_product", "group_norm", "group_norm", "norm_product"])
    kind_type = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "quantize_tokens":
        k = _log_int(rng, 1, 16384)
        return {"kind": kind, "m": _log_int(rng, 1, max(2, 33554432 // k)), "k": k, "type": kind_type, "extra": rng.choice([0, 0, 1, 8, 64])}
    if kind == "token_product":
        return {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 1, 8192), "k": _log_int(rng, 1, 8192), "type": kind_type,
                "bias": rng.choice([True, False]), "act": rng.choice(["none", "relu", "leaky_relu", "silu", "mish_fast"]),
                "extra": rng.choice([0, 0, 1, 8, 64])}
    groups = rng.choice([1, 2, 3, 8, 16, 32])
    c = groups * _log_int(rng, 1, 1 + 1280 // groups)
    batch = _log_int(rng, 1, 16)
    side = _log_int(rng, 1, max(1, int(math.sqrt((134217728 if kind == "group_norm" else 16777216) / (batch * c)))))
    side = min(side, 512)
    case = {"kind": kind, "batch": batch, "h": side, "w": max(1, side - rng.choice([0, 0, 1, 3])), "c": c, "groups": groups, "type": kind_type,
            "act": rng.choice(["none", "relu", "leaky_relu", "silu", "mish_fast"])}
    if kind == "norm_product":
        case["n"] = _log_int(rng, 16, 4096)
        case["type"] = rng.choice(["f16", "bf16"])      # fp32 values next to a rounding border of int8 go either way
    return case


# ---------------------------------------------------------------------------------------------- what a program holds

SLOPE = 0.1
EPSILON = 1e-5


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32) * (hi - lo) + lo
    t = _TYPES[case["type"]]
    state = {"case": case}
    if case["kind"] in ("quantize_tokens", "token_product"):
        m, k = case["m"], case["k"]
        # activations: tokens of different size, a few channels far larger than the others
        x = normal(m, k + case["extra"]) * torch.exp(0.5 * normal(m, 1))
        x *= torch.where(uniform(0, 1, k + case["extra"]) < 0.01, 8.0, 1.0)
        state["x"] = x.to(t)[:, :k]
    else:
        b, h, w, c = case["batch"], case["h"], case["w"], case["c"]
        x = normal(b, h, w, c)
        x *= uniform(0.5, 2.0, c)
        x += normal(c)
        state["x"] = x.to(t)
        state["gamma"], state["beta"] = 1.0 + 0.2 * normal(c), 0.2 * normal(c)
        k = c
    if case["kind"] in ("token_product", "norm_product"):
        # weights as a quantized layer stores them: int8 [n][k] with a scale for each of the n channels
        w = normal(case["n"], k)
        w /= w.abs().amax(1, keepdim=True)
        state["w"] = (w * 127.0).round().to(torch.int8)
        state["w_scales"] = uniform(0.5, 1.5, case["n"]) * (3.0 / 127.0 / math.sqrt(k))
        state["bias"] = normal(case["n"]) if case.get("bias") else None
    return state


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from tennis_amd import capi
    case, x = state["case"], state["x"]
    if "w" in state and "layer" not in state:      # a program makes the layer once and keeps it: its weights packed
        state["layer"] = capi.TokenGemmI8(state["w"], state["w_scales"], bias=state["bias"])
    if case["kind"] == "quantize_tokens":
        return capi.quantize_tokens(x)
    if case["kind"] == "token_product":
        return state["layer"](x, act=case["act"], slope=SLOPE)
    if case["kind"] == "group_norm":
        return capi.group_norm(x, case["groups"], state["gamma"], state["beta"], EPSILON, act=case["act"], slope=SLOPE)
    q, scales = capi.group_norm_tokens(x, case["groups"], state["gamma"], state["beta"], EPSILON, act=case["act"], slope=SLOPE)
    return state["layer"](q, x_scales=scales, out_dtype=x.dtype)


def _run_plain(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "quantize_tokens":
        return _quantized(x.float())
    if case["kind"] == "token_product":
        return _product(state, x.float(), case["act"]).to(x.dtype)
    y = _normed(x, state["gamma"], state["beta"], case["groups"], case["act"])
    if case["kind"] == "group_norm":
        return y.to(x.dtype)
    return _product(state, y, "none").to(x.dtype)


def _quantized(x):
    # 64 bits: the product is rounded to a whole number once
    top = x.abs().amax(-1, keepdim=True)
    lift = torch.where(top < 2.0 ** -64, 2.0 ** 64, 1.0)
    reciprocal = (127.0 / (top.double() * lift)).float()
    reciprocal = torch.where((top > 0) & torch.isfinite(top), reciprocal, torch.zeros_like(reciprocal))
    q = torch.where(torch.isfinite(top), (x.double() * lift) * reciprocal.double(), 0.0)
    scales = torch.where(torch.isfinite(top), (top.double() / 127.0).float(), math.nan)
    return torch.round(q).to(torch.int8), scales.squeeze(-1)


def _product(state, x, act):
    q, scales = _quantized(x)
    y = torch.matmul(q.float(), state["w"].float().t()) * state["w_scales"] * scales.unsqueeze(-1)
    if state["bias"] is not None:
        y = y + state["bias"]
    return _activated(y, act)


def _normed(x, gamma, beta, groups, act):
    b, c = x.shape[0], x.shape[-1]
    v = x.float().reshape(b, -1, groups, c // groups)
    d = v - v.mean((1, 3), keepdim=True)
    y = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + EPSILON)
    return _activated(y.reshape(x.shape) * gamma + beta, act)


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
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "quantize_tokens":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (size + 1) + 4 * m, "flops": 2 * m * k}
    if case["kind"] == "token_product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * size + n * k + n * (8 if case["bias"] else 4) + m * n * size, "flops": 2 * m * n * k}
    pixels, c = case["batch"] * case["h"] * case["w"], case["c"]
    if case["kind"] == "group_norm":
        return {"bytes": 2 * pixels * c * size + 8 * c, "flops": 8 * pixels * c}
    n = case["n"]
    return {"bytes": pixels * c * size + 8 * c + n * c + 4 * n + pixels * n * size, "flops": 2 * pixels * n * c + 8 * pixels * c}


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"].double()
    if case["kind"] == "quantize_tokens":
        return _tokens64(x)
    if case["kind"] != "token_product":
        b, c, groups = case["batch"], case["c"], case["groups"]
        flat = x.view(b, -1, groups, c // groups).transpose(1, 2).reshape(b * groups, -1)
        count = flat.shape[1]
        mean = flat.sum(1) / count
        variance = (flat - mean[:, None]).square_().sum(1) / count
        scale = (1.0 / torch.sqrt(variance + EPSILON)).view(b, groups, 1) * state["gamma"].double().view(1, groups, -1)
        shift = state["beta"].double().view(1, groups, -1) - mean.view(b, groups, 1) * scale
        del flat
        x = x.view(b, -1, c) * scale.view(b, 1, c) + shift.view(b, 1, c)
        x = _activated64(x, case["act"]).view(case["batch"], case["h"], case["w"], c)
        if case["kind"] == "group_norm":
            return x
    q, scales = _tokens64(x)
    y = (q.double().view(-1, q.shape[-1]) @ state["w"].double().t().contiguous()).view(q.shape[:-1] + (case["n"],))
    y *= scales[..., None]
    y *= state["w_scales"].double()
    if case["kind"] == "norm_product":
        return y
    if state["bias"] is not None:
        y += state["bias"].double()
    return _activated64(y, case["act"])


def _tokens64(x):
    # the multiplier is defined as the fp32 number next to 127 / max; the products with it are exact in 64 bits
    top = x.abs().max(-1).values
    lift = 1.0 + (top < 2.0 ** -64).double() * (2.0 ** 64 - 1.0)
    multiplier = torch.where(top > 0, 127.0 / (top * lift).clamp(min=1e-300), 0.0).to(torch.float32).double()
    return (x * lift[..., None] * multiplier[..., None]).round().to(torch.int8), top / 127.0


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
