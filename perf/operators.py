"""The operators of a quantised linear layer, as a program meets them: inputs, one pass, exact values.

  norm      h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight; y in 8 bits with a scale per row
  linear8   out = x_scale[t] * w_scale[n] * sum_k x[t, k] w[n, k], 8-bit operands (int8 or e4m3)
  linear4   out = sum_k x[t, k] * w_scale[n, k / group] * (w[n, k] - zero[n, k / group]), 4-bit weights

`own = False` computes them with elementary torch operations in 32 bits; `own = True` makes the calls of
immerdink_b200."""
import math

import torch

own = False

if torch.cuda.is_available():
    torch.backends.cuda.matmul.allow_tf32 = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one generated token: the layer's input after the residual stream of the block before it
        {"name": "norm_token", "op": "norm", "rows": 1, "dim": 4096, "type": "bf16", "to": "e4m3", "residual": True},
        # sequences that decode together, at the first layer (no residual yet), int8 rows for an int8 product
        {"name": "norm_batch_i8", "op": "norm", "rows": 250, "dim": 5120, "type": "f16", "to": "i8", "residual": False},
        # a long prompt inside a model
        {"name": "norm_prompt", "op": "norm", "rows": 8191, "dim": 8192, "type": "bf16", "to": "e4m3", "residual": True},
        # one token through an int8 projection: the weights' bytes are the whole cost
        {"name": "linear8_token", "op": "linear8", "rows": 1, "n": 6144, "k": 4096, "kind": "i8", "out": "bf16"},
        # a decode batch through a wide e4m3 projection
        {"name": "linear8_batch", "op": "linear8", "rows": 48, "n": 28672, "k": 8192, "kind": "e4m3", "out": "bf16"},
        # a prompt of odd length, odd output width, 16-bit floats out
        {"name": "linear8_ragged", "op": "linear8", "rows": 1999, "n": 5003, "k": 4176, "kind": "e4m3", "out": "f16"},
        # a large prompt batch: tensor-core bound
        {"name": "linear8_prompt", "op": "linear8", "rows": 8192, "n": 8192, "k": 8192, "kind": "i8", "out": "bf16"},
        # one token, symmetric 4-bit weights with groups of 128
        {"name": "linear4_token", "op": "linear4", "rows": 1, "n": 4096, "k": 4096, "group": 128, "zeros": False, "type": "bf16", "out": "bf16"},
        # one token through the widest projection of a large model, groups of 64 with zero points
        {"name": "linear4_token_wide", "op": "linear4", "rows": 1, "n": 28672, "k": 8192, "group": 64, "zeros": True, "type": "f16", "out": "f16"},
        # a small decode batch, fine groups
        {"name": "linear4_batch", "op": "linear4", "rows": 13, "n": 14336, "k": 4096, "group": 32, "zeros": True, "type": "bf16", "out": "f32"},
        # a prompt through 4-bit weights
        {"name": "linear4_prompt", "op": "linear4", "rows": 2048, "n": 8192, "k": 8192, "group": 128, "zeros": False, "type": "bf16", "out": "bf16"},
        # sizes that are multiples of nothing
        {"name": "linear4_odd", "op": "linear4", "rows": 5, "n": 5001, "k": 4091, "group": 64, "zeros": False, "type": "f16", "out": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear8", "linear4"])
    if op == "norm":
        dim = _log(rng, 64, 16384)
        dim = dim if rng.random() < 0.3 else max(8, dim // 8 * 8)
        return {"op": op, "rows": _log(rng, 1, min(16384, 67_000_000 // dim)), "dim": dim, "type": rng.choice(["bf16", "f16", "f32"]),
                "to": rng.choice(["e4m3", "e4m3", "i8"]), "residual": rng.random() < 0.7}
    k = _log(rng, 128, 28672)
    n = _log(rng, 64, min(28672, 234_000_000 // k))
    if op == "linear8":
        if rng.random() < 0.85:  # rows of whole 16-byte units, as weights are stored; the others are multiples of nothing
            k = k // 16 * 16
        rows = _log(rng, 1, min(8192, 540_000_000_000 // (n * k)))
        return {"op": op, "rows": rows, "n": n, "k": k, "kind": rng.choice(["i8", "e4m3"]), "out": rng.choice(["bf16", "f16", "f32"])}
    if rng.random() < 0.7:
        k = max(128, k // 128 * 128)
    rows = _log(rng, 1, min(2048, 137_000_000_000 // (n * k)))
    if rng.random() < 0.4:
        rows = min(rows, rng.randint(1, 16))
    return {"op": op, "rows": rows, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
            "type": rng.choice(["bf16", "f16"]), "out": rng.choice(["same", "f32"])}


def _out_type(case):
    return TYPES[case["type"] if case["out"] == "same" else case["out"]]


def _value_type(case):
    """The 16-bit type that int8 codes times their scale are handed back in."""
    return TYPES["bf16" if case["type"] == "f32" else case["type"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    rows = case["rows"]
    s = {"case": case}
    if case["op"] == "norm":
        dim, t = case["dim"], TYPES[case["type"]]
        x = normal(rows, dim)
        # a few channels are much larger than the others, as in a trained model's residual stream
        x[:, torch.randint(dim, (max(1, dim // 512),), generator=g, device="cuda")] *= 20.0
        s["x"] = x.to(t)
        s["residual"] = (normal(rows, dim) * 3.0).to(t) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * normal(dim)).to(t)
        s["h"] = torch.empty(rows, dim, dtype=t, device="cuda") if case["residual"] else None
        s["q"] = torch.empty(rows, dim, dtype=torch.int8 if case["to"] == "i8" else torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty(rows, dtype=torch.float32, device="cuda")
        s["values"] = torch.empty(rows, dim, dtype=_value_type(case), device="cuda") if case["to"] == "i8" else None
        return s
    n, k = case["n"], case["k"]
    s["y"] = torch.empty(rows, n, dtype=_out_type(case), device="cuda")
    if case["op"] == "linear8":
        if case["kind"] == "i8":
            s["x"] = (normal(rows, k) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
            s["w"] = (normal(n, k) * 32.0).round_().clamp_(-127, 127).to(torch.int8)
        else:
            s["x"] = (normal(rows, k) * 100.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
            s["w"] = (normal(n, k) * 100.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s["x_scale"] = 0.01 + 0.02 * torch.rand(rows, generator=g, device="cuda")
        s["w_scale"] = (0.5 + torch.rand(n, generator=g, device="cuda")) * (0.001 / math.sqrt(k))
        return s
    groups = -(-k // case["group"])
    s["x"] = normal(rows, k).to(TYPES[case["type"]])
    s["w"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    s["w_scale"] = ((0.5 + torch.rand(n, groups, generator=g, device="cuda")) * (0.2 / math.sqrt(k))).to(TYPES[case["type"]])
    s["zeros"] = torch.randint(4, 12, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return s


def run(s):
    case = s["case"]
    if own:
        import immerdink_b200 as imd
        if case["op"] == "norm":
            imd.norm_quantize(s["x"], s["weight"], s["q"], s["scale"], eps=EPS, residual=s["residual"], residual_out=s["h"])
            # int8 codes are handed back as the values they stand for
            q = s["q"] if case["to"] == "e4m3" else torch.mul(s["q"], s["scale"][:, None], out=s["values"])
            return [q, s["scale"], s["h"]]
        if case["op"] == "linear8":
            return imd.scaled_linear(s["x"], s["w"], s["y"], s["x_scale"], s["w_scale"])
        return imd.linear_w4(s["x"], s["w"], s["y"], s["w_scale"], zeros=s["zeros"], group=case["group"])
    if case["op"] == "norm":
        h = s["x"].float()
        stored = None
        if s["residual"] is not None:
            h = h + s["residual"].float()
            stored = h.to(s["x"].dtype)
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
        top = y.abs().amax(1, keepdim=True)
        if case["to"] == "e4m3":
            return [(y * (448.0 / top)).clamp(-448, 448).to(torch.float8_e4m3fn), top[:, 0] / 448.0, stored]
        scale = top / 127.0
        return [((y * (127.0 / top)).round() * scale).to(_value_type(case)), scale[:, 0], stored]
    if case["op"] == "linear8":
        y = s["x"].float() @ s["w"].float().t()
        return (y * s["x_scale"][:, None] * s["w_scale"]).to(s["y"].dtype)
    k, group = case["k"], case["group"]
    q = torch.stack((s["w"] & 15, s["w"] >> 4), 2).flatten(1)[:, :k].float()
    at = torch.arange(k, device="cuda") // group
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, at]
    return (s["x"].float() @ ((q - zero) * s["w_scale"].float()[:, at]).t()).to(s["y"].dtype)


def work(case):
    rows = case["rows"]
    if case["op"] == "norm":
        b = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
        each = b * (3 if case["residual"] else 1) + 1
        return {"bytes": rows * case["dim"] * each + b * case["dim"] + 4 * rows, "flops": 8 * rows * case["dim"]}
    n, k = case["n"], case["k"]
    out = rows * n * torch.empty(0, dtype=_out_type(case)).element_size()
    if case["op"] == "linear8":
        return {"bytes": (rows + n) * k + 4 * (rows + n) + out, "flops": 2 * rows * n * k}
    groups = -(-k // case["group"])
    return {"bytes": 2 * rows * k + n * ((k + 1) // 2) + n * groups * (3 if case["zeros"] else 2) + out, "flops": 2 * rows * n * k}


def exact(case, seed):
    """From the definitions, in 64 bits. The 8-bit codes of `norm` are rounded to the nearest code, ties to the even one,
    so that they stand for the same values; they follow from the row's scale."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "norm":
        if s["residual"] is not None:
            x = x + s["residual"].double()
        y = s["weight"].double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
        largest = y.abs().max(-1, keepdim=True).values
        if case["to"] == "i8":
            step = largest / 127
            codes = torch.round(y / step) * step
        else:
            # e4m3: 4 significant bits, exponents from -6 (2^-9 is the smallest step) to 8
            v = y * 448 / largest
            _, e = torch.frexp(v)
            step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
            codes = torch.round(v / step) * step
        return [codes, (largest / (127 if case["to"] == "i8" else 448))[:, 0], x if s["residual"] is not None else None]
    if case["op"] == "linear8":
        return torch.einsum("tk,nk->tn", x * s["x_scale"].double()[:, None], s["w"].double() * s["w_scale"].double()[:, None])
    n, k, group = case["n"], case["k"], case["group"]
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2] = (s["w"] % 16).double()[:, :(k + 1) // 2]
    w[:, 1::2] = (s["w"] // 16).double()[:, :k // 2]
    w -= 8.0 if s["zeros"] is None else s["zeros"].double().repeat_interleave(group, 1)[:, :k]
    w *= s["w_scale"].double().repeat_interleave(group, 1)[:, :k]
    return torch.einsum("tk,nk->tn", x, w)
