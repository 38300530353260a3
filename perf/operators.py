"""Cases of the 8-bit activation operators: what they compute, in plain torch, and how they are called.

Training keeps activations of the forward pass for the backward pass.  Kept in 8 bits they are
E4M3 numbers with one power-of-two scale for every block of 128 consecutive features of a row:

    k = the smallest integer with  max |x| <= 448 * 2^k  in the block, limited to -117 .. 119
    q = x / 2^k rounded to E4M3 (nearest even);    the value kept is  q * 2^k

The operators:

  pack        x -> (values, exponents) and back: an activation's way through the checkpoint
  norm_fwd    h = x + residual, n = h / sqrt(mean(h^2) + eps), y = n * weight; n is kept in 8 bits,
              and read back as n * weight (what the linear layers behind the norm take as input)
  norm_bwd    the gradients of the norm from n in 8 bits
  wgrad       a linear layer's weight gradient  grad_out^T . input  from the input in 8 bits

Sums and statistics are held in 32 bits and every output is rounded once.
"""

import math
import random

import torch

own = False

BLOCK = 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
MOST_ELEMENTS = 8192 * 14336
MOST_FLOPS = 2 * 8192 * 14336 * 4096


def listed():
    return [
        # a micro-batch of a few tokens in single precision: the call itself is the cost
        {"name": "pack fp32 16x768", "op": "pack", "dtype": "fp32", "rows": 16, "features": 768, "row_pad": 0},
        # a view into a wider projection whose rows start at odd places
        {"name": "pack fp32 2047x1001 strided", "op": "pack", "dtype": "fp32", "rows": 2047, "features": 1001, "row_pad": 24},
        # the input of an 8-billion-parameter model's down projection, 8192 tokens
        {"name": "pack bf16 8192x14336", "op": "pack", "dtype": "bf16", "rows": 8192, "features": 14336, "row_pad": 0},
        # one short sequence of a small model, no residual stream (the first norm)
        {"name": "norm_fwd fp32 33x768", "op": "norm_fwd", "dtype": "fp32", "rows": 33, "features": 768, "residual": False, "row_pad": 0},
        # a ragged batch with a hidden size that is no multiple of the block
        {"name": "norm_fwd fp16 5001x1000", "op": "norm_fwd", "dtype": "fp16", "rows": 5001, "features": 1000, "residual": True, "row_pad": 0},
        # the norm before a block's projections, 16384 tokens
        {"name": "norm_fwd bf16 16384x4096", "op": "norm_fwd", "dtype": "bf16", "rows": 16384, "features": 4096, "residual": True, "row_pad": 0},
        # the same norms on the way back
        {"name": "norm_bwd fp32 257x2048", "op": "norm_bwd", "dtype": "fp32", "rows": 257, "features": 2048, "residual": False, "row_pad": 0},
        {"name": "norm_bwd bf16 8192x4096", "op": "norm_bwd", "dtype": "bf16", "rows": 8192, "features": 4096, "residual": True, "row_pad": 0},
        # a projection of a small model, fp16 with a scaled loss
        {"name": "wgrad fp16 64x768x768", "op": "wgrad", "dtype": "fp16", "rows": 64, "out": 768, "features": 768, "scaled": False, "row_pad": 0},
        # a classifier with an odd number of classes in single precision
        {"name": "wgrad fp32 1000x1001x768", "op": "wgrad", "dtype": "fp32", "rows": 1000, "out": 1001, "features": 768, "scaled": False, "row_pad": 0},
        # key or value projection behind a norm: few output tiles, a long sum
        {"name": "wgrad bf16 4096x1024x4096", "op": "wgrad", "dtype": "bf16", "rows": 4096, "out": 1024, "features": 4096, "scaled": True, "row_pad": 0},
        # gate or up projection, 8192 tokens: the largest product of a layer
        {"name": "wgrad bf16 8192x14336x4096", "op": "wgrad", "dtype": "bf16", "rows": 8192, "out": 14336, "features": 4096, "scaled": True, "row_pad": 0},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """Spread over the logarithm; half of them multiples of 64 as models have them, the rest as they fall."""
    n = _log_uniform(rng, low, high)
    return max(low, n // 64 * 64) if n >= 64 and rng.random() < 0.5 else n


def draw(rng: random.Random):
    op = rng.choice(["pack", "norm_fwd", "norm_bwd", "wgrad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = _size(rng, 1, 16384)
    features = _size(rng, 16, 14336)
    case = {"op": op, "dtype": dtype, "rows": rows, "features": features,
            "row_pad": rng.choice([0, 0, 0, 8, 64, 3])}
    if op == "wgrad":
        case["out"] = _size(rng, 16, 14336)
        case["scaled"] = rng.random() < 0.5
        most = MOST_FLOPS // (4 if dtype == "fp32" else 2 if dtype == "fp16" else 1)
        if 2 * rows * features * case["out"] > most:
            case["rows"] = max(1, most // (2 * features * case["out"]))
    else:
        if op != "pack":
            case["residual"] = rng.random() < 0.6
        most = MOST_ELEMENTS // (2 if dtype == "fp32" else 1) // (1 if op == "pack" else 2)
        if rows * features > most:
            case["rows"] = max(1, most // features)
    return case


# --- inputs -----------------------------------------------------------------------------------


def _device():
    return torch.device("cuda", 0)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=_device(), dtype=torch.float32)


def _strided(values, dtype, row_pad):
    """The values with ``row_pad`` elements of other data behind every row."""
    rows, n = values.shape
    if not row_pad:
        return values.to(dtype)
    wide = torch.full((rows, n + row_pad), 7.0, device=values.device, dtype=dtype)
    wide[:, :n] = values
    return wide[:, :n]


def _activations(gen, rows, features):
    """Rows of differing size with a few features that stand out, as hidden states have them."""
    x = _normal(gen, rows, features)
    x *= torch.exp(0.5 * _normal(gen, features))
    x[:, :: max(1, features // 5)] *= 12.0
    x *= torch.exp(0.3 * _normal(gen, rows, 1))
    return x


def _gradients(gen, rows, n, dtype):
    """Small gradients; every seventh token is masked out of the loss."""
    g = _normal(gen, rows, n) * (0.02 if dtype == "fp16" else 1e-3)
    g *= torch.exp(0.5 * _normal(gen, rows, 1))
    if rows >= 7:
        g[::7] = 0.0
    return g


def _blocks(features):
    return -(-features // BLOCK)


def _pitch(features):
    """Rows of kept values start at multiples of 16 bytes."""
    return -(-features // 16) * 16


def _quantise(x):
    """(q as fp32 numbers, k) of fp32 rows."""
    rows, features = x.shape
    nb = _blocks(features)
    x = torch.nn.functional.pad(x, (0, nb * BLOCK - features)).view(rows, nb, BLOCK)
    m, p = torch.frexp(x.abs().amax(dim=2))
    k = (p - 9 + (m > 0.875).to(p.dtype)).clamp(-117, 119)
    q = torch.ldexp(x, -k.unsqueeze(2)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return q.view(rows, nb * BLOCK)[:, :features], k


def _kept(x):
    """What x becomes in 8 bits, in fp32."""
    q, k = _quantise(x)
    return torch.ldexp(q, k.repeat_interleave(BLOCK, dim=1)[:, : x.shape[1]])


def _stored(x):
    """(values [rows, pitch] E4M3, exponents [rows, blocks] uint8) of fp32 rows, as they are kept."""
    q, k = _quantise(x)
    values = torch.zeros(x.shape[0], _pitch(x.shape[1]), device=x.device, dtype=torch.float32)
    values[:, : x.shape[1]] = q
    return values.to(torch.float8_e4m3fn), (k + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(seed)
    dtype, rows, features = DTYPES[case["dtype"]], case["rows"], case["features"]
    state = {"case": dict(case)}
    if case["op"] == "pack":
        state["x"] = _strided(_activations(gen, rows, features), dtype, case["row_pad"])
        return state
    weight = 1.0 + 0.2 * _normal(gen, features)
    if case["op"] == "norm_fwd":
        state["x"] = _strided(_activations(gen, rows, features), dtype, case["row_pad"])
        state["residual"] = _activations(gen, rows, features).to(dtype) if case["residual"] else None
        state["weight"] = weight.to(dtype)
        return state
    h = _activations(gen, rows, features)
    rstd = torch.rsqrt(h.square().mean(dim=1) + EPS)
    state["values"], state["exponents"] = _stored(h * rstd[:, None])
    if case["op"] == "norm_bwd":
        state["rstd"] = rstd
        state["weight"] = weight.to(dtype)
        state["grad_y"] = _strided(_gradients(gen, rows, features, case["dtype"]), dtype, case["row_pad"])
        state["grad_h"] = _gradients(gen, rows, features, case["dtype"]).to(dtype) if case["residual"] else None
    else:
        state["weight"] = weight.to(dtype) if case["scaled"] else None
        state["grad_out"] = _strided(_gradients(gen, rows, case["out"], case["dtype"]), dtype, case["row_pad"])
    return state


# --- one pass ---------------------------------------------------------------------------------


def _read_back(state):
    """The kept input in fp32 (exact: an E4M3 number times a power of two)."""
    features = state["case"]["features"]
    k = state["exponents"].to(torch.int32) - 127
    return torch.ldexp(state["values"][:, :features].float(), k.repeat_interleave(BLOCK, dim=1)[:, :features])


def _run_plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "pack":
        return _kept(state["x"].float()).to(dtype)
    if case["op"] == "norm_fwd":
        h = state["x"]
        if state["residual"] is not None:
            h = (h.float() + state["residual"].float()).to(dtype)
        wide, w = h.float(), state["weight"].float()
        rstd = torch.rsqrt(wide.square().mean(dim=1) + EPS)
        n = wide * rstd[:, None]
        out = {"y": (n * w).to(dtype), "rstd": rstd, "kept": (_kept(n) * w).to(torch.bfloat16)}
        if state["residual"] is not None:
            out["h"] = h
        return out
    x = _read_back(state)
    if case["op"] == "norm_bwd":
        gy = state["grad_y"].float()
        g = gy * state["weight"].float()
        gx = state["rstd"][:, None] * (g - x * (g * x).mean(dim=1, keepdim=True))
        if state["grad_h"] is not None:
            gx = gx + state["grad_h"].float()
        return {"grad_x": gx.to(dtype), "grad_weight": (gy * x).sum(dim=0).to(dtype)}
    if state["weight"] is not None:
        x = x * state["weight"].float()
    return (state["grad_out"].float().t() @ x).to(dtype)


def _run_own(state):
    from torchft_amd import activations

    case = state["case"]
    if case["op"] == "pack":
        return activations.pack(state["x"]).unpack()
    if case["op"] == "norm_fwd":
        y, h, kept, rstd = activations.rms_norm_forward(
            state["x"], state["weight"], EPS, residual=state["residual"])
        out = {"y": y, "rstd": rstd, "kept": kept.unpack(torch.bfloat16)}
        if state["residual"] is not None:
            out["h"] = h
        return out
    kept = activations.PackedActivation(
        state["values"], state["exponents"], case["features"], column_scale=state["weight"])
    if case["op"] == "norm_bwd":
        gx, gw = activations.rms_norm_backward(
            state["grad_y"], kept, state["rstd"], grad_h=state["grad_h"])
        return {"grad_x": gx, "grad_weight": gw}
    return activations.linear_weight_grad(state["grad_out"], kept)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    rows, features, size = case["rows"], case["features"], SIZE[case["dtype"]]
    n = rows * features
    kept = n + rows * _blocks(features)
    if case["op"] == "pack":  # x in, kept out; kept in, x out
        return {"bytes": 2 * (n * size + kept), "flops": 4 * n}
    if case["op"] == "norm_fwd":  # reading back what was kept: kept in, 16 bits out
        streams = 4 if case["residual"] else 2
        return {"bytes": streams * n * size + kept + 4 * rows + features * size + kept + 2 * n, "flops": 8 * n}
    if case["op"] == "norm_bwd":
        streams = 3 if case["residual"] else 2
        return {"bytes": streams * n * size + kept + 4 * rows + 2 * features * size, "flops": 10 * n}
    return {"bytes": rows * case["out"] * size + kept + case["out"] * features * size,
            "flops": 2 * n * case["out"]}


# --- the same from the definition, in 64 bits ---------------------------------------------------


def _in_8_bits(x):
    """Nearest kept value of every element of fp64 rows: the block's scale by comparison with
    448 * 2^k, the grid of E4M3 from the binary exponent (steps of 2^-3 of it, none below 2^-9)."""
    out = torch.empty_like(x)
    for start in range(0, x.shape[1], BLOCK):
        b = x[:, start:start + BLOCK]
        top = b.abs().amax(dim=1, keepdim=True)
        k = torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / 448.0))
        k = torch.where(top > 448.0 * torch.exp2(k), k + 1, k)
        k = torch.where(top <= 448.0 * torch.exp2(k - 1), k - 1, k).clamp(-117, 119)
        v = (b / torch.exp2(k)).clamp(-448.0, 448.0)
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        out[:, start:start + BLOCK] = torch.round(v / step) * step * torch.exp2(k)
    return out


def _kept_in_64(state):
    values = state["values"].double()[:, : state["case"]["features"]]
    return torch.cat([values[:, j * BLOCK:(j + 1) * BLOCK] * torch.exp2(state["exponents"][:, j:j + 1].double() - 127)
                      for j in range(state["exponents"].shape[1])], dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        return _in_8_bits(s["x"].double())
    if case["op"] == "norm_fwd":
        h = s["x"]
        if s["residual"] is not None:  # what is normed is the rounded sum
            h = (h.double() + s["residual"].double()).to(h.dtype)
        root = (h.double().pow(2).sum(dim=1) / case["features"] + EPS).sqrt()
        n = h.double() / root[:, None]
        w = s["weight"].double()
        out = {"y": n * w, "rstd": 1.0 / root, "kept": _in_8_bits(n) * w}
        if s["residual"] is not None:
            out["h"] = s["x"].double() + s["residual"].double()
        return out
    n = _kept_in_64(s)
    if case["op"] == "norm_bwd":
        gy = s["grad_y"].double()
        g = gy * s["weight"].double()
        gx = (g - n * ((g * n).sum(dim=1, keepdim=True) / case["features"])) * s["rstd"].double()[:, None]
        if s["grad_h"] is not None:
            gx += s["grad_h"].double()
        return {"grad_x": gx, "grad_weight": torch.einsum("td,td->d", gy, n)}
    out = torch.mm(s["grad_out"].double().t().contiguous(), n)
    return out if s["weight"] is None else out * s["weight"].double()
