"""The 4-bit operators of the framework as measured work: cases, inputs, plain forms, exact values.

Three operators of a served language model whose weights are held in 4 bits:

* ``quantize_fp4`` / ``dequantize_fp4`` -- activations to microscaled 4-bit floating point (E2M1
  codes with E4M3 scales per 16 and an fp32 scale per row, or E8M0 scales per 32) and back;
* ``w4a4_linear`` -- quantise the activations, multiply by 4-bit weights on the tensor cores, bias
  and activation in the epilogue;
* ``moe_layer`` -- a mixture-of-experts layer for a few tokens: router, top-k, the experts'
  gate / up products, SwiGLU, down product and the weighted sum, weights in NVFP4.

The plain form of each is elementary torch in 32 bits (64 where a selection hangs on a border).
Weights are held as a user's program holds them: natural E2M1 codes, and for the GEMM the scale
bytes in tiles of 128 rows x 4 scales.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MIDPOINTS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
MIN_ROW_SCALE = 2.0 ** -120


# ------------------------------------------------------------------------------------- cases

def _round_trip(rows, k, fmt, dtype):
    return {"op": "round_trip", "rows": rows, "k": k, "fmt": fmt, "dtype": dtype}


def _linear(m, n, k, fmt, dtype, out, epilogue):
    return {"op": "linear", "m": m, "n": n, "k": k, "fmt": fmt, "dtype": dtype, "out": out,
            "epilogue": epilogue}


def _moe(tokens, hidden, inter, experts, top_k, scoring, dtype):
    return {"op": "moe", "tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts,
            "top_k": top_k, "scoring": scoring, "dtype": dtype}


def listed():
    return [
        # the values of a few decoded tokens' activations in 4 bits: latency only
        dict(_round_trip(5, 4096, "nvfp4", "bf16"), name="round_trip_decode"),
        # a prompt's activations before the down projection, for an accuracy study of MXFP4
        dict(_round_trip(4099, 14336, "mxfp4", "f32"), name="round_trip_prompt"),
        # one token through the gate / up projection: the weights are read once
        dict(_linear(1, 14336, 4096, "nvfp4", "bf16", "bf16", "none"), name="linear_1_token"),
        # a decode batch through the down projection, MXFP4 weights
        dict(_linear(32, 4096, 14336, "mxfp4", "bf16", "bf16", "bias"), name="linear_32_tokens"),
        # a small batch on a square projection
        dict(_linear(128, 4096, 4096, "nvfp4", "bf16", "f16", "none"), name="linear_128_tokens"),
        # a ragged batch on a ragged layer with bias and activation
        dict(_linear(333, 1000, 1056, "nvfp4", "f32", "bf16", "bias_silu"), name="linear_ragged"),
        # a prompt of 8192 tokens through both projections of an MLP
        dict(_linear(8192, 14336, 4096, "nvfp4", "bf16", "bf16", "none"), name="linear_prefill_up"),
        dict(_linear(8192, 4096, 14336, "mxfp4", "bf16", "bf16", "none"),
             name="linear_prefill_down"),
        # one token through many small experts
        dict(_moe(1, 2048, 768, 64, 8, "softmax", "bf16"), name="moe_1_token"),
        # a few sequences with speculated tokens; sigmoid router with a selection bias
        dict(_moe(7, 4096, 1408, 128, 6, "sigmoid", "f16"), name="moe_7_tokens"),
        # a decode batch that touches nearly every small expert
        dict(_moe(48, 2048, 1024, 128, 8, "softmax", "bf16"), name="moe_48_tokens"),
        # the largest: a full batch on eight large experts
        dict(_moe(64, 4096, 14336, 8, 2, "softmax", "bf16"), name="moe_large_experts"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("round_trip", "linear", "linear", "moe", "moe"))
    fmt = rng.choice(("nvfp4", "mxfp4"))
    if op == "round_trip":
        return _round_trip(_log_int(rng, 1, 4096), _log_int(rng, 32, 14336, 32), fmt,
                           rng.choice(("f32", "bf16", "f16")))
    if op == "linear":
        n = _log_int(rng, 16, 14336, rng.choice((1, 8, 128)))
        return _linear(_log_int(rng, 1, 8192), max(n, 1), _log_int(rng, 32, 4096, 32), fmt,
                       rng.choice(("f32", "bf16", "f16")), rng.choice(("bf16", "f16")),
                       rng.choice(("none", "bias", "bias_relu", "bias_silu", "bias_gelu")))
    experts = _log_int(rng, 4, 128)
    return _moe(_log_int(rng, 1, 64), _log_int(rng, 128, 4096, 128),
                _log_int(rng, 128, 2048, 128), experts, rng.randint(1, min(8, experts)),
                rng.choice(("softmax", "sigmoid")), rng.choice(("bf16", "f16")))


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "round_trip":
        n = case["rows"] * case["k"]
        four = n // 2 + n // (16 if case["fmt"] == "nvfp4" else 32)
        return {"bytes": n * size[case["dtype"]] + 2 * four + 4 * n, "flops": 4 * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        weights = n * k // 2 + n * k // (16 if case["fmt"] == "nvfp4" else 32)
        return {"bytes": m * k * size[case["dtype"]] + weights + m * n * size[case["out"]],
                "flops": 2 * m * n * k}
    t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "inter", "experts", "top_k"))
    touched = e * (1.0 - (1.0 - k / e) ** t)  # experts that at least one token takes
    return {"bytes": touched * 3 * h * i * 9 / 16 + e * h * 2 + t * h * 4,
            "flops": 2 * t * (e * h + k * 3 * h * i)}


# ------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, k, dtype, g):
    """N(0, 1) with one channel in a thousand twenty times as large."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    loud = torch.randperm(k, device="cuda", generator=g)[: max(1, k // 1000)]
    x[:, loud] *= 20.0
    return x.to(DTYPES[dtype])


def _encode(w, fmt):
    """(N, K) fp32 weights -> packed codes (N, K/2), natural scale bytes, tensor scale: round to
    nearest, block maxima near 6 times the block's scale."""
    n, k = w.shape
    block = 16 if fmt == "nvfp4" else 32
    tensor_scale = float(w.abs().max()) / 2688.0 if fmt == "nvfp4" else 1.0
    v = (w / tensor_scale).reshape(n, k // block, block)
    top = v.abs().amax(dim=2) / 6.0
    if fmt == "nvfp4":
        scale = top.clamp(2.0 ** -6, 448.0).to(torch.float8_e4m3fn)
        value, byte = scale.float(), scale.view(torch.uint8)
    else:
        exponent = torch.ceil(torch.log2(top.clamp_min(2.0 ** -40))).clamp(-40, 40)
        value, byte = torch.exp2(exponent), (exponent + 127).to(torch.uint8)
    edges = torch.tensor(MIDPOINTS, device=w.device)
    code = torch.bucketize(v.abs() / value[..., None], edges, out_int32=True).to(torch.uint8)
    code |= (v < 0).to(torch.uint8) << 3
    code = code.reshape(n, k)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte, tensor_scale


def _tile_scales(byte):
    """Natural scale bytes (N, S) -> tiles [N/128][S/4] of 512 bytes: row r of a tile at
    16 (r % 32) + 4 (r / 32), its four scales side by side; zeros where the matrix ends."""
    n, s = byte.shape
    rows, words = -(-n // 128), -(-s // 4)
    full = torch.zeros(rows * 128, words * 4, dtype=torch.uint8, device=byte.device)
    full[:n, :s] = byte
    return full.view(rows, 4, 32, words, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "round_trip":
        return {"case": case, "x": _activations(case["rows"], case["k"], case["dtype"], g)}
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        w = torch.randn(n, k, device="cuda", generator=g) * 0.02
        codes, byte, tensor_scale = _encode(w, case["fmt"])
        bias = None
        if case["epilogue"] != "none":
            bias = torch.randn(n, device="cuda", generator=g).to(torch.bfloat16)
        return {"case": case, "x": _activations(case["m"], k, case["dtype"], g),
                "codes": codes.contiguous(), "scales": _tile_scales(byte),
                "tensor_scale": tensor_scale, "bias": bias}
    t, h, i, e = (case[x] for x in ("tokens", "hidden", "inter", "experts"))
    state = {"case": case, "x": torch.randn(t, h, device="cuda", generator=g).to(
        DTYPES[case["dtype"]])}
    router = torch.randn(e, h, device="cuda", generator=g) * (1.5 / math.sqrt(h))
    state["router"] = router.to(DTYPES[case["dtype"]])
    state["bias"] = None
    if case["scoring"] == "sigmoid":
        state["bias"] = torch.randn(e, device="cuda", generator=g) * 0.05
    for name, n, k in (("gate_up", 2 * i, h), ("down", h, i)):
        codes = torch.empty(e, n, k // 2, dtype=torch.uint8, device="cuda")
        byte = torch.empty(e, n, k // 16, dtype=torch.uint8, device="cuda")
        scale = []
        for j in range(e):
            w = torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)
            codes[j], byte[j], s = _encode(w, "nvfp4")
            scale.append(s)
        state[name] = (codes, byte, torch.tensor(scale, device="cuda"))
    return state


# ------------------------------------------------------------------------------- plain forms

def _e2m1_nearest(a):
    """Nearest E2M1 magnitude of a >= 0, a tie to the lower one."""
    levels = torch.tensor(E2M1, device=a.device)
    return levels[torch.bucketize(a, torch.tensor(MIDPOINTS, device=a.device), out_int32=True)]


def _power_of_two(e):
    """2^e in fp32, exactly, for integer e in [-126, 127]."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize(x, fmt):
    """(rows, K) -> (E2M1 value x block scale, row scale): the rule of quantize_fp4 in 32 bits."""
    rows, k = x.shape
    x = x.float()
    if fmt == "mxfp4":
        b = x.reshape(rows, k // 32, 32)
        mantissa, exponent = torch.frexp(b.abs().amax(dim=2))
        # the smallest e with 6 * 2^e >= amax; amax = mantissa * 2^exponent, mantissa in [.5, 1)
        e = (exponent - 3 + (mantissa > 0.75)).clamp(-40, 40)
        e = torch.where(mantissa == 0, torch.zeros_like(e), e)[..., None]
        y = b * _power_of_two(-e)
        value = torch.copysign(_e2m1_nearest(y.abs()), y) * _power_of_two(e)
        return value.reshape(rows, k), None
    amax = x.abs().amax(dim=1, keepdim=True)
    # divisors as tensors: torch multiplies by the rounded reciprocal of a number
    s = (amax / torch.full_like(amax, 2688.0)).clamp_min(MIN_ROW_SCALE)
    s = torch.where(amax == 0, torch.ones_like(amax), s)
    inverse = 1.0 / s
    b = x.reshape(rows, k // 16, 16)
    top = b.abs().amax(dim=2) * inverse
    # the smallest E4M3 normal B with 6 B >= top: a 3-bit mantissa, compared exactly in 64 bits
    top6 = top.double() / torch.full_like(top, 6.0, dtype=torch.float64)
    mantissa, exponent = torch.frexp(top6)
    scale = torch.ldexp(torch.ceil(mantissa * 16.0), exponent - 4).clamp(2.0 ** -6, 448.0).float()
    scale = torch.where(top == 0, torch.ones_like(scale), scale)[..., None]
    y = b * (inverse[..., None] / scale)
    value = torch.copysign(_e2m1_nearest(y.abs()), y) * scale
    return value.reshape(rows, k), s


def _codes_to_values(codes):
    """Packed nibbles (..., K/2) -> fp32 values (..., K)."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    return table[pair.int()]


def _weights(state, case):
    """The 4-bit weights of a linear case as fp32 values, without the tensor scale."""
    n, k = case["n"], case["k"]
    block = 16 if case["fmt"] == "nvfp4" else 32
    rows, words = -(-n // 128), -(-k // (4 * block))
    byte = state["scales"].view(rows, words, 32, 4, 4).permute(0, 3, 2, 1, 4)
    byte = byte.reshape(rows * 128, words * 4)[:n, : k // block]
    if case["fmt"] == "nvfp4":
        scale = byte.contiguous().view(torch.float8_e4m3fn).float()
    else:
        scale = _power_of_two(byte.int() - 127)
    return (_codes_to_values(state["codes"]).view(n, k // block, block) * scale[..., None]).view(
        n, k)


def _activate(y, epilogue):
    if epilogue == "bias_relu":
        return y.clamp_min(0.0)
    if epilogue == "bias_silu":
        return y / (1.0 + torch.exp(-y))
    if epilogue == "bias_gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(state, case):
    value, row_scale = _quantize(state["x"], case["fmt"])
    y = value @ _weights(state, case).t()
    y = y * state["tensor_scale"] if row_scale is None else y * (row_scale * state["tensor_scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return _activate(y, case["epilogue"]).to(DTYPES[case["out"]])


def _expert_weights(codes, byte, scale):
    """(E, N, K) fp32 weights of all experts."""
    e, n, half = codes.shape
    value = _codes_to_values(codes).view(e, n, half // 8, 16)
    value *= byte.view(torch.float8_e4m3fn).float()[..., None]
    return value.view(e, n, 2 * half) * scale[:, None, None]


def _plain_moe(state, case):
    x, inter = state["x"].float(), case["inter"]
    # the selection in 64 bits: two scores may lie next to one another
    logits = x.double() @ state["router"].double().t()
    score = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    score = score / score.sum(dim=1, keepdim=True)
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    rank_by = logits if state["bias"] is None else score + state["bias"].double()
    ids = torch.sort(rank_by, dim=1, descending=True, stable=True).indices[:, : case["top_k"]]
    weight = score.gather(1, ids)
    weight = (weight / weight.sum(dim=1, keepdim=True)).float()
    gate_up = torch.matmul(x, _expert_weights(*state["gate_up"]).transpose(1, 2))
    gate, up = gate_up[..., :inter], gate_up[..., inter:]
    hidden = gate / (1.0 + torch.exp(-gate)) * up
    y = torch.matmul(hidden, _expert_weights(*state["down"]).transpose(1, 2))
    share = torch.zeros(x.shape[0], case["experts"], device=x.device).scatter_(1, ids, weight)
    y = (y * share.t()[..., None]).sum(dim=0)
    return {"y": y.to(state["x"].dtype), "ids": ids.int(), "weights": weight}


def run(state):
    case = state["case"]
    if own:
        import bitdance_b200 as bd
        if case["op"] == "round_trip":
            return bd.dequantize_fp4(bd.quantize_fp4(state["x"], case["fmt"]))
        if case["op"] == "linear":
            weights = bd.Fp4Operand(state["codes"], state["scales"], case["n"], case["k"],
                                    case["fmt"], tensor_scale=state["tensor_scale"])
            return bd.w4a4_linear(state["x"], weights, bias=state["bias"],
                                  out_dtype=DTYPES[case["out"]], epilogue=case["epilogue"])
        experts = bd.MoeWeights(*state["gate_up"], *state["down"])
        y, ids, weight = bd.moe_layer(state["x"], state["router"], experts, case["top_k"],
                                      scoring=case["scoring"], selection_bias=state["bias"],
                                      return_routing=True)
        return {"y": y, "ids": ids, "weights": weight}
    if case["op"] == "round_trip":
        value, row_scale = _quantize(state["x"], case["fmt"])
        return value if row_scale is None else value * row_scale
    if case["op"] == "linear":
        return _plain_linear(state, case)
    return _plain_moe(state, case)


# ------------------------------------------------------------------------------ exact values

def _f32(v):
    """A 64-bit result rounded once to 32 bits, where the definition stores 32."""
    return v.float().double()


def _exact_quantize(x, fmt):
    """(rows, K) quantised values in 64 bits, block by block from the definition: block scale
    from the list of all scales, code from the distance to every level."""
    rows, k = x.shape
    x = x.double()
    block = 16 if fmt == "nvfp4" else 32
    b = x.view(rows, k // block, block)
    if fmt == "nvfp4":
        amax = x.abs().amax(dim=1)
        s = _f32(amax / torch.full_like(amax, 2688.0)).clamp_min(MIN_ROW_SCALE)
        s = torch.where(amax > 0, s, torch.ones_like(s))
        inverse = _f32(1.0 / s)[:, None]
        top = _f32(b.abs().amax(dim=2) * inverse)
        book = torch.tensor([(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1],
                            dtype=torch.float64, device=x.device)
    else:
        s = torch.ones(rows, dtype=torch.float64, device=x.device)
        inverse = s[:, None]
        top = b.abs().amax(dim=2)
        book = torch.tensor([2.0 ** e for e in range(-40, 41)], dtype=torch.float64,
                            device=x.device)
    pick = torch.searchsorted(6.0 * book, top).clamp_max(book.numel() - 1)
    scale = torch.where(top > 0, book[pick], torch.ones_like(top))
    y = _f32(b * _f32(inverse / scale)[..., None]).abs()
    best = torch.zeros_like(y)
    for lower, upper in zip(E2M1, E2M1[1:]):
        best = torch.where(y - lower > upper - y, torch.full_like(y, upper), best)
    value = best * torch.sign(b) * scale[..., None]
    return value.view(rows, k) * s[:, None]


def _exact_values(codes, scale):
    """Packed codes (N, K/2) and block scales (N, blocks) in 64 bits -> (N, K)."""
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        nibble = ((codes >> (4 * half)) & 15).int()
        level = (nibble & 7).double()
        big = torch.exp2(torch.floor(level / 2) - 1) * (1 + (level % 2) / 2)
        value = torch.where(level < 2, level / 2, big)
        out[:, half::2] = torch.where(nibble >= 8, -value, value)
    return out * scale.repeat_interleave(out.shape[1] // scale.shape[1], dim=1)


def _e4m3_in_64(byte):
    e, m = (byte >> 3).double(), (byte & 7).double()
    return torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e - 7))


def _exact_linear(state, case):
    n, k, fmt = case["n"], case["k"], case["fmt"]
    block = 16 if fmt == "nvfp4" else 32
    row = torch.arange(n, device="cuda")[:, None]
    col = torch.arange(k // block, device="cuda")[None, :]
    words = -(-(k // block) // 4)
    at = ((row // 128) * words + col // 4) * 512 + row % 32 * 16 + row % 128 // 32 * 4 + col % 4
    byte = state["scales"][at]
    scale = _e4m3_in_64(byte) if fmt == "nvfp4" else torch.exp2(byte.double() - 127)
    w = _exact_values(state["codes"], scale) * state["tensor_scale"]
    y = _exact_quantize(state["x"], fmt) @ w.t()
    if state["bias"] is not None:
        y += state["bias"].double()
    if case["epilogue"] == "bias_relu":
        y = torch.relu(y)
    elif case["epilogue"] == "bias_silu":
        y = y * torch.sigmoid(y)
    elif case["epilogue"] == "bias_gelu":
        y = y / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _exact_moe(state, case):
    x, k, inter = state["x"].double(), case["top_k"], case["inter"]
    logits = x @ state["router"].double().t()
    sigmoid = case["scoring"] == "sigmoid"
    score = torch.sigmoid(logits) if sigmoid else torch.softmax(logits, dim=1)
    rank_by = score if state["bias"] is None else score + state["bias"].double()
    index = torch.arange(case["experts"], device=x.device)
    ids = []
    for _ in range(k):
        top = rank_by.amax(dim=1, keepdim=True)
        first = torch.where(rank_by == top, index, case["experts"]).amin(dim=1, keepdim=True)
        rank_by = rank_by.scatter(1, first, -math.inf)
        ids.append(first)
    ids = torch.cat(ids, dim=1)
    weight = score.gather(1, ids)
    weight = weight / weight.sum(dim=1, keepdim=True)
    y = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        w = [_exact_values(state[m][0][e], _e4m3_in_64(state[m][1][e])) * state[m][2][e].double()
             for m in ("gate_up", "down")]
        both = x[token] @ w[0].t()
        hidden = both[:, :inter] * torch.sigmoid(both[:, :inter]) * both[:, inter:]
        y.index_add_(0, token, hidden @ w[1].t() * weight[token, slot, None])
    return {"y": y, "ids": ids.int(), "weights": weight}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "round_trip":
        return _exact_quantize(state["x"], case["fmt"])
    return _exact_linear(state, case) if case["op"] == "linear" else _exact_moe(state, case)
