"""Performance cases of microscaled 4-bit floating point and of the norms around a block.

A program whose weights are kept in blocks of 32 e2m1 codes with a power of two each makes four kinds
of call: it turns rows into such blocks (`quantize_mx4`, read back through `dequant_mx4`), multiplies
rows that it has in blocks already (`linear_mx4`: gate and up share them) or rows of floats
(`linear_mx4_fused`), and passes from one block of a layer to the next (`block_norm`: the norm behind a
block, its gate, the scaled residual, the norm in front of the next one).  `draw` spreads over the same
ranges.

codes [rows, k/2]: element 2j in the low nibble of byte j; nibble = sign, two bits of exponent, one of
mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  scales [rows, k/32]: byte E stands for 2^(E - 127).
"""
from __future__ import annotations

import math

import torch

own = False

_DEVICE = "cuda"
_DTYPES = {"f16": torch.float16, "f32": torch.float32}
_SIZES = {"f16": 2, "f32": 4}
_EPS = 1e-5


# ---------------------------------------------------------------------------------- the cases
def _quantize(name, rows, dim, rule, io):
    return {"name": name, "op": "quantize", "rows": rows, "dim": dim, "rule": rule, "io": io}


def _norm(name, rows, dim, post, gate, span, io, norm):
    """`span` rows share a row of gates (0: all of them)."""
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "post": post, "gate": gate,
            "span": span, "io": io, "norm": norm}


def _linear(name, m, n, k, pairs, bias, residual, rule, io, out):
    """`n` rows of weights; `pairs`: they are (gate, up) in turn, and silu(gate) * up comes out."""
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "pairs": pairs, "bias": bias,
            "residual": residual, "rule": rule, "io": io, "out": out}


def _product(name, m, n, k, pairs, bias, residual, out):
    return {"name": name, "op": "product", "m": m, "n": n, "k": k, "pairs": pairs, "bias": bias,
            "residual": residual, "rule": "floor", "io": "f32", "out": out}


def listed():
    return [
        # the rows of a decode batch: latency alone
        _quantize("quantize_decode", 16, 4096, "floor", "f16"),
        # the rows of a long prompt in front of a down projection, f32, without clipping
        _quantize("quantize_prompt", 4099, 11008, "ceil", "f32"),
        # one token between attention and feed-forward of the default decoder shape
        _norm("norm_decode", 1, 2048, True, "none", 0, "f16", "f16"),
        # a prompt's rows between two blocks
        _norm("norm_prompt", 8192, 4096, True, "none", 0, "f16", "f16"),
        # f32 rows whose block is gated element by element, into fp16 for the next product
        _norm("norm_gated", 1023, 5632, False, "sigmoid", 1, "f32", "f16"),
        # one token through a square projection: the smallest product
        _linear("linear_decode", 1, 4096, 4096, False, False, False, "floor", "f16", "f16"),
        # eight tokens through gate and up
        _linear("linear_gate_up", 8, 22016, 4096, True, False, False, "floor", "f16", "f16"),
        # 64 sequences through the down projection, added to the stream
        _linear("linear_down", 64, 4096, 11008, False, False, True, "floor", "f16", "f16"),
        # an odd chunk of a prompt through the default decoder's q, k and v, f32 with a bias
        _linear("linear_chunk", 509, 2560, 2048, False, True, False, "ceil", "f32", "f32"),
        # a speculative batch through the vocabulary
        _linear("linear_head", 16, 32000, 2048, False, False, False, "floor", "f32", "f32"),
        # a long prompt through gate and up: the largest product
        _product("product_prompt", 4096, 22016, 4096, True, False, False, "f16"),
        # rows that end inside a tile, a length that ends inside a step
        _product("product_ragged", 1001, 4100, 11040, False, True, True, "f16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cost(case):
    if case["op"] in ("quantize", "norm"):
        return case["rows"] * case["dim"] * _SIZES[case["io"]]
    # the plain form's product, its expanded weights and its rows
    return (case["m"] * case["n"] * case["k"] + 64 * case["n"] * case["k"]
            + 64 * case["m"] * case["k"])


def draw(rng):
    op = rng.choice(("quantize", "norm", "linear", "linear", "product", "product"))
    io = rng.choice(("f16", "f16", "f32"))
    most = {c["op"]: max(_cost(d) for d in listed() if d["op"] == c["op"]) for c in listed()}
    while True:
        if op == "quantize":
            case = _quantize("", _log_int(rng, 1, 16384), 32 * _log_int(rng, 1, 344),
                             rng.choice(("floor", "ceil")), io)
            limit = most[op]
        elif op == "norm":
            rows = _log_int(rng, 1, 16384)
            dim = rng.choice((64 * _log_int(rng, 1, 172), _log_int(rng, 64, 11008)))
            gate = rng.choice(("none", "plain", "sigmoid"))
            case = _norm("", rows, dim, rng.random() < 0.7, gate,
                         rng.choice((0, 1, rng.randrange(1, rows + 1))) if gate != "none" else 0,
                         io, rng.choice((io, "f16")))
            limit = most[op]
        else:
            m = rng.choice((1, rng.randrange(2, 17), _log_int(rng, 17, 4096)))
            pairs = rng.random() < 0.3
            n = rng.choice((16 * _log_int(rng, 4, 2000), 2 * _log_int(rng, 32, 16000)))
            k = 32 * rng.choice((_log_int(rng, 2, 512), 4 * _log_int(rng, 1, 128)))
            bias, residual = rng.random() < 0.3, rng.random() < 0.3
            if op == "linear":
                case = _linear("", m, n, k, pairs, bias, residual, rng.choice(("floor", "ceil")),
                               io, rng.choice((io, "f16")))
            else:
                case = _product("", m, n, k, pairs, bias, residual, rng.choice(("f16", "f32")))
            limit = max(most["linear"], most["product"])
        case.pop("name", None)
        if _cost(case) <= limit:
            return case


# --------------------------------------------------------------------------------- preparation
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=_DEVICE)


def _activations(gen, rows, dim):
    """Rows in which some channels are far larger than others."""
    return _normal(gen, rows, dim) * torch.exp(0.8 * _normal(gen, dim))


def _quantised(x, rule):
    """e2m1 codes (uint8, one an element) and scale bytes of f32 rows."""
    x = x.unflatten(-1, (-1, 32))
    fraction, exponent = torch.frexp(x.abs().amax(-1))      # the largest is fraction * 2^exponent
    power = exponent - 3                                    # it comes to stand between 4 and 8
    if rule == "ceil":
        power = power + (fraction > 0.75).to(power.dtype)   # or at 6 at most
    power = torch.where(fraction == 0, -127, power).clamp(min=-127)
    size = torch.ldexp(x, -power.unsqueeze(-1))
    sign, size = (torch.signbit(size) * 8).to(torch.uint8), size.abs()
    code = torch.zeros_like(sign)
    for edge, with_edge in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False),
                            (3.5, True), (5.0, False)):     # a tie goes to the even code
        code += (size >= edge) if with_edge else (size > edge)
    return (code | sign).flatten(-2), (power + 127).to(torch.uint8)


def _packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


_gpu = None


def _context():
    """The package's context, on the stream that torch works on."""
    global _gpu
    if _gpu is None:
        import karume_amd
        _gpu = karume_amd.acquire_gpu(0, stream=torch.cuda.current_stream().cuda_stream)
    return _gpu


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    io = _DTYPES[case["io"]]
    empty = lambda *shape, dtype=torch.uint8: torch.empty(shape, dtype=dtype, device=_DEVICE)  # noqa: E731
    if case["op"] == "quantize":
        rows, dim = case["rows"], case["dim"]
        return {"case": case, "x": _activations(gen, rows, dim).to(io), "codes": empty(rows, dim // 2),
                "scales": empty(rows, dim // 32), "values": empty(rows, dim, dtype=io)}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        state = {"case": case, "y": _normal(gen, rows, dim).to(io),
                 "residual": (3 * _activations(gen, rows, dim)).to(io), "gate": None,
                 "post": 1 + 0.2 * _normal(gen, dim) if case["post"] else None,
                 "pre": 1 + 0.2 * _normal(gen, dim), "sum": empty(rows, dim, dtype=io),
                 "out": empty(rows, dim, dtype=_DTYPES[case["norm"]]),
                 "scales": (0.22, 0.95)}      # of the block and of the stream
        if case["gate"] != "none":
            count = -(-rows // case["span"]) if case["span"] else 1
            state["gate"] = _normal(gen, count, dim).to(io)
        return state
    m, n, k = case["m"], case["n"], case["k"]
    width, out = n // 2 if case["pairs"] else n, _DTYPES[case["out"]]
    codes, scales = _quantised(_normal(gen, n, k) * 0.02, "floor")
    state = {"case": case, "w": _packed(codes), "w_scales": scales, "bias": None, "residual": None,
             "xq": empty(m, k // 2), "xs": empty(m, k // 32), "out": empty(m, width, dtype=out)}
    if case["bias"]:
        state["bias"] = 0.1 * _normal(gen, n)
    if case["residual"]:
        state["residual"] = _normal(gen, m, width).to(out)
    x = _activations(gen, m, k)
    if case["op"] == "linear":
        state["x"] = x.to(io)
    else:
        codes, state["xs"] = _quantised(x, case["rule"])
        state["xq"] = _packed(codes)
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"quantize": _plain_quantize, "norm": _plain_norm, "linear": _plain_linear,
            "product": _plain_linear}[state["case"]["op"]](state)


def _run_own(state):
    import karume_amd as ka
    case, gpu = state["case"], _context()
    code = {"f16": ka.F16, "f32": ka.F32}
    rule = {"floor": ka.MX4_FLOOR, "ceil": ka.MX4_CEIL}.get(case.get("rule"))
    at = lambda name: None if state[name] is None else state[name].data_ptr()  # noqa: E731
    if case["op"] == "quantize":
        shape = dict(rows=case["rows"], dim=case["dim"])
        gpu.quantize_mx4(at("x"), at("codes"), at("scales"), x_dtype=code[case["io"]],
                         scale_rule=rule, **shape)
        gpu.dequant_mx4(at("codes"), at("scales"), at("values"), out_dtype=code[case["io"]], **shape)
        return state["values"]
    if case["op"] == "norm":
        kind = {"none": ka.GATE_PLAIN, "plain": ka.GATE_PLAIN, "sigmoid": ka.GATE_SIGMOID}
        block_scale, residual_scale = state["scales"]
        gpu.block_norm(at("y"), rows=case["rows"], dim=case["dim"], post_weight=at("post"),
                       gate=at("gate"), gate_span=case["span"], gate_kind=kind[case["gate"]],
                       residual=at("residual"), pre_weight=at("pre"), sum_out=at("sum"),
                       norm_out=at("out"), eps=_EPS, block_scale=block_scale,
                       residual_scale=residual_scale, io_dtype=code[case["io"]],
                       norm_dtype=code[case["norm"]])
        return [state["sum"], state["out"]]
    rest = dict(bias=at("bias"), residual=at("residual"), out_dtype=code[case["out"]],
                epilogue=ka.EPILOGUE_SILU_PAIRS if case["pairs"] else ka.EPILOGUE_NONE)
    m, n, k = case["m"], case["n"], case["k"]
    if case["op"] == "linear":
        gpu.linear_mx4_fused(at("x"), at("w"), at("w_scales"), at("out"), m, n, k, xq=at("xq"),
                             xs=at("xs"), x_dtype=code[case["io"]], scale_rule=rule, **rest)
    else:
        gpu.linear_mx4(at("xq"), at("xs"), at("w"), at("w_scales"), at("out"), m, n, k, **rest)
    return state["out"]


def _values(codes, scales):
    """f32 values of one code an element and scale bytes."""
    size = codes & 7
    value = torch.where(size < 2, 0.5 * size, torch.ldexp(1 + 0.5 * (size & 1), (size >> 1) - 1))
    value = torch.where(codes > 7, -value, value).unflatten(-1, (-1, 32))
    return torch.ldexp(value, scales.to(torch.int32).unsqueeze(-1) - 127).flatten(-2)


def _plain_quantize(state):
    return _values(*_quantised(state["x"].float(), state["case"]["rule"])).to(state["x"].dtype)


def _plain_rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight


def _plain_norm(state):
    case, t = state["case"], state["y"].float()
    if case["post"]:
        t = _plain_rms(t, state["post"])
    if state["gate"] is not None:
        gate = state["gate"].float()
        if case["gate"] == "sigmoid":
            gate = 1 / (1 + torch.exp(-gate))
        if case["span"] > 1:
            gate = gate.repeat_interleave(case["span"], 0)[:case["rows"]]
        t = t * gate
    block_scale, residual_scale = state["scales"]
    total = residual_scale * state["residual"].float() + block_scale * t
    return [total.to(state["sum"].dtype), _plain_rms(total, state["pre"]).to(state["out"].dtype)]


def _unpacked(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _plain_linear(state):
    case = state["case"]
    if case["op"] == "linear":
        codes, scales = _quantised(state["x"].float(), case["rule"])
    else:
        codes, scales = _unpacked(state["xq"]), state["xs"]
    out = torch.mm(_values(codes, scales), _values(_unpacked(state["w"]), state["w_scales"]).t())
    if state["bias"] is not None:
        out = out + state["bias"]
    if case["pairs"]:
        gate, up = out[:, 0::2], out[:, 1::2]
        out = gate / (1 + torch.exp(-gate)) * up
    if state["residual"] is not None:
        out = out + state["residual"].float()
    return out.to(state["out"].dtype)


# -------------------------------------------------------------------------- work and exactness
def work(case):
    if case["op"] == "quantize":
        size = case["rows"] * case["dim"]
        held = size // 2 + size // 32      # written, and read for the values that come back
        return {"bytes": 2 * size * _SIZES[case["io"]] + 2 * held, "flops": 4 * size}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        gates = 0 if case["gate"] == "none" else (-(-rows // case["span"]) if case["span"] else 1)
        size = (3 * rows + gates) * dim * _SIZES[case["io"]] + rows * dim * _SIZES[case["norm"]]
        return {"bytes": size + dim * 4 * (2 if case["post"] else 1), "flops": 12 * rows * dim}
    m, n, k = case["m"], case["n"], case["k"]
    x = m * k * _SIZES[case["io"]] if case["op"] == "linear" else m * (k // 2 + k // 32)
    out = m * (n // 2 if case["pairs"] else n) * _SIZES[case["out"]]
    return {"bytes": n * (k // 2 + k // 32) + x + out * (2 if case["residual"] else 1)
            + (n * 4 if case["bias"] else 0), "flops": 2 * m * n * k}


def _exact_block(x, rule):
    """What blocks of 32 elements of 64-bit rows stand for."""
    shape, x = x.shape, x.reshape(-1, 32)
    top = x.abs().max(1, keepdim=True)[0]
    power = torch.floor(torch.log2(top)).nan_to_num(neginf=0.0)
    # (a logarithm may be off at a power of two itself)
    power = power + (2.0 ** (power + 1) <= top).double() - (2.0 ** power > top).double()
    unit = 2.0 ** (power - 2)
    if rule == "ceil":
        unit = torch.where(top > 6 * unit, 2 * unit, unit)
    v = (x / unit).clamp(-6, 6)
    # spacing of the numbers around v: 0.5 below 2, 1 below 4, 2 from there on
    step = 0.5 + 0.5 * (v.abs() >= 2) + (v.abs() >= 4)
    return (torch.round(v / step) * step * unit).reshape(shape)


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _exact_stored(codes, scales):
    grid = torch.tensor(_GRID, dtype=torch.float64, device=codes.device)
    rows, half = codes.shape
    out = torch.empty((rows, half, 2), dtype=torch.float64, device=codes.device)
    out[:, :, 0] = grid[(codes % 16).long()]
    out[:, :, 1] = grid[torch.div(codes, 16, rounding_mode="floor").long()]
    scale = torch.exp2(scales.double() - 127)
    return (out.view(rows, half // 16, 32) * scale[:, :, None]).view(rows, 2 * half)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_block(state["x"].double(), case["rule"])
    if case["op"] == "norm":
        y = state["y"].double()
        if case["post"]:
            root = torch.sqrt(y.pow(2).sum(1, keepdim=True) / case["dim"] + _EPS)
            y = y / root * state["post"].double()
        if state["gate"] is not None:
            row = torch.arange(case["rows"], device=y.device)
            gate = state["gate"].double()[row // case["span"] if case["span"] else row * 0]
            y = y * (torch.sigmoid(gate) if case["gate"] == "sigmoid" else gate)
        total = state["residual"].double() * state["scales"][1] + y * state["scales"][0]
        root = torch.sqrt(total.pow(2).sum(1, keepdim=True) / case["dim"] + _EPS)
        return [total, total / root * state["pre"].double()]
    x = (_exact_block(state["x"].double(), case["rule"]) if case["op"] == "linear"
         else _exact_stored(state["xq"], state["xs"]))
    out = x @ _exact_stored(state["w"], state["w_scales"]).t()
    if state["bias"] is not None:
        out += state["bias"].double()
    if case["pairs"]:
        pair = out.view(case["m"], -1, 2)
        out = pair[:, :, 0] * torch.sigmoid(pair[:, :, 0]) * pair[:, :, 1]
    return out if state["residual"] is None else out + state["residual"].double()
