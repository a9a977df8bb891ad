"""Performance cases of the paged 4-bit K/V cache and of the rotary operators beside it.

A program that serves growing sequences makes four kinds of call: it builds rotation tables once
for its longest context (`rope_tables`), rotates rows (`rope_rows`), appends a step's keys and
values to pages of 4-bit codes with the rotation applied on the way (`kv4_append`, read back
through `kv4_read`), and attends over those pages (`kv4_attention`), with one row a sequence
(decode) or many (chunks of prompts).  `draw` spreads over the same ranges.

A page holds, for every kv head in turn, four blocks (P rows, depth D, groups of g elements):
  key codes     [P, 4, D/32] words: word (c, s) of a row has elements 32s + 8c .. + 7, element 2i
                in nibble i, element 2i + 1 in nibble 4 + i
  key params    [P, D/g, 2] fp16: step, minimum
  value codes   [P/4, D/8, 4] words: word (b, w, t) has elements 8w .. 8w + 7 of row 4b + t, in order
  value params  [P/4, D/g, 2, 4] fp16: steps of the four rows, then their minima
and an element stands for step * code + minimum.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DEVICE = "cuda"
_DTYPES = {"f16": torch.float16, "f32": torch.float32}
_SIZES = {"f16": 2, "f32": 4}
_VALUE_LIMIT = 32640.0   # a group with a larger magnitude in it reads as NaN


# ---------------------------------------------------------------------------------- the cases
def _attention(name, nseq, query, low, high, heads, kv_heads, depth, group, page, window, io):
    """`nseq` sequences with up to `query` rows each over `low` to `high` cached columns."""
    return {"name": name, "op": "attention", "nseq": nseq, "query": query, "low": low,
            "high": high, "heads": heads, "kv_heads": kv_heads, "depth": depth, "group": group,
            "page": page, "window": window, "io": io}


def _append(name, nseq, query, low, high, heads, kv_heads, depth, group, page, rotary, layout, io):
    return {"name": name, "op": "append", "nseq": nseq, "query": query, "low": low, "high": high,
            "heads": heads, "kv_heads": kv_heads, "depth": depth, "group": group, "page": page,
            "rotary": rotary, "layout": layout, "io": io}


def listed():
    return [
        # one sequence early in its life: the smallest step, latency alone
        _attention("decode_one", 1, 1, 500, 500, 32, 8, 128, 32, 16, 0, "f16"),
        # a serving step of 32 sequences of 128 to 4096 cached columns
        _attention("decode_ragged", 32, 1, 128, 4096, 32, 8, 128, 32, 64, 0, "f16"),
        # one sequence at the end of a long context
        _attention("decode_long", 1, 1, 131000, 131000, 32, 8, 128, 64, 256, 0, "f16"),
        # f32 activations, wide heads that share one kv head, a sliding window (odd lengths)
        _attention("decode_window_f32", 24, 1, 300, 3001, 8, 1, 256, 128, 16, 512, "f32"),
        # a 128-row chunk of the default decoder shape in the middle of a prompt, f32 activations
        _attention("chunk_f32", 1, 128, 1152, 1152, 32, 4, 64, 32, 64, 0, "f32"),
        # prompts of four requests, up to 512 rows each behind what they share with earlier ones
        _attention("prompts_f16", 4, 512, 700, 4608, 32, 8, 128, 32, 64, 0, "f16"),
        # keys and values of one decode step of 64 sequences
        _append("append_decode", 64, 1, 1, 4000, 32, 8, 128, 32, 16, 128, "half", "f16"),
        # the rows of two long prompts, interleaved pairs in half of each head, f32 activations
        _append("append_prompts", 2, 4096, 4096, 5000, 32, 8, 128, 64, 64, 64, "interleaved",
                "f32"),
        # the query rows of one decode step, rotated in part
        {"name": "rope_decode", "op": "rope", "rows": 16, "heads": 32, "depth": 128, "rotary": 64,
         "layout": "interleaved", "span": 8192, "head_major": False, "io": "f16"},
        # all heads of a long prompt, into the layout that the states-form attention reads
        {"name": "rope_prompt", "op": "rope", "rows": 5003, "heads": 40, "depth": 128,
         "rotary": 128, "layout": "half", "span": 131072, "head_major": True, "io": "f16"},
        # tables of a short context (the default decoder shape)
        {"name": "tables_short", "op": "tables", "rows": 512, "pairs": 32, "both": True,
         "first": 0, "base": 10000.0, "amplitude": 1.0},
        # tables of a stretched long context
        {"name": "tables_long", "op": "tables", "rows": 131072, "pairs": 64, "both": False,
         "first": 0, "base": 500000.0, "amplitude": 1.2079},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_SHAPES = ((32, 8, 128), (32, 4, 64), (8, 1, 256), (16, 16, 64), (28, 4, 128), (64, 8, 128))


def _cost(case):
    """Elements that the plain form goes through, in units of one number of a score or a row."""
    if case["op"] == "attention":
        rows, columns = _lengths(case)
        padded = case["nseq"] * (int(columns.max()) + case["page"])
        return (padded * case["kv_heads"] * case["depth"] * 2
                + padded * case["heads"] * int(rows.max()))
    if case["op"] == "append":
        return int(_lengths(case)[0].sum()) * (case["heads"] + 2 * case["kv_heads"]) * case["depth"]
    if case["op"] == "rope":
        return case["rows"] * case["heads"] * case["depth"]
    return case["rows"] * case["pairs"]


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "rope", "tables"))
    io = rng.choice(("f16", "f16", "f32"))
    heads, kv_heads, depth = rng.choice(_SHAPES)
    group = rng.choice([g for g in (32, 64, 128) if g <= depth])
    page = rng.choice((16, 32, 64, 128, 256))
    most = {c["op"]: max(_cost(d) for d in listed() if d["op"] == c["op"]) for c in listed()}[op]
    while True:
        if op == "attention":
            query = rng.choice((1, 1, rng.randrange(2, 9), _log_int(rng, 9, 512)))
            nseq = _log_int(rng, 1, 64)
            high = max(query, _log_int(rng, 1, 131000))
            low = max(1, int(high * rng.uniform(0.03, 1.0)))
            case = _attention("", nseq, query, low, high, heads, kv_heads, depth, group, page,
                              rng.choice((0, 0, 0, _log_int(rng, 1, 4096))), io)
        elif op == "append":
            query, nseq = rng.choice((1, _log_int(rng, 2, 4096))), _log_int(rng, 1, 64)
            high = max(query, _log_int(rng, 1, 8192))
            case = _append("", nseq, query, max(1, high // rng.randrange(1, 9)), high, heads,
                           kv_heads, depth, group, page,
                           rng.choice((depth, depth // 2, 2 * rng.randrange(1, depth // 2))),
                           rng.choice(("half", "interleaved")), io)
        elif op == "rope":
            case = {"op": "rope", "rows": _log_int(rng, 1, 5003), "heads": heads, "depth": depth,
                    "rotary": rng.choice((depth, depth // 2, 2 * rng.randrange(1, depth // 2))),
                    "layout": rng.choice(("half", "interleaved")),
                    "span": _log_int(rng, 64, 131072), "head_major": rng.random() < 0.5, "io": io}
        else:
            case = {"op": "tables", "rows": _log_int(rng, 64, 131072),
                    "pairs": rng.choice((16, 24, 32, 48, 64, 128)), "both": rng.random() < 0.5,
                    "first": rng.choice((0, rng.randrange(1 << 20))),
                    "base": rng.choice((10000.0, 500000.0, 1000000.0)),
                    "amplitude": rng.choice((1.0, 1.2079))}
        case.pop("name", None)
        if _cost(case) <= most:
            return case


def _lengths(case):
    """(rows of this step, columns with them) of each sequence: whole numbers that a case fixes."""
    rs = np.random.RandomState(case["nseq"] * 7919 + case["high"])
    columns = rs.randint(case["low"], case["high"] + 1, size=case["nseq"])
    columns[0] = case["high"]
    rows = np.full(case["nseq"], case["query"])
    if case["query"] > 8:   # prompts differ in length
        rows = rs.randint(max(1, case["query"] // 4), case["query"] + 1, size=case["nseq"])
        rows[0] = case["query"]
    return np.minimum(rows, columns), columns


# --------------------------------------------------------------------------------- preparation
def _quantised(x, group):
    """Codes and fp16 (step, minimum) of groups along the last axis of f32 rows."""
    x = x.unflatten(-1, (-1, group))
    low, high = x.amin(-1), x.amax(-1)
    bad = ~(x.abs().amax(-1) <= _VALUE_LIMIT)
    low, high = low.masked_fill(bad, 0.0), high.masked_fill(bad, 0.0)
    minimum = low.half()   # the largest fp16 number that is not above it
    minimum = torch.where(minimum.float() > low, _next_half(minimum, False), minimum)
    # (a true quotient: torch multiplies by the reciprocal of a plain number)
    raw = (high - minimum.float()) / torch.full_like(low, 15.0)
    step = raw.half()      # the smallest that is not below it
    step = torch.where(step.float() < raw, _next_half(step, True), step)
    wide = torch.where(step == 0, 1.0, step.float()).unsqueeze(-1)
    codes = torch.round((x - minimum.float().unsqueeze(-1)) / wide).clamp(0, 15)
    codes = codes.masked_fill(bad.unsqueeze(-1), 0.0).to(torch.uint8).flatten(-2)
    return codes, step.masked_fill(bad, math.nan), minimum


def _next_half(x, up):
    """The fp16 number next to `x` above or below (never called at an end of the range)."""
    bits = x.view(torch.int16)
    away = (x > 0) if up else (x < 0)
    moved = torch.where(away, bits + 1, bits - 1)
    first = torch.full_like(bits, 1 if up else -32767)   # from zero: the least subnormal
    return torch.where(x == 0, first, moved).view(torch.float16)


def _key_bytes(codes):
    """[..., P, D] codes -> [..., P, D/2] bytes."""
    c = codes.unflatten(-1, (-1, 4, 4, 2))               # step, column, i, parity
    c = c.movedim(-4, -3).transpose(-1, -2).flatten(-2)  # column, step, nibble
    return (c[..., 0::2] | (c[..., 1::2] << 4)).flatten(-3)


def _value_bytes(codes):
    """[..., P, D] codes -> [..., P/4, D/8, 4, 4] bytes."""
    c = codes.unflatten(-1, (-1, 8)).unflatten(-3, (-1, 4))
    return (c[..., 0::2] | (c[..., 1::2] << 4)).transpose(-2, -3)


def _pages_of(k, v, group):
    """[pages, kv heads, P, D] f32 keys and values -> [pages, bytes] as the cache holds them."""
    (kc, ks, km), (vc, vs, vm) = _quantised(k, group), _quantised(v, group)
    vp = torch.stack([vs, vm], -1).unflatten(-3, (-1, 4)).movedim(-3, -1)   # P/4, D/g, 2, 4
    parts = [_key_bytes(kc), torch.stack([ks, km], -1).contiguous().view(torch.uint8),
             _value_bytes(vc), vp.contiguous().view(torch.uint8)]
    return torch.cat([p.flatten(2) for p in parts], -1).flatten(1)


def _block_sizes(case):
    page, depth, groups = case["page"], case["depth"], case["depth"] // case["group"]
    return [page * depth // 2, page * groups * 4, page * depth // 2, page * groups * 4]


def _prepare_cache(case, seed, gen):
    rows, columns = _lengths(case)
    nseq, page, depth = case["nseq"], case["page"], case["depth"]
    need = -(-columns // page)
    stride = int(need.max()) + 1          # a table has room to grow
    order = np.random.RandomState(seed % (1 << 31)).permutation(int(need.sum()) + 3)
    table, at = np.full((nseq, stride), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(_DEVICE)  # noqa: E731
    return {"case": case, "table": to(table), "cu": to(cu), "lens": to(columns),
            "total": int(cu[-1]), "query": int(rows.max()), "columns": int(columns.max()),
            "pages": len(order), "stride": stride}


def _normal(gen, shape):
    return torch.randn(shape, generator=gen, device=_DEVICE)


def _frequencies(pairs, base):
    return base ** -(np.arange(pairs, dtype=np.float64) / pairs)


def _table(rows, pairs, base=10000.0, amplitude=1.0, first=0):
    """cos and sin rows as a program has them in hand, from angles in 64 bits."""
    angle = torch.arange(first, first + rows, device=_DEVICE, dtype=torch.float64)[:, None] \
        * torch.from_numpy(_frequencies(pairs, base)).to(_DEVICE)
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()


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
    if case["op"] == "tables":
        # (another seed: another stretch of the context)
        factor = 1.0 + (seed % 1000) / 250.0
        freq = torch.from_numpy(_frequencies(case["pairs"], case["base"]) / factor).to(_DEVICE)
        width = case["pairs"] * (2 if case["both"] else 1)
        return {"case": case, "freq": freq, "width": width,
                "cos": torch.empty((case["rows"], width), device=_DEVICE),
                "sin": torch.empty((case["rows"], width), device=_DEVICE)}
    io = _DTYPES[case["io"]]
    if case["op"] == "rope":
        rows, heads, depth = case["rows"], case["heads"], case["depth"]
        cos, sin = _table(case["span"], case["rotary"] // 2)
        shape = (heads, rows, depth) if case["head_major"] else (rows, heads, depth)
        return {"case": case, "cos": cos, "sin": sin, "x": _normal(gen, (rows, heads, depth)).to(io),
                "positions": torch.randint(0, case["span"], (rows,), generator=gen,
                                           device=_DEVICE, dtype=torch.int32),
                "out": torch.empty(shape, device=_DEVICE, dtype=io)}
    state = _prepare_cache(case, seed, gen)
    heads, kv_heads, depth, total = case["heads"], case["kv_heads"], case["depth"], state["total"]
    if case["op"] == "append":
        cos, sin = _table(case["high"], case["rotary"] // 2)
        size = sum(_block_sizes(case)) * kv_heads
        # one projection writes [q; k; v] rows; some channels of keys are far larger than others
        qkv = _normal(gen, (total, heads + 2 * kv_heads, depth))
        qkv[:, heads:heads + kv_heads] *= torch.exp(0.7 * _normal(gen, (kv_heads, depth)))
        state.update(cos=cos, sin=sin, qkv=qkv.to(io),
                     cache=torch.zeros((state["pages"], size), dtype=torch.uint8, device=_DEVICE),
                     q_out=torch.empty((total, heads, depth), dtype=io, device=_DEVICE),
                     k_read=torch.empty((total, kv_heads, depth), dtype=torch.float16,
                                        device=_DEVICE),
                     v_read=torch.empty((total, kv_heads, depth), dtype=torch.float16,
                                        device=_DEVICE))
        return state
    shape = (state["pages"], kv_heads, case["page"], depth)
    k = _normal(gen, shape) * torch.exp(0.5 * _normal(gen, (kv_heads, 1, depth)))
    cache = _pages_of(k, _normal(gen, shape), case["group"])
    state.update(cache=cache, q=_normal(gen, (total, heads, depth)).to(io),
                 out=torch.empty((total, heads, depth), dtype=io, device=_DEVICE),
                 scale=float(np.float32(depth ** -0.25)), workspace=None)
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    return {"attention": _plain_attention, "append": _plain_append, "rope": _plain_rope,
            "tables": _plain_tables}[case["op"]](state)


def _shape_of(state):
    case = state["case"]
    return dict(nseq=case["nseq"], max_query=state["query"], total_rows=state["total"],
                kv_heads=case["kv_heads"], depth=case["depth"], group=case["group"],
                page_rows=case["page"], pages=state["pages"], table_stride=state["stride"])


def _run_own(state):
    import karume_amd as ka
    case, gpu = state["case"], _context()
    io = ka.F16 if case.get("io") == "f16" else ka.F32
    if case["op"] == "tables":
        gpu.rope_tables(state["freq"].data_ptr(), state["cos"].data_ptr(), state["sin"].data_ptr(),
                        first=case["first"], rows=case["rows"], pairs=case["pairs"],
                        width=state["width"], amplitude=case["amplitude"])
        return [state["cos"], state["sin"]]
    layout = {"half": ka.ROPE_HALF, "interleaved": ka.ROPE_INTERLEAVED}.get(case.get("layout"))
    if case["op"] == "rope":
        gpu.rope_rows(state["x"].data_ptr(), state["positions"].data_ptr(), state["cos"].data_ptr(),
                      state["sin"].data_ptr(), state["out"].data_ptr(), rows=case["rows"],
                      heads=case["heads"], head_dim=case["depth"], rotary_dim=case["rotary"],
                      layout=layout, table_rows=case["span"], table_width=case["rotary"] // 2,
                      to_head_major=case["head_major"], io_dtype=io)
        return state["out"]
    cache, table, cu, lens = (state[n].data_ptr() for n in ("cache", "table", "cu", "lens"))
    shape = _shape_of(state)
    if case["op"] == "append":
        qkv, eb = state["qkv"].data_ptr(), _SIZES[case["io"]]
        heads, kv_heads, depth = case["heads"], case["kv_heads"], case["depth"]
        row = (heads + 2 * kv_heads) * depth
        gpu.kv4_append(qkv + heads * depth * eb, qkv + (heads + kv_heads) * depth * eb, cache, table,
                       cu, lens, q=qkv, q_out=state["q_out"].data_ptr(), heads=heads,
                       cos_table=state["cos"].data_ptr(), sin_table=state["sin"].data_ptr(),
                       q_stride=row, k_stride=row, v_stride=row, rotary_dim=case["rotary"],
                       layout=layout, table_rows=case["high"], table_width=case["rotary"] // 2,
                       io_dtype=io, **shape)
        gpu.kv4_read(cache, table, cu, lens, state["k_read"].data_ptr(), state["v_read"].data_ptr(),
                     out_dtype=ka.F16, **shape)
        return [state["q_out"], state["k_read"], state["v_read"]]
    limits = dict(heads=case["heads"], max_columns=state["columns"], window=case["window"])
    if state["workspace"] is None:
        need = gpu.kv4_attention_workspace(io_dtype=io, **limits, **shape)
        state["workspace"] = torch.empty(max(16, need), dtype=torch.uint8, device=_DEVICE)
    gpu.kv4_attention(state["q"].data_ptr(), cache, table, cu, lens, state["out"].data_ptr(),
                      half_scale=state["scale"], io_dtype=io,
                      workspace=state["workspace"].data_ptr(),
                      workspace_bytes=state["workspace"].numel(), **limits, **shape)
    return state["out"]


def _plain_tables(state):
    case = state["case"]
    at = torch.arange(case["first"], case["first"] + case["rows"], device=_DEVICE,
                      dtype=torch.float64)
    angle = at[:, None] * state["freq"]
    if case["both"]:
        angle = torch.cat([angle, angle], 1)
    return [(angle.cos() * case["amplitude"]).float(), (angle.sin() * case["amplitude"]).float()]


def _rotated(x, cos, sin, rotary, layout):
    """f32 rows [rows, heads, D] rotated in their first `rotary` elements; cos, sin [rows, R/2]."""
    turned, rest = x[..., :rotary], x[..., rotary:]
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_rope(state):
    case, at = state["case"], state["positions"].long()
    out = _rotated(state["x"].float(), state["cos"][at], state["sin"][at], case["rotary"],
                   case["layout"]).to(state["x"].dtype)
    return out.transpose(0, 1).contiguous() if case["head_major"] else out


def _row_places(state):
    """(sequence, row in its step, column) of every row of the step."""
    cu, lens = state["cu"].long(), state["lens"].long()
    row = torch.arange(state["total"], device=cu.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    inner = row - cu[seq]
    return seq, inner, lens[seq] - (cu[1:] - cu[:-1])[seq] + inner


def _plain_append(state):
    case, cache = state["case"], state["cache"]
    heads, kv_heads, depth, page = case["heads"], case["kv_heads"], case["depth"], case["page"]
    qkv = state["qkv"].float()
    seq, _, column = _row_places(state)
    cos, sin = state["cos"][column], state["sin"][column]
    turned = _rotated(qkv[:, :heads + kv_heads], cos, sin, case["rotary"], case["layout"])
    # each kv head's codes and parameters, then their places in the page
    (kc, ks, km), (vc, vs, vm) = (_quantised(x, case["group"]) for x in
                                  (turned[:, heads:], qkv[:, heads + kv_heads:]))
    sizes = _block_sizes(case)
    start = np.concatenate([[0], np.cumsum(sizes)])
    at = (state["table"].long()[seq, column // page] * cache.shape[1])[:, None] \
        + torch.arange(kv_heads, device=cache.device) * int(start[4])
    inner, groups = (column % page)[:, None, None], depth // case["group"]
    flat, span = cache.view(-1), lambda n: torch.arange(n, device=cache.device)  # noqa: E731
    at = at[..., None]
    flat[at + inner * (depth // 2) + span(depth // 2)] = _key_bytes(kc)
    params = torch.stack([ks, km], -1).view(torch.uint8).flatten(-2)
    flat[at + int(start[1]) + inner * groups * 4 + span(groups * 4)] = params
    words = (vc[..., 0::2] | (vc[..., 1::2] << 4)).unflatten(-1, (-1, 4))
    place = at + int(start[2]) + inner // 4 * (depth * 2) + inner % 4 * 4 + span(depth // 8) * 16
    flat[place[..., None] + span(4)] = words
    place = at + int(start[3]) + inner // 4 * (groups * 16) + inner % 4 * 2 + span(groups) * 16
    params = torch.stack([vs, vm], -1).view(torch.uint8).unflatten(-1, (2, 2))
    flat[place[..., None, None] + (span(2) * 8)[:, None] + span(2)] = params
    stands = [(s.float().repeat_interleave(case["group"], -1) * c.float()
               + m.float().repeat_interleave(case["group"], -1)).half()
              for c, s, m in ((kc, ks, km), (vc, vs, vm))]
    return [turned[:, :heads].to(state["qkv"].dtype)] + stands


def _read_pages(pages, case):
    """[n, bytes] pages -> f32 keys and values [n, kv heads, P, D]."""
    groups, page, group = case["depth"] // case["group"], case["page"], case["group"]
    kc, kp, vc, vp = pages.unflatten(-1, (case["kv_heads"], -1)).split(_block_sizes(case), -1)
    c = torch.stack([kc & 15, kc >> 4], -1).flatten(-2)
    c = c.unflatten(-1, (page, 4, -1, 2, 4)).transpose(-1, -2).movedim(-4, -3)
    k = c.reshape(*c.shape[:-5], page, case["depth"]).float()
    p = kp.contiguous().view(torch.float16).float().unflatten(-1, (page, groups, 2))
    k = k.unflatten(-1, (-1, group)) * p[..., :1] + p[..., 1:]
    c = torch.stack([vc & 15, vc >> 4], -1).flatten(-2)
    c = c.unflatten(-1, (page // 4, -1, 4, 8)).transpose(-2, -3)
    v = c.reshape(*c.shape[:-4], page, case["depth"]).float()
    p = vp.contiguous().view(torch.float16).float().unflatten(-1, (page // 4, groups, 2, 4))
    p = p.movedim(-1, -3).flatten(-4, -3)
    v = v.unflatten(-1, (-1, group)) * p[..., :1] + p[..., 1:]
    return k.flatten(-2), v.flatten(-2)


def _plain_attention(state):
    case, lens, cu = state["case"], state["lens"].long(), state["cu"].long()
    nseq, heads, kv_heads, depth = (case[n] for n in ("nseq", "heads", "kv_heads", "depth"))
    used = -(-state["columns"] // case["page"])
    table = state["table"][:, :used].long().clamp(min=0)
    k, v = (x.unflatten(0, (nseq, used)).transpose(1, 2).flatten(2, 3)
            for x in _read_pages(state["cache"][table.flatten()], case))
    # rows of a sequence beside its kv heads: [nseq, kv heads, G * rows, D]
    most, share = state["query"], heads // kv_heads
    rows = cu[1:] - cu[:-1]
    inner = torch.arange(most, device=cu.device)
    at = (cu[:-1, None] + inner).clamp(max=state["total"] - 1)
    q = state["q"].float()[at].unflatten(2, (kv_heads, share)).permute(0, 2, 3, 1, 4)
    q = q.reshape(nseq, kv_heads, share * most, depth) * (state["scale"] * state["scale"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).unflatten(2, (share, most))
    column = torch.arange(scores.shape[-1], device=cu.device)
    position = (lens - rows)[:, None] + inner
    behind = position[:, :, None] - column
    seen = behind >= 0
    if case["window"]:
        seen &= behind < case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), v).unflatten(2, (share, most)) / total
    seq, inner, _ = _row_places(state)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, inner].to(state["q"].dtype)


# -------------------------------------------------------------------------- work and exactness
def work(case):
    if case["op"] == "tables":
        count = case["rows"] * case["pairs"]
        return {"bytes": count * 8 * (2 if case["both"] else 1) + case["pairs"] * 8,
                "flops": count * 30}
    eb = _SIZES[case["io"]]
    if case["op"] == "rope":
        size = case["rows"] * case["heads"] * case["depth"]
        angles = min(case["rows"], case["span"]) * case["rotary"] * 4
        return {"bytes": 2 * size * eb + angles + case["rows"] * 4, "flops": 3 * size}
    rows, columns = _lengths(case)
    heads, kv_heads, depth = case["heads"], case["kv_heads"], case["depth"]
    held = 2 * kv_heads * (depth // 2 + depth // case["group"] * 4)   # of one column
    if case["op"] == "append":
        total = int(rows.sum())
        values = 2 * kv_heads * depth
        # (the written rows come back as values)
        size = total * ((2 * heads + 2 * kv_heads) * depth * eb + 2 * held + values * 2)
        angles = min(total, int(columns.max())) * case["rotary"] * 4
        return {"bytes": size + angles, "flops": total * (3 * heads * depth + 8 * values)}
    window = case["window"] or int(columns.max()) + 1
    size = pairs = 0
    for q, c in zip(rows.tolist(), columns.tolist()):
        first = max(0, c - q - window + 1)
        size += (c - first) * held + 2 * q * heads * depth * eb
        ends = np.arange(c - q + 1, c + 1)
        pairs += int(np.minimum(ends, window).sum())
    return {"bytes": size, "flops": 4 * heads * depth * pairs}


def _exact_turn(x, angles_cos, angles_sin, rotary, layout):
    """One rotation per pair of indices, in 64 bits."""
    j = torch.arange(rotary // 2, device=x.device)
    first, second = (j, j + rotary // 2) if layout == "half" else (2 * j, 2 * j + 1)
    out = x.clone()
    c, s = angles_cos.double()[:, None], angles_sin.double()[:, None]
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def _exact_held(x, group):
    """What a row of 64-bit values reads back as."""
    x = x.reshape(*x.shape[:-1], -1, group)
    low, high = x.min(-1, keepdim=True)[0], x.max(-1, keepdim=True)[0]
    halves = torch.arange(1 << 16, device=x.device).to(torch.int16).view(torch.float16)
    halves = halves[torch.isfinite(halves)].double().unique()    # every finite fp16, ascending
    minimum = halves[torch.searchsorted(halves, low.contiguous(), right=True) - 1]
    step = halves[torch.searchsorted(halves, ((high - minimum) / 15).contiguous())]
    code = torch.where(step > 0, ((x - minimum) / step.clamp(min=1e-30)).round().clamp(0, 15), 0.0)
    return (code * step + minimum).flatten(-2)


def _exact_column(state, seq, columns, head):
    """Keys and values [columns, D] of one sequence and kv head, byte by byte from their places."""
    case = state["case"]
    depth, group, page = case["depth"], case["group"], case["page"]
    groups, size = depth // group, sum(_block_sizes(case))
    start = np.concatenate([[0], np.cumsum(_block_sizes(case))]).tolist()
    flat = state["cache"].reshape(-1)
    halves = flat.view(torch.float16)
    c = torch.arange(columns, device=flat.device)[:, None]
    d = torch.arange(depth, device=flat.device)[None]
    at = state["table"][seq].long()[c // page] * (size * case["kv_heads"]) + head * size
    r, e, g = c % page, d % 8, d // group
    nibble = (e % 2) * 4 + e // 2
    byte = at + r * (depth // 2) + ((d // 8 % 4) * (depth // 32) + d // 32) * 4 + nibble // 2
    key = (flat[byte].long() >> (nibble % 2 * 4)) & 15
    par = (at + start[1]) // 2 + (r * groups + g) * 2
    key = key.double() * halves[par].double() + halves[par + 1].double()
    byte = at + start[2] + ((r // 4 * (depth // 8) + d // 8) * 4 + r % 4) * 4 + e // 2
    value = (flat[byte].long() >> (e % 2 * 4)) & 15
    par = (at + start[3]) // 2 + (r // 4 * groups + g) * 8 + r % 4
    return key, value.double() * halves[par].double() + halves[par + 4].double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "tables":
        at = torch.arange(case["rows"], device=_DEVICE, dtype=torch.float64) + case["first"]
        turns = torch.outer(at, state["freq"])
        turns = turns - 2 * math.pi * torch.round(turns / (2 * math.pi))
        both = (torch.cos(turns) * case["amplitude"], torch.sin(turns) * case["amplitude"])
        return [t.tile(1, 2) if case["both"] else t for t in both]
    if case["op"] == "rope":
        at = state["positions"].long()
        out = _exact_turn(state["x"].double(), state["cos"][at], state["sin"][at], case["rotary"],
                          case["layout"])
        return out.permute(1, 0, 2) if case["head_major"] else out
    heads, kv_heads, share = case["heads"], case["kv_heads"], case["heads"] // case["kv_heads"]
    rows, columns = _lengths(case)
    if case["op"] == "append":
        at = torch.from_numpy(np.concatenate([np.arange(c - q, c) for q, c in zip(rows, columns)]))
        at = at.to(_DEVICE)
        x = state["qkv"].double()
        turned = _exact_turn(x[:, :heads + kv_heads], state["cos"][at], state["sin"][at],
                             case["rotary"], case["layout"])
        return [turned[:, :heads], _exact_held(turned[:, heads:], case["group"]),
                _exact_held(x[:, heads + kv_heads:], case["group"])]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=_DEVICE)
    first = 0
    for i, (n, c) in enumerate(zip(rows.tolist(), columns.tolist())):
        far = torch.arange(c - n, c, device=_DEVICE)[:, None] - torch.arange(c, device=_DEVICE)
        seen = (far >= 0) & (far < (case["window"] or c + 1))
        for head in range(kv_heads):
            key, value = _exact_column(state, i, c, head)
            mine = slice(head * share, (head + 1) * share)
            q = state["q"][first:first + n, mine].double().transpose(0, 1).reshape(share * n, -1)
            s = (q @ key.t()).reshape(share, n, c) * state["scale"] ** 2
            p = torch.softmax(torch.where(seen, s, -math.inf), -1)
            out[first:first + n, mine] = (p.reshape(share * n, c) @ value).reshape(share, n, -1).transpose(0, 1)
        first += n
    return out
