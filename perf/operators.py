"""The products of a model's routed experts on microscaled 4-bit (MXFP4) and on unquantized (bfloat16) banks, with the
quantizer that makes the former: what they are measured on.

  quantize    mx.quantize, then mx.dequantize: rows to e2m1 or e4m3 codes with a power-of-two scale per 32 columns, and
              the values that they stand for
  mx_line     mx.gemv: the chosen experts of a few decode lines, each row through its own top-8
  mx_prompt   mx.grouped: a prompt's (row, expert) pairs, grouped by expert
  bf16_line   kernels.gemv_bf16: the same for banks as they are before conversion
  bf16_prompt kernels.grouped_bf16

`bank` says which of a layer's products it is: gate_up reads the rows of hidden size 2048 and ends with SiLU(gate) * up
in bfloat16; down reads a row per pair, the FFN's width, and gives float32. `bits` is the rows' element size in the
microscaled products (8: e4m3, 4: e2m1). Hidden size 2048, top-8 of 128 experts with FFN 768 or of 256 with FFN 512;
drawn cases have other FFN widths and expert counts too. Weights are N(0, 0.02), activations N(0, 1) with a few channels
eight times as large, routing even or Zipf(1.1) over a random order of the experts.
"""
import functools
import math
import pathlib
import sys

import torch

own = False

H, TOPK, BLOCK, STAGE = 2048, 8, 32, 256
FFN = {128: 768, 256: 512}
MAX_PROMPT = 4096
BANK_ROWS = 128 * 1536
DEV = "cuda:0"


def listed():
    return [
        # one decode line's row, between two launches of its layer: latency
        {"name": "quantize_line", "op": "quantize", "rows": 1, "cols": 2048, "bits": 8, "type": "bf16"},
        # a layer's gate_up bank at conversion
        {"name": "quantize_bank", "op": "quantize", "rows": BANK_ROWS, "cols": 2048, "bits": 4, "type": "bf16"},
        # one voice, frame by frame
        {"name": "mx_line1", "op": "mx_line", "bank": "gate_up", "rows": 1, "experts": 128, "ffn": 768, "bits": 8,
         "routing": "even"},
        # five lines of a story decoded together, at the model's shape
        {"name": "mx_lines5_down", "op": "mx_line", "bank": "down", "rows": 5, "experts": 256, "ffn": 512, "bits": 4,
         "routing": "even"},
        # a short text chunk
        {"name": "mx_prompt77", "op": "mx_prompt", "bank": "gate_up", "rows": 77, "experts": 256, "ffn": 512,
         "bits": 8, "routing": "even"},
        # the benchmark's prompt, skewed routing, second bank
        {"name": "mx_prompt256_down", "op": "mx_prompt", "bank": "down", "rows": 256, "experts": 128, "ffn": 768,
         "bits": 8, "routing": "zipf"},
        # a long prompt
        {"name": "mx_prompt4096", "op": "mx_prompt", "bank": "gate_up", "rows": 4096, "experts": 128, "ffn": 768,
         "bits": 4, "routing": "even"},
        # one voice on the banks before conversion
        {"name": "bf16_line1", "op": "bf16_line", "bank": "gate_up", "rows": 1, "experts": 128, "ffn": 768,
         "routing": "even"},
        # three lines, second bank
        {"name": "bf16_lines3_down", "op": "bf16_line", "bank": "down", "rows": 3, "experts": 256, "ffn": 512,
         "routing": "even"},
        # a short text chunk, second bank
        {"name": "bf16_prompt77_down", "op": "bf16_prompt", "bank": "down", "rows": 77, "experts": 128, "ffn": 768,
         "routing": "even"},
        # a reference voice's frames as the prompt (odd length), skewed routing
        {"name": "bf16_prompt1391", "op": "bf16_prompt", "bank": "gate_up", "rows": 1391, "experts": 128, "ffn": 768,
         "routing": "zipf"},
        # a long prompt
        {"name": "bf16_prompt4096", "op": "bf16_prompt", "bank": "gate_up", "rows": 4096, "experts": 128, "ffn": 768,
         "routing": "even"},
    ]


def _spread(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    op = rng.choices(("quantize", "mx_line", "mx_prompt", "bf16_line", "bf16_prompt"), (2, 2, 4, 2, 4))[0]
    if op == "quantize":
        of = rng.choice(("bf16", "f32"))
        return {"op": op, "rows": _spread(rng, 1, BANK_ROWS // (1 if of == "bf16" else 2)),
                "cols": 32 * rng.randint(1, 64), "bits": rng.choice((4, 8)), "type": of}
    case = {"op": op, "bank": rng.choice(("gate_up", "down")),
            "rows": rng.randint(1, 16) if op.endswith("line") else _spread(rng, 17, MAX_PROMPT),
            "experts": rng.choice((128, 256, rng.randint(8, 127)))}
    step = 32 if op.startswith("mx") else 64
    case["ffn"] = FFN.get(case["experts"]) or step * rng.randint(256 // step, 768 // step)
    case["routing"] = rng.choice(("even", "zipf"))
    if op.startswith("mx"):
        case["bits"] = rng.choice((4, 8))
    return case


def _shape(case):
    """(rows of an expert's weight, columns) of the case's bank."""
    return (2 * case["ffn"], H) if case["bank"] == "gate_up" else (H, case["ffn"])


# ---------------------------------------------------------------------------------------------------------- inputs
def _activations(gen, rows, cols):
    x = torch.randn((rows, cols), generator=gen, device=DEV)
    x[:, torch.randperm(cols, generator=gen, device=DEV)[:max(1, cols // 256)]] *= 8
    return x


def _routes(gen, case):
    """The top-8 experts [rows, 8] of each row."""
    T, E = case["rows"], case["experts"]
    base = torch.zeros(E, device=DEV)
    if case["routing"] == "zipf":
        base[torch.randperm(E, generator=gen, device=DEV)] = -1.1 * torch.arange(
            1, E + 1, device=DEV, dtype=torch.float32).log()
    u = torch.rand((T, E), generator=gen, device=DEV).clamp_(1e-12, 1 - 1e-7)
    return (base - torch.log(-torch.log(u))).topk(TOPK, dim=-1).indices


def _codes(x, bits):
    """Rows x in the microscaled format: codes [R, C * bits / 8] and scales [R, C / 32], both uint8, C the columns
    rounded up to whole stages of 256 (zeros there)."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % STAGE))
    value, exponent = _microscaled(x, bits)
    scale = (exponent + 127).to(torch.uint8).squeeze(-1)
    if bits == 8:
        return value.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2), scale
    grid = torch.tensor(_E2M1, device=DEV)
    code = torch.bucketize(value.abs(), (grid[1:] + grid[:-1]) / 2, out_int32=True).to(torch.uint8)
    code = (code | (value.signbit().to(torch.uint8) << 3)).flatten(-2)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def _tiled(codes, scale):
    """A bank's rows as the products read them: codes in tiles of 16 rows x 256 columns, by half of a block pair, the
    pair, the row; scales by tile, block pair of a stage, row and stage, the stages rounded up to an even number."""
    tiles, stages = codes.shape[0] // 16, codes.shape[1] // 128
    codes = codes.view(tiles, 16, stages, 4, 2, 16).permute(0, 2, 4, 3, 1, 5).reshape(tiles * 16, -1)
    scale = scale.view(tiles, 16, stages, 4, 2).permute(0, 3, 1, 2, 4)
    scale = torch.nn.functional.pad(scale, (0, 0, 0, stages % 2))
    return codes.contiguous(), scale.reshape(tiles * 16, -1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1000003 * seed + 29)
    state = dict(case)
    if case["op"] == "quantize":
        x = _activations(gen, case["rows"], case["cols"])
        state["x"] = x if case["type"] == "f32" else x.to(torch.bfloat16)
        return state
    E, (n, k) = case["experts"], _shape(case)
    ids = _routes(gen, case)
    P = ids.numel()
    gate_up = case["bank"] == "gate_up"
    x = _activations(gen, case["rows"] if gate_up else P, k)
    w = torch.randn((E * n, k), generator=gen, device=DEV) * 0.02
    if case["op"].startswith("mx"):
        state["codes"], state["scale"] = _codes(x, case["bits"])
        parts = [_codes(part, 4) for part in w.split(max(1, E // 8) * n)]  # a few experts at a time: less memory
        state["w_codes"], state["w_scale"] = (torch.cat(t) for t in zip(*parts))
        state["w_tiled"], state["w_scale_tiled"] = _tiled(state["w_codes"], state["w_scale"])
    else:
        state["x"], state["w"] = x.to(torch.bfloat16), w.to(torch.bfloat16)
    state["ids"] = ids.flatten()
    if case["op"].endswith("prompt"):
        # the pairs sorted by expert, as the layer's grouping gives them to both of its products
        order = torch.sort(state["ids"], stable=True).indices
        counts = torch.bincount(state["ids"], minlength=E)
        first = counts.cumsum(0) - counts
        e = torch.arange(E, device=DEV)
        state["groups"] = torch.stack((e, e, torch.zeros_like(e), first, counts), dim=1).to(torch.int32)
        state["order"] = order
        # where each pair lies when every expert has room for as many rows as the fullest one
        state["room"] = int(counts.max())
        sorted_ids = state["ids"][order]
        state["place"] = sorted_ids * state["room"] + torch.arange(P, device=DEV) - first[sorted_ids]
    return state


# ------------------------------------------------------------------------------------------------- the plain form
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# largest exponent, mantissa bits, smallest normal exponent and largest value of an element
_ELEMENT = {4: (2, 1, 0, 6.0), 8: (8, 3, -6, 448.0)}


def _power(exponent):
    """2^exponent in float32, exactly, for exponents from -127 (the scale code 0) to 127."""
    e = exponent.int()
    return torch.where(e < -126, 1 << 22, (e + 127) << 23).int().view(torch.float32)


def _microscaled(x, bits):
    """(elements [R, C / 32, 32], their blocks' exponents [R, C / 32, 1]) of rows x: the block's scale is the power of two
    at or below its largest magnitude, over the element's largest; elements to nearest, ties to even, saturated."""
    top, mantissa, low, most = _ELEMENT[bits]
    x = x.float().unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(dim=-1, keepdim=True)
    exponent = (torch.frexp(amax).exponent - 1 - top).clamp(-127, 127)
    exponent = torch.where(amax == 0, -127, exponent)
    v = x * _power(-exponent)
    step = _power((torch.frexp(v).exponent - 1).clamp_min(low) - mantissa)
    return (torch.round(v / step) * step).clamp(-most, most), exponent


def _elements(codes, bits):
    if bits == 8:
        return codes.view(torch.float8_e4m3fn).float()
    table = torch.tensor(_E2M1, device=DEV)
    table = torch.cat((table, -table))
    return table[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]


def _values(codes, scale, bits):
    """float32 values of microscaled rows (any leading dimensions)."""
    v = _elements(codes, bits).unflatten(-1, (-1, BLOCK))
    return (v * _power(scale.int() - 127)[..., None]).flatten(-2)


def _finish(y, bank):
    if bank == "down":
        return y
    gate, up = y.chunk(2, dim=-1)
    return (gate / (1 + torch.exp(-gate)) * up).to(torch.bfloat16)


def _plain(state):
    bits = state.get("bits")
    if state["op"] == "quantize":
        value, exponent = _microscaled(state["x"], state["bits"])
        return {"values": (value * _power(exponent)).flatten(-2).to(torch.bfloat16)}
    E, (n, _) = state["experts"], _shape(state)
    x = _values(state["codes"], state["scale"], bits) if bits else state["x"].float()
    if state["op"].endswith("line"):
        ids, x = state["ids"], x.repeat_interleave(state["ids"].numel() // x.shape[0], dim=0)
        if bits:
            w = _values(*(state[f].unflatten(0, (E, n)).index_select(0, ids) for f in ("w_codes", "w_scale")), 4)
        else:
            w = state["w"].unflatten(0, (E, n)).index_select(0, ids).float()
        return {"out": _finish(torch.bmm(w, x.unsqueeze(-1)).squeeze(-1), state["bank"])}
    w = _values(state["w_codes"], state["w_scale"], 4) if bits else state["w"].float()
    if state["bank"] == "gate_up":
        x = x[state["order"] // TOPK]
    rows = torch.zeros((E * state["room"], x.shape[1]), device=DEV).index_copy_(0, state["place"], x)
    y = torch.bmm(rows.unflatten(0, (E, -1)), w.unflatten(0, (E, n)).transpose(1, 2))
    return {"out": _finish(y.flatten(0, 1).index_select(0, state["place"]), state["bank"])}


# ------------------------------------------------------------------------------------------------ the framework's
@functools.cache
def _package():
    path = str(pathlib.Path(__file__).resolve().parents[1] / "comfyui-drama3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from drama3 import kernels, mx
    return kernels, mx


def _own(state):
    kernels, mx = _package()
    op = state["op"]
    if op == "quantize":
        return {"values": mx.dequantize(mx.quantize(state["x"], state["bits"]), torch.bfloat16)}
    (n, k), gate_up = _shape(state), state["bank"] == "gate_up"
    how = {"order": state["order"], "k": TOPK} if op.endswith("prompt") and gate_up else {}
    if op.startswith("mx"):
        rows = mx.MxRows(state["codes"], state["scale"], state["bits"], k)
        bank = mx.MxBank(state["w_tiled"], state["w_scale_tiled"], state["experts"], n, k)
        if op == "mx_line":
            return {"out": mx.gemv(rows, state["ids"], bank, swiglu=gate_up)}
        return {"out": mx.grouped(rows, state["groups"], bank, swiglu=gate_up, **how)}
    if op == "bf16_line":
        return {"out": kernels.gemv_bf16(state["x"], state["ids"], state["w"], n, swiglu=gate_up)}
    return {"out": kernels.grouped_bf16(state["x"], state["groups"], state["w"], n, swiglu=gate_up, **how)}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------- work
def _expected_experts(case):
    """The experts that the rows' routes are expected to touch."""
    E, T = case["experts"], case["rows"]
    if case["routing"] == "even":
        return E * (1 - (1 - TOPK / E) ** T)
    p = [r ** -1.1 for r in range(1, E + 1)]
    total = sum(p)
    return max(min(E, TOPK), sum(1 - (1 - min(1.0, TOPK * v / total)) ** T for v in p))


def work(case):
    if case["op"] == "quantize":
        R, C, bits = case["rows"], case["cols"], case["bits"]
        packed = R * C * (bits / 8 + 1 / BLOCK)
        return {"bytes": R * C * (2 if case["type"] == "bf16" else 4) + packed + R * C * 2, "flops": 6 * R * C}
    (n, k), P = _shape(case), case["rows"] * TOPK
    rows = case["rows"] if case["bank"] == "gate_up" else P
    weight, row = (17 / 32, case["bits"] / 8 + 1 / BLOCK) if case["op"].startswith("mx") else (2, 2)
    out = P * (case["ffn"] * 2 if case["bank"] == "gate_up" else H * 4)
    return {"bytes": _expected_experts(case) * n * k * weight + rows * k * row + out, "flops": 2 * P * n * k}


# ------------------------------------------------------------------------------------------------ 64-bit results
def _e2m1_64(codes):
    """e2m1 from its definition: sign, two exponent bits biased by one, one mantissa bit."""
    c = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2)
    e, m = ((c // 2) % 4).double(), (c % 2).double()
    v = torch.where(e == 0, m / 2, 2.0 ** (e - 1) * (1 + m / 2))
    return torch.where(c >= 8, -v, v)


def _dequantized_64(codes, scale, bits):
    v = _e2m1_64(codes) if bits == 4 else codes.view(torch.float8_e4m3fn).double()
    return v * torch.ldexp(torch.ones_like(scale, dtype=torch.float64), scale.int() - 127).repeat_interleave(BLOCK, -1)


def _quantized_64(x, bits):
    """The nearest of the format's values, found among all of them; a tie goes to the one with an even code."""
    if bits == 4:
        grid = torch.tensor(_E2M1, dtype=torch.float64, device=DEV)
    else:
        grid = torch.arange(127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
    block = x.double().unflatten(-1, (-1, BLOCK))
    amax = block.abs().amax(dim=-1, keepdim=True)
    top = math.frexp(float(grid[-1]))[1]  # the block's largest magnitude comes into the binade of the largest element
    scale = torch.where(amax == 0, 1.0, torch.ldexp(torch.ones_like(amax), torch.frexp(amax).exponent - top))
    v = block / scale
    high = torch.searchsorted(grid, v.abs()).clamp_max(len(grid) - 1)
    low = (high - 1).clamp_min(0)
    down, up = v.abs() - grid[low], grid[high] - v.abs()
    pick = torch.where((down < up) | ((down == up) & (low % 2 == 0)), low, high)
    return (grid[pick] * torch.sign(v) * scale).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return {"values": torch.cat([_quantized_64(part, case["bits"]) for part in s["x"].split(16384)])}
    (n, k), gate_up, ids = _shape(case), case["bank"] == "gate_up", s["ids"]
    order = s["order"] if "order" in s else torch.arange(ids.numel(), device=DEV)
    x = _dequantized_64(s["codes"], s["scale"], case["bits"]) if "codes" in s else s["x"].double()
    out = torch.empty((ids.numel(), n), dtype=torch.float64, device=DEV)
    for e in ids.unique().tolist():
        at = (ids[order] == e).nonzero().squeeze(-1)
        rows = slice(e * n, (e + 1) * n)
        w = _dequantized_64(s["w_codes"][rows], s["w_scale"][rows], 4) if "codes" in s else s["w"][rows].double()
        # pair p of the prompt's second product is its row p; of the lines', and of a first product, it is the token's
        source = order[at] // TOPK if gate_up else at
        out[at] = x[source] @ w.T
    if not gate_up:
        return {"out": out}
    gate, up = out[:, :n // 2], out[:, n // 2:]
    return {"out": gate * torch.sigmoid(gate) * up}
