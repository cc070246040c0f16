"""What stands around a block's routed experts, on unquantized (bfloat16) weights: what it is measured on.

  ffn         block.gated_ffn: the gated feed-forward (a layer's shared expert, or a dense layer), down(SiLU(gate) * up)
  ffn_train   block.gated_ffn_forward, then gated_ffn_backward: the same with the gradients of the rows and both weights
  norm        block.add_norm: the end of one block and the start of the next, h = residual + scale * gate * norm(y), norm(h)
  norm_train  block.add_norm_forward, then add_norm_backward: the same with every gradient
  lora        block.lora_linear: a projection that all rows share, beside the low-rank adapter of each row's own request

`stream` is the type of the residual stream and of the norms' weights, `y` the type of the block's output; `gate` is none,
or one value per row, per channel, or per element. Hidden size 2048 and FFN 512 or 768 are the model's; the other sizes are
generic. Weights are N(0, 0.02) (norms' around 1), activations N(0, 1) with a few channels eight times as large. Requests'
rows follow each other, as prompts packed into one pass do; in decode lines every row is a request of its own. Some requests
have no adapter (id -1).
"""
import math

import torch

own = False

H = 2048
EPS = 1e-6
DEV = "cuda:0"


def listed():
    return [
        # one voice, frame by frame: the shared expert of one layer
        {"name": "ffn_line1", "op": "ffn", "rows": 1, "hidden": H, "ffn": 512},
        # a reference voice's frames as the prompt (odd length), the benchmark's FFN width
        {"name": "ffn_prompt1391", "op": "ffn", "rows": 1391, "hidden": H, "ffn": 768},
        # a long prompt through a dense layer of a large model
        {"name": "ffn_dense4096", "op": "ffn", "rows": 4096, "hidden": 4096, "ffn": 11008},
        # fine-tuning the shared expert on one short take
        {"name": "ffn_train509", "op": "ffn_train", "rows": 509, "hidden": H, "ffn": 512},
        # a training step's micro-batch through a dense layer
        {"name": "ffn_train4096", "op": "ffn_train", "rows": 4096, "hidden": H, "ffn": 6144},
        # between two blocks of a decode line: latency
        {"name": "norm_line1", "op": "norm", "rows": 1, "hidden": H, "stream": "bf16", "y": "bf16", "gate": "none",
         "post": False, "scale": 1.0},
        # a long prompt, sandwich norms and a gate per row, float32 stream
        {"name": "norm_prompt8192", "op": "norm", "rows": 8192, "hidden": H, "stream": "f32", "y": "bf16", "gate": "row",
         "post": True, "scale": 1.0},
        # training, residual scale only
        {"name": "norm_train4096", "op": "norm_train", "rows": 4096, "hidden": H, "stream": "bf16", "y": "bf16",
         "gate": "none", "post": False, "scale": 0.22},
        # training with sandwich norms and a learned gate per channel, odd sizes
        {"name": "norm_train1391", "op": "norm_train", "rows": 1391, "hidden": 5120, "stream": "bf16", "y": "bf16",
         "gate": "channel", "post": True, "scale": 1.0},
        # eight lines decoded together, each in a voice of its own
        {"name": "lora_lines8", "op": "lora", "rows": 8, "inner": H, "outer": 1024, "rank": 16, "adapters": 8,
         "requests": 8},
        # a server's decode step: many requests, some with the same adapter
        {"name": "lora_lines61", "op": "lora", "rows": 61, "inner": H, "outer": 4096, "rank": 64, "adapters": 24,
         "requests": 61},
        # a dozen prompts in one pass
        {"name": "lora_prompts5000", "op": "lora", "rows": 5000, "inner": H, "outer": 4096, "rank": 32, "adapters": 16,
         "requests": 12},
    ]


def _spread(rng, low, high, step=1):
    return step * max(1, round(math.exp(rng.uniform(math.log(low), math.log(high))) / step))


def draw(rng):
    op = rng.choices(("ffn", "ffn_train", "norm", "norm_train", "lora"), (4, 3, 2, 3, 4))[0]
    if op == "ffn":
        return {"op": op, "rows": _spread(rng, 1, 4096), "hidden": rng.choice((H, _spread(rng, 256, 4096, 8))),
                "ffn": rng.choice((512, 768, _spread(rng, 256, 8192, 8)))}
    if op == "ffn_train":
        return {"op": op, "rows": _spread(rng, 16, 4096), "hidden": rng.choice((H, _spread(rng, 256, 2048, 8))),
                "ffn": rng.choice((512, 768, _spread(rng, 256, 6144, 8)))}
    if op.startswith("norm"):
        stream = rng.choice(("bf16", "f32"))
        return {"op": op, "rows": _spread(rng, 1, 8192), "hidden": rng.choice((H, _spread(rng, 64, 4096, 8),
                                                                              _spread(rng, 65, 4095))),
                "stream": stream, "y": "bf16" if stream == "bf16" else rng.choice(("bf16", "f32")),
                "gate": rng.choice(("none", "row", "channel", "full")), "post": rng.random() < 0.5,
                "scale": rng.choice((1.0, 0.22))}
    rows = _spread(rng, 1, 5000)
    return {"op": op, "rows": rows, "inner": rng.choice((H, _spread(rng, 256, 4096, 8))),
            "outer": rng.choice((1024, 2048, _spread(rng, 256, 4096, 8))), "rank": rng.choice((8, 16, 32, 64, 128)),
            "adapters": rng.randint(1, 32), "requests": rows if rows <= 64 else rng.randint(1, 64)}


# ---------------------------------------------------------------------------------------------------------- inputs
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _activations(gen, rows, cols):
    x = torch.randn((rows, cols), generator=gen, device=DEV)
    x[:, torch.randperm(cols, generator=gen, device=DEV)[:max(1, cols // 256)]] *= 8
    return x


def _weights(gen, *shape):
    return (torch.randn(shape, generator=gen, device=DEV) * 0.02).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1000003 * seed + 31)
    op, T = case["op"], case["rows"]
    state = dict(case)
    if op.startswith("ffn"):
        h, i = case["hidden"], case["ffn"]
        state["x"] = _activations(gen, T, h).to(torch.bfloat16)
        state["gate_up"], state["down"] = _weights(gen, 2 * i, h), _weights(gen, h, i)
        if op == "ffn_train":
            state["dout"] = torch.randn((T, h), generator=gen, device=DEV).to(torch.bfloat16)
    elif op.startswith("norm"):
        h, stream, of = case["hidden"], _TYPES[case["stream"]], _TYPES[case["y"]]
        state["residual"] = _activations(gen, T, h).to(stream)
        state["y"] = torch.randn((T, h), generator=gen, device=DEV).to(of)
        near_one = lambda n: (1 + 0.1 * torch.randn(n, generator=gen, device=DEV)).to(stream)  # noqa: E731
        state["weight"] = near_one(h)
        state["post_weight"] = near_one(h) if case["post"] else None
        shape = {"none": None, "row": (T, 1), "channel": (h,), "full": (T, h)}[case["gate"]]
        state["gate_value"] = None if shape is None else torch.rand(shape, generator=gen, device=DEV).to(of)
        if op == "norm_train":
            state["dh"] = torch.randn((T, h), generator=gen, device=DEV).to(stream)
            state["dn"] = torch.randn((T, h), generator=gen, device=DEV).to(of)
    else:
        k, n, rank, count = case["inner"], case["outer"], case["rank"], case["adapters"]
        state["x"], state["weight"] = _activations(gen, T, k).to(torch.bfloat16), _weights(gen, n, k)
        state["a"], state["b"] = _weights(gen, count, rank, k), _weights(gen, count, n, rank)
        state["alpha"] = 0.5 + torch.rand(count, generator=gen, device=DEV)
        # requests of random lengths one after the other, one in eight of them without an adapter
        requests = case["requests"]
        ends = torch.sort(torch.randperm(max(T - 1, 0), generator=gen, device=DEV)[:requests - 1]).values
        which = torch.randint(0, count, (requests,), generator=gen, device=DEV)
        which = torch.where(torch.rand(requests, generator=gen, device=DEV) < 0.125, -1, which)
        state["ids"] = which[torch.searchsorted(ends, torch.arange(T, device=DEV))]
    return state


# ------------------------------------------------------------------------------------------------- the plain form
def _ffn(s):
    x, down = s["x"].float(), s["down"].float()
    gate, up = (x @ s["gate_up"].float().T).chunk(2, dim=1)
    sig = torch.sigmoid(gate)
    return x, down, gate, up, sig, gate * sig * up


def _plain_ffn(s):
    _, down, _, _, _, hidden = _ffn(s)
    return (hidden @ down.T).to(torch.bfloat16)


def _plain_ffn_train(s):
    x, down, gate, up, sig, hidden = _ffn(s)
    dout = s["dout"].float()
    dhidden = dout @ down
    dgate = dhidden * up * sig * (1 + gate * (1 - sig))
    dboth = torch.cat((dgate, dhidden * gate * sig), dim=1)
    grads = dboth @ s["gate_up"].float(), dboth.T @ x, dout.T @ hidden
    return ((hidden @ down.T).to(torch.bfloat16),) + tuple(g.to(torch.bfloat16) for g in grads)


def _norm(s):
    y = s["y"].float()
    post_rstd = normed = None
    v = y
    if s["post_weight"] is not None:
        post_rstd = torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS)
        normed = y * post_rstd
        v = normed * s["post_weight"].float()
    gate = 1.0 if s["gate_value"] is None else s["gate_value"].float()
    h = s["residual"].float() + s["scale"] * (gate * v)
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    return post_rstd, normed, v, gate, h, rstd


def _plain_norm(s):
    *_, h, rstd = _norm(s)
    return h.to(s["residual"].dtype), (h * rstd * s["weight"].float()).to(s["y"].dtype)


def _plain_norm_train(s):
    post_rstd, normed, v, gate, h, rstd = _norm(s)
    stream, of = s["residual"].dtype, s["y"].dtype
    dn, hat = s["dn"].float(), h * rstd
    dweight = (dn * hat).sum(dim=0)
    dhat = dn * s["weight"].float()
    dh = s["dh"].float() + rstd * (dhat - hat * (dhat * hat).mean(dim=1, keepdim=True))
    dv = s["scale"] * dh
    dgate = dpost = None
    if s["gate_value"] is not None:
        dgate = dv * v
        if s["gate"] != "full":
            dgate = dgate.sum(dim=1, keepdim=True) if s["gate"] == "row" else dgate.sum(dim=0)
        dgate = dgate.to(of)
        dv = dv * gate
    if s["post_weight"] is not None:
        dpost = (dv * normed).sum(dim=0).to(stream)
        dnormed = dv * s["post_weight"].float()
        dv = post_rstd * (dnormed - normed * (dnormed * normed).mean(dim=1, keepdim=True))
    return (h.to(stream), (hat * s["weight"].float()).to(of), dv.to(of), dh.to(stream), dweight.to(stream)) + tuple(
        g for g in (dpost, dgate) if g is not None)


def _plain_lora(s):
    x, ids = s["x"].float(), s["ids"]
    out = x @ s["weight"].float().T
    # every adapter's inner product for all rows at once, the row's own adapter then picked by a mask
    count, rank, _ = s["a"].shape
    inner = (x @ s["a"].float().flatten(0, 1).T).view(-1, count, rank)
    mine = (ids[:, None] == torch.arange(count, device=ids.device)) * s["alpha"]
    inner = (inner * mine[:, :, None]).flatten(1)
    return (out + inner @ s["b"].float().transpose(1, 2).flatten(0, 1)).to(torch.bfloat16)


def run(state):
    op, s = state["op"], state
    if not own:
        return {"ffn": _plain_ffn, "ffn_train": _plain_ffn_train, "norm": _plain_norm, "norm_train": _plain_norm_train,
                "lora": _plain_lora}[op](s)
    block = _block()
    if op == "ffn":
        return block.gated_ffn(s["x"], s["gate_up"], s["down"])
    if op == "ffn_train":
        out, saved = block.gated_ffn_forward(s["x"], s["gate_up"], s["down"])
        return (out,) + tuple(block.gated_ffn_backward(s["dout"], s["x"], s["gate_up"], s["down"], saved))
    if op == "lora":
        return block.lora_linear(s["x"], s["weight"], s["a"], s["b"], s["alpha"], s["ids"])
    options = {"post": s["post_weight"], "gate": s["gate_value"], "scale": s["scale"]}
    if op == "norm":
        return block.add_norm(s["y"], s["residual"], s["weight"], eps=EPS, **options)
    h, n, rstd = block.add_norm_forward(s["y"], s["residual"], s["weight"], eps=EPS, **options)
    grads = block.add_norm_backward(s["dh"], s["dn"], s["y"], h, rstd, s["weight"], **options)
    return (h, n) + tuple(g for g in grads if g is not None)


def _block():
    import pathlib
    import sys
    package = str(pathlib.Path(__file__).resolve().parents[1] / "comfyui-drama3_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from drama3 import block
    return block


# ------------------------------------------------------------------------------------------ floors and exact results
def work(case):
    op, T = case["op"], case["rows"]
    if op.startswith("ffn"):
        h, i = case["hidden"], case["ffn"]
        weights, rows = 2 * 3 * h * i, 2 * T * h
        if op == "ffn":
            return {"bytes": weights + 2 * rows, "flops": 6 * T * h * i}
        return {"bytes": 2 * weights + 4 * rows, "flops": 18 * T * h * i}
    if op.startswith("norm"):
        h, size = case["hidden"], {"bf16": 2, "f32": 4}
        stream, of = size[case["stream"]], size[case["y"]]
        gate = of * {"none": 0, "row": T, "channel": h, "full": T * h}[case["gate"]]
        weights = stream * h * (2 if case["post"] else 1)
        if op == "norm":
            return {"bytes": 2 * T * h * (stream + of) + weights + gate, "flops": 12 * T * h}
        return {"bytes": 4 * T * h * (stream + of) + 2 * weights + 2 * gate, "flops": 40 * T * h}
    k, n, rank = case["inner"], case["outer"], case["rank"]
    adapters = min(case["adapters"], case["requests"])
    return {"bytes": 2 * (k * n + T * (k + n) + adapters * rank * (k + n)) + 8 * T,
            "flops": 2 * T * (k * n + rank * (k + n))}


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    op = case["op"]
    if op.startswith("ffn"):
        i = case["ffn"]
        wg, wu, wd = d["gate_up"][:i], d["gate_up"][i:], d["down"]
        g, u = torch.matmul(d["x"], wg.t()), torch.matmul(d["x"], wu.t())
        silu = g / (1 + torch.exp(-g))
        out = torch.matmul(silu * u, wd.t())
        if op == "ffn":
            return out
        # d silu / dg = silu / g + silu (1 - sigmoid): sigmoid and its complement each from its own exponential
        p, not_p = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
        da = torch.matmul(d["dout"], wd)
        dg, du = da * u * (p + silu * not_p), da * silu
        return (out, torch.matmul(dg, wg) + torch.matmul(du, wu),
                torch.cat((torch.matmul(dg.t(), d["x"]), torch.matmul(du.t(), d["x"]))),
                torch.matmul(d["dout"].t(), silu * u))
    if op.startswith("norm"):
        # the gradients by autograd, of the formula as it is defined
        train = op == "norm_train"
        names = ("y", "residual", "weight", "post_weight", "gate_value")
        leaves = {k: d[k].requires_grad_(train) for k in names if d[k] is not None}
        unit = lambda t: t / torch.sqrt((t ** 2).sum(-1, keepdim=True) / t.shape[-1] + EPS)  # noqa: E731
        v = leaves["y"]
        if "post_weight" in leaves:
            v = unit(v) * leaves["post_weight"]
        if "gate_value" in leaves:
            v = v * leaves["gate_value"]
        h = leaves["residual"] + case["scale"] * v
        n = unit(h) * leaves["weight"]
        if not train:
            return h, n
        grads = torch.autograd.grad((h, n), list(leaves.values()), (d["dh"], d["dn"]))
        return (h.detach(), n.detach()) + tuple(grads)
    out = torch.matmul(d["x"], d["weight"].t())
    for j in range(case["adapters"]):
        rows = (d["ids"] == j).nonzero().flatten()
        low = torch.matmul(d["x"][rows], d["a"][j].t())
        out[rows] += d["alpha"][j] * torch.matmul(low, d["b"][j].t())
    return out
