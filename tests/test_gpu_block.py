"""The parts around a block's routed experts (drama3.block) against their definitions in float64.

Tolerances count roundings, each at most half a step (bf16 2^-8, float32 2^-24 of the value), carried through the formulas entry by
entry. A float32 sum of n products is taken to be off by at most n 2^-23 of the sum of their magnitudes, whatever its order
(the matrix cores may cut instead of round); exp and the reciprocal add 2^-21 + |g| 2^-23 of the sigmoid."""
import pytest
import torch

from drama3 import _lib, block, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}
SUM = 2.0 ** -23


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(gen, *shape, dtype=BF, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def within(got, want, bound, what=""):
    got = got.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1
    assert worst <= 0 and torch.isfinite(got).all(), (what, worst, off.max().item())


def dot(a, b, ea=None, eb=None):
    """(a @ b, its error bound as a float32 sum) in float64, with bounds ea, eb of the operands' own errors."""
    size = a.abs() @ b.abs()
    err = a.shape[1] * SUM * size
    if ea is not None:
        err = err + ea @ b.abs()
    if eb is not None:
        err = err + a.abs() @ eb
    return a @ b, err


def rounded(v, err, dtype=BF):
    return err + HALF[dtype] * (v.abs() + err) + 1e-40


# ------------------------------------------------------------------------------------------------- gated feed-forward
class Ffn:
    """The definition and its error bounds."""

    def __init__(self, x, gate_up, down, lora=(None, None), ids=None):
        self.x, self.w, self.d = (t.to(F64) for t in (x, gate_up, down))
        I = down.shape[1]
        pre, e_pre = dot(self.x, self.w.T)
        if lora[0] is not None:
            more, e_more = adapter(self.x, *lora[0], ids)
            pre, e_pre = pre + more, e_pre + e_more
        self.pre, self.e_pre = pre, e_pre
        (g, u), (eg, eu) = pre.split(I, 1), e_pre.split(I, 1)
        s = torch.sigmoid(g)
        e_s = s * (2.0 ** -21 + g.abs() * 2.0 ** -23 + 2.0 ** -23)  # with the products' roundings
        self.hidden = g * s * u
        # |d silu / dg| <= 1.1
        e_h = 1.1 * eg * (u.abs() + eu) + (g * s).abs() * eu + (g * u).abs() * e_s + 2.0 ** -22 * self.hidden.abs()
        self.e_h = rounded(self.hidden, e_h)
        self.g, self.u, self.s, self.eg, self.eu, self.e_s = g, u, s, eg, eu, e_s
        self.out, e_out = dot(self.hidden, self.d.T, self.e_h)
        if lora[1] is not None:
            more, e_more = adapter(self.hidden, *lora[1], ids, self.e_h)
            self.out, e_out = self.out + more, e_out + e_more
        self.e_out = rounded(self.out, e_out)

    def grads(self, dout):
        dout, g, u, s = dout.to(F64), self.g, self.u, self.s
        dh, e_dh = dot(dout, self.d)
        slope = s * (1 + g * (1 - s))
        # |d slope / dg| <= 0.5, |slope| <= 1.1; its own roundings: of s and 1 - s (in absolute terms), and of the products
        e_slope = 0.5 * self.eg + self.e_s * (1 + g.abs()) + (1 + g.abs()) * s * 2.0 ** -22
        dg, du = dh * u * slope, dh * g * s
        e_dg = e_dh * u.abs() * 1.1 + dh.abs() * (1.1 * self.eu + u.abs() * e_slope) + 2.0 ** -22 * dg.abs()
        e_du = e_dh * (g * s).abs() + dh.abs() * (1.1 * self.eg + g.abs() * self.e_s) + 2.0 ** -22 * du.abs()
        both, e_both = torch.cat((dg, du), 1), torch.cat((rounded(dg, e_dg), rounded(du, e_du)), 1)
        found = dot(both, self.w, e_both), dot(both.T, self.x, e_both.T), dot(dout.T, self.hidden, None, self.e_h)
        return [(v, rounded(v, e)) for v, e in found]


def adapter(x, a, b, alpha, ids, ex=None):
    """What the adapters add to the rows' product, and its error bound."""
    out = torch.zeros((x.shape[0], b.shape[1]), dtype=F64, device=x.device)
    err = torch.zeros_like(out)
    for j in range(a.shape[0]):
        rows = (ids == j).nonzero().flatten()
        low, e = dot(x[rows], a[j].to(F64).T, None if ex is None else ex[rows])
        al = alpha[j].to(F64)
        low, e = low * al, e * al.abs() + 2.0 ** -23 * (low * al).abs()
        out[rows], err[rows] = dot(low, b[j].to(F64).T, rounded(low, e))
    return out, err


def close_on_the_whole(got, want, what):
    # independent roundings of the operand and of the result: each at most 2^-8 / sqrt(3) of the norm on the average
    rel = ((got.to(F64) - want).norm() / want.norm()).item()
    assert rel < 2.0 ** -8, (what, rel)


def ffn_inputs(T, H, I, O, seed=0):
    gen = gen_of(seed)
    x = randn(gen, T, H)
    return x, randn(gen, 2 * I, H, scale=0.5 / H ** 0.5), randn(gen, O, I, scale=0.5 / I ** 0.5), randn(gen, T, O)


FFN_SHAPES = [  # rows, hidden, ffn, out: row counts at every kernel's borders, widths that end inside a tile, a stage and a step
    (1, 8, 8, 8), (1, 2048, 512, 2048), (2, 72, 24, 40), (15, 2048, 768, 2048), (16, 264, 136, 264), (17, 512, 64, 8), (31, 64, 72, 520),
    (33, 200, 8, 1000), (63, 1000, 264, 64), (64, 2048, 512, 2048), (65, 2048, 512, 2048), (100, 8, 2048, 16), (127, 136, 128, 128),
    (128, 64, 64, 72), (129, 72, 1032, 200), (255, 320, 200, 256), (256, 256, 256, 256), (257, 1000, 264, 520), (300, 2048, 768, 2048),
    (509, 2048, 512, 2048), (1391, 2048, 768, 2048), (2050, 2056, 2056, 2064),
    # every size of tile in every product, with ends inside tiles and stages
    (777, 4104, 4104, 4104), (1500, 1032, 2056, 1544), (2600, 2568, 2056, 4104), (3333, 2056, 3976, 2056), (4000, 3080, 1000, 2056)]


@pytest.mark.parametrize("T, H, I, O", FFN_SHAPES)
def test_gated_ffn(T, H, I, O):
    x, gate_up, down, dout = ffn_inputs(T, H, I, O)
    ref = Ffn(x, gate_up, down)
    out = block.gated_ffn(x, gate_up, down)
    assert out.dtype == BF
    within(out, ref.out, ref.e_out, "out")
    out2, saved = block.gated_ffn_forward(x, gate_up, down)
    assert torch.equal(out, out2)
    within(saved[0], ref.pre, ref.e_pre + 1e-40, "pre")
    within(saved[1], ref.hidden, ref.e_h, "hidden")
    grads = block.gated_ffn_backward(dout, x, gate_up, down, saved)
    for name, got, (want, bound) in zip(("dx", "dgate_up", "ddown"), grads, ref.grads(dout)):
        assert got.dtype == BF
        within(got, want, bound, name)
        if T * H >= 4096:
            close_on_the_whole(got, want, name)
    again = block.gated_ffn_backward(dout, x, gate_up, down, saved)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_gated_ffn_rows_do_not_depend_on_each_other():
    """A row with infinities or NaN stays in its own row, at row counts of every kernel."""
    for T in (3, 20, 50, 200):
        x, gate_up, down, _ = ffn_inputs(T, 264, 136, 72, seed=T)
        want = block.gated_ffn(x, gate_up, down)
        bad = x.clone()
        bad[1, 5], bad[T - 1, 263] = float("inf"), float("nan")
        got = block.gated_ffn(bad, gate_up, down)
        keep = [t for t in range(T) if t not in (1, T - 1)]
        assert torch.equal(got[keep], want[keep]) and got[T - 1].isnan().all(), T


def test_gated_ffn_large_gates():
    """Gates far out: SiLU is the gate or zero, its slope one or zero, without NaN."""
    T, H, I = 70, 64, 64
    x = torch.zeros((T, H), device=DEV, dtype=BF)
    x[:, 0] = torch.linspace(-300, 300, T, device=DEV).to(BF)
    gate_up = torch.zeros((2 * I, H), device=DEV, dtype=BF)
    gate_up[:, 0] = 1
    down = torch.eye(I, device=DEV, dtype=BF)
    for rows in (x, x[:9]):
        out, saved = block.gated_ffn_forward(rows, gate_up, down)
        dx, dw, dd = block.gated_ffn_backward(torch.ones_like(out), rows, gate_up, down, saved)
        ref = Ffn(rows, gate_up, down)
        within(out, ref.out, ref.e_out)
        for got, (want, bound) in zip((dx, dw, dd), ref.grads(torch.ones_like(out))):
            within(got, want, bound)


@pytest.mark.parametrize("T", [0, 1, 5, 200])
def test_gated_ffn_autograd(T):
    """The autograd form: the explicit pair's numbers, strided rows and gradients, and only what is asked for."""
    x, gate_up, down, dout = ffn_inputs(T, 136, 72, 64, seed=3)
    wide = torch.zeros((T, 3 * 136), device=DEV, dtype=BF)
    wide[:, 136:272] = x
    leaves = [wide.requires_grad_(), gate_up.requires_grad_(), down.requires_grad_()]
    out = block.gated_ffn(wide[:, 136:272], gate_up, down)
    want_out, saved = block.gated_ffn_forward(x, gate_up, down)
    assert torch.equal(out, want_out)
    grads = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    want = block.gated_ffn_backward(dout, x, gate_up, down, saved)
    assert torch.equal(grads[0][:, 136:272], want[0]) and torch.equal(grads[1], want[1]) and torch.equal(grads[2], want[2])
    if T == 0:
        assert not grads[1].any() and not grads[2].any()
    only, = torch.autograd.grad(out, (down,), dout, retain_graph=True)
    assert torch.equal(only, want[2])
    # a gradient that is one value for all (out.sum()) and one that is stored transposed
    summed, = torch.autograd.grad(out.sum(), (down,), retain_graph=True)
    assert torch.equal(summed, block.gated_ffn_backward(torch.ones_like(dout), x, gate_up, down, saved)[2])
    turned = dout.t().contiguous().t()
    assert torch.equal(torch.autograd.grad(out, (gate_up,), turned)[0], want[1])
    with torch.no_grad():
        assert not block.gated_ffn(x, gate_up, down).requires_grad


@pytest.mark.parametrize("T", [9, 150])
def test_gated_ffn_gradients_against_differences(T):
    """The output's change from one point to a near one against the mean of the gradients at both (the trapezoid rule, off by the
    third order). The outputs' roundings, at most 2^-8 of each, are taken as independent: six times their standard deviation."""
    x, gate_up, down, dout = ffn_inputs(T, 256, 128, 192, seed=5)
    gen = gen_of(6)
    near = [(t.float() * (1 + 0.02 * torch.randn(t.shape, generator=gen, device=DEV))).to(BF) for t in (x, gate_up, down)]
    points = [(x, gate_up, down), near]
    outs, grads = [], []
    for p in points:
        out, saved = block.gated_ffn_forward(*p)
        outs.append(out.to(F64))
        grads.append(block.gated_ffn_backward(dout, *p, saved))
    change = ((outs[1] - outs[0]) * dout.to(F64)).sum().item()
    told = sum((0.5 * (a.to(F64) + b.to(F64)) * (q.to(F64) - p.to(F64))).sum().item()
               for a, b, p, q in zip(grads[0], grads[1], *points))
    noise = (dout.to(F64) * outs[0]).norm().item() * 2.0 ** -8 / 3 ** 0.5 * 2  # hidden and out, at both points
    assert abs(change - told) < 6 * noise + 1e-3 * abs(change), (change, told, noise)


def test_gated_ffn_unaligned_and_strided():
    x, gate_up, down, dout = ffn_inputs(40, 136, 72, 64, seed=9)
    want, saved = block.gated_ffn_forward(x, gate_up, down)
    odd = torch.zeros(40 * 136 + 1, device=DEV, dtype=BF)
    odd[1:] = x.flatten()
    for rows in (odd[1:].view(40, 136), x.t().contiguous().t(), x.repeat(1, 2)[:, :136], x.repeat_interleave(2, 0)[::2]):
        assert torch.equal(block.gated_ffn(rows, gate_up, down), want)
        for a, b in zip(block.gated_ffn_backward(dout, rows, gate_up, down, saved),
                        block.gated_ffn_backward(dout, x, gate_up, down, saved)):
            assert torch.equal(a, b)
    assert torch.equal(block.gated_ffn(x, gate_up.t().contiguous().t(), down.t().contiguous().t()), want)
    same = x[:1].expand(40, 136)
    assert torch.equal(block.gated_ffn(same, gate_up, down), block.gated_ffn(same.contiguous(), gate_up, down))


def test_more_rows_than_65536_tiles():
    """Grids whose tiles or rows pass 2^16, and rows past 4 GiB: each row is its own product, checked where they start, end and pass
    the borders."""
    gen = gen_of(11)
    T = 64 * 65536 + 70
    x, w = randn(gen, T, 8), randn(gen, 16, 8)
    out = block.linear(x, w)
    some = torch.cat([torch.arange(a, a + 70, device=DEV) for a in (0, 64 * 65535, 64 * 65536, T - 70)])
    v, e = dot(x[some].to(F64), w.to(F64).T)
    within(out[some], v, rounded(v, e))
    wide = torch.zeros((70000, 32768), device=DEV, dtype=BF)  # 4.6 GB
    at = [0, 65535, 65536, 69999]
    wide[at] = randn(gen, 4, 32768)
    w = randn(gen, 8, 32768, scale=0.01)
    v, e = dot(wide[at].to(F64), w.to(F64).T)
    within(block.linear(wide, w)[at], v, rounded(v, e))


# ---------------------------------------------------------------------------------------------------------- adapters
def lora_inputs(T, K, N, rank, count, seed=0):
    gen = gen_of(seed)
    return (randn(gen, T, K), randn(gen, N, K, scale=K ** -0.5), randn(gen, count, rank, K, scale=K ** -0.5),
            randn(gen, count, N, rank, scale=rank ** -0.5), 0.5 + torch.rand(count, generator=gen, device=DEV))


def ids_of(kind, T, count, seed=0):
    gen = gen_of(seed)
    if kind == "none":
        return torch.full((T,), -1, dtype=torch.int64, device=DEV)
    if kind == "one":
        return torch.full((T,), count - 1, dtype=torch.int64, device=DEV)
    if kind == "each":
        return torch.arange(T, device=DEV) % count
    ids = torch.randint(-1, count, (T,), generator=gen, device=DEV)
    if kind == "runs":
        return ids.sort().values
    if kind == "outside":
        ids[::3] = count + ids[::3].abs()
        ids[1::4] = -7
        ids[2::5] = 2 ** 40 + 1
        ids[4::7] = -2 ** 40
    return ids


@pytest.mark.parametrize("kind", ["none", "one", "each", "runs", "mixed", "outside"])
@pytest.mark.parametrize("T, K, N, rank, count", [
    (1, 8, 8, 8, 1), (1, 2048, 1024, 16, 4), (8, 2048, 1024, 16, 8), (15, 72, 24, 24, 20), (17, 520, 40, 8, 3), (33, 264, 1000, 40, 40),
    (61, 2048, 512, 64, 24), (64, 128, 128, 128, 64), (65, 264, 136, 16, 70), (130, 72, 264, 72, 7), (257, 1000, 520, 32, 300),
    (700, 512, 256, 8, 5)])
def test_lora_linear(T, K, N, rank, count, kind):
    x, w, a, b, alpha = lora_inputs(T, K, N, rank, count)
    ids = ids_of(kind, T, count)
    out = block.lora_linear(x, w, a, b, alpha, ids)
    base, e_base = dot(x.to(F64), w.to(F64).T)
    more, e_more = adapter(x.to(F64), a, b, alpha, ids)
    assert out.dtype == BF
    within(out, base + more, rounded(base + more, e_base + e_more), kind)


@pytest.mark.parametrize("T", [5, 30, 60, 200])
def test_lora_linear_bad_adapters_stay_in_their_rows(T):
    """An adapter of infinities and NaN, and NaN rows, change their own rows alone; so does an adapter that no row names."""
    x, w, a, b, alpha = lora_inputs(T, 72, 40, 24, 4, seed=T)
    ids = torch.arange(T, device=DEV) % 4 - 1  # -1, 0, 1, 2
    want = block.lora_linear(x, w, a, b, alpha, ids)
    a2, b2, x2 = a.clone(), b.clone(), x.clone()
    a2[1], b2[1, ::2], b2[3], a2[3] = float("inf"), float("nan"), float("nan"), float("nan")
    x2[3] = float("nan")
    got = block.lora_linear(x2, w, a2, b2, alpha, ids)
    keep = (ids != 1) & (torch.arange(T, device=DEV) != 3)
    assert torch.equal(got[keep], want[keep])
    assert not got[ids == 1].isfinite().all(1).any() and got[3].isnan().all()


def test_lora_linear_without_adapters():
    x, w, _, _, _ = lora_inputs(70, 64, 40, 8, 1)
    none = [torch.empty(s, device=DEV, dtype=t) for s, t in (((0, 8, 64), BF), ((0, 40, 8), BF), ((0,), F32))]
    for rows in (x, x[:3], x[:0]):
        ids = torch.zeros(rows.shape[0], dtype=torch.int64, device=DEV)
        v, e = dot(rows.to(F64), w.to(F64).T)
        within(block.lora_linear(rows, w, *none, ids), v, rounded(v, e))


@pytest.mark.parametrize("T", [1, 8, 40, 200])
@pytest.mark.parametrize("which", [(True, False), (False, True), (True, True)])
def test_gated_ffn_with_adapters(T, which):
    x, gate_up, down, _ = ffn_inputs(T, 264, 136, 72, seed=T)
    _, _, a1, b1, alpha1 = lora_inputs(T, 264, 272, 16, 5, seed=1)
    _, _, a2, b2, alpha2 = lora_inputs(T, 136, 72, 40, 5, seed=2)
    lora = ((a1, b1, alpha1) if which[0] else None, (a2, b2, alpha2) if which[1] else None)
    ids = ids_of("mixed", T, 5)
    ref = Ffn(x, gate_up, down, lora, ids)
    out = block.gated_ffn(x, gate_up, down, gate_up_lora=lora[0], down_lora=lora[1], ids=ids)
    within(out, ref.out, ref.e_out)


# ------------------------------------------------------------------------------------------------------------- norms
def norm_inputs(T, H, of, stream, gate, post, weights, seed=0):
    gen = gen_of(seed)
    y, residual = randn(gen, T, H, dtype=of), randn(gen, T, H, dtype=stream)
    weight = randn(gen, H, dtype=weights)
    shape = {"none": None, "row": (T, 1), "channel": (H,), "full": (T, H)}[gate]
    return (y, residual, weight, randn(gen, H, dtype=weights) if post else None, None if shape is None else randn(gen, *shape, dtype=of),
            randn(gen, T, H, dtype=stream), randn(gen, T, H, dtype=of))


def norm_formula(y, residual, weight, post, gate, scale, eps, offset):
    unit = lambda t: t / torch.sqrt((t * t).mean(1, keepdim=True) + eps)  # noqa: E731
    v = y
    if post is not None:
        v = unit(v) * (post + offset)
    if gate is not None:
        v = gate * v
    h = residual + scale * v
    return h, None if weight is None else unit(h) * (weight + offset)


def norm_sizes(y, residual, weight, post, gate, dh, dn, scale, eps, offset):
    """The magnitudes of the terms that each gradient is the sum of."""
    rstd = lambda t: 1 / torch.sqrt((t * t).mean(1, keepdim=True) + eps)  # noqa: E731
    h, _ = norm_formula(y, residual, None, post, gate, scale, eps, offset)
    r, hat = rstd(h), (h * rstd(h)).abs()
    a = (dn * (weight + offset)).abs()
    res = dh.abs() + r * (a + hat * (a * hat).mean(1, keepdim=True))
    v, gates = y.abs(), 1.0 if gate is None else gate.abs()
    normed = v * rstd(y)
    if post is not None:
        v = normed * (post + offset).abs()
    dgate = None if gate is None else (abs(scale) * res * v)
    if gate is not None and gate.dim() == 1:
        dgate = dgate.sum(0)
    elif gate is not None and gate.shape[1] == 1:
        dgate = dgate.sum(1, keepdim=True)
    dy = abs(scale) * res * gates
    dpost = None
    if post is not None:
        dpost = (dy * normed).sum(0)
        b = dy * (post + offset).abs()
        dy = rstd(y) * (b + normed * (b * normed).mean(1, keepdim=True))
    return {"y": dy, "residual": res, "weight": (dn.abs() * hat).sum(0), "post": dpost, "gate": dgate}


def norm_check(T, H, of, stream, gate="none", post=False, weights=None, scale=1.0, offset=False, eps=1e-6, seed=0):
    weights = stream if weights is None else weights
    y, residual, weight, post_w, g, dh, dn = norm_inputs(T, H, of, stream, gate, post, weights, seed)
    names = ("y", "residual", "weight", "post", "gate")
    doubles = [None if t is None else t.to(F64).requires_grad_() for t in (y, residual, weight, post_w, g)]
    want_h, want_n = norm_formula(*doubles, scale, eps, float(offset))
    opt = {"post": post_w, "gate": g, "scale": scale, "unit_offset": offset}
    h, n = block.add_norm(y, residual, weight, eps=eps, **opt)
    h2, n2, rstd = block.add_norm_forward(y, residual, weight, eps=eps, **opt)
    assert torch.equal(h, h2) and torch.equal(n, n2) and h.dtype == stream and n.dtype == of
    # a row's sum of squares, its mean, root and reciprocal are off by less than 96 steps of 2^-24 (at most 32 in a lane, 6 + 16 between
    # lanes, a few more); h by that much of what the norm gives plus two roundings of its terms
    u = 2.0 ** -24
    part = ((want_h - doubles[1]).abs() + (doubles[1].abs() if not post else 0)).detach()
    e_h = 100 * u * (part + doubles[1].abs().detach())
    within(h, want_h.detach(), rounded(want_h.detach(), e_h, stream), "h")
    rms = (want_h * want_h).mean(1, keepdim=True).add(eps).sqrt().detach()
    factor = (doubles[2].detach() + float(offset)).abs() / rms
    # the mean square of h moves by at most 2 |h| e_h / mean: less than the mean of e_h's own row against its rms
    moved = (e_h * want_h.detach().abs()).mean(1, keepdim=True) / rms ** 2
    e_n = factor * (e_h + want_h.detach().abs() * (moved + 100 * u))
    within(n, want_n.detach(), rounded(want_n.detach(), e_n, of), "n")
    grads = block.add_norm_backward(dh, dn, y, h, rstd, weight, **opt)
    again = block.add_norm_backward(dh, dn, y, h, rstd, weight, **opt)
    used = [t for t in doubles if t is not None]
    want = dict(zip([k for k, t in zip(names, doubles) if t is not None],
                    torch.autograd.grad((want_h, want_n), used, (dh.to(F64), dn.to(F64)))))
    sizes = norm_sizes(*(None if t is None else t.detach() for t in doubles), dh.to(F64), dn.to(F64), scale, eps, float(offset))
    for name, got, twice, inp in zip(names, grads, again, (y, residual, weight, post_w, g)):
        if inp is None:
            assert got is None
            continue
        assert got.dtype == inp.dtype and got.shape == inp.shape, name
        assert torch.equal(got, twice), name
        w, size = want[name], sizes[name]
        # Half a step of the result's type, and float32 sums over H columns and T rows. A gradient is a sum of products of a few
        # factors of which each may be off by that much: taken on the whole, against the norm of the terms' magnitudes. (Not
        # against the gradient's own: of one column y^ is 1 - eps / (2 y^2), and dy = rstd b (1 - y^2 rstd^2) is 1e-6 of the two
        # terms that it is the difference of, each of which float32 holds to 6e-8.)
        rel = ((got.to(F64) - w).norm() / size.norm().clamp_min(1e-30)).item()
        limit = HALF[inp.dtype] + 2.0 ** -17
        if w.numel() * T >= 16:
            assert rel < limit, (name, rel, limit)
        assert got.isfinite().all()


WIDTHS = [1, 2, 7, 8, 9, 64, 65, 511, 512, 513, 1000, 1001, 1024, 1032, 2048, 2049, 4096, 4100, 5120, 8192, 8200, 16383, 16384]


@pytest.mark.parametrize("H", WIDTHS)
def test_add_norm_widths(H):
    for stream, of in ((BF, BF), (F32, BF), (F32, F32)):
        norm_check(5, H, of, stream, "channel", True, seed=H)
        norm_check(3, H, of, stream, "none", False, scale=0.22, seed=H + 1)


@pytest.mark.parametrize("gate", ["none", "row", "channel", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("of, stream, weights", [(BF, BF, BF), (BF, BF, F32), (BF, F32, F32), (BF, F32, BF), (F32, F32, F32), (F32, BF, BF)])
def test_add_norm_forms(gate, post, of, stream, weights):
    norm_check(37, 264, of, stream, gate, post, weights, scale=0.5, offset=post, eps=1e-5, seed=1)
    norm_check(6, 2048, of, stream, gate, post, weights, offset=not post, seed=2)
    norm_check(3, 1001, of, stream, gate, post, weights, seed=3)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 63, 1023, 1024, 1025, 1391, 4096, 8192])
def test_add_norm_rows(T):
    norm_check(T, 512, BF, BF, "channel", True, seed=T)
    norm_check(T, 72, F32, F32, "row", False, seed=T)


def test_add_norm_more_rows_than_a_dimension_has_threads():
    """2^24 + 3 rows (of whole workgroups: 2^33 threads), checked at their ends."""
    T, H = 2 ** 24 + 3, 520
    gen = gen_of(12)
    residual = torch.ones((T, H), device=DEV, dtype=BF)
    some = torch.tensor([0, 1, 2 ** 23, 2 ** 24 - 1, 2 ** 24, T - 1], device=DEV)
    residual[some] = randn(gen, 6, H)
    weight = randn(gen, H)
    out = block.norm(residual, weight)
    want = residual[some].to(F64)
    want = want / (want ** 2).mean(1, keepdim=True).add(1e-6).sqrt() * weight.to(F64)
    within(out[some], want, rounded(want, want.abs() * 100 * 2.0 ** -24))


def test_add_norm_without_rows():
    z = lambda *s: torch.ones(s, device=DEV, dtype=BF)  # noqa: E731
    h, n, rstd = block.add_norm_forward(z(0, 64), z(0, 64), z(64), post=z(64), gate=z(64))
    assert h.shape == n.shape == (0, 64)
    grads = block.add_norm_backward(h, n, z(0, 64), h, rstd, z(64), post=z(64), gate=z(64))
    assert grads[0].shape == (0, 64) and not any(g.any() for g in grads[2:])


def test_add_norm_parts_alone():
    """No next norm; either gradient alone; norm by itself; only the gradients that are asked for."""
    y, residual, weight, post, gate, dh, dn = norm_inputs(20, 200, BF, F32, "full", True, F32, 4)
    h, n, rstd = block.add_norm_forward(y, residual, weight, post=post, gate=gate)
    h1, none = block.add_norm(y, residual, None, post=post, gate=gate)
    assert none is None and torch.equal(h, h1)
    args = (y, h, rstd, weight)
    zero_h, zero_n = torch.zeros_like(dh), torch.zeros_like(dn)
    for a, b in zip(block.add_norm_backward(dh, None, *args, post=post, gate=gate), block.add_norm_backward(dh, zero_n, *args, post=post, gate=gate)):
        assert torch.equal(a, b)
    for a, b in zip(block.add_norm_backward(None, dn, *args, post=post, gate=gate), block.add_norm_backward(zero_h, dn, *args, post=post, gate=gate)):
        assert torch.equal(a, b)
    whole = block.add_norm_backward(dh, dn, *args, post=post, gate=gate)
    for i in range(5):
        one = block.add_norm_backward(dh, dn, *args, post=post, gate=gate, needs=tuple(j == i for j in range(5)))
        assert torch.equal(one[i], whole[i]) and all(g is None for j, g in enumerate(one) if j != i)
    x = residual.to(BF)
    for src, dtype in ((residual, F32), (residual, BF), (x, BF), (x, F32)):
        got = block.norm(src, weight, dtype=dtype)
        want = src.to(F64) / (src.to(F64) ** 2).mean(1, keepdim=True).add(1e-6).sqrt() * weight.to(F64)
        assert got.dtype == dtype
        within(got, want, rounded(want, want.abs() * 100 * 2.0 ** -24, dtype))


@pytest.mark.parametrize("T", [1, 40])
def test_add_norm_autograd(T):
    """The autograd forms: the explicit pair's numbers, broadcast gates, strided inputs, one output used alone."""
    y, residual, weight, post, _, dh, dn = norm_inputs(T, 136, BF, BF, "none", True, BF, 5)
    gate = torch.rand((1, 136), device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (y, residual, weight, post, gate)]
    h, n = block.add_norm(y, residual, weight, post=post, gate=gate, scale=0.3)
    _, _, rstd = block.add_norm_forward(y, residual, weight, post=post, gate=gate, scale=0.3)
    for grads in ((dh, dn), (dh, None), (None, dn)):
        outs = [o for o, g in zip((h, n), grads) if g is not None]
        got = torch.autograd.grad(outs, leaves, [g for g in grads if g is not None], retain_graph=True, allow_unused=True)
        want = block.add_norm_backward(*grads, y, h.detach(), rstd, weight, post=post, gate=gate, scale=0.3)
        for a, b, leaf in zip(got, want, leaves):
            if a is None:
                assert leaf is weight and grads[1] is None
                continue
            assert torch.equal(a, b) and a.shape == leaf.shape
    x = torch.randn((T, 300), device=DEV).requires_grad_()
    part = x[:, 7:7 + 136]
    out = block.norm(part, weight, dtype=BF)
    got = torch.autograd.grad(out, (x, weight), dn)
    ref = part.detach().to(F64).requires_grad_()
    w64 = weight.detach().to(F64).requires_grad_()
    want = torch.autograd.grad(ref / (ref ** 2).mean(1, keepdim=True).add(1e-6).sqrt() * w64, (ref, w64), dn.to(F64))
    assert (got[0][:, 7:143].to(F64) - want[0]).norm() < 2.0 ** -17 * want[0].norm()
    assert (got[1].to(F64) - want[1]).norm() < (2.0 ** -8 + 2.0 ** -17) * want[1].norm()


def test_add_norm_gradients_against_differences():
    """float32 throughout: the change between two near points against the mean gradient (the trapezoid rule)."""
    T, H = 6, 200
    y, residual, weight, post, gate, dh, dn = norm_inputs(T, H, F32, F32, "channel", True, F32, 6)
    gen = gen_of(7)
    points = [(y, residual, weight, post, gate)]
    points.append(tuple(t + 0.02 * torch.randn(t.shape, generator=gen, device=DEV) for t in points[0]))
    values, grads = [], []
    for p in points:
        h, n, rstd = block.add_norm_forward(*p[:3], post=p[3], gate=p[4], scale=0.7)
        values.append(((h.to(F64) * dh.to(F64)).sum() + (n.to(F64) * dn.to(F64)).sum()).item())
        grads.append(block.add_norm_backward(dh, dn, p[0], h, rstd, p[2], post=p[3], gate=p[4], scale=0.7))
    told = sum((0.5 * (a.to(F64) + b.to(F64)) * (q.to(F64) - p.to(F64))).sum().item() for a, b, p, q in zip(*grads, *points))
    # third order of steps of 2%: 1e-5 of the sum of the terms' magnitudes, of which there are T H 2 of about one
    assert abs(values[1] - values[0] - told) < 1e-5 * 2 * T * H + 1e-3 * abs(told), (values, told)


def test_add_norm_bad_rows_stay_alone():
    y, residual, weight, post, gate, dh, dn = norm_inputs(9, 300, BF, BF, "row", True, BF, 8)
    h, n = block.add_norm(y, residual, weight, post=post, gate=gate)
    y2, r2 = y.clone(), residual.clone()
    y2[2, 7], r2[5, 299], y2[7], r2[8] = float("nan"), float("inf"), 0, 0
    h2, n2 = block.add_norm(y2, r2, weight, post=post, gate=gate)
    keep = [0, 1, 3, 4, 6]
    assert torch.equal(h[keep], h2[keep]) and torch.equal(n[keep], n2[keep])
    assert n2[2].isnan().all() and n2[5, 299].isnan() and n2[7:].isfinite().all()
    zero, _ = block.add_norm(torch.zeros_like(y), torch.zeros_like(residual), weight, post=post)
    assert not zero.any()


# -------------------------------------------------------------------------------------------------- streams and graphs
def a_step(x, residual, weight, post, gate, gate_up, down, lora, ids, dout):
    """A block's parts as they are used: norm, feed-forward with its gradients, adapters, the next norm with its gradients."""
    n = block.norm(x, weight)
    y, saved = block.gated_ffn_forward(n, gate_up, down)
    z = block.lora_linear(y, down.new_ones(1) * gate_up[:gate_up.shape[0] // 2], *lora, ids)
    h, n2, rstd = block.add_norm_forward(y, residual, weight, post=post, gate=gate, scale=0.5)
    grads = block.add_norm_backward(dout, dout, y, h, rstd, weight, post=post, gate=gate, scale=0.5)
    return [n, y, z, h, n2, *grads, *block.gated_ffn_backward(grads[0], n, gate_up, down, saved)]


def step_inputs(T, seed=0):
    x, gate_up, down, dout = ffn_inputs(T, 264, 136, 264, seed)
    gen = gen_of(seed + 50)
    _, _, a, b, alpha = lora_inputs(T, 264, 136, 16, 3, seed)
    return [x, randn(gen, T, 264), randn(gen, 264), randn(gen, 264), randn(gen, 264), gate_up, down, (a, b, alpha),
            ids_of("mixed", T, 3, seed), dout]


@pytest.mark.parametrize("T", [1, 20, 50, 300])
def test_captured_steps(T):
    """Two graphs of a step on one memory pool each, replayed in turn with eager work and synchronizations between, on new inputs."""
    sets = [step_inputs(T, 0), step_inputs(T, 1)]
    a_step(*sets[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(a_step(*s))
        graphs.append(g)
    for turn in range(4):
        for s in sets:
            s[0].copy_(torch.randn(s[0].shape, device=DEV))
            s[-1].copy_(torch.randn(s[-1].shape, device=DEV))
            s[-2].copy_(ids_of("mixed", T, 3, turn))
        want = [a_step(*s) for s in sets]
        torch.cuda.synchronize()
        for g in graphs if turn % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_two_streams_at_once():
    sets = [step_inputs(T, T) for T in (40, 300)]
    want = [a_step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i] = a_step(*s)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("T", [0, 1, 3, 40, 300])
@pytest.mark.parametrize("with_shared", [False, True])
def test_sparse_block(T, with_shared):
    """A block's expert half: router, routed experts, the shared expert with its rows' adapters and its gate, the residual stream
    in float32 and the next norm. The routed experts' own error is taken from their layer (tested in test_gpu_direct_layer.py)."""
    H, I, E, k, S = 512, 192, 16, 4, 136
    gen = gen_of(T)
    n, h = randn(gen, T, H), randn(gen, T, H, dtype=F32)
    router, gate = randn(gen, E, H, scale=0.05), randn(gen, H, scale=0.05)
    banks = randn(gen, E * 2 * I, H, scale=0.05), randn(gen, E * H, I, scale=0.05)
    shared = randn(gen, 2 * S, H, scale=0.05), randn(gen, H, S, scale=0.05)
    loras = lora_inputs(max(T, 1), H, 2 * S, 8, 3)[2:], lora_inputs(max(T, 1), S, H, 16, 3, seed=1)[2:]
    ids = ids_of("mixed", T, 3)
    weight = randn(gen, H, dtype=F32)
    options = dict(shared=shared, shared_gate=block.gate_weight(gate), shared_lora=loras, ids=ids) if with_shared else {}
    got_h, got_n = block.sparse_block(n, h, router, *banks, k, next_weight=weight, scale=0.5, **options)
    assert got_h.dtype == F32 and got_n.dtype == BF and got_h.shape == got_n.shape == (T, H)
    if T == 0:
        return
    experts, weights = kernels.route(block.linear(n, router), k)
    routed = kernels.bf16_layer(n, experts, weights, *banks, E).to(F64)
    want, err = h.to(F64) + 0.5 * routed, 4 * HALF[F32] * (h.to(F64).abs() + routed.abs())
    if with_shared:
        ref = Ffn(n, *shared, loras, ids)
        v, e = dot(n.to(F64), gate.to(F64)[:, None])
        e = rounded(v, e)  # the logit is rounded, and so is its sigmoid, whose slope is at most 1 / 4
        g = torch.sigmoid(v)
        want, err = want + 0.5 * g * ref.out, err + 0.5 * (g * ref.e_out + (0.25 * e + HALF[BF] * g) * (ref.out.abs() + ref.e_out)) \
            + 8 * HALF[F32] * (want.abs() + ref.out.abs())
    within(got_h, want, err + 1e-30)
    rms = (want * want).mean(1, keepdim=True).sqrt()
    rel = ((got_n.to(F64) - want / rms * weight.to(F64)).norm() / (want / rms * weight.to(F64)).norm()).item()
    assert rel < 2.0 ** -8 + (err.norm() / want.norm()).item()


def test_sparse_block_captured():
    H, I, E = 512, 192, 16
    gen = gen_of(3)
    n, h = randn(gen, 20, H), randn(gen, 20, H)
    args = randn(gen, E, H), randn(gen, E * 2 * I, H, scale=0.05), randn(gen, E * H, I, scale=0.05), 4
    options = dict(shared=(randn(gen, 2 * I, H, scale=0.05), randn(gen, H, I, scale=0.05)), shared_gate=block.gate_weight(randn(gen, H)),
                   next_weight=randn(gen, H))
    block.sparse_block(n, h, *args, **options)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.sparse_block(n, h, *args, **options)
    for _ in range(3):
        n.copy_(torch.randn(n.shape, device=DEV))
        want = block.sparse_block(n, h, *args, **options)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_training_step_by_autograd():
    """Two layers by autograd against the same in float64: the operators in a row, as a model trains with them."""
    T, H, I = 90, 136, 72
    gen = gen_of(0)
    x = randn(gen, T, H)
    layers = [dict(gu=randn(gen, 2 * I, H, scale=0.1), dn=randn(gen, H, I, scale=0.1), w=randn(gen, H) + 2, g=randn(gen, H)) for _ in range(2)]
    leaves = [t.requires_grad_() for layer in layers for t in layer.values()]
    first = (torch.ones(H, device=DEV, dtype=BF)).requires_grad_()
    h, n = x, block.norm(x, first)
    for p in layers:
        h, n = block.add_norm(block.gated_ffn(n, p["gu"], p["dn"]), h, p["w"], gate=p["g"], scale=0.5)
    dout = randn(gen, T, H)
    got = torch.autograd.grad(n, [first, *leaves], dout)
    d_leaves = [t.detach().to(F64).requires_grad_() for t in [first, *leaves]]
    it = iter(d_leaves[1:])
    unit = lambda t: t / torch.sqrt((t * t).mean(1, keepdim=True) + 1e-6)  # noqa: E731
    h, n = x.to(F64), unit(x.to(F64)) * d_leaves[0]
    for _ in layers:
        gu, dn, w, g = (next(it) for _ in range(4))
        pre = n @ gu.T
        h = h + 0.5 * g * ((pre[:, :I] * torch.sigmoid(pre[:, :I]) * pre[:, I:]) @ dn.T)
        n = unit(h) * w
    want = torch.autograd.grad(n, d_leaves, dout.to(F64))
    # some ten roundings to bf16 on the longest way, each at most 2^-8 / sqrt(3) of the norm on the average: 2^-8 sqrt(10 / 3)
    for a, b in zip(got, want):
        assert ((a.to(F64) - b).norm() / b.norm()).item() < 2.0 ** -8 * (10 / 3) ** 0.5


@pytest.mark.parametrize("stream, dtype", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
def test_norm_pair_captured(stream, dtype):
    """The explicit pair of a model's first norm: autograd's numbers, eager and in a graph that is replayed on new rows."""
    gen = gen_of(2)
    x, weight, dn = randn(gen, 37, 264, dtype=stream), randn(gen, 264, dtype=stream), randn(gen, 37, 264, dtype=dtype)

    def step():
        n, saved = block.norm_forward(x, weight, unit_offset=True, dtype=dtype)
        return (n, *block.norm_backward(dn, x, saved, weight, unit_offset=True))

    leaves = [t.clone().requires_grad_() for t in (x, weight)]
    out = block.norm(*leaves, unit_offset=True, dtype=dtype)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip((out, *torch.autograd.grad(out, leaves, dn)), want))
    n, saved = block.norm_forward(x, weight, unit_offset=True, dtype=dtype)
    for i in range(2):
        one = block.norm_backward(dn, x, saved, weight, unit_offset=True, needs=(i == 0, i == 1))
        assert torch.equal(one[i], want[1 + i]) and one[1 - i] is None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device=DEV))
        dn.copy_(torch.randn(dn.shape, device=DEV))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_adapters_by_turns_have_no_cliff():
    """Rows that name 32 adapters by turns: one row more than 256 takes about as long (it took five times as long where the rule of
    the workgroups an adapter tile gets went by the rows alone)."""
    times = {}
    for T in (256, 257, 500):
        x, w, a, b, alpha = lora_inputs(T, 2048, 1024, 32, 32)
        ids = ids_of("each", T, 32)
        for _ in range(3):
            block.lora_linear(x, w, a, b, alpha, ids)
        best = float("inf")
        for _ in range(8):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(20):
                block.lora_linear(x, w, a, b, alpha, ids)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        times[T] = best
    assert times[257] < 2.5 * times[256] and times[500] < 3 * times[256], times


@pytest.mark.parametrize("kind", ["each", "runs", "mixed", "outside"])
@pytest.mark.parametrize("T, K, N, rank, count", [(300, 136, 72, 40, 70), (517, 264, 136, 8, 33), (1100, 72, 264, 160, 3), (2100, 64, 64, 96, 90)])
def test_lora_linear_many_rows(T, K, N, rank, count, kind):
    """More rows than 256 and adapters by turns: tiles of rows that name more adapters than they have workgroups, or fewer."""
    x, w, a, b, alpha = lora_inputs(T, K, N, rank, count, seed=T)
    ids = ids_of(kind, T, count)
    base, e_base = dot(x.to(F64), w.to(F64).T)
    more, e_more = adapter(x.to(F64), a, b, alpha, ids)
    within(block.lora_linear(x, w, a, b, alpha, ids), base + more, rounded(base + more, e_base + e_more), kind)


# --------------------------------------------------------------------- many rows: sums over them, and every size of tile
def norm_bounds(doubles, dh, dn, scale, offset, eps, additions):
    """(gradients, bounds) in float64 of dresidual and of what is summed over the rows, for float32 work on a stream that is not
    rounded on the way: a row's sums and their roots off by 100 steps u = 2^-24 (as in norm_check), each product by one; a
    sum over the rows by `additions` steps of its terms' magnitudes."""
    u = 2.0 ** -24
    y, residual, weight, post, gate = doubles
    rms = lambda t: (t * t).mean(1, keepdim=True).add(eps).sqrt()  # noqa: E731
    yhat = y if post is None else y / rms(y)
    v = yhat if post is None else yhat * (post + offset)
    g = 1.0 if gate is None else gate
    h = residual + scale * g * v
    e_h = 100 * u * ((h - residual).abs() + residual.abs())
    r = 1 / rms(h)
    e_r = 100 * u + (e_h * h.abs()).mean(1, keepdim=True) * r ** 2  # relative
    hat = h * r
    e_hat = e_h * r + hat.abs() * e_r
    a = dn * (weight + offset)
    m = (a * hat).mean(1, keepdim=True)
    e_m = 100 * u * (a * hat).abs().mean(1, keepdim=True) + (a.abs() * e_hat).mean(1, keepdim=True)
    dr = dh + r * (a - hat * m)
    e_dr = (8 * u + e_r) * (dh.abs() + r * (a.abs() + (hat * m).abs())) + r * (e_hat * m.abs() + hat.abs() * e_m)

    def summed(terms, err):
        return terms.sum(0), err.sum(0) + additions * u * terms.abs().sum(0)

    def product(factor):  # of dv = scale dr and a factor that is off by 100 steps and a few
        return scale * dr * factor, abs(scale) * factor.abs() * (e_dr + 110 * u * dr.abs())

    found = {"residual": (dr, e_dr), "weight": summed(dn * hat, dn.abs() * (e_hat + 2 * u * hat.abs()))}
    if post is not None:
        found["post"] = summed(*product(g * yhat))
    if gate is not None and gate.dim() == 1:
        found["gate"] = summed(*product(v))
    elif gate is not None and gate.shape[1] == 1:
        terms, err = product(v)  # a row's sum over its columns
        found["gate"] = terms.sum(1, keepdim=True), (err + 100 * u * terms.abs()).sum(1, keepdim=True)
    elif gate is not None:
        found["gate"] = product(v)
    return found


@pytest.mark.parametrize("of, stream, weights", [(BF, BF, BF), (BF, F32, F32), (F32, F32, F32), (F32, BF, F32)])
@pytest.mark.parametrize("gate, post", [("none", False), ("channel", True), ("row", True), ("full", True), ("channel", False)])
@pytest.mark.parametrize("T, H", [(8192, 512), (4099, 72), (5000, 1000), (1600, 2048), (1391, 5120), (601, 8200), (600, 16384)])
def test_add_norm_sums_over_many_rows(T, H, gate, post, of, stream, weights):
    """More rows than a backward pass has groups, so that each walks several, at widths of every form of the kernel. Every sum over
    the rows is held to half a step of itself and to float32's steps, which a row left out, or h read back as it was rounded to a
    bfloat16 stream, exceeds by far."""
    scale, offset = 0.7, not post
    y, residual, weight, post_w, g, dh, dn = norm_inputs(T, H, of, stream, gate, post, weights, seed=T + H)
    opt = {"post": post_w, "gate": g, "scale": scale, "unit_offset": offset}
    h, _, saved = block.add_norm_forward(y, residual, weight, **opt)
    grads = dict(zip(("y", "residual", "weight", "post", "gate"), block.add_norm_backward(dh, dn, y, h, saved, weight, **opt)))
    groups = _lib.lib().d3_add_norm_partials(T, H) // H
    assert T > groups
    # a group's rows one after the other, every 128th group, 4 of those and 32 of these
    additions = -(-T // groups) + -(-groups // 128) + 4 + 32
    found = norm_bounds([None if t is None else t.to(F64) for t in (y, residual, weight, post_w, g)], dh.to(F64), dn.to(F64), scale,
                        float(offset), 1e-6, additions)
    for name, (want, err) in found.items():
        within(grads[name], want, rounded(want, err, grads[name].dtype), name)
    norm_check(T, H, of, stream, gate, post, weights, scale=scale, offset=offset, seed=T + H)


@pytest.mark.parametrize("T, H, I, O", [
    (900, 72, 520, 264),       # gate and up by 64 x 64
    (4001, 1032, 6152, 4040),  # the second product, gate's and up's gradients and the set of gradients by 256 x 256
    (2500, 264, 4072, 72),     # gate's and up's gradients: 128 x 256 for whole turns, then 64 x 64
    (3300, 72, 3080, 520),     # then 128 x 128
    (5000, 136, 3080, 264),    # then 32 x 64
])
def test_gated_ffn_by_other_tiles(T, H, I, O):
    test_gated_ffn(T, H, I, O)


@pytest.mark.parametrize("kind", ["runs", "each", "outside"])
@pytest.mark.parametrize("T, K, N, rank, count", [
    (700, 72, 1032, 40, 9),      # 64 x 64
    (700, 200, 3080, 72, 5),     # 128 x 128
    (1900, 136, 3080, 136, 7),   # 128 x 256
    (2500, 72, 4072, 16, 12),    # 128 x 256 for whole turns, then 64 x 64
    (3300, 264, 3080, 64, 6),    # then 128 x 128
    (5000, 64, 3080, 96, 4),     # then 64 x 32
])
def test_lora_linear_by_other_tiles(T, K, N, rank, count, kind):
    test_lora_linear(T, K, N, rank, count, kind)


@pytest.mark.parametrize("kind", ["runs", "each"])
@pytest.mark.parametrize("T, H, I, O", [
    (700, 72, 520, 1032),     # gate and up by 64 x 64, down too
    (1100, 136, 1032, 2056),  # 128 x 128
    (3300, 72, 776, 3080),    # 128 x 256, down 128 x 256 for whole turns, then 128 x 128
    (2500, 72, 2056, 264),    # 128 x 256 for whole turns, then 128 x 128
    (5000, 64, 776, 136),     # then 64 x 64
    (5000, 72, 1544, 72),     # then 64 x 32
])
def test_gated_ffn_with_adapters_by_other_tiles(T, H, I, O, kind):
    x, gate_up, down, _ = ffn_inputs(T, H, I, O, seed=T)
    lora = lora_inputs(T, H, 2 * I, 40, 6, seed=1)[2:], lora_inputs(T, I, O, 72, 6, seed=2)[2:]
    ids = ids_of(kind, T, 6)
    ref = Ffn(x, gate_up, down, lora, ids)
    within(block.gated_ffn(x, gate_up, down, gate_up_lora=lora[0], down_lora=lora[1], ids=ids), ref.out, ref.e_out)


@pytest.mark.parametrize("T, K, N", [(300, 72, 2056), (700, 72, 3080), (1900, 72, 3080), (5000, 72, 3080)])
def test_lora_linear_bad_adapters_stay_in_their_rows_of_other_tiles(T, K, N):
    """As above, at 64 x 64, 128 x 128, 128 x 256 and the latter followed by 64 x 32."""
    x, w, a, b, alpha = lora_inputs(T, K, N, 72, 4, seed=T)
    ids = torch.arange(T, device=DEV) % 4 - 1
    want = block.lora_linear(x, w, a, b, alpha, ids)
    a2, b2 = a.clone(), b.clone()
    a2[1], b2[1, ::2], b2[3], a2[3] = float("inf"), float("nan"), float("nan"), float("nan")
    got = block.lora_linear(x, w, a2, b2, alpha, ids)
    assert torch.equal(got[ids != 1], want[ids != 1])
    assert not got[ids == 1].isfinite().all(1).any()
