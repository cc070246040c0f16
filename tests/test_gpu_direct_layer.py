"""The routed layer on bfloat16 and on microscaled banks (kernels.bf16_layer, mx.moe_layer) and its ways in
(offload.resident_decode, routed_decode, resident_prefill, ExpertTable): the operators in a row, as they are used."""
import numpy as np
import pytest
import torch

from drama3 import kernels, mx, offload

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


class Layer:
    def __init__(self, kind, E, H, I, seed=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.kind, self.E, self.H, self.I = kind, E, H, I
        w = [torch.randn((E, n, k), generator=gen, device=DEV) * 0.05 for n, k in ((2 * I, H), (H, I))]
        if kind == "bf16":
            self.banks = [{"weight": v.to(torch.bfloat16).flatten(0, 1)} for v in w]
        else:
            self.mx = [mx.quantize_bank(v) for v in w]
            self.banks = [{"weight": b.weight, "scale": b.scale} for b in self.mx]
        self.rows = (2 * I, H)

    def inputs(self, T, k, seed=1):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn((T, self.H), generator=gen, device=DEV).to(torch.bfloat16)
        ids = torch.rand((T, self.E), generator=gen, device=DEV).topk(k, dim=1).indices
        weights = torch.softmax(torch.randn((T, k), generator=gen, device=DEV), dim=1).to(torch.bfloat16)
        return x, ids, weights

    def __call__(self, x, ids, weights):
        if self.kind == "bf16":
            return kernels.bf16_layer(x, ids, weights, *(b["weight"] for b in self.banks), self.E)
        return mx.moe_layer(x, ids, weights, *self.mx, bits=int(self.kind[2]))

    def parts(self, x, ids):
        """The pairs' outputs [T, k, H] float32 from the products for single pairs."""
        T, k = ids.shape
        flat = ids.flatten()
        if self.kind == "bf16":
            h = kernels.gemv_bf16(x, flat, self.banks[0]["weight"], 2 * self.I, swiglu=True)
            return kernels.gemv_bf16(h, flat, self.banks[1]["weight"], self.H).view(T, k, -1)
        bits = int(self.kind[2])
        h = mx.gemv(mx.quantize(x, bits), flat, self.mx[0], swiglu=True)
        return mx.gemv(mx.quantize(h, bits), flat, self.mx[1]).view(T, k, -1)


@pytest.mark.parametrize("T, k", [(1, 8), (1, 1), (3, 8), (4, 2), (5, 8), (40, 3), (300, 8), (1100, 8)])
@pytest.mark.parametrize("kind", ["bf16", "mx4", "mx8"])
def test_layer_is_its_products_in_a_row(kind, T, k):
    """The layer at every way it takes (lines, streamed and wide passes, either grouping) against the single pairs' products,
    which are bit for bit its own, weighted and summed over k: k products and sums in float32 (each within 2^-24 of sum
    |w y|), the result rounded to bfloat16."""
    layer = Layer(kind, 12, 512, 192)
    x, ids, weights = layer.inputs(T, k)
    got = layer(x, ids, weights)
    assert got.shape == x.shape and got.dtype == torch.bfloat16
    pairs = layer.parts(x, ids).double() * weights.double()[..., None]
    want, size = pairs.sum(1), pairs.abs().sum(1)
    off = 2 * k * 2.0 ** -24 * size
    assert torch.all((got.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off) + 1e-37)


def test_bf16_layer_against_64_bits():
    """The whole layer from the formula: float32 sums of 32 products a step (2 units of the last place each), SiLU within
    2^-21 + |g| 2^-23 and |SiLU'| <= 1.1, the hidden values rounded to bfloat16, their errors through the second product."""
    layer = Layer("bf16", 6, 1024, 256)
    x, ids, weights = layer.inputs(50, 4)
    wg, wd = (b["weight"].double().view(6, n, -1) for b, n in zip(layer.banks, layer.rows))
    x64 = x.double()
    want, allowed = torch.zeros((50, 1024), dtype=torch.float64, device=DEV), 0
    for j in range(4):
        w = wg[ids[:, j]]
        gu, size = (torch.einsum("tk,tnk->tn", a, b) for a, b in ((x64, w), (x64.abs(), w.abs())))
        d = (1024 // 32 + 3) * 2.0 ** -22 * size
        (g, u), (dg, du) = gu.chunk(2, 1), d.chunk(2, 1)
        silu = g * torch.sigmoid(g)
        h = silu * u
        dh = 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + (2.0 ** -21 + g.abs() * 2.0 ** -23) * h.abs()
        dh = dh + 2.0 ** -8 * (h.abs() + dh)
        w = wd[ids[:, j]]
        y, size = torch.einsum("tk,tnk->tn", h, w), torch.einsum("tk,tnk->tn", h.abs() + dh, w.abs())
        dy = torch.einsum("tk,tnk->tn", dh, w.abs()) + (256 // 32 + 3) * 2.0 ** -22 * size
        share = weights[:, j:j + 1].double()
        want += share * y
        allowed = allowed + share * (dy + 8 * 2.0 ** -24 * (y.abs() + dy))
    got = layer(x, ids, weights).double()
    assert torch.all((got - want).abs() <= allowed + 2.0 ** -8 * (want.abs() + allowed))


@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_a_row_does_not_depend_on_the_others(kind):
    layer = Layer(kind, 8, 256, 128)
    x, ids, weights = layer.inputs(2000, 4)
    whole = layer(x, ids, weights)
    for part in (slice(0, 1), slice(7, 11), slice(100, 105), slice(3, 900)):
        assert torch.equal(layer(x[part], ids[part], weights[part]), whole[part])


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_ways_in(kind):
    """ExpertTable and the resident entries with the two kinds; routed_decode routes as kernels.route does."""
    E, H, I, k = 16, 512, 256, 4
    layer = Layer(kind, E, H, I)
    run = Layer.__call__ if kind == "bf16" else lambda s, *a: mx.moe_layer(*a, *s.mx, bits=8)
    x, ids, weights = layer.inputs(60, k)
    table = offload.ExpertTable(DEV)
    table.place(0, kind, *layer.banks)
    assert table.bytes == sum(t.nbytes for b in layer.banks for t in b.values())
    assert torch.equal(table.prefill(0, x, ids, weights, E), run(layer, x, ids, weights))
    one = run(layer, x[:1], ids[:1], weights[:1])
    assert torch.equal(table.decode(0, x[:1], ids[0], weights[0], E), one)
    assert torch.equal(offload.resident_prefill(x, ids, weights, layer.banks, layer.rows, kind, (None, None), E),
                       run(layer, x, ids, weights))
    logits = torch.randn((1, E), device=DEV).to(torch.bfloat16)
    out, got_ids, got_w = offload.routed_decode(x[:1], logits, k, layer.banks, layer.rows, kind, (None, None))
    want_ids, want_w = kernels.route(logits, k)
    assert torch.equal(got_ids, want_ids) and torch.equal(got_w, want_w)
    assert torch.equal(out, run(layer, x[:1], want_ids, want_w))


@pytest.mark.parametrize("kind", ["bf16", "mx8"])
@pytest.mark.parametrize("T", [1, 30, 1500])
def test_captured_layer(kind, T):
    """Captured, and replayed with other rows and routes in place, with eager calls between; two graphs of one layer."""
    layer = Layer(kind, 8, 256, 128)
    a, b = layer.inputs(T, 8), layer.inputs(T, 8, seed=2)
    want = [layer(*a), layer(*b)]
    held = [t.clone() for t in a]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                out = layer(*held)
            graphs.append((g, out))
    torch.cuda.current_stream().wait_stream(stream)
    for turn in range(6):
        for h, t in zip(held, (a, b)[turn % 2]):
            h.copy_(t)
        g, out = graphs[turn // 2 % 2]
        g.replay()
        assert torch.equal(layer(*held), want[turn % 2])
        torch.cuda.synchronize()
        assert torch.equal(out, want[turn % 2])


def test_empty_and_refused():
    layer = Layer("bf16", 4, 128, 64)
    x, ids, weights = layer.inputs(3, 2)
    assert layer(x[:0], ids[:0], weights[:0]).shape == (0, 128)
    with pytest.raises(ValueError):
        layer(x, ids[:2], weights)
    with pytest.raises(ValueError):
        kernels.bf16_layer(x, ids, weights, layer.banks[0]["weight"], layer.banks[1]["weight"], 3)
    bad = mx.quantize_bank(torch.randn((4, 64, 128), device=DEV))
    with pytest.raises(ValueError):
        mx.moe_layer(x, ids, weights, bad, bad)
    # routes outside the bank are left out of the sum
    out_of = ids.clone()
    out_of[:, 1] = 9
    alone = layer(x, ids[:, :1], weights[:, :1])
    assert torch.equal(layer(x, out_of, weights), alone)
    big = layer.inputs(50, 2, seed=3)
    out_of = big[1].clone()
    out_of[:, 1] = -1
    assert torch.equal(layer(big[0], out_of, big[2]), layer(big[0], big[1][:, :1], big[2][:, :1]))


@pytest.mark.parametrize("E, P", [(1, 1), (7, 1023), (128, 30011), (1024, 70000)])
def test_prompt_expert_groups(E, P):
    """The grouping over many workgroups gives expert_groups' groups and, within them, its pairs."""
    rng = np.random.default_rng(P)
    ids = rng.integers(0, E, P)
    ids[rng.random(P) < 0.01] = -3
    t = torch.from_numpy(ids).to(DEV).view(-1, 1)
    order, inverse, groups = kernels.prompt_expert_groups(t, E)
    _, _, want = kernels.expert_groups(t, E)
    assert torch.equal(groups, want)
    order, inverse = order.cpu().numpy(), inverse.cpu().numpy()
    assert np.array_equal(np.sort(order), np.arange(P))
    for e, _, _, first, n in groups.cpu().numpy()[:: max(1, E // 50)]:
        assert np.all(ids[order[first:first + n]] == e)
    valid = ids >= 0
    assert np.array_equal(order[inverse[valid]], np.arange(P)[valid]) and np.all(inverse[~valid] == -1)
