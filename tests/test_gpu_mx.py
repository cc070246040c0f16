"""The quantizer of microscaled rows bit for bit against its definition, and the expert products on microscaled and on
bfloat16 banks against 64-bit sums of the values that their operands hold."""
import numpy as np
import pytest
import torch

from drama3 import kernels, mx
from oracle import mx as omx

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


# ------------------------------------------------------------------------------------------------------- quantizer
def _blocks():
    """Rows of 32 columns that a quantizer can get wrong: zeros, powers of two, the borders between elements and around
    saturation, subnormal maxima, the ends of float32's range, and blocks with an infinity or NaN."""
    rng = np.random.default_rng(3)
    rows = [np.zeros(32), -np.zeros(32), np.full(32, 1.0), np.full(32, -0.75)]
    for g in (omx.E2M1, omx.E4M3):
        mid = (g[1:] + g[:-1]) / 2
        every = np.concatenate([g, mid, np.nextafter(mid.astype(np.float32), np.float32(0)).astype(np.float64),
                                np.nextafter(mid.astype(np.float32), np.float32(1e9)).astype(np.float64)])
        for part in np.array_split(every, -(-len(every) // 31)):
            row = np.zeros(32)
            row[:len(part)] = part * np.where(np.arange(len(part)) % 2, -1, 1)
            row[31] = 1.875 * 2.0 ** np.floor(np.log2(g[-1]))  # in the largest element's binade: scale 1, and saturated
            rows += [row, row * 2.0 ** 40, row * 2.0 ** -70]
    for top in (2.0 ** -149, 2.0 ** -126, 2.0 ** -120, 3.4028234663852886e38):
        row = rng.uniform(-1, 1, 32)
        row[rng.integers(32)] = 1.0
        rows += [row * top, row * top * 0.7]
    for bad in (np.inf, -np.inf, np.nan):
        row = rng.standard_normal(32)
        row[7] = bad
        rows.append(row)
    return np.array(rows).astype(np.float32)


def _check_quantized(x, got, bits):
    """codes and scales equal the definition's (the sign of a zero and the elements of a NaN block aside)."""
    want, scale = omx.quantize(x, bits)
    cols = x.shape[1]
    assert np.array_equal(got.scale.cpu().numpy()[:, :cols // 32], scale)
    codes = omx.unpack(got.codes.cpu().numpy(), bits)
    assert not codes[:, cols:].any() and not got.scale[:, cols // 32:].any()
    fine = np.repeat(scale, 32, axis=1) != 255
    a, b = (omx.values(c, np.full_like(scale, 127), bits)[fine] for c in (codes[:, :cols], want))
    assert np.array_equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_edges(bits):
    x = _blocks()
    got = mx.quantize(dev(x), bits)
    _check_quantized(x, got, bits)
    # the same blocks side by side in one row, and in bfloat16
    wide = x.reshape(1, -1)
    _check_quantized(wide, mx.quantize(dev(wide), bits), bits)
    half = dev(x).to(torch.bfloat16)
    _check_quantized(half.float().cpu().numpy(), mx.quantize(half, bits), bits)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_every_bfloat16(bits):
    """Every finite bfloat16 value in a block of each scale that it may meet: its own, and eight binades more."""
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    v = v[torch.isfinite(v)].numpy()
    v = v[np.abs(v) < 2.0 ** 100]
    for up in (0, 1, 4, 8):
        x = np.zeros((len(v), 32), np.float32)
        x[:, 3] = v
        x[:, 20] = np.exp2(np.frexp(v)[1] - 1 + up)
        h = dev(x).to(torch.bfloat16)
        _check_quantized(x, mx.quantize(h, bits), bits)


@pytest.mark.parametrize("R, cols", [(0, 64), (1, 32), (3, 96), (1, 2048), (37, 800), (1000, 768), (5, 4096)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_and_back(R, cols, dtype, bits):
    gen = torch.Generator().manual_seed(R + cols)
    x = (torch.randn((R, cols), generator=gen) * torch.randn((R, 1), generator=gen).exp2()).to(dtype)
    got = mx.quantize(x.to(DEV), bits)
    assert got.codes.shape == (R, -(-cols // 256) * 32 * bits) and got.scale.shape == (R, -(-cols // 256) * 8)
    if R:
        _check_quantized(x.float().numpy(), got, bits)
    want = omx.values(*omx.quantize(x.float().numpy(), bits), bits) if R else np.zeros((0, cols))
    assert np.array_equal(mx.dequantize(got).double().cpu().numpy(), want)
    # an element has 2 or 4 significant bits: bfloat16 holds its value too
    assert np.array_equal(mx.dequantize(got, torch.bfloat16).double().cpu().numpy(), want)


def test_quantize_strided_rows():
    """Rows further apart than their columns, a view at an offset that is not 16-byte aligned, transposed and expanded."""
    x = torch.randn((40, 300), device=DEV)
    for view in (x[:, :96], x[::2, 4:132], x[1:, 3:99], x[:32].t()[:64], x[:1, :64].expand(8, 64)):
        a, b = mx.quantize(view, 8), mx.quantize(view.clone(memory_format=torch.contiguous_format), 8)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)


def test_dequantize_every_scale_code():
    """Every e2m1 and e4m3 code at every scale code: float32 exactly where it holds the value."""
    for bits, n in ((4, 16), (8, 256)):
        codes = np.zeros((256, 256), np.uint8)
        codes[:, :n] = np.arange(n)
        scale = np.repeat(np.arange(256)[:, None], 8, axis=1).astype(np.uint8)
        rows = mx.rows_from(dev(omx.pack(codes, bits)), dev(scale), bits)
        want = omx.values(codes, scale, bits)
        with np.errstate(over="ignore"):
            single = want.astype(np.float32)
        assert np.array_equal(mx.dequantize(rows).cpu().numpy(), single, equal_nan=True)
        got = mx.dequantize(rows, torch.bfloat16).float().cpu().numpy()
        normal = np.isnan(want) | (want == 0) | ((np.abs(want) >= 2.0 ** -126) & (np.abs(want) < 3e38))
        assert np.array_equal(got[normal], single[normal], equal_nan=True)


# -------------------------------------------------------------------------------------------------------- products
FORMATS = ["mx4", "mx8", "bf16"]


class Case:
    """A bank of E experts [n, K] and R rows in a format, their values in 64 bits, and the products on them."""

    def __init__(self, fmt, E, n, K, R, seed=0, spread=0.0):
        rng = np.random.default_rng(seed + 7919 * n + K)
        self.fmt, self.E, self.n, self.K, self.R = fmt, E, n, K, R
        x = rng.standard_normal((R, K)) * np.exp2(spread * rng.standard_normal((R, K // 32)).repeat(32, 1))
        w = rng.standard_normal((E * n, K)) * 0.02 * np.exp2(spread * rng.standard_normal((E * n, K // 32)).repeat(32, 1))
        if fmt == "bf16":
            self.x, self.w = dev(x).to(torch.bfloat16), dev(w).to(torch.bfloat16)
            self.xv, self.wv = self.x.double(), self.w.double().view(E, n, K)
        else:
            bits = int(fmt[2])
            (xc, xs), (wc, ws) = omx.quantize(x, bits), omx.quantize(w, 4)
            self.x = mx.rows_from(dev(omx.pack(xc, bits)), dev(xs), bits)
            self.w = mx.bank(mx.rows_from(dev(omx.pack(wc, 4)), dev(ws), 4), E)
            self.xv, self.wv = dev(omx.values(xc, xs, bits)), dev(omx.values(wc, ws, 4)).view(E, n, K)

    def gemv(self, ids, **how):
        if self.fmt == "bf16":
            return kernels.gemv_bf16(self.x, ids, self.w, self.n, **how)
        return mx.gemv(self.x, ids, self.w, **how)

    def grouped(self, groups, **how):
        if self.fmt == "bf16":
            return kernels.grouped_bf16(self.x, groups, self.w, self.n, **how)
        return mx.grouped(self.x, groups, self.w, **how)

    def want(self, row, expert, swiglu, rounded):
        """(values, allowed error before the output's own rounding) of pairs (row, expert), in 64 bits. Products are exact;
        a step adds its 32 (bf16) or 128 of them to the sum with one rounding of what it aligns to 24 bits or more: at most
        2 units of the last place of the largest partial sum, below sum |x w|, for each of the steps (two to a step of e4m3
        rows). Results from e4m3 rows that are rounded to bf16: the instruction aligns a block's 32 products to the largest
        one's exponent e and cuts what lies below 2^(e - 13). With 4 and 2 significant bits a product p's last place is at
        least 2^-4 of its power of two, so only products below 2^(e - 8) are cut, each by less than 2^(e - 13) and |p|, and
        2^e is at most the largest product."""
        x, w = self.xv[row], self.wv[expert]
        p = x[:, None] * w
        out, size = p.sum(-1), p.abs().sum(-1)
        off = (self.K // (32 if self.fmt == "bf16" else 64) + 3) * 2.0 ** -22 * size
        if self.fmt == "mx8" and rounded:
            p = p.abs().unflatten(-1, (-1, 32))
            top = p.amax(-1, keepdim=True)
            off += torch.where(p < top * 2.0 ** -8, torch.minimum(p, top * 2.0 ** -13), 0.0).sum((-2, -1))
        if not swiglu:
            return out, off
        (g, u), (dg, du) = out.chunk(2, dim=1), off.chunk(2, dim=1)
        silu = g * torch.sigmoid(g)
        # |SiLU'| <= 1.1; SiLU in float32: exp within 2 ulp and of an argument rounded to |g| 2^-24, a sum, a division, a product
        return silu * u, 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + \
            (2.0 ** -21 + g.abs() * 2.0 ** -23) * (silu * u).abs()

    def check(self, got, row, expert, swiglu=False):
        for part in range(0, len(row), 32):
            at = slice(part, part + 32)
            want, off = self.want(row[at], expert[at], swiglu, got.dtype == torch.bfloat16)
            eps = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
            err = (got[at].double() - want).abs()
            allowed = off + eps * (want.abs() + off) + 1e-37
            assert torch.all(err <= allowed), (self.fmt, float((err / allowed).max()))


@pytest.mark.parametrize("n, K", [(16, 64), (32, 256), (48, 320), (96, 768), (160, 2048), (32, 2368), (64, 5120)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_gemv(fmt, n, K):
    """Decode lines: one row for all its experts, a row per pair, repeated experts, ids outside the bank (zeros)."""
    case = Case(fmt, 5, n, K, 3, spread=1.0)
    ids = dev(np.array([4, 0, 2, 2, -1, 1, 5, 3, 0], np.int64))
    row = torch.arange(9, device=DEV) // 3
    ok = (ids >= 0) & (ids < 5)
    for how in ({}, {"dtype": torch.bfloat16}, {"swiglu": True}):
        if n % 32 and "swiglu" in how:
            continue
        got = case.gemv(ids, **how)
        assert not got[~ok].any()
        case.check(got[ok], row[ok], ids[ok], "swiglu" in how)
    one = case.gemv(ids[:3])
    assert torch.equal(one, case.gemv(ids)[[0]].new_tensor(one.tolist()))
    assert case.gemv(ids[:0]).shape == (0, n)


# rows of the experts: few on average, and many (around a pass's 128 and 256 rows)
COUNTS = [0, 1, 15, 16, 17, 31, 33, 0, 64, 65, 130, 3]
MANY = [0, 1, 127, 128, 129, 255, 256, 257, 0, 300, 513, 33, 16, 191]
FEW = [0, 1, 3, 16, 17, 0, 2, 5, 33, 1]


def _pairs(E, counts, seed=1):
    """The pairs of `counts` rows an expert in random order, grouped: (ids, order, groups)."""
    ids = torch.from_numpy(np.random.default_rng(seed).permutation(np.repeat(np.arange(E), counts))).to(DEV)
    order, inverse, groups = kernels.expert_groups(ids.view(-1, 1), E)
    return ids, order, inverse, groups


@pytest.mark.parametrize("counts, n, K", [
    (COUNTS, 16, 64), (COUNTS, 32, 256), (COUNTS, 96, 320), (COUNTS, 288, 768), (COUNTS, 160, 2048), (COUNTS, 32, 2368),
    (FEW, 32, 64), (FEW, 288, 512), (FEW, 160, 2368), (MANY, 16, 64), (MANY, 32, 192), (MANY, 288, 256), (MANY, 544, 320), (MANY, 160, 2048), (MANY, 256, 1344)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_grouped_ragged(fmt, counts, n, K):
    E, P = len(counts), sum(counts)
    case = Case(fmt, E, n, K, P, spread=1.0)
    ids, order, _, groups = _pairs(E, counts)
    for how in ({}, {"dtype": torch.bfloat16}, {"swiglu": True}):
        if n % 32 and "swiglu" in how:
            continue
        case.check(case.grouped(groups, order=order, **how), order, ids[order], "swiglu" in how)
    # without order: place p is row p
    case.check(case.grouped(groups), torch.arange(P, device=DEV), ids[order])


@pytest.mark.parametrize("fmt", FORMATS)
def test_grouped_top_k(fmt):
    """A prompt's pairs: row order[p] // k, several experts to a row."""
    E, T, k = 12, 100, 3
    case = Case(fmt, E, 64, 512, T)
    ids = torch.from_numpy(np.argsort(np.random.default_rng(5).random((T, E)), axis=1)[:, :k].copy()).to(DEV)
    order, inverse, groups = kernels.expert_groups(ids, E)
    got = case.grouped(groups, order=order, k=k, swiglu=True)
    case.check(got, order // k, ids.flatten()[order], True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_results_do_not_depend_on_the_other_rows(fmt):
    """A pair's result, bit for bit: as a decode line's, alone in its group, and among few and many other rows."""
    E, n, K, R = 4, 320, 1024, 700
    case = Case(fmt, E, n, K, R)
    everything = torch.empty((R, n), device=DEV)
    ids = torch.from_numpy(np.random.default_rng(2).integers(0, E, R)).to(DEV)
    line = case.gemv(ids)
    for counts in (R, 100, 17, 1):
        rows = torch.arange(counts, device=DEV)
        order, _, groups = kernels.expert_groups(ids[:counts].view(-1, 1), E)
        for how in ({}, {"swiglu": True}):
            got = case.grouped(groups, order=order, **how)
            want = line if not how else case.gemv(ids, swiglu=True)
            assert torch.equal(got, want[:counts][order])


@pytest.mark.parametrize("E, rows, n", [(10, 300, 800), (70, 33, 800), (100, 34, 800), (300, 34, 96)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_more_items_than_workgroups(fmt, E, rows, n):
    """Wide passes where a workgroup walks several of them, with a last turn that is shared and one that is not, more
    than 256 groups, and a last column that is not full: bit for bit the single pairs' results, some of them checked."""
    K = 128 if fmt == "bf16" else 512
    counts = np.random.default_rng(E).integers(rows - 1, rows + 2, E)
    counts[3], counts[5] = 0, 7 * rows
    P = int(counts.sum())
    case = Case(fmt, E, n, K, P)
    ids, order, _, groups = _pairs(E, counts)
    for how in ({}, {"swiglu": True}, {"dtype": torch.bfloat16}):
        got = case.grouped(groups, order=order, **how)
        assert torch.equal(got, case.gemv(ids, **how)[order])
        at = torch.arange(0, P, 499, device=DEV)
        case.check(got[at], order[at], ids[order[at]], "swiglu" in how)


@pytest.mark.parametrize("fmt", FORMATS)
def test_groups_outside_are_left_alone(fmt):
    """Places in no group and groups whose expert or places lie outside keep what `out` held; order's values outside
    the rows read the nearest row."""
    case = Case(fmt, 3, 32, 512, 40)
    groups = torch.tensor([[0, 0, 0, 5, 7], [3, 0, 0, 12, 4], [-1, 0, 0, 16, 4], [1, 0, 0, 38, 3], [2, 0, 0, -2, 3],
                           [1, 0, 0, 20, 0], [2, 0, 0, 30, 2], [1, 0, 0, 25, -1], [2, 0, 0, 2 ** 31 - 1, 2],
                           [0, 0, 0, 2, 2 ** 31 - 1]], dtype=torch.int32, device=DEV)
    out = torch.full((40, 32), -7.0, device=DEV)
    got = case.grouped(groups, out=out)
    assert got is out
    touched = torch.zeros(40, dtype=torch.bool, device=DEV)
    touched[5:12] = touched[30:32] = True
    assert torch.all(got[~touched] == -7)
    rows = torch.arange(40, device=DEV)
    case.check(got[5:12], rows[5:12], rows[5:12] * 0)
    case.check(got[30:32], rows[30:32], rows[30:32] * 0 + 2)
    # the same groups in wide passes (40 places an entry)
    wide, far = torch.full((400, 32), -7.0, device=DEV), torch.arange(400, device=DEV) % 40
    case.grouped(groups, order=far, out=wide)
    touched = torch.zeros(400, dtype=torch.bool, device=DEV)
    for first, n, e in ((5, 7, 0), (30, 2, 2), (38, 3, 1)):
        touched[first:first + n] = True
        case.check(wide[first:first + n], far[first:first + n], far[first:first + n] * 0 + e)
    assert torch.all(wide[~touched] == -7)
    order = torch.tensor([-5, 2 ** 40, 79, 0], device=DEV)
    one = torch.tensor([[0, 0, 0, 0, 4]], dtype=torch.int32, device=DEV)
    case.check(case.grouped(one, order=order, k=2), torch.tensor([0, 39, 39, 0], device=DEV), order * 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_is_not_finite_stays_in_its_row(fmt):
    """A NaN row and an infinite weight reach their own results only, also within a tile."""
    case = Case(fmt, 2, 64, 512, 20)
    ids = torch.arange(20, device=DEV) % 2
    order, _, groups = kernels.expert_groups(ids.view(-1, 1), 2)
    before = case.grouped(groups, order=order)
    if fmt == "bf16":
        case.x[6, 100] = float("nan")
        case.w[64 + 9, 3] = float("inf")
    else:
        case.x.scale[6, 3] = 255
        rows = mx.bank_rows(case.w)
        rows.scale[64 + 9, 0] = 255
        case.w = mx.bank(rows, 2)
    for got, pair in ((case.grouped(groups, order=order), order), (case.gemv(ids), torch.arange(20, device=DEV))):
        before_here = before[torch.argsort(order)][pair]
        bad = (pair == 6)[:, None] | ((ids[pair] == 1)[:, None] & (torch.arange(64, device=DEV) == 9))
        assert not torch.isfinite(got[bad]).any()
        assert torch.equal(got[~bad], before_here[~bad])


@pytest.mark.parametrize("fmt", FORMATS)
def test_capture_and_streams(fmt):
    """Captured in a graph and replayed with other inputs in place and eager work between, and run on a side stream."""
    case = Case(fmt, 6, 96, 768, 50)
    other = Case(fmt, 6, 96, 768, 50, seed=1)
    ids = torch.from_numpy(np.random.default_rng(3).integers(0, 6, 50)).to(DEV)
    order, _, groups = kernels.expert_groups(ids.view(-1, 1), 6)

    def run(c):
        return c.grouped(groups, order=order, swiglu=True), c.gemv(ids)

    want, want2 = run(case), run(other)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert all(torch.equal(a, b) for a, b in zip(run(case), want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run(case)
    torch.cuda.current_stream().wait_stream(stream)
    tensors = [(case.x, other.x)] if fmt == "bf16" else [(case.x.codes, other.x.codes), (case.x.scale, other.x.scale)]
    kept = [a.clone() for a, _ in tensors]
    for turn in range(4):
        graph.replay()
        torch.cuda.synchronize()
        if turn % 2 == 0:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        else:
            row = torch.arange(50, device=DEV)
            mixed = Case.__new__(Case)
            mixed.__dict__.update(case.__dict__, xv=other.xv)
            mixed.check(got[1], row, ids)
        for (a, b), k in zip(tensors, kept):
            a.copy_(b if turn % 2 == 0 else k)
        run(other)
        torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", ["mx8", "bf16"])
def test_banks_beyond_32_bit_offsets(fmt):
    """The last experts of a bank of more than 4 GiB."""
    n, K = 2048, 2048
    E = 560 if fmt == "bf16" else 2100
    small = Case(fmt, 2, n, K, 6)
    if fmt == "bf16":
        w = torch.zeros((E * n, K), dtype=torch.bfloat16, device=DEV)
        w[-2 * n:] = small.w
    else:
        w = mx.MxBank(torch.zeros((E * n, K // 2), dtype=torch.uint8, device=DEV),
                      torch.zeros((E * n, K // 32), dtype=torch.uint8, device=DEV), E, n, K)
        w.weight[-2 * n:], w.scale[-2 * n:] = small.w.weight, small.w.scale
    assert (w if fmt == "bf16" else w.weight).nbytes > 2 ** 32
    ids = torch.tensor([E - 1, E - 2, E - 1, E - 2, E - 2, E - 1], device=DEV)
    groups = torch.tensor([[E - 2, 0, 0, 0, 2], [E - 1, 0, 0, 2, 4]], dtype=torch.int32, device=DEV)
    want = small.gemv(ids - (E - 2))
    want_grouped = small.grouped(groups - torch.tensor([E - 2, 0, 0, 0, 0], dtype=torch.int32, device=DEV))
    small.w, small.E = w, E
    assert torch.equal(small.gemv(ids), want)
    assert torch.equal(small.grouped(groups), want_grouped)


@pytest.mark.parametrize("K", [64, 256, 512, 768, 1024, 1280, 2048, 2368])
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_few_pairs_of_many_experts(fmt, K):
    """Decode lines of fewer pairs than a sixth of the experts, at every number of stages that their loads go by, the same
    expert twice, ids outside; bit for bit the results of the same pairs among more. And groups of few rows."""
    case = Case(fmt, 48, 96, K, 2, spread=1.0)
    ids = torch.tensor([47, 3, 3, 0, 20, 48, 47, -1], device=DEV)
    row, ok = torch.arange(8, device=DEV) // 4, (ids >= 0) & (ids < 48)
    many = ids.view(2, 4).repeat_interleave(4, dim=1).flatten()  # four times each
    for how in ({}, {"dtype": torch.bfloat16}, {"swiglu": True}):
        got = case.gemv(ids, **how)
        assert not got[~ok].any()
        case.check(got[ok], row[ok], ids[ok], "swiglu" in how)
        assert torch.equal(case.gemv(many, **how)[::4], got)
    one = Case(fmt, 48, 96, K, 1)
    assert torch.equal(one.gemv(ids), torch.cat([one.gemv(ids[i:i + 1]) for i in range(8)]))
    rows = Case(fmt, 10, 96, K, sum(FEW))
    ids, order, _, groups = _pairs(10, FEW)
    for how in ({}, {"swiglu": True}):
        rows.check(rows.grouped(groups, order=order, **how), order, ids[order], "swiglu" in how)


@pytest.mark.parametrize("n, K", [(96, 320), (544, 512), (288, 2048)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_experts_of_many_passes(fmt, n, K):
    """More rows to an expert than a wide pass takes, on average too: several passes read an expert's weights. Bit for bit what
    the pairs give one by one."""
    counts = [700, 0, 1301]
    case = Case(fmt, 3, n, K, sum(counts))
    ids, order, _, groups = _pairs(3, counts)
    for how in ({}, {"dtype": torch.bfloat16}, {"swiglu": True}):
        got = case.grouped(groups, order=order, **how)
        assert torch.equal(got, case.gemv(ids, **how)[order])
        case.check(got[::37], order[::37], ids[order[::37]], "swiglu" in how)


# per number of rows: streamed (20 rows an expert), and wide passes
SUMS = [[20, 19], [300, 77]]


@pytest.mark.parametrize("counts", SUMS)
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_bfloat16_result_is_the_float32_one_rounded(fmt, counts):
    """Sums are the same whatever becomes of them: a bfloat16 result is the float32 one to nearest, ties to even, bit for bit."""
    case = Case(fmt, 2, 96, 832, sum(counts), spread=2.0)
    ids, order, _, groups = _pairs(2, counts)
    assert torch.equal(case.gemv(ids, dtype=torch.bfloat16), case.gemv(ids).to(torch.bfloat16))
    assert torch.equal(case.grouped(groups, order=order, dtype=torch.bfloat16),
                       case.grouped(groups, order=order).to(torch.bfloat16))


def _cancelling(bits, E, n, K, R):
    """A Case whose every fourth block holds two products of the formats' largest elements that cancel, beside 30 that are a
    thousandth of them or less, as the other blocks' are."""
    case = Case(f"mx{bits}", E, n, K, R)
    rng = np.random.default_rng(41)
    big = np.arange(K) // 32 % 4 == 1
    x = rng.uniform(-1, 1, (R, K)) * (0.0625 if bits == 8 else 0.5)
    w = rng.uniform(-1, 1, (E * n, K)) * 6
    x[:, big & (np.arange(K) % 32 < 2)] = 448.0 if bits == 8 else 6.0
    w[:, big & (np.arange(K) % 32 == 0)], w[:, big & (np.arange(K) % 32 == 1)] = 6.0, -6.0
    w[:, ~big & (np.arange(K) % 32 == 0)] = 6.0  # (the weights' scales are 1)
    (xc, xs), (wc, ws) = omx.quantize(x, bits), omx.quantize(w, 4)
    case.x = mx.rows_from(dev(omx.pack(xc, bits)), dev(xs), bits)
    case.w = mx.bank(mx.rows_from(dev(omx.pack(wc, 4)), dev(ws), 4), E)
    case.xv, case.wv = dev(omx.values(xc, xs, bits)), dev(omx.values(wc, ws, 4)).view(E, n, K)
    return case


@pytest.mark.parametrize("how", [{}, {"dtype": torch.bfloat16}, {"swiglu": True}])
@pytest.mark.parametrize("counts", SUMS)
@pytest.mark.parametrize("bits", [4, 8])
def test_small_products_beside_large_ones_that_cancel(bits, counts, how):
    """A result is what the small products of its blocks add up to, within the bound of float32 sums (`want`'s for results that
    are kept) and the result's own rounding."""
    case = _cancelling(bits, 2, 96, 768, sum(counts))
    ids, order, _, groups = _pairs(2, counts)
    rows = torch.arange(sum(counts), device=DEV)
    for got, row in ((case.gemv(ids, **how), rows), (case.grouped(groups, order=order, **how), order)):
        for part in range(0, len(row), 32):
            at = row[part:part + 32]
            want, off = case.want(at, ids[at], "swiglu" in how, False)
            eps = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
            assert torch.all((got[part:part + 32].double() - want).abs() <= off + eps * (want.abs() + off) + 1e-37)


@pytest.mark.parametrize("down", [4, 10, 16])
@pytest.mark.parametrize("apart", [1, 2, 8])
@pytest.mark.parametrize("bits", [4, 8])
def test_small_blocks_beside_large_ones_that_cancel(bits, apart, down):
    """The same across blocks: a block of the formats' largest products and, `apart` blocks on (in the same step's products or
    another's), its negative; what is between them and behind is 2^-down as large in its scales."""
    E, n, K, R = 2, 32, 512, 80
    case = Case(f"mx{bits}", E, n, K, R)
    rng = np.random.default_rng(100 * apart + down)
    first = 2
    x = rng.uniform(-1, 1, (R, K)) * 2.0 ** -down
    w = rng.uniform(-1, 1, (E * n, K)) * 6
    large = 32 * first + np.arange(32)
    x[:, large] = rng.uniform(0.5, 1, (R, 32)) * (448 if bits == 8 else 6)
    x[:, large + 32 * apart] = -x[:, large]
    w[:, large + 32 * apart] = w[:, large]
    (xc, xs), (wc, ws) = omx.quantize(x, bits), omx.quantize(w, 4)
    case.x = mx.rows_from(dev(omx.pack(xc, bits)), dev(xs), bits)
    case.w = mx.bank(mx.rows_from(dev(omx.pack(wc, 4)), dev(ws), 4), E)
    case.xv, case.wv = dev(omx.values(xc, xs, bits)), dev(omx.values(wc, ws, 4)).view(E, n, K)
    ids = torch.arange(R, device=DEV) % E
    order, _, groups = kernels.expert_groups(ids.view(-1, 1), E)
    rows = torch.arange(R, device=DEV)
    for got, row in ((case.gemv(ids), rows), (case.grouped(groups, order=order), order)):
        want, off = case.want(row, ids[row], False, False)
        err = (got.double() - want).abs()
        assert torch.all(err <= off + 2.0 ** -24 * want.abs()), float((err / off).max())


@pytest.mark.parametrize("bits", [4, 8])
def test_products_at_every_scale_code(bits):
    """Rows of every scale code from 0 to 254 against weights of codes that bring the products back into float32's range,
    the smallest and the largest code among both."""
    E, n, K, R = 8, 32, 512, 255
    case = Case(f"mx{bits}", E, n, K, R)
    codes, _ = omx.quantize(case.xv.cpu().numpy(), bits)
    wcodes, _ = omx.quantize(case.wv.flatten(0, 1).cpu().numpy(), 4)
    xs = np.repeat(np.arange(255)[:, None], K // 32, axis=1).astype(np.uint8)
    level = np.array([0, 1, 60, 120, 134, 190, 253, 254])
    ws = np.repeat(level, n)[:, None].repeat(K // 32, axis=1).astype(np.uint8)
    case.x = mx.rows_from(dev(omx.pack(codes, bits)), dev(xs), bits)
    case.w = mx.bank(mx.rows_from(dev(omx.pack(wcodes, 4)), dev(ws), 4), E)
    case.xv, case.wv = dev(omx.values(codes, xs, bits)), dev(omx.values(wcodes, ws, 4)).view(E, n, K)
    # (row, expert) of products between 2^-100 and 2^90 a scale
    row, expert = (torch.from_numpy(a).to(DEV) for a in np.nonzero(np.abs(np.arange(255)[:, None] + level - 249) <= 95))
    ids = torch.full((R * E,), -1, dtype=torch.int64, device=DEV)
    ids[row * E + expert] = expert
    got = case.gemv(ids)[row * E + expert]
    case.check(got, row, expert)
    # the same pairs grouped, in wide passes
    order = row * E + expert
    order = order[torch.argsort(expert, stable=True)]
    counts = torch.bincount(expert, minlength=E)
    groups = torch.stack([torch.arange(E, device=DEV)] * 2 + [torch.zeros_like(counts), counts.cumsum(0) - counts, counts],
                         dim=1).to(torch.int32)
    grouped = case.grouped(groups, order=order, k=E)
    assert torch.equal(grouped, case.gemv(ids)[order])


@pytest.mark.parametrize("fmt", FORMATS)
def test_pairs_of_a_row(fmt):
    """How many pairs each row has follows from the ids' number: three rows with one expert each, then with three."""
    case = Case(fmt, 5, 96, 320, 3, spread=1.0)
    ids = dev(np.array([4, 0, 2, 2, 4, 1, 0, 3, 2], np.int64))
    row = torch.arange(3, device=DEV)
    one, three = case.gemv(ids[[0, 4, 8]]), case.gemv(ids)
    case.check(one, row, ids[[0, 4, 8]])
    assert torch.equal(one, three[[0, 4, 8]])


@pytest.mark.parametrize("n, K", [(288, 768), (96, 1280), (160, 2368)])
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_wide_passes_of_an_odd_number_of_stages(fmt, n, K):
    """Wide passes where an item ends inside a pair of stages, whose scale words lie together: the next item's start in the other
    buffer."""
    case = Case(fmt, len(MANY), n, K, sum(MANY), spread=1.0)
    ids, order, _, groups = _pairs(len(MANY), MANY)
    for how in ({}, {"dtype": torch.bfloat16}, {"swiglu": True}):
        got = case.grouped(groups, order=order, **how)
        case.check(got, order, ids[order], "swiglu" in how)
        assert torch.equal(got, case.gemv(ids, **how)[order])


@pytest.mark.parametrize("E, rows, n", [(10, 300, 800), (70, 33, 800), (300, 34, 96)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_more_items_of_an_odd_number_of_stages(fmt, E, rows, n):
    """The same where a workgroup walks several items."""
    K = 192 if fmt == "bf16" else 768
    counts = np.random.default_rng(E).integers(rows - 1, rows + 2, E)
    counts[3], counts[5] = 0, 7 * rows
    case = Case(fmt, E, n, K, int(counts.sum()))
    ids, order, _, groups = _pairs(E, counts)
    for how in ({}, {"swiglu": True}, {"dtype": torch.bfloat16}):
        got = case.grouped(groups, order=order, **how)
        assert torch.equal(got, case.gemv(ids, **how)[order])
        at = torch.arange(0, len(order), 499, device=DEV)
        case.check(got[at], order[at], ids[order[at]], "swiglu" in how)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_is_not_finite_stays_in_its_row_of_a_wide_pass(fmt):
    """A NaN row and an infinite (microscaled: NaN) weight beside the rows of a pass whose last tile is not full."""
    case = Case(fmt, 2, 64, 768, 150)
    pair = torch.arange(150, device=DEV)
    ids = pair % 2
    order, _, groups = kernels.expert_groups(ids.view(-1, 1), 2)
    before = case.grouped(groups, order=order)[torch.argsort(order)]
    if fmt == "bf16":
        case.x[6, 100] = float("nan")
        case.w[64 + 9, 3] = float("inf")
    else:
        case.x.scale[6, 3] = 255
        rows = mx.bank_rows(case.w)
        rows.scale[64 + 9, 0] = 255
        case.w = mx.bank(rows, 2)
    got = case.grouped(groups, order=order)[torch.argsort(order)]
    bad = (pair == 6)[:, None] | ((ids == 1)[:, None] & (torch.arange(64, device=DEV) == 9))
    assert not torch.isfinite(got[bad]).any()
    assert torch.equal(got[~bad], before[~bad])


@pytest.mark.parametrize("fmt", ["mx8", "bf16"])
def test_wide_passes_beyond_32_bit_offsets(fmt):
    """The last experts of a bank of more than 4 GiB, 40 rows each."""
    n, K = 2048, 2048
    E = 560 if fmt == "bf16" else 2100
    small = Case(fmt, 2, n, K, 80)
    groups = torch.tensor([[0, 0, 0, 0, 39], [1, 0, 0, 39, 41]], dtype=torch.int32, device=DEV)
    want = small.grouped(groups)
    at = torch.tensor([0, 38, 39, 79], device=DEV)
    small.check(want[at], at, (at >= 39).long())
    if fmt == "bf16":
        w = torch.zeros((E * n, K), dtype=torch.bfloat16, device=DEV)
        w[-2 * n:] = small.w
    else:
        w = mx.MxBank(torch.zeros((E * n, K // 2), dtype=torch.uint8, device=DEV),
                      torch.zeros((E * n, K // 32), dtype=torch.uint8, device=DEV), E, n, K)
        w.weight[-2 * n:], w.scale[-2 * n:] = small.w.weight, small.w.scale
    assert (w if fmt == "bf16" else w.weight).nbytes > 2 ** 32
    small.w, small.E = w, E
    assert torch.equal(small.grouped(groups + torch.tensor([E - 2, 0, 0, 0, 0], dtype=torch.int32, device=DEV)), want)


@pytest.mark.parametrize("fmt", ["mx8", "bf16"])
def test_rows_beyond_32_bit_offsets(fmt):
    """The last rows of more than 4 GiB of them, some with an expert of few pairs and some with one of many."""
    K, last = 2048, 64
    R = 2 ** 32 // (K * (2 if fmt == "bf16" else 1)) + last
    case = Case(fmt, 2, 64, K, last)
    for counts in ((3, 5), (64, 64)):
        pairs = torch.cat([torch.arange(c, device=DEV) for c in counts])
        groups = torch.tensor([[0, 0, 0, 0, counts[0]], [1, 0, 0, counts[0], counts[1]]], dtype=torch.int32, device=DEV)
        want = case.grouped(groups, order=pairs)
        case.check(want, pairs, torch.arange(2, device=DEV).repeat_interleave(torch.tensor(counts, device=DEV)))
        many = Case.__new__(Case)
        many.__dict__.update(case.__dict__, R=R)
        if fmt == "bf16":
            many.x = torch.zeros((R, K), dtype=torch.bfloat16, device=DEV)
            many.x[-last:] = case.x
            assert many.x.nbytes > 2 ** 32
        else:
            many.x = mx.MxRows(torch.zeros((R, K), dtype=torch.uint8, device=DEV),
                               torch.zeros((R, K // 32), dtype=torch.uint8, device=DEV), 8, K)
            many.x.codes[-last:], many.x.scale[-last:] = case.x.codes, case.x.scale
            assert many.x.codes.nbytes > 2 ** 32
        assert torch.equal(many.grouped(groups, order=R - last + pairs), want)
        del many


@pytest.mark.parametrize("fmt, n, P", [("mx4", 16, 2 ** 24 + 16), ("bf16", 128, 2 ** 23 + 5)])
def test_lines_of_more_than_2_32_threads(fmt, n, P):
    """A gemv of more pairs than one dimension of a launch has threads for: all of them come out, as the first ones do."""
    case = Case(fmt, 2, n, 64, 1)
    ids = torch.arange(P, device=DEV) % 2
    out = torch.full((P, n), float("nan"), dtype=torch.bfloat16, device=DEV)
    case.gemv(ids, dtype=torch.bfloat16, out=out)
    case.check(out[:2], torch.zeros(2, dtype=torch.int64, device=DEV), ids[:2])
    for part in (out[:P // 2 * 2].view(-1, 2 * n), out[P - 2:][ids[P - 2:]].view(-1, 2 * n)):
        assert torch.all(part == out[:2].view(-1))


def test_groups_of_more_than_2_32_threads():
    """The same of a grouped product: 2^24 and some passes of 32 rows."""
    P, E = 2 ** 29 + 100, 7
    case = Case("bf16", E, 16, 64, 1)
    counts = torch.full((E,), P // E, dtype=torch.int64, device=DEV)
    counts[-1] += P - int(counts.sum())
    first = counts.cumsum(0) - counts
    e = torch.arange(E, device=DEV)
    groups = torch.stack((e, e, e * 0, first, counts), dim=1).to(torch.int32)
    out = torch.full((P, 16), float("nan"), dtype=torch.bfloat16, device=DEV)
    case.grouped(groups, order=torch.zeros(P, dtype=torch.int64, device=DEV), dtype=torch.bfloat16, out=out)
    case.check(out[first], e * 0, e)
    for g in range(E):
        assert torch.all(out[first[g]:first[g] + counts[g]] == out[first[g]])
