"""Argument checks of drama3.block that run before any launch (no GPU needed), and of its C entries and descriptors."""
import pathlib
import struct
import subprocess

import pytest
import torch

from drama3 import _lib, block

BF, F32 = torch.bfloat16, torch.float32
HEADER = pathlib.Path(__file__).resolve().parents[1] / "include" / "drama3_moe.h"


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("error, match, call", [
    (TypeError, "x .T, K. bfloat16", lambda: block.gated_ffn(z(2, 16, dtype=F32), z(32, 16), z(16, 16))),
    (TypeError, "x .T, K. bfloat16", lambda: block.gated_ffn(z(2, 2, 16), z(32, 16), z(16, 16))),
    (ValueError, "multiple of 8 columns", lambda: block.gated_ffn(z(2, 20), z(32, 20), z(16, 16))),
    (ValueError, "gate_up", lambda: block.gated_ffn(z(2, 16), z(32, 24), z(16, 16))),
    (TypeError, "gate_up bfloat16", lambda: block.gated_ffn(z(2, 16), z(32, 16, dtype=F32), z(16, 16))),
    (ValueError, "multiples of 8 each", lambda: block.gated_ffn(z(2, 16), z(24, 16), z(16, 8))),
    (ValueError, "down", lambda: block.gated_ffn(z(2, 16), z(32, 16), z(16, 32))),
    (ValueError, "down", lambda: block.gated_ffn(z(2, 16), z(32, 16), z(12, 16))),
    (ValueError, "ids go with", lambda: block.gated_ffn(z(2, 16), z(32, 16), z(16, 16), ids=torch.zeros(2, dtype=torch.int64))),
    (ValueError, "on a GPU", lambda: block.gated_ffn(z(2, 16), z(32, 16), z(16, 16))),
    (ValueError, "dout", lambda: block.gated_ffn_backward(z(2, 24), z(2, 16), z(32, 16), z(16, 16), (z(2, 32, dtype=F32), z(2, 16)))),
    (ValueError, "dout", lambda: block.gated_ffn_backward(z(3, 16), z(2, 16), z(32, 16), z(16, 16), (z(2, 32, dtype=F32), z(2, 16)))),
    (ValueError, "saved", lambda: block.gated_ffn_backward(z(2, 16), z(2, 16), z(32, 16), z(16, 16), (z(2, 32), z(2, 16)))),
    (ValueError, "saved", lambda: block.gated_ffn_backward(z(2, 16), z(2, 16), z(32, 16), z(16, 16), (z(1, 32, dtype=F32), z(2, 16)))),
])
def test_gated_ffn_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def lora(T=2, K=16, N=24, rank=8, count=3, **changed):
    args = {"x": z(T, K), "weight": z(N, K), "a": z(count, rank, K), "b": z(count, N, rank), "alpha": z(count, dtype=F32),
            "ids": torch.zeros(T, dtype=torch.int64)}
    return block.lora_linear(**{**args, **changed})


@pytest.mark.parametrize("error, match, changed", [
    (ValueError, "rank a multiple of 8", {"a": z(3, 12, 16), "b": z(3, 24, 12)}),
    (ValueError, "adapters a", {"a": z(3, 8, 24)}),
    (ValueError, "adapters a", {"b": z(2, 24, 8)}),
    (TypeError, "adapters a", {"a": z(3, 8, 16, dtype=F32)}),
    (ValueError, "alpha", {"alpha": z(3)}),
    (ValueError, "alpha", {"alpha": z(4, dtype=F32)}),
    (ValueError, "ids", {"ids": torch.zeros(2, dtype=torch.int32)}),
    (ValueError, "ids", {"ids": torch.zeros(3, dtype=torch.int64)}),
    (ValueError, "ids", {"ids": None}),
    (ValueError, "weight", {"weight": z(24, 24)}),
    (RuntimeError, "no backward", {"a": z(3, 8, 16).requires_grad_()}),
    (ValueError, "on a GPU", {}),
])
def test_lora_linear_refusals(error, match, changed):
    with pytest.raises(error, match=match):
        lora(**changed)


def test_gated_ffn_with_adapters_has_no_backward():
    with pytest.raises(RuntimeError, match="no backward"):
        block.gated_ffn(z(2, 16).requires_grad_(), z(32, 16), z(16, 16), ids=torch.zeros(2, dtype=torch.int64),
                        down_lora=(z(1, 8, 16), z(1, 16, 8), z(1, dtype=F32)))


def norm(**changed):
    args = {"y": z(3, 10), "residual": z(3, 10, dtype=F32), "weight": z(10, dtype=F32)}
    return block.add_norm(**{**args, **changed})


@pytest.mark.parametrize("error, match, changed", [
    (TypeError, "y .T, H.", {"y": None}),
    (TypeError, "y .T, H.", {"y": z(3, 10, dtype=torch.float16)}),
    (ValueError, "y .3, 10.", {"y": z(3, 12)}),
    (TypeError, "residual", {"residual": z(3, 10, dtype=torch.float64)}),
    (TypeError, "residual", {"residual": z(30)}),
    (ValueError, "weight", {"weight": z(12)}),
    (ValueError, "weight", {"weight": z(1, 10)}),
    (ValueError, "post", {"post": z(10, dtype=torch.float16)}),
    (ValueError, "gate", {"gate": z(3)}),
    (ValueError, "gate", {"gate": z(2, 1)}),
    (ValueError, "gate", {"gate": z(3, 10, dtype=torch.float16)}),
    (ValueError, "1 to 16384 columns", {"y": z(1, 16385), "residual": z(1, 16385), "weight": z(16385)}),
    (ValueError, "on a GPU", {}),
])
def test_add_norm_refusals(error, match, changed):
    with pytest.raises(error, match=match):
        norm(**changed)


@pytest.mark.parametrize("match, changed", [
    ("dh or dn", {"dh": None, "dn": None}),
    ("dh of", {"dh": z(3, 10)}),
    ("dn of", {"dn": z(3, 10, dtype=F32)}),
    ("dn goes with weight", {"weight": None}),
    ("rstd", {"saved": (z(3, dtype=F32), None)}),
    ("rstd", {"saved": (None, None)}),
    ("saved", {"h": z(3, 10), "dh": z(3, 10), "saved": (z(2, 3, dtype=F32), z(3, 12))}),
    ("saved", {"h": z(3, 10), "dh": z(3, 10), "saved": (z(2, 3, dtype=F32), z(3, 10, dtype=F32))}),
])
def test_add_norm_backward_refusals(match, changed):
    args = {"dh": z(3, 10, dtype=F32), "dn": z(3, 10), "y": z(3, 10), "h": z(3, 10, dtype=F32), "saved": (z(2, 3, dtype=F32), None),
            "weight": z(10)}
    with pytest.raises(ValueError, match=match):
        block.add_norm_backward(**{**args, **changed})


def test_norm_refusals():
    with pytest.raises(TypeError):
        block.norm(z(2, 8), z(8), dtype=torch.float16)
    with pytest.raises(ValueError, match="weight"):
        block.norm(z(2, 8), None)


@pytest.mark.parametrize("error, match, call", [
    (RuntimeError, "no backward", lambda: block.linear(z(2, 16).requires_grad_(), z(8, 16))),
    (ValueError, "rows", lambda: block.linear(z(1, 16).expand(2 ** 30 + 1, 16), z(8, 16))),
    (ValueError, "weight", lambda: block.linear(z(2, 16), z(12, 16))),
    (TypeError, "shared_gate", lambda: block.gate_weight(z(16, dtype=F32))),
    (ValueError, "go with shared", lambda: block.sparse_block(z(2, 16), z(2, 16), z(8, 16), z(8, 16), z(8, 16), 2, shared_gate=z(8, 16))),
    (ValueError, "gate_weight", lambda: block.sparse_block(z(2, 16), z(2, 16), z(8, 16), z(8, 16), z(8, 16), 2, shared=(z(16, 16), z(16, 8)),
                                                          shared_gate=z(16))),
    (RuntimeError, "no backward", lambda: block.sparse_block(z(2, 16), z(2, 16).requires_grad_(), z(8, 16), z(8, 16), z(8, 16), 2)),
])
def test_sparse_block_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


@pytest.mark.parametrize("form, name", [(block._GatedFfn, "gated_ffn"), (block._AddNorm, "add_norm"), (block._Norm, "add_norm")])
def test_autograd_backward_is_refused_under_capture(form, name, monkeypatch):
    """The autograd forms' backward passes, of which this is the first check."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    grads = (z(2, 8),) * (2 if form is block._AddNorm else 1)
    with pytest.raises(RuntimeError, match=f"{name}_backward"):
        form.backward(None, *grads)


def call(entry, layout, **fields):
    """The entry's return code for a descriptor of these fields, zeros elsewhere."""
    left = dict(fields)
    data = layout.pack(*(left.pop(name, None) or (0.0 if code == "f" else 0) for name, code in layout.fields))
    assert not left, left
    return getattr(_lib.lib(), entry)(data, None)


P = 1 << 20  # an address that passes the checks of alignment; nothing is launched on it


@pytest.mark.parametrize("match, changed", [
    (b"multiples of 8", {"K": 12}),
    (b"multiples of 8", {"N": 20}),
    (b"multiples of 8 each", {"N": 24, "swiglu": 1}),
    (b"2^30 rows", {"T": -1}),
    (b"2^30 rows", {"T": 2 ** 30 + 1}),
    (b"2\\^31", {"N": 1 << 20, "K": 1 << 12}),
    (b"null pointer", {"x": None}),
    (b"null pointer", {"w": P + 8}),
    (b"null pointer", {"x_stride": 12}),
    (b"null pointer", {"x_stride": 8}),
    (b"rank", {"adapters": 1, "rank": 12}),
    (b"null pointer", {"adapters": 1, "rank": 8}),
    (b"aligned", {"adapters": 1, "rank": 8, "a": P + 2, "b": P, "alpha": P, "ids": P, "inner": P}),
])
def test_dense_entry_refuses(match, changed):
    assert call("d3_dense", _lib.DENSE, **{**dict(x=P, w=P, out=P, x_stride=16, T=2, N=16, K=16), **changed}) == -1
    assert match.replace(b"\\", b"") in _lib.lib().d3_last_error()


def test_entries_refuse_null_descriptors():
    for name in ("d3_dense", "d3_gated_ffn_backward", "d3_add_norm", "d3_add_norm_backward"):
        assert getattr(_lib.lib(), name)(None, None) == -1, name


@pytest.mark.parametrize("changed", [{"H": 12}, {"I": 4}, {"O": 0}, {"T": -1}, {"dout": None}, {"pre": P + 4}, {"dx": P, "gate_up": None},
                                     {"dgate_up": P, "x": None}, {"ddown": P, "hidden": None}, {"I": 1 << 20, "H": 1 << 12}])
def test_ffn_backward_entry_refuses(changed):
    args = dict(dout=P, x=P, gate_up=P, down=P, pre=P, hidden=P, dgate_up_rows=P, x_stride=16, T=2, H=16, I=16, O=16)
    assert call("d3_gated_ffn_backward", _lib.GATED_FFN_BACKWARD, **{**args, **changed}) == -1


@pytest.mark.parametrize("changed", [{"H": 0}, {"H": 16385}, {"T": -1}, {"y_type": 2}, {"gate_kind": 4}, {"gate_kind": 1},
                                     {"residual": None}, {"h": None}, {"n": None}, {"y": None, "post": P}, {"y": None, "weight": None}])
def test_add_norm_entry_refuses(changed):
    args = dict(y=P, residual=P, weight=P, h=P, n=P, T=2, H=16, y_stride=16, residual_stride=16, scale=1.0, eps=1e-6)
    assert call("d3_add_norm", _lib.ADD_NORM, **{**args, **changed}) == -1


@pytest.mark.parametrize("changed", [{"dh": None, "dn": None}, {"weight": None}, {"rstd": None}, {"h": None}, {"partials_floats": 31},
                                     {"partials": None}, {"dpost": P}, {"dgate": P}, {"y": None},
                                     {"stream_type": 1}])
def test_add_norm_backward_entry_refuses(changed):
    args = dict(y=P, h=P, weight=P, dh=P, dn=P, rstd=P, dy=P, dresidual=P, dweight=P, partials=P, partials_floats=32, T=2, H=16,
                y_stride=16, residual_stride=16, scale=1.0)
    assert call("d3_add_norm_backward", _lib.ADD_NORM, **{**args, **changed}) == -1


@pytest.mark.parametrize("layout, cname", [(_lib.ADD_NORM, "d3_add_norm_desc"), (_lib.DENSE, "d3_dense_desc"),
                                           (_lib.GATED_FFN_BACKWARD, "d3_gated_ffn_backward_desc")])
def test_descriptor_layout_matches_header(layout, cname, tmp_path):
    """Every field sits at the offset and has the size that the C compiler gives it in the header."""
    prog = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {", f"  {cname} d;",
             '  printf("size %zu 0\\n", sizeof(d));']
    lines += [f'  printf("{f} %zu %zu\\n", offsetof({cname}, {f}), sizeof(d.{f}));' for f, _ in layout.fields]
    prog.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(prog)], check=True, capture_output=True)
    got = {n: (int(a), int(b)) for n, a, b in (line.split() for line in subprocess.run(
        [str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())}
    size = got.pop("size")[0]
    assert 0 <= size - layout.struct.size < 8  # (the end of the struct is padded to its alignment)
    codes = "".join(code for _, code in layout.fields)
    for i, (name, code) in enumerate(layout.fields):
        assert got[name] == (struct.calcsize(codes[:i + 1]) - struct.calcsize(code), struct.calcsize(code)), name
    assert len(got) == len(layout.fields)


@pytest.mark.parametrize("layout, cname", [(_lib.ADD_NORM, "d3_add_norm_desc"), (_lib.DENSE, "d3_dense_desc"),
                                           (_lib.GATED_FFN_BACKWARD, "d3_gated_ffn_backward_desc")])
def test_descriptors_are_whole(layout, cname, tmp_path):
    """A packed descriptor has as many bytes as the header's struct, of which the C entries read every one."""
    prog = tmp_path / "size.c"
    prog.write_text(f'#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{ printf("%zu\\n", sizeof({cname})); return 0; }}\n')
    exe = tmp_path / "size"
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(prog)], check=True, capture_output=True)
    size = int(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout)
    assert layout.struct.size == size == len(layout.pack(*(0.0 if code == "f" else 0 for _, code in layout.fields)))


@pytest.mark.parametrize("stream", [BF, F32])
def test_add_norm_backward_refuses_a_changed_residual(stream, monkeypatch):
    """A bfloat16 stream's gradients read the residual again: one written to between the explicit pair's calls is refused."""
    launched = []
    monkeypatch.setattr(block.kernels, "launch", lambda name, *args: launched.append(name))
    residual, y, weight = z(3, 16, dtype=stream), z(3, 16), z(16)
    h, n, saved = block.add_norm_forward(y, residual, weight)
    assert len(saved) == 2 and saved[1] is residual
    block.add_norm_backward(h, n, y, h, saved, weight)
    residual.add_(1)
    if stream is F32:
        block.add_norm_backward(h, n, y, h, saved, weight)
    else:
        with pytest.raises(RuntimeError, match="residual was changed"):
            block.add_norm_backward(h, n, y, h, saved, weight)
    with torch.inference_mode():  # (keeps no versions)
        residual = z(3, 16, dtype=stream)
        h, n, saved = block.add_norm_forward(y, residual, weight)
        block.add_norm_backward(h, n, y, h, saved, weight)
    assert launched.count("d3_add_norm") == 2


DUAL_CALLS = {
    "linear": (lambda *t: block.linear(*t), [(2, 16), (8, 16)]),
    "lora_linear": (lambda *t: block.lora_linear(*t, torch.zeros(2, dtype=torch.int64)),
                    [(2, 16), (24, 16), (3, 8, 16), (3, 24, 8), (3,)]),
    "gated_ffn": (lambda *t: block.gated_ffn(*t), [(2, 16), (32, 16), (16, 16)]),
    "gated_ffn with adapters": (lambda x, g, d, *t: block.gated_ffn(x, g, d, down_lora=t, ids=torch.zeros(2, dtype=torch.int64)),
                                [(2, 16), (32, 16), (16, 16), (1, 8, 16), (1, 16, 8), (1,)]),
    "add_norm": (lambda y, r, w, p, g: block.add_norm(y, r, w, post=p, gate=g), [(2, 16), (2, 16), (16,), (16,), (2, 1)]),
    "norm": (lambda *t: block.norm(*t), [(2, 16), (16,)]),
    "sparse_block": (lambda n, h, r, gu, d, sgu, sd, sg, w, a, b, al: block.sparse_block(
        n, h, r, gu, d, 2, shared=(sgu, sd), shared_gate=sg, next_weight=w, shared_lora=(None, (a, b, al)),
        ids=torch.zeros(2, dtype=torch.int64)),
        [(2, 16), (2, 16), (8, 16), (256, 16), (128, 16), (32, 16), (16, 16), (8, 16), (16,), (1, 8, 16), (1, 16, 8), (1,)]),
}


@pytest.mark.parametrize("name, which", [(name, i) for name, (_, shapes) in DUAL_CALLS.items() for i in range(len(shapes))])
def test_forward_mode_is_refused(name, which, monkeypatch):
    """A tangent is never dropped: a dual tensor (whose requires_grad is False) in any place is refused before any launch."""
    monkeypatch.setattr(block.kernels, "launch", lambda *args: pytest.fail("launched"))
    call, shapes = DUAL_CALLS[name]
    tensors = [z(*s, dtype=F32 if s in ((1,), (3,)) else BF) for s in shapes]
    with torch.autograd.forward_ad.dual_level():
        tensors[which] = torch.autograd.forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        assert not tensors[which].requires_grad
        with pytest.raises(RuntimeError, match=f"{name.split()[0]} has no forward-mode"):
            call(*tensors)


def test_norm_backward_under_capture_names_its_own_pair(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="^norm: .*norm_forward and norm_backward"):
        block._Norm.backward(None, z(2, 8))


@pytest.mark.parametrize("match, changed", [
    ("dn", {"dn": None}),
    ("dn", {"dn": z(3, 10, dtype=torch.float16)}),
    ("dn of", {"dn": z(2, 10)}),
    ("weight", {"weight": None}),
    ("weight", {"weight": z(12)}),
    ("rstd", {"saved": None}),
    ("rstd", {"saved": z(1, 3, dtype=F32)}),
    ("on a GPU", {}),
])
def test_norm_backward_refusals(match, changed):
    with pytest.raises(ValueError, match=match):
        block.norm_backward(**{**{"dn": z(3, 10), "x": z(3, 10, dtype=F32), "saved": z(2, 3, dtype=F32), "weight": z(10)}, **changed})


def test_norm_forward_refusals():
    with pytest.raises(TypeError):
        block.norm_forward(z(2, 8), z(8), dtype=torch.float16)
    with pytest.raises(ValueError, match="weight"):
        block.norm_forward(z(2, 8), None)


@pytest.mark.parametrize("changed", [{"y_stride": 0}, {"y_stride": 15}, {"residual_stride": -16}, {"residual_stride": 8}, {"gate_kind": 3, "gate": P},
                                     {"gate_kind": 3, "gate": P, "gate_stride": -16}, {"gate_kind": 1, "gate": P}])
@pytest.mark.parametrize("entry", ["d3_add_norm", "d3_add_norm_backward"])
def test_add_norm_entries_refuse_strides(entry, changed):
    """A descriptor whose strides were left out, or run backwards, is refused and not read."""
    args = dict(y=P, residual=P, weight=P, dh=P, dn=P, h=P, n=P, rstd=P, dy=P, T=2, H=16, y_stride=16, residual_stride=16, scale=1.0, eps=1e-6)
    assert call(entry, _lib.ADD_NORM, **{**args, **changed}) == -1
    assert b"apart" in _lib.lib().d3_last_error()


def test_route_goes_to_its_logits_device(monkeypatch):
    """sparse_block's routing, as its products, runs with the rows' device as the current one, whichever that is."""
    seen = []

    class Device:
        def __init__(self, index):
            seen.append(index)

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *_):
            seen.append("out")

    class Lib:
        def d3_route(self, *args):
            seen.append(args[-1])
            return 0

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: ("stream of", index), raising=False)
    monkeypatch.setattr(block.kernels._lib, "lib", Lib)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 1)
    block.kernels.route(z(2, 16), 4)
    assert seen == [1, "in", ("stream of", 1), "out"]


def test_dense_entry_refuses_an_unaligned_pre():
    """Gate and up are stored 16 bytes at a time, as the backward entry reads them."""
    assert call("d3_dense", _lib.DENSE, x=P, w=P, out=P, pre=P + 4, x_stride=16, T=2, N=16, K=16, swiglu=1) == -1
    assert b"pre must be" in _lib.lib().d3_last_error()


def test_add_norm_backward_takes_a_residual_that_it_does_not_read_or_that_stayed(monkeypatch):
    """Neither a write to other rows of the buffer that residual is a part of, nor one to a residual that dh alone needs not, is refused."""
    monkeypatch.setattr(block.kernels, "launch", lambda *args: None)
    buffer, y, weight = z(2, 3, 16), z(3, 16), z(16)
    h, n, saved = block.add_norm_forward(y, buffer[0], weight)
    buffer[1].add_(1)
    block.add_norm_backward(h, n, y, h, saved, weight)
    residual = z(3, 16)
    h, n, saved = block.add_norm_forward(y, residual, weight)
    residual.add_(1)
    block.add_norm_backward(h, None, y, h, saved, weight)
