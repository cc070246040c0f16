"""Microscaled rows and banks without a GPU: the oracle's formats, the banks' layout, and what the entry points refuse."""
import ctypes
import pathlib
import subprocess
import sys

import numpy as np
import pytest
import torch

from drama3 import _lib, kernels, loader, mx, offload
from oracle import mx as omx


def test_element_grids():
    """e4m3's codes are torch's; e2m1's grid is 0, 0.5 .. 6."""
    codes = torch.arange(127, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), omx.E4M3)
    assert omx.E2M1.tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]


@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_rounds_to_even_and_saturates(bits):
    g = omx.grid(bits)
    middle = (g[1:] + g[:-1]) / 2
    got = omx.element(middle, bits)
    assert np.all(got % 2 == 0) and np.all(np.abs(got - np.arange(len(g) - 1)) <= 1)
    assert np.array_equal(omx.element(np.nextafter(middle, 0), bits), np.arange(len(g) - 1))
    assert np.array_equal(omx.element(np.nextafter(middle, 1e9), bits), np.arange(1, len(g)))
    assert omx.element(np.array([g[-1] * 1.3, -g[-1] * 2]), bits).tolist() == [
        len(g) - 1, (len(g) - 1) | 1 << (bits - 1)]


@pytest.mark.parametrize("E, N, K", [(1, 16, 32), (3, 48, 96), (2, 32, 256), (2, 16, 800), (2, 64, 2048)])
def test_bank_layout(E, N, K):
    """A bank's tiles hold every code and scale where the layout says, and bank_rows undoes bank."""
    rng = np.random.default_rng(K)
    codes = rng.integers(0, 256, (E * N, K // 2)).astype(np.uint8)
    scale = rng.integers(0, 256, (E * N, K // 32)).astype(np.uint8)
    rows = mx.rows_from(torch.from_numpy(codes), torch.from_numpy(scale), 4)
    bank = mx.bank(rows, E)
    stages = -(-K // 256)
    assert (bank.experts, bank.rows, bank.cols) == (E, N, K)
    assert bank.weight.shape == (E * N, stages * 128) and bank.scale.shape == (E * N, 8 * (stages + stages % 2))
    w = bank.weight.view(-1, stages, 2, 4, 16, 16).numpy()
    s = bank.scale.view(E * N // 16, 4, 16, -1, 2).numpy()
    for r in (0, 5, 16 * (E * N // 16) - 1):
        for b in range(K // 32):
            st, q, half = b // 8, b % 8 // 2, b % 2
            assert np.array_equal(w[r // 16, st, half, q, r % 16], codes[r, 16 * b:16 * b + 16])
            assert s[r // 16, q, r % 16, st, half] == scale[r, b]
    back = mx.bank_rows(bank)
    assert torch.equal(back.codes, rows.codes) and torch.equal(back.scale, rows.scale)
    assert bank.expert_bytes() == N * stages * 128 + N * 8 * (stages + stages % 2)


def _rows(R=4, cols=256, bits=8):
    C = -(-cols // 256) * 256
    return mx.MxRows(torch.zeros((R, C * bits // 8), dtype=torch.uint8), torch.zeros((R, C // 32), dtype=torch.uint8),
                     bits, cols)


def _bank(E=2, N=32, K=256):
    return mx.bank(_rows(E * N, K, 4), E)


def _groups(*rows):
    return torch.tensor([[e, e, 0, first, n] for e, first, n in rows], dtype=torch.int32)


@pytest.mark.parametrize("call, error", [
    (lambda: mx.quantize(torch.zeros(2, 48)), ValueError),
    (lambda: mx.quantize(torch.zeros(2, 0)), ValueError),
    (lambda: mx.quantize(torch.zeros(2, 64), 6), ValueError),
    (lambda: mx.quantize(torch.zeros(64)), TypeError),
    (lambda: mx.quantize(torch.zeros(2, 64, dtype=torch.float16)), TypeError),
    (lambda: mx.quantize(torch.zeros(2, 64)), ValueError),                      # not on a GPU
    (lambda: mx.dequantize(_rows(), torch.float16), TypeError),
    (lambda: mx.dequantize(mx.MxRows(torch.zeros(2, 100, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.uint8), 8,
                                     256)), ValueError),
    (lambda: mx.rows_from(torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), 4), ValueError),
    (lambda: mx.bank(_rows(24, 256, 4), 2), ValueError),                        # 12 rows an expert
    (lambda: mx.bank(_rows(32, 256, 8), 2), ValueError),                        # e4m3 rows
    (lambda: mx.gemv(_rows(), torch.zeros(6, dtype=torch.int64), _bank()), ValueError),   # 6 pairs of 4 rows
    (lambda: mx.gemv(_rows(), torch.zeros(8, dtype=torch.int32), _bank()), ValueError),
    (lambda: mx.gemv(_rows(cols=512), torch.zeros(8, dtype=torch.int64), _bank()), ValueError),
    (lambda: mx.gemv(_rows(), torch.zeros(8, dtype=torch.int64), _bank(N=16), swiglu=True), ValueError),
    (lambda: mx.gemv(_rows(), torch.zeros(8, dtype=torch.int64), _bank(), dtype=torch.float16), TypeError),
    (lambda: mx.gemv(_rows(), torch.zeros(8, dtype=torch.int64), _bank(), out=torch.zeros(8, 31)), ValueError),
    (lambda: mx.gemv(_rows(), torch.zeros(8, dtype=torch.int64), mx.MxBank(torch.zeros(64, 128, dtype=torch.uint8),
                     torch.zeros(64, 8, dtype=torch.uint8), 2, 32, 256)), ValueError),    # scales not laid out
    (lambda: mx.grouped(_rows(), torch.zeros(2, 4, dtype=torch.int32), _bank()), ValueError),
    (lambda: mx.grouped(_rows(), _groups((0, 0, 4)).long(), _bank()), ValueError),
    (lambda: mx.grouped(_rows(), _groups((0, 0, 4)), _bank(), k=2), ValueError),
    (lambda: mx.grouped(_rows(), _groups((0, 0, 4)), _bank(), order=torch.zeros(4, dtype=torch.int32)), ValueError),
    (lambda: mx.grouped(_rows(), _groups((0, 0, 4)), _bank(), order=torch.zeros(4, dtype=torch.int64), k=0), ValueError),
    (lambda: mx.grouped(_rows(), _groups((0, 0, 4)), _bank()), ValueError),     # not on a GPU
    (lambda: kernels.gemv_bf16(torch.zeros(1, 64), torch.zeros(1, dtype=torch.int64),
                               torch.zeros(16, 64, dtype=torch.bfloat16), 16), TypeError),
    (lambda: kernels.gemv_bf16(torch.zeros(1, 96).bfloat16(), torch.zeros(1, dtype=torch.int64),
                               torch.zeros(16, 96, dtype=torch.bfloat16), 16), ValueError),
    (lambda: kernels.gemv_bf16(torch.zeros(1, 64).bfloat16(), torch.zeros(1, dtype=torch.int64),
                               torch.zeros(24, 64, dtype=torch.bfloat16), 16), ValueError),
    (lambda: kernels.gemv_bf16(torch.zeros(1, 64).bfloat16(), torch.zeros(1, dtype=torch.int64),
                               torch.zeros(24, 64, dtype=torch.bfloat16), 24), ValueError),
    (lambda: kernels.grouped_bf16(torch.zeros(1, 64).bfloat16(), _groups((0, 0, 1)),
                                  torch.zeros(16, 128, dtype=torch.bfloat16)[:, :64], 16), ValueError),
    (lambda: kernels.grouped_bf16(torch.zeros(1, 64).bfloat16(), _groups((0, 0, 1)),
                                  torch.zeros(16, 64, dtype=torch.bfloat16), 16), ValueError),  # not on a GPU
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_c_entries_refuse():
    """The C entries' own checks, which launch nothing: D3_EINVAL with a message."""
    lib, p = _lib.lib(), ctypes.c_void_p(4096)
    odd = ctypes.c_void_p(4104)
    calls = {
        "d3_mx_quantize": [(p, 2, 64, 1, 64, 4, p, p), (p, 0, 64, 1, 48, 4, p, p), (p, 0, 63, 1, 32, 4, p, p),
                           (p, 0, 64, 1, 64, 5, p, p), (odd, 0, 64, 1, 64, 4, p, p), (None, 0, 64, 1, 64, 4, p, p),
                           (p, 0, 2048, 1 << 30, 2048, 4, p, p), (p, 0, 64, -1, 64, 4, p, p)],
        "d3_mx_dequantize": [(p, p, 1, 64, 4, 7, p), (p, p, 1, 33, 4, 0, p), (p, p, 1, 64, 4, 0, odd)],
        "d3_mx_gemv": [(p, p, 3, 1, p, 1, p, p, 1, 16, 32, 0, 0, p), (p, p, 4, 1, p, 1, p, p, 1, 24, 32, 0, 0, p),
                       (p, p, 4, 1, p, 1, p, p, 1, 16, 32, 1, 0, p), (p, p, 4, 1, p, 1, p, p, 1, 16, 40, 0, 0, p),
                       (p, p, 4, 2, p, 3, p, p, 1, 16, 32, 0, 0, p), (p, None, 4, 1, p, 1, p, p, 1, 16, 32, 0, 0, p),
                       (odd, p, 4, 1, p, 1, p, p, 1, 16, 32, 0, 0, p), (p, p, 4, 0, p, 1, p, p, 1, 16, 32, 0, 0, p)],
        "d3_mx_grouped": [(p, p, 4, 1, None, 1, 2, p, 1, p, p, 1, 16, 32, 0, 0, p),
                          (p, p, 4, 1, p, 0, 2, p, 1, p, p, 1, 16, 32, 0, 0, p),
                          (p, p, 4, 1, p, 1, 2, None, 1, p, p, 1, 16, 32, 0, 0, p)],
        "d3_bf16_gemv": [(p, 1, p, 1, p, 1, 16, 32, 0, 0, p), (p, 1, p, 1, p, 1, 8, 64, 0, 0, p),
                         (p, 1, p, 1, None, 1, 16, 64, 0, 0, p)],
        "d3_bf16_grouped": [(p, 1, None, 1, 2, p, 1, p, 1, 16, 64, 0, 0, p), (p, 1, p, 1, 2, p, 0, p, 1, 16, 64, 0, 0, p),
                            (p, 1, p, 1, -1, p, 1, p, 1, 16, 64, 0, 0, p)],
    }
    for name, args in calls.items():
        for a in args:
            assert getattr(lib, name)(*a, None) == -1, (name, a)
            assert name.encode() in lib.d3_last_error()
    # nothing to do: no pointer is looked at
    assert lib.d3_mx_quantize(None, 0, 64, 0, 64, 4, None, None, None) == 0
    assert lib.d3_mx_grouped(None, None, 4, 0, None, 1, 0, None, 0, None, None, 0, 16, 32, 0, 0, None, None) == 0
    assert lib.d3_bf16_gemv(None, 0, None, 0, None, 0, 16, 64, 0, 0, None, None) == 0


def test_sizes_past_32_bits_are_refused():
    """The C entries take 32-bit sizes, which ctypes would cut to their low bits."""
    far = 2 ** 32
    with pytest.raises(ValueError):
        mx.quantize(torch.zeros(1, device="meta").expand(1, far + 32))
    with pytest.raises(ValueError):
        mx.gemv(mx.MxRows(torch.empty(1, far // 2 + 128, dtype=torch.uint8, device="meta"),
                          torch.empty(1, far // 32 + 8, dtype=torch.uint8, device="meta"), 4, far + 256),
                torch.zeros(1, dtype=torch.int64), _bank())
    with pytest.raises(ValueError):
        kernels.pair_ids(torch.empty(far + 1, dtype=torch.int64, device="meta"), 1, -1)
    order = torch.empty(4, dtype=torch.int64)
    assert kernels.check_groups(_groups((0, 0, 4)), order, 2, 2, -1) == 4
    for groups, order, k in ((_groups((0, 0, 4)), order, far + 1),
                             (_groups((0, 0, 4)), torch.empty(far + 1, dtype=torch.int64, device="meta"), 2),
                             (torch.empty(far + 1, 5, dtype=torch.int32, device="meta"), order, 2)):
        with pytest.raises(ValueError):
            kernels.check_groups(groups, order, k, 2, -1)
    lib, p = _lib.lib(), ctypes.c_void_p(4096)
    for cols in (2 ** 31 - 32, 2 ** 31 - 224):
        assert lib.d3_mx_quantize(p, 0, 64, 1, cols, 4, p, p, None) == -1
        assert lib.d3_mx_dequantize(p, p, 1, cols, 4, 0, p, None) == -1


def test_layer_refuses_routes_elsewhere():
    """Routes or weights that are not on the rows' device would be read through a pointer of another memory."""
    x, ids, weights = torch.zeros(2, 64), torch.zeros(2, 1, dtype=torch.int64), torch.ones(2, 1)

    class OnGpu(torch.Tensor):  # rows that say they are on a GPU
        def get_device(self):
            return 0

        @property
        def device(self):
            return torch.device("cuda:0")

    with pytest.raises(ValueError, match="topk_idx and topk_weight"):
        kernels.direct_layer(x.as_subclass(OnGpu), ids, weights, 2, None, None)


def test_modules_import_without_gpu_bindings():
    """A torch built without GPU support has no current stream or device to ask for: the package imports there, and the
    products refuse rows that are not on a GPU."""
    code = """
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from drama3 import formats, kernels, loader, moe, mx, offload
try:
    mx.quantize(torch.zeros(2, 64))
except ValueError as e:
    assert "GPU" in str(e)
else:
    raise AssertionError("not refused")
"""
    root = pathlib.Path(mx.__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("kind", ["bf16", "mx4", "int4"])
def test_store_refuses_kinds_it_does_not_take(kind):
    """A store's slot cache reads the four reference formats: the other kinds are refused by name, and nothing is added."""
    fields = {"weight": torch.zeros((64, 256), dtype=torch.uint8), "scale": torch.zeros((64, 16), dtype=torch.uint8)}
    store = offload.ExpertStore(0, False)
    with pytest.raises(ValueError, match=kind):
        store.add_fields(kind, fields, fields, 2)
    assert not store.banks


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_files_refuse_kinds_they_do_not_hold(kind, tmp_path):
    fields = {"weight": torch.zeros((64, 256), dtype=torch.uint8), "scale": torch.zeros((64, 16), dtype=torch.uint8)}
    with pytest.raises(ValueError, match=kind):
        loader.write_experts(tmp_path / "x.safetensors", kind, {0: ((fields, fields), (None, None))}, {"num_experts": 2})
    assert not list(tmp_path.iterdir())
