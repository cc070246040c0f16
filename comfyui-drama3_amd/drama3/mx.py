"""Microscaled 4-bit expert banks (OCP MX): the quantizer, the banks' layout and the products that read them.

A microscaled row holds elements of 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) or 8 (e4m3) with one
power-of-two scale (e8m0) per 32 columns. MI355X multiplies both operands as they are stored, scales included, so a bank
of e2m1 weights costs 17/32 byte a weight and no decoding. Sums are float32, also of results that are then rounded to bfloat16:

    gate_up, down = mx.quantize_bank(w_gate_up), mx.quantize_bank(w_down)   # [E, 2I, H], [E, H, I] float -> MxBank
    rows = mx.quantize(x, 8)                                                # [T, H] -> MxRows (e4m3; 4: e2m1)
    h = mx.gemv(rows, ids, gate_up, swiglu=True)                            # decode lines: ids [T * k] int64
    h = mx.grouped(rows, groups, gate_up, order=order, k=k, swiglu=True)    # a prompt (kernels.expert_groups)
    out = mx.moe_layer(x, topk_idx, topk_weight, gate_up, down)             # the routed layer, rows of any number

`rows_from` and `bank` take rows and weights that a checkpoint already holds in the format. The C entries are in
include/drama3_moe.h (d3_mx_*); nothing waits on the host, and outputs are the only allocations, so a call can be captured
in a graph. The reference has no counterpart.
"""
import dataclasses

import torch

from . import _lib, kernels

BLOCK, STAGE = 32, 256
MAX_COLS = 2 ** 31 - 2 * STAGE  # (whole stages of them in 32 bits)
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _stages(cols):
    return -(-cols // STAGE)


@dataclasses.dataclass
class MxRows:
    """Rows of `cols` columns: codes [R, C * bits / 8] and scale [R, C / 32], uint8, C = cols rounded up to a multiple
    of 256 (zeros there). e2m1 codes are two to a byte, column 2 j in the low half."""
    codes: torch.Tensor
    scale: torch.Tensor
    bits: int
    cols: int


@dataclasses.dataclass
class MxBank:
    """E experts of `rows` e2m1 weight rows over `cols` columns, in the tiles that the products read (`bank` lays them
    out): weight [E * rows, C / 2], scale [E * rows, 8 * stages], uint8, the stages of 256 columns rounded up to an
    even number."""
    weight: torch.Tensor
    scale: torch.Tensor
    experts: int
    rows: int
    cols: int

    def to(self, device):
        return dataclasses.replace(self, weight=self.weight.to(device), scale=self.scale.to(device))

    def expert_bytes(self):
        return (self.weight.numel() + self.scale.numel()) // self.experts


def _check_cols(cols):
    if cols < BLOCK or cols % BLOCK or cols > MAX_COLS:
        raise ValueError(f"microscaled rows have a positive multiple of {BLOCK} columns, up to {MAX_COLS}, not {cols}")


def _check_rows(r):
    """(codes, scale, R, device index) of MxRows, checked."""
    codes, scale, bits = r.codes, r.scale, r.bits
    if bits != 8 and bits != 4:
        raise ValueError(f"microscaled rows have 4 or 8 bits an element, not {bits}")
    if r.cols > MAX_COLS:
        raise ValueError(f"microscaled rows have up to {MAX_COLS} columns, not {r.cols}")
    if codes.dtype is not torch.uint8 or scale.dtype is not torch.uint8:
        raise TypeError("codes and scale must be uint8")
    R, C, index = codes.size(0), -(-r.cols // STAGE) * STAGE, codes.get_device()
    if codes.shape != (R, C * bits // 8) or scale.shape != (R, C // BLOCK):
        raise ValueError(f"codes [R, {C * bits // 8}] and scale [R, {C // BLOCK}] expected for {r.cols} columns")
    if not (codes.is_contiguous() and scale.is_contiguous()):
        raise ValueError("codes and scale must be contiguous")
    if scale.get_device() != index:
        raise ValueError("codes and scale must be on one device")
    return codes, scale, R, index


def quantize(x, bits=4):
    """Rows x [R, C] (float32 or bfloat16, any row stride) as MxRows: per 32 columns the scale is the power of two
    2^(floor(log2 max|v|) - m), m = 2 for 4 bits and 8 for 8, the elements v / scale to nearest, ties to even, saturated
    at +-6 or +-448. A block with an infinity or NaN reads as NaN."""
    if x.dim() != 2 or x.dtype not in _TYPES:
        raise TypeError("x [R, C] float32 or bfloat16 expected")
    R, cols = x.shape
    _check_cols(cols)
    if bits not in (4, 8):
        raise ValueError(f"4 or 8 bits an element, not {bits}")
    if x.stride(1) != 1 or x.stride(0) < cols or x.stride(0) * x.element_size() % 16 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    C = _stages(cols) * STAGE
    codes = x.new_empty((R, C * bits // 8), dtype=torch.uint8)
    scale = x.new_empty((R, C // BLOCK), dtype=torch.uint8)
    kernels.launch("d3_mx_quantize", x.get_device(), x.data_ptr(), _TYPES[x.dtype], x.stride(0), R, cols, bits,
                   codes.data_ptr(), scale.data_ptr())
    return MxRows(codes, scale, bits, cols)


def dequantize(rows, dtype=torch.float32):
    """The values of MxRows: [R, cols] float32 or bfloat16."""
    codes, scale, R, index = _check_rows(rows)
    _check_cols(rows.cols)
    if dtype not in _TYPES:
        raise TypeError("float32 or bfloat16 expected")
    out = codes.new_empty((R, rows.cols), dtype=dtype)
    kernels.launch("d3_mx_dequantize", index, codes.data_ptr(), scale.data_ptr(), R, rows.cols, rows.bits, _TYPES[dtype],
                   out.data_ptr())
    return out


def rows_from(codes, scale, bits):
    """MxRows of codes [R, cols * bits / 8] and scale codes [R, cols / 32] (uint8), as a checkpoint holds them."""
    R, cols = codes.shape[0], codes.shape[1] * 8 // bits
    _check_cols(cols)
    if codes.dtype != torch.uint8 or scale.dtype != torch.uint8 or scale.shape != (R, cols // BLOCK):
        raise ValueError("codes [R, cols * bits / 8] and scale [R, cols / 32], uint8, expected")
    more = -cols % STAGE
    pad = torch.nn.functional.pad
    return MxRows(pad(codes, (0, more * bits // 8)).contiguous(), pad(scale, (0, more // BLOCK)).contiguous(), bits, cols)


def bank(rows, experts):
    """MxRows of e2m1 weights (experts * N rows, N % 16 == 0) laid out for the products, once: tile t holds 16 rows, their
    codes by stage of 256 columns, half s of the block pairs, pair q, row; their scales by pair, row, stage and s, where
    block 2 q + s of a stage's eight is pair q's half s."""
    R = _check_rows(rows)[2]
    if rows.bits != 4 or experts < 1 or R % experts or (R // experts) % 16:
        raise ValueError("a bank holds experts of e2m1 rows, a multiple of 16 each")
    tiles, stages = R // 16, _stages(rows.cols)
    codes = rows.codes.view(tiles, 16, stages, 4, 2, 16).permute(0, 2, 4, 3, 1, 5).reshape(R, -1)
    scale = rows.scale.view(tiles, 16, stages, 4, 2).permute(0, 3, 1, 2, 4)
    scale = torch.nn.functional.pad(scale, (0, 0, 0, stages % 2)).reshape(R, -1)
    return MxBank(codes.contiguous(), scale.contiguous(), experts, R // experts, rows.cols)


def bank_rows(b):
    """The MxRows of a bank: `bank`'s inverse."""
    tiles, stages = b.weight.shape[0] // 16, _stages(b.cols)
    codes = b.weight.view(tiles, stages, 2, 4, 16, 16).permute(0, 4, 1, 3, 2, 5).reshape(16 * tiles, -1)
    scale = b.scale.view(tiles, 4, 16, -1, 2)[:, :, :, :stages].permute(0, 2, 3, 1, 4).reshape(16 * tiles, -1)
    return MxRows(codes.contiguous(), scale.contiguous(), 4, b.cols)


def quantize_bank(w):
    """Float weights [E, N, K] as an MxBank (N a multiple of 16, K of 32)."""
    E, n, k = w.shape
    return bank(quantize(w.reshape(E * n, k), 4), E)


def _check_bank(b, cols, index):
    """(weight, scale) of a bank that rows of `cols` columns on device `index` go through, checked."""
    weight, scale = b.weight, b.scale
    if cols != b.cols:
        raise ValueError(f"rows of {cols} columns for a bank of {b.cols}")
    if weight.dtype is not torch.uint8 or scale.dtype is not torch.uint8:
        raise TypeError("a bank's weight and scale must be uint8")
    stages, R = -(-cols // STAGE), b.experts * b.rows
    if weight.shape != (R, stages * STAGE // 2) or scale.shape != (R, 8 * (stages + stages % 2)):
        raise ValueError("the bank's tensors do not have its shape (mx.bank lays them out)")
    if not (weight.is_contiguous() and scale.is_contiguous()):
        raise ValueError("a bank's tensors must be contiguous")
    if weight.get_device() != index or scale.get_device() != index:
        raise ValueError("rows and bank must be on one device")
    return weight, scale


def gemv(rows, ids, bank, swiglu=False, dtype=torch.float32, out=None):
    """[P, N] of P pairs of rows and experts ids [P] (int64): pair p is row p // (P / R) of the R rows with expert
    ids[p] of `bank`; float32 or bfloat16. With `swiglu` (gate rows, then up rows) [P, N / 2] bfloat16 = SiLU(gate) * up.
    An id outside the bank gives zeros. For decode lines: every pair reads its expert by itself."""
    codes, scale, R, index = _check_rows(rows)
    weight, wscale = _check_bank(bank, rows.cols, index)
    ids, P = kernels.pair_ids(ids, R, index)
    out = kernels.product_out(codes, P, bank.rows, swiglu, dtype, out)
    kernels.launch("d3_mx_gemv", index, codes.data_ptr(), scale.data_ptr(), rows.bits, R, ids.data_ptr(), P,
                   weight.data_ptr(), wscale.data_ptr(), bank.experts, bank.rows, bank.cols, swiglu,
                   out.dtype is torch.bfloat16, out.data_ptr())
    return out


def grouped(rows, groups, bank, order=None, k=1, swiglu=False, dtype=torch.float32, out=None):
    """[P, N] of pairs grouped by expert: groups [g, 5] int32 (expert, ., ., first place, rows) and order [P] int64 as
    kernels.expert_groups makes them; place p multiplies row order[p] // k (its own row p without order; an order outside the
    rows reads the nearest one) with its group's expert. dtype and `swiglu` as for gemv. Places in no group are left as `out` had them (unset without it), as are groups
    whose expert or places lie outside the bank or the pairs. Groups must not share places."""
    codes, scale, R, index = _check_rows(rows)
    weight, wscale = _check_bank(bank, rows.cols, index)
    P = kernels.check_groups(groups, order, k, R, index)
    out = kernels.product_out(codes, P, bank.rows, swiglu, dtype, out)
    kernels.launch("d3_mx_grouped", index, codes.data_ptr(), scale.data_ptr(), rows.bits, R, _lib.ptr(order), k, P,
                   groups.data_ptr(), groups.size(0), weight.data_ptr(), wscale.data_ptr(), bank.experts, bank.rows,
                   bank.cols, swiglu, out.dtype is torch.bfloat16, out.data_ptr())
    return out


def moe_layer(x, topk_idx, topk_weight, gate_up, down, bits=8):
    """The routed layer on MxBanks (gate_up [E, 2I, H], down [E, H, I]): rows x [T, H] bfloat16 or float32, topk_idx [T, k],
    topk_weight [T, k] -> [T, H] in x's dtype. The rows, and the hidden rows SiLU(gate) * up in bfloat16, are quantized to
    `bits` (8: e4m3, 4: e2m1). A row's result does not depend on the other rows."""
    banks = (gate_up, down)
    if down.experts != gate_up.experts or down.rows != x.shape[-1] or gate_up.rows != 2 * down.cols:
        raise ValueError("gate_up [E, 2I, H] and down [E, H, I] expected")
    return kernels.direct_layer(
        x, topk_idx, topk_weight, gate_up.experts,
        lambda i, rows, ids: gemv(quantize(rows, bits), ids, banks[i], swiglu=i == 0),
        lambda i, rows, groups, order, k: grouped(quantize(rows, bits), groups, banks[i], order, k, swiglu=i == 0))
