"""What stands around a block's routed experts, on unquantized (bfloat16) weights.

    out = block.gated_ffn(n, gate_up, down)                          # a layer's shared expert, or a dense layer
    out = block.lora_linear(x, weight, a, b, alpha, ids)             # a projection beside every row's own adapter
    h, n = block.add_norm(y, residual, weight)                       # end of one block, start of the next

The reference has no kernels for these. Nothing waits on the host; outputs and workspaces are allocated per call, so calls on
different streams are independent and each can be captured in a graph. The C entries are in include/drama3_moe.h.

Gradients: gated_ffn (without adapters), add_norm and norm are differentiable (torch.autograd, first order). Under graph capture
their autograd backward is refused, since torch may then touch a stream outside the capture; a captured training step calls
gated_ffn_forward and gated_ffn_backward, add_norm_forward and add_norm_backward, which the autograd forms are made of.
"""
import ctypes

import torch

from . import _lib, kernels

MAX_NORM_COLS = 16384
_INT_MAX = 2 ** 31 - 1
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _no_capture(name):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: autograd's backward pass is not captured; call {name}_backward in the captured step")


# ---------------------------------------------------------------------------------------------------------- products
MAX_ROW_STRIDE = 2 ** 23  # of a product's rows, in elements


def _rows(x, what, cols=None, rows=None, index=None):
    """Rows [T, K] bfloat16 as the products read them: columns side by side, 16-byte aligned (else a copy that is so)."""
    if x.dim() != 2 or x.dtype is not torch.bfloat16:
        raise TypeError(f"{what} [T, K] bfloat16 expected")
    T, K = x.shape
    if cols is not None and K != cols or rows is not None and T != rows:
        raise ValueError(f"{what} [{'T' if rows is None else rows}, {'K' if cols is None else cols}] expected, not {[T, K]}")
    if K < 8 or K % 8 or K > MAX_ROW_STRIDE or T > _INT_MAX:
        raise ValueError(f"{what} has a positive multiple of 8 columns up to {MAX_ROW_STRIDE}, not {K}")
    if index is not None and x.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    if T == 1:
        return x if x.stride(1) == 1 and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)
    stride = x.stride(0)
    if x.stride(1) != 1 or stride < K or stride % 8 or stride > MAX_ROW_STRIDE or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _stride(x):
    return x.stride(0) if x.size(0) > 1 else x.size(1)


def _weight(w, what, n, k, index):
    """A weight [n, k] bfloat16, contiguous, 16-byte aligned (n None: any multiple of 8)."""
    if w.dim() != 2 or w.dtype is not torch.bfloat16:
        raise TypeError(f"{what} bfloat16, two-dimensional, expected")
    if w.size(1) != k or (n is not None and w.size(0) != n) or w.size(0) < 8 or w.size(0) % 8:
        raise ValueError(f"{what} [{'a multiple of 8' if n is None else n}, {k}] expected, not {list(w.shape)}")
    if w.numel() > _INT_MAX:
        raise ValueError(f"{what}: fewer than 2^31 elements expected")
    if w.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    return w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)


def _adapters(lora, ids, T, n, k, index):
    """(a, b, alpha, ids, rank, adapters) of rows' adapters, checked."""
    a, b, alpha = lora
    if a.dim() != 3 or b.dim() != 3 or a.dtype is not torch.bfloat16 or b.dtype is not torch.bfloat16:
        raise TypeError("adapters a [A, rank, K] and b [A, N, rank] bfloat16 expected")
    count, rank, _ = a.shape
    if a.shape != (count, rank, k) or b.shape != (count, n, rank) or rank < 8 or rank % 8:
        raise ValueError(f"adapters a [A, rank, {k}] and b [A, {n}, rank] expected, rank a multiple of 8, not {list(a.shape)} and "
                         f"{list(b.shape)}")
    if rank * max(n, k) > _INT_MAX or count > _INT_MAX:
        raise ValueError("an adapter of fewer than 2^31 elements expected")
    if alpha.dtype is not torch.float32 or alpha.shape != (count,):
        raise ValueError(f"alpha [{count}] float32 expected")
    if ids is None or ids.dtype is not torch.int64 or ids.shape != (T,):
        raise ValueError(f"ids [{T}] int64 expected: every row's adapter")
    if any(t.get_device() != index for t in (a, b, alpha, ids)):
        raise ValueError("adapters and ids on the rows' device expected")
    a, b = (t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format) for t in (a, b))
    return a, b, alpha.contiguous(), ids.contiguous(), rank, count


def _dense(x, w, index, swiglu=False, pre=None, lora=None, ids=None):
    """[T, N] bfloat16 of checked rows and weight (swiglu: [T, N / 2])."""
    (T, K), N = x.shape, w.size(0)
    out = x.new_empty((T, N // 2 if swiglu else N))
    d = _lib.DenseDesc(x=x.data_ptr(), w=w.data_ptr(), out=out.data_ptr(), pre=_lib.ptr(pre), x_stride=_stride(x), T=T, N=N, K=K,
                       swiglu=swiglu)
    if lora is not None:
        a, b, alpha, ids, d.rank, d.adapters = _adapters(lora, ids, T, N, K, index)
        inner = x.new_empty((T, d.rank))
        d.a, d.b, d.alpha, d.ids, d.inner = (t.data_ptr() for t in (a, b, alpha, ids, inner))
    kernels.launch("d3_dense", index, ctypes.byref(d))
    return out


def lora_linear(x, weight, a, b, alpha, ids):
    """x weight^T for rows x [T, K] of many requests and a weight [N, K] that they share, with every row's own low-rank adapter
    added: alpha[i] (x[t] a[i]^T) b[i]^T for i = ids[t], a [A, rank, K], b [A, N, rank] (all bfloat16), alpha [A] float32, ids [T]
    int64; a row whose id is outside 0 .. A - 1 (-1, say) has none. [T, N] bfloat16, rounded once; sums in float32, the inner
    product x a^T alpha rounded to bfloat16 between its two products. Widths and rank are multiples of 8 (pad adapters of smaller
    rank with zeros). For decode lines and for prompts packed into one pass."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, weight, a, b, alpha)):
        raise RuntimeError("lora_linear has no backward pass: call it under torch.no_grad()")
    index = x.get_device()
    x = _rows(x, "x")
    return _dense(x, _weight(weight, "weight", None, x.size(1), index), index, lora=(a, b, alpha), ids=ids)


def _ffn_operands(x, gate_up, down):
    index = x.get_device()
    x = _rows(x, "x")
    gate_up = _weight(gate_up, "gate_up", None, x.size(1), index)
    if gate_up.size(0) % 16:
        raise ValueError(f"gate and up rows are multiples of 8 each, not {gate_up.size(0)} in all")
    return x, gate_up, _weight(down, "down", None, gate_up.size(0) // 2, index), index


def gated_ffn_forward(x, gate_up, down):
    """gated_ffn's output and what gated_ffn_backward needs of it: (pre [T, 2 I] float32, hidden [T, I] bfloat16). The gate and up
    sums are kept unrounded: their rounding to bfloat16 would add as much error to the gradients as the gradients' own. Autograd does
    not see it."""
    with torch.no_grad():
        x, gate_up, down, index = _ffn_operands(x, gate_up, down)
        pre = x.new_empty((x.size(0), gate_up.size(0)), dtype=torch.float32)
        hidden = _dense(x, gate_up, index, swiglu=True, pre=pre)
        return _dense(hidden, down, index), (pre, hidden)


def gated_ffn_backward(dout, x, gate_up, down, saved, needs=(True, True, True)):
    """(dx, dgate_up, ddown) bfloat16 of gated_ffn for the gradient dout [T, O] bfloat16 of its output, with x, gate_up and down as
    they went in and `saved` as gated_ffn_forward returned it; None where `needs` says so. Sums in float32; the gradients of gate
    and up are rounded to bfloat16 as the operands of the products that follow. The same bits from call to call."""
    with torch.no_grad():
        x, gate_up, down, index = _ffn_operands(x, gate_up, down)
        (T, H), I, O = x.shape, down.size(1), down.size(0)
        pre, hidden = saved
        dout = _rows(dout, "dout", O, T, index)
        dout = dout if dout.is_contiguous() else dout.contiguous()
        if pre.shape != (T, 2 * I) or pre.dtype is not torch.float32 or hidden.shape != (T, I) or \
                hidden.dtype is not torch.bfloat16 or not (pre.is_contiguous() and hidden.is_contiguous()) or \
                pre.get_device() != index or hidden.get_device() != index:
            raise ValueError(f"saved (pre [{T}, {2 * I}] float32, hidden [{T}, {I}] bfloat16) of gated_ffn_forward expected")
        new = x.new_zeros if T == 0 else x.new_empty
        dx, dgate_up, ddown = (new(shape) if need else None for need, shape in zip(needs, ((T, H), (2 * I, H), (O, I))))
        rows = x.new_empty((T, 2 * I))
        d = _lib.GatedFfnBackwardDesc(
            dout=dout.data_ptr(), x=x.data_ptr(), gate_up=gate_up.data_ptr(), down=down.data_ptr(), pre=pre.data_ptr(),
            hidden=hidden.data_ptr(), dgate_up_rows=rows.data_ptr(), dx=_lib.ptr(dx), dgate_up=_lib.ptr(dgate_up),
            ddown=_lib.ptr(ddown), x_stride=_stride(x), T=T, H=H, I=I, O=O)
        kernels.launch("d3_gated_ffn_backward", index, ctypes.byref(d))
        return dx, dgate_up, ddown


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up, down):
        out, saved = gated_ffn_forward(x, gate_up, down)
        ctx.save_for_backward(x, gate_up, down, *saved)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _no_capture("gated_ffn")
        x, gate_up, down, *saved = ctx.saved_tensors
        return gated_ffn_backward(dout, x, gate_up, down, saved, ctx.needs_input_grad)


def gated_ffn(x, gate_up, down, *, gate_up_lora=None, down_lora=None, ids=None):
    """The gated feed-forward, SiLU(x gate^T) * (x up^T) down^T, of rows x [T, H]: a layer's shared expert, or a dense layer. gate_up
    [2 I, H] holds the gate rows, then the up rows, down [O, I] (all bfloat16): [T, O] bfloat16. Sums and the activation in float32,
    the hidden rows rounded to bfloat16 between the products; widths are multiples of 8. Rows of any number: a decode line, lines
    decoded together, a prompt, a training batch. Differentiable.
    gate_up_lora, down_lora = (a, b, alpha) with `ids` [T]: the rows' adapters beside either projection, as lora_linear's (then not
    differentiable)."""
    if gate_up_lora is None and down_lora is None:
        if ids is not None:
            raise ValueError("ids go with gate_up_lora or down_lora")
        if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad):
            return _GatedFfn.apply(x, gate_up, down)
    elif torch.is_grad_enabled() and any(
            t.requires_grad for t in (x, gate_up, down, *(gate_up_lora or ()), *(down_lora or ()))):
        raise RuntimeError("gated_ffn with adapters has no backward pass: call it under torch.no_grad()")
    x, gate_up, down, index = _ffn_operands(x, gate_up, down)
    hidden = _dense(x, gate_up, index, swiglu=True, lora=gate_up_lora, ids=ids)
    return _dense(hidden, down, index, lora=down_lora, ids=ids)


# ------------------------------------------------------------------------------------------------------------- norms
def _float_rows(t, what, shape=None):
    """Rows [T, H] float32 or bfloat16 with columns side by side (else a copy that has them so)."""
    if t.dim() != 2 or t.dtype not in _TYPES:
        raise TypeError(f"{what} [T, H] float32 or bfloat16 expected")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} {list(shape)} expected, not {list(t.shape)}")
    return t if t.stride(1) == 1 and t.stride(0) >= t.size(1) else t.contiguous()


def _norm_weight(w, what, H, index):
    if w is None:
        return None
    if w.dtype not in _TYPES or w.shape != (H,):
        raise ValueError(f"{what} [{H}] float32 or bfloat16 expected")
    if w.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    return w.contiguous()


def _norm_gate(gate, T, H, index):
    """(gate, kind): 1 a value per row ([T, 1]), 2 per channel ([H] or [1, H]), 3 per element."""
    if gate is None:
        return None, 0
    if gate.dtype not in _TYPES or gate.get_device() != index:
        raise ValueError("gate float32 or bfloat16 on the rows' device expected")
    if gate.dim() == 1 and gate.shape == (H,):
        return gate.contiguous(), 2
    if gate.dim() == 2:
        if gate.shape == (T, H):
            return (gate if gate.stride(1) == 1 and gate.stride(0) >= H else gate.contiguous()), 3
        if gate.shape == (T, 1):
            return gate.contiguous(), 1
        if gate.shape == (1, H):
            return gate.contiguous(), 2
    raise ValueError(f"gate [{T}, 1], [{H}], [1, {H}] or [{T}, {H}] expected, not {list(gate.shape)}")


def _norm_desc(y, residual, weight, post, gate, scale, eps, unit_offset, out_dtype=None):
    """(descriptor, tensors that it points to, device index) of a call's inputs, checked."""
    residual = _float_rows(residual, "residual")
    (T, H), index = residual.shape, residual.get_device()
    if not 1 <= H <= MAX_NORM_COLS or T > _INT_MAX:
        raise ValueError(f"rows of 1 to {MAX_NORM_COLS} columns, not {H}")
    if y is not None:
        y = _float_rows(y, "y", (T, H))
        if y.get_device() != index:
            raise ValueError("y on residual's device expected")
        out_dtype = y.dtype
    weight, post = _norm_weight(weight, "weight", H, index), _norm_weight(post, "post", H, index)
    gate, kind = _norm_gate(gate, T, H, index)
    d = _lib.AddNormDesc(
        y=_lib.ptr(y), residual=residual.data_ptr(), weight=_lib.ptr(weight), post=_lib.ptr(post), gate=_lib.ptr(gate),
        y_stride=0 if y is None else y.stride(0), residual_stride=residual.stride(0),
        gate_stride=0 if gate is None else gate.stride(0), y_type=_TYPES[out_dtype], stream_type=_TYPES[residual.dtype],
        weight_type=0 if weight is None else _TYPES[weight.dtype], post_type=0 if post is None else _TYPES[post.dtype],
        gate_type=0 if gate is None else _TYPES[gate.dtype], gate_kind=kind, T=T, H=H, scale=float(scale), eps=float(eps),
        unit_offset=bool(unit_offset))
    return d, (y, residual, weight, post, gate), index


def _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, stats):
    if y is None:
        raise TypeError("y [T, H] float32 or bfloat16 expected")
    d, (y, residual, weight, post, gate), index = _norm_desc(y, residual, weight, post, gate, scale, eps, unit_offset)
    T, H = d.T, d.H
    h = residual.new_empty((T, H))
    n = None if weight is None else y.new_empty((T, H))
    rstd = residual.new_empty((2, T), dtype=torch.float32) if stats else None
    d.h, d.n, d.rstd = h.data_ptr(), _lib.ptr(n), _lib.ptr(rstd)
    kernels.launch("d3_add_norm", index, ctypes.byref(d))
    return h, n, rstd


def add_norm_forward(y, residual, weight, *, post=None, gate=None, scale=1.0, eps=1e-6, unit_offset=False):
    """add_norm's (h, n) and rstd [2, T] float32, which add_norm_backward takes; autograd does not see it."""
    with torch.no_grad():
        return _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, True)


def add_norm_backward(dh, dn, y, h, rstd, weight, *, post=None, gate=None, scale=1.0, unit_offset=False,
                      needs=(True, True, True, True, True)):
    """(dy, dresidual, dweight, dpost, dgate) of add_norm for the gradients dh and dn of its outputs (either may be None: zero),
    with y, weight, post, gate, scale and unit_offset as they went in and h and rstd as add_norm_forward returned them. Each
    gradient has its input's type and shape; None where the input is absent or `needs` says so. Float32 inside, from h as it is
    stored; sums over the rows (dweight, dpost, a gate per channel) are the same bits from call to call."""
    with torch.no_grad():
        return _add_norm_backward(dh, dn, y, h, rstd, weight, post, gate, scale, unit_offset, needs,
                                  h.dtype if y is None else y.dtype)


def _add_norm_backward(dh, dn, y, h, rstd, weight, post, gate, scale, unit_offset, needs, out_dtype):
    gate_in = gate
    d, (y, h, weight, post, gate), index = _norm_desc(y, h, weight, post, gate, scale, 0.0, unit_offset, out_dtype)
    T, H = d.T, d.H
    if dh is None and dn is None:
        raise ValueError("dh or dn expected")
    if weight is None and dn is not None:
        raise ValueError("dn goes with weight")
    if rstd is None or rstd.dtype != torch.float32 or rstd.shape != (2, T) or not rstd.is_contiguous() or rstd.get_device() != index:
        raise ValueError(f"rstd [2, {T}] float32 of add_norm_forward expected")
    if dh is not None and (dh.dtype != h.dtype or dh.shape != (T, H) or dh.get_device() != index):
        raise ValueError("dh of h's type and shape, on its device, expected")
    if dn is not None and (dn.dtype != out_dtype or dn.shape != (T, H) or dn.get_device() != index):
        raise ValueError("dn of n's type and shape, on its device, expected")
    dh, dn = (None if t is None else t.contiguous() for t in (dh, dn))
    if not any(needs):
        return (None,) * 5
    new = lambda like, need, *shape: h.new_empty(shape, dtype=like.dtype) if like is not None and need else None  # noqa: E731
    dy, dresidual = new(y, needs[0], T, H), new(h, needs[1], T, H)
    dweight, dpost = new(weight, needs[2], H), new(post, needs[3], H)
    dgate = new(gate, needs[4], *gate_in.shape) if gate_in is not None else None
    floats = _lib.lib().d3_add_norm_partials(T, H)
    partials = h.new_empty(floats, dtype=torch.float32) if any(t is not None for t in (dweight, dpost, dgate)) else None
    d.dh, d.dn, d.h, d.rstd = _lib.ptr(dh), _lib.ptr(dn), h.data_ptr(), rstd.data_ptr()
    d.dy, d.dresidual, d.dweight, d.dpost, d.dgate = (_lib.ptr(t) for t in (dy, dresidual, dweight, dpost, dgate))
    d.partials, d.partials_floats = _lib.ptr(partials), floats
    kernels.launch("d3_add_norm_backward", index, ctypes.byref(d))
    return dy, dresidual, dweight, dpost, dgate


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, post, gate, scale, eps, unit_offset):
        h, n, rstd = _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, True)
        ctx.save_for_backward(y, h, rstd, weight, post, gate)
        ctx.options = scale, unit_offset
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        _no_capture("add_norm")
        if dh is None and dn is None:
            return (None,) * 8
        y, h, rstd, weight, post, gate = ctx.saved_tensors
        grads = _add_norm_backward(dh, dn, y, h, rstd, weight, post, gate, *ctx.options, ctx.needs_input_grad[:5], y.dtype)
        return grads + (None,) * 3


def add_norm(y, residual, weight, *, post=None, gate=None, scale=1.0, eps=1e-6, unit_offset=False):
    """The end of one block and the start of the next, in one pass: (h, n) with h = residual + scale * gate * v, in residual's
    type, and n = h / rms(h) * weight, in y's type; v is the block's output y, or y / rms(y) * post with `post` (a norm after the
    block as well). y and residual [T, H], float32 or bfloat16 each; weight and post [H]; gate a value per row [T, 1], per
    channel [H] or per element [T, H]. rms(z) = sqrt(mean(z^2) + eps); with unit_offset weight and post are read as 1 + w.
    weight None: n is None. Float32 inside, h and n each rounded once (n comes from h before its rounding). Differentiable."""
    wants = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, residual, weight, post, gate))
    if wants:
        return _AddNorm.apply(y, residual, weight, post, gate, scale, eps, unit_offset)
    return _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, False)[:2]


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, unit_offset, dtype):
        n, rstd = _norm(x, weight, eps, unit_offset, dtype, True)
        ctx.save_for_backward(x, rstd, weight)
        ctx.options = unit_offset, dtype
        return n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dn):
        _no_capture("add_norm")
        x, rstd, weight = ctx.saved_tensors
        needs = ctx.needs_input_grad
        unit_offset, dtype = ctx.options
        _, dx, dweight, _, _ = _add_norm_backward(None, dn, None, x, rstd, weight, None, None, 1.0, unit_offset,
                                                  (False, needs[0], needs[1], False, False), dtype)
        return dx, dweight, None, None, None


def _norm(x, weight, eps, unit_offset, dtype, stats):
    if weight is None:
        raise ValueError("weight [H] expected")
    d, (_, x, weight, _, _), index = _norm_desc(None, x, weight, None, None, 1.0, eps, unit_offset, dtype)
    n = x.new_empty((d.T, d.H), dtype=dtype)
    rstd = x.new_empty((2, d.T), dtype=torch.float32) if stats else None
    d.n, d.rstd = n.data_ptr(), _lib.ptr(rstd)
    kernels.launch("d3_add_norm", index, ctypes.byref(d))
    return n, rstd


def norm(x, weight, *, eps=1e-6, unit_offset=False, dtype=None):
    """x / rms(x) * weight of rows x [T, H] (float32 or bfloat16), in `dtype` (x's without it): the norm before a model's first
    block; add_norm makes the others. Differentiable."""
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _TYPES or x.dtype not in _TYPES:
        raise TypeError("float32 or bfloat16 expected")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)):
        return _Norm.apply(x, weight, eps, unit_offset, dtype)
    return _norm(x, weight, eps, unit_offset, dtype, False)[0]
