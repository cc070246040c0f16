"""What stands around a block's routed experts, on unquantized (bfloat16) weights.

    out = block.gated_ffn(n, gate_up, down)                          # a layer's shared expert, or a dense layer
    out = block.lora_linear(x, weight, a, b, alpha, ids)             # a projection beside every row's own adapter
    h, n = block.add_norm(y, residual, weight)                       # end of one block, start of the next
    h, n = block.sparse_block(n, h, router, gate_up, down, 8, shared=(s_gate_up, s_down), next_weight=weight)  # all of it

The reference has no kernels for these. Nothing waits on the host; outputs and workspaces are allocated per call, so calls on
different streams are independent and each can be captured in a graph. The C entries are in include/drama3_moe.h.

Gradients: gated_ffn (without adapters), add_norm and norm are differentiable (torch.autograd, reverse mode, first order); inputs
with a forward-mode tangent are refused, here and in what has no backward pass. Under graph capture
their autograd backward is refused, since torch may then touch a stream outside the capture; a captured training step calls
gated_ffn_forward and gated_ffn_backward, add_norm_forward and add_norm_backward, norm_forward and norm_backward, which the
autograd forms are made of.
"""
import torch
from torch.autograd import forward_ad

from . import _lib, kernels

MAX_NORM_COLS = 16384
_INT_MAX = 2 ** 31 - 1
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _no_capture(name):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name}: autograd's backward pass is not captured; call the explicit pairs in the captured step "
                           "(gated_ffn_forward and gated_ffn_backward, add_norm_forward and add_norm_backward, norm_forward and "
                           "norm_backward)")


def _any_grad(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _no_tangent(name, *tensors):
    """Refuses forward-mode AD's dual tensors, whose requires_grad is False: their tangents would be dropped, as if zero. (Outside a
    dual level there are none; asking each of five tensors would cost 4 us a call.)"""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


def _at(t):
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------- products
MAX_ROW_STRIDE = 2 ** 23  # of a product's rows, in elements
MAX_ROWS = 2 ** 30


def _rows(x, what, index, cols=None, rows=None):
    """Rows x [T, K] bfloat16, checked, and as the products read them, (x, T, K, row stride): columns side by side, 16-byte aligned
    (else a copy that is so)."""
    if x.dtype is not torch.bfloat16 or x.dim() != 2:
        raise TypeError(f"{what} [T, K] bfloat16 expected")
    T, K = x.shape
    if cols is not None and (K != cols or T != rows):
        raise ValueError(f"{what} [{rows}, {cols}] expected, not {[T, K]}")
    if K < 8 or K % 8 or K > MAX_ROW_STRIDE or T > MAX_ROWS:
        raise ValueError(f"{what} has up to {MAX_ROWS} rows of a positive multiple of 8 columns up to {MAX_ROW_STRIDE}, not {[T, K]}")
    if x.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    at = x.data_ptr()
    if x.is_contiguous():
        return (x if at % 16 == 0 else x.clone()), T, K, K
    stride = x.stride(0)
    if x.stride(1) != 1 or stride < K or stride % 8 or stride > MAX_ROW_STRIDE or at % 16:
        return x.clone(memory_format=torch.contiguous_format), T, K, K
    return x, T, K, stride


def _weight(w, what, n, k, index):
    """(w, its rows): a weight [n, k] bfloat16, checked, contiguous and 16-byte aligned (n None: any multiple of 8)."""
    if w.dtype is not torch.bfloat16 or w.dim() != 2:
        raise TypeError(f"{what} bfloat16, two-dimensional, expected")
    N, K = w.shape
    if K != k or N < 8 or N % 8 or (n is not None and N != n):
        raise ValueError(f"{what} [{'a multiple of 8' if n is None else n}, {k}] expected, not {[N, K]}")
    if N * K > _INT_MAX:
        raise ValueError(f"{what}: fewer than 2^31 elements expected")
    if w.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    return (w if w.is_contiguous() and w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)), N


def _adapters(lora, ids, T, n, k, index):
    """(a, b, alpha, ids, rank, adapters) of rows' adapters, checked."""
    a, b, alpha = lora
    if a.dtype is not torch.bfloat16 or b.dtype is not torch.bfloat16 or a.dim() != 3 or b.dim() != 3:
        raise TypeError("adapters a [A, rank, K] and b [A, N, rank] bfloat16 expected")
    count, rank, K = a.shape
    if K != k or b.shape != (count, n, rank) or rank < 8 or rank % 8:
        raise ValueError(f"adapters a [A, rank, {k}] and b [A, {n}, rank] expected, rank a multiple of 8, not {list(a.shape)} and "
                         f"{list(b.shape)}")
    if rank * max(n, k) > _INT_MAX or count > _INT_MAX:
        raise ValueError("an adapter of fewer than 2^31 elements expected")
    if alpha.dtype is not torch.float32 or alpha.shape != (count,):
        raise ValueError(f"alpha [{count}] float32 expected")
    if ids is None or ids.dtype is not torch.int64 or ids.shape != (T,):
        raise ValueError(f"ids [{T}] int64 expected: every row's adapter")
    if a.get_device() != index or b.get_device() != index or alpha.get_device() != index or ids.get_device() != index:
        raise ValueError("adapters and ids on the rows' device expected")
    if not a.is_contiguous() or a.data_ptr() % 16:
        a = a.clone(memory_format=torch.contiguous_format)
    if not b.is_contiguous() or b.data_ptr() % 16:
        b = b.clone(memory_format=torch.contiguous_format)
    return a, b, alpha.contiguous(), ids.contiguous(), rank, count


def _dense(x, T, K, stride, w, N, index, swiglu=False, pre=None, lora=None, ids=None):
    """[T, N] bfloat16 of checked rows and weight (swiglu: [T, N / 2])."""
    out = x.new_empty((T, N // 2 if swiglu else N))
    if lora is None:
        kernels.launch("d3_dense", index, _lib.DENSE.pack(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), 0 if pre is None else pre.data_ptr(), 0, 0, 0, 0, 0, stride, T, N, K, swiglu,
            0, 0))
    else:
        a, b, alpha, ids, rank, count = _adapters(lora, ids, T, N, K, index)
        inner = x.new_empty((T, rank))
        kernels.launch("d3_dense", index, _lib.DENSE.pack(
            x.data_ptr(), w.data_ptr(), out.data_ptr(), 0, a.data_ptr(), b.data_ptr(), alpha.data_ptr(), ids.data_ptr(),
            inner.data_ptr(), stride, T, N, K, swiglu, rank, count))
    return out


def linear(x, weight):
    """x weight^T of rows x [T, K] and a weight [N, K] (bfloat16): [T, N] bfloat16, float32 sums rounded once. A router's logits,
    say; widths are multiples of 8. No backward pass."""
    _no_tangent("linear", x, weight)
    if torch.is_grad_enabled() and _any_grad(x, weight):
        raise RuntimeError("linear has no backward pass: call it under torch.no_grad()")
    index = x.get_device()
    x, T, K, stride = _rows(x, "x", index)
    weight, N = _weight(weight, "weight", None, K, index)
    return _dense(x, T, K, stride, weight, N, index)


def lora_linear(x, weight, a, b, alpha, ids):
    """x weight^T for rows x [T, K] of many requests and a weight [N, K] that they share, with every row's own low-rank adapter
    added: alpha[i] (x[t] a[i]^T) b[i]^T for i = ids[t], a [A, rank, K], b [A, N, rank] (all bfloat16), alpha [A] float32, ids [T]
    int64; a row whose id is outside 0 .. A - 1 (-1, say) has none. [T, N] bfloat16, rounded once; sums in float32, the inner
    product x a^T alpha rounded to bfloat16 between its two products. Widths and rank are multiples of 8 (pad adapters of smaller
    rank with zeros). For decode lines and for prompts packed into one pass."""
    _no_tangent("lora_linear", x, weight, a, b, alpha)
    if torch.is_grad_enabled() and _any_grad(x, weight, a, b, alpha):
        raise RuntimeError("lora_linear has no backward pass: call it under torch.no_grad()")
    index = x.get_device()
    x, T, K, stride = _rows(x, "x", index)
    weight, N = _weight(weight, "weight", None, K, index)
    return _dense(x, T, K, stride, weight, N, index, lora=(a, b, alpha), ids=ids)


def _ffn_weights(gate_up, down, H, index):
    """(gate_up, down, I, O), checked."""
    gate_up, N = _weight(gate_up, "gate_up", None, H, index)
    if N % 16:
        raise ValueError(f"gate and up rows are multiples of 8 each, not {N} in all")
    return (gate_up, N // 2) + _weight(down, "down", None, N // 2, index)


def gated_ffn_forward(x, gate_up, down):
    """gated_ffn's output and what gated_ffn_backward needs of it: (pre [T, 2 I] float32, hidden [T, I] bfloat16). The gate and up
    sums are kept unrounded: their rounding to bfloat16 would add as much error to the gradients as the gradients' own. Autograd does
    not see it."""
    with torch.no_grad():
        index = x.get_device()
        x, T, H, stride = _rows(x, "x", index)
        gate_up, I, down, O = _ffn_weights(gate_up, down, H, index)
        pre = x.new_empty((T, 2 * I), dtype=torch.float32)
        hidden = _dense(x, T, H, stride, gate_up, 2 * I, index, True, pre)
        return _dense(hidden, T, I, I, down, O, index), (pre, hidden)


def gated_ffn_backward(dout, x, gate_up, down, saved, needs=(True, True, True)):
    """(dx, dgate_up, ddown) bfloat16 of gated_ffn for the gradient dout [T, O] bfloat16 of its output, with x, gate_up and down as
    they went in and `saved` as gated_ffn_forward returned it; None where `needs` says so. Sums in float32; the gradients of gate
    and up are rounded to bfloat16 as the operands of the products that follow. The same bits from call to call."""
    with torch.no_grad():
        index = x.get_device()
        x, T, H, stride = _rows(x, "x", index)
        gate_up, I, down, O = _ffn_weights(gate_up, down, H, index)
        pre, hidden = saved
        dout = _rows(dout, "dout", index, O, T)[0].contiguous()
        if pre.shape != (T, 2 * I) or pre.dtype is not torch.float32 or hidden.shape != (T, I) or \
                hidden.dtype is not torch.bfloat16 or not (pre.is_contiguous() and hidden.is_contiguous()) or \
                pre.get_device() != index or hidden.get_device() != index:
            raise ValueError(f"saved (pre [{T}, {2 * I}] float32, hidden [{T}, {I}] bfloat16) of gated_ffn_forward expected")
        new = x.new_zeros if T == 0 else x.new_empty
        dx, dgate_up, ddown = (new(shape) if need else None for need, shape in zip(needs, ((T, H), (2 * I, H), (O, I))))
        rows = x.new_empty((T, 2 * I))
        kernels.launch("d3_gated_ffn_backward", index, _lib.GATED_FFN_BACKWARD.pack(
            dout.data_ptr(), x.data_ptr(), gate_up.data_ptr(), down.data_ptr(), pre.data_ptr(), hidden.data_ptr(), rows.data_ptr(),
            _at(dx), _at(dgate_up), _at(ddown), stride, T, H, I, O))
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
    _no_tangent("gated_ffn", x, gate_up, down, *(gate_up_lora or ()), *(down_lora or ()))
    if gate_up_lora is None and down_lora is None:
        if ids is not None:
            raise ValueError("ids go with gate_up_lora or down_lora")
        if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad):
            return _GatedFfn.apply(x, gate_up, down)
    elif torch.is_grad_enabled() and _any_grad(x, gate_up, down, *(gate_up_lora or ()), *(down_lora or ())):
        raise RuntimeError("gated_ffn with adapters has no backward pass: call it under torch.no_grad()")
    index = x.get_device()
    x, T, H, stride = _rows(x, "x", index)
    gate_up, I, down, O = _ffn_weights(gate_up, down, H, index)
    hidden = _dense(x, T, H, stride, gate_up, 2 * I, index, True, lora=gate_up_lora, ids=ids)
    return _dense(hidden, T, I, I, down, O, index, lora=down_lora, ids=ids)


# ------------------------------------------------------------------------------------------------------------- norms
def _float_rows(t, what, index, shape=None):
    """(rows [T, H], their stride, type), checked, float32 or bfloat16, with columns side by side (else a copy that has them so)."""
    kind = _TYPES.get(t.dtype)
    if kind is None or t.dim() != 2:
        raise TypeError(f"{what} [T, H] float32 or bfloat16 expected")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} {list(shape)} expected, not {list(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    if t.is_contiguous():
        return t, t.size(1), kind
    if t.stride(1) == 1 and t.stride(0) >= t.size(1):
        return t, t.stride(0), kind
    return t.contiguous(), t.size(1), kind


def _norm_weight(w, what, H, index):
    """(weight, type), checked; (None, 0) without one."""
    if w is None:
        return None, 0
    kind = _TYPES.get(w.dtype)
    if kind is None or w.dim() != 1 or w.size(0) != H:
        raise ValueError(f"{what} [{H}] float32 or bfloat16 expected")
    if w.get_device() != index:
        raise ValueError(f"{what} on the rows' device expected")
    return w.contiguous(), kind


def _norm_gate(gate, T, H, index):
    """(gate, type, kind, row stride): 1 a value per row ([T, 1]), 2 per channel ([H] or [1, H]), 3 per element, 0 without one."""
    if gate is None:
        return None, 0, 0, 0
    dtype, shape = _TYPES.get(gate.dtype), gate.shape
    if dtype is None or gate.get_device() != index:
        raise ValueError("gate float32 or bfloat16 on the rows' device expected")
    if shape == (T, H):
        gate, stride, _ = _float_rows(gate, "gate", index)
        return gate, dtype, 3, stride
    if shape == (T, 1):
        return gate.contiguous(), dtype, 1, 1
    if shape == (H,) or shape == (1, H):
        return gate.contiguous(), dtype, 2, 0
    raise ValueError(f"gate [{T}, 1], [{H}], [1, {H}] or [{T}, {H}] expected, not {list(shape)}")


def _norm_launch(name, index, y, residual, weight, post, gate, T, H, out_type, scale, eps, unit_offset, dh=0, dn=0, h=0, n=0, rstd=0,
                 dy=0, dresidual=0, dweight=0, dpost=0, dgate=0, partials=0, floats=0):
    """C entry `name` on inputs as the functions above return them."""
    (y, y_stride, _), (residual, stride, stream_type) = y, residual
    (weight, weight_type), (post, post_type), (gate, gate_type, gate_kind, gate_stride) = weight, post, gate
    kernels.launch(name, index, _lib.ADD_NORM.pack(
        _at(y), residual.data_ptr(), _at(weight), _at(post), _at(gate), dh, dn, h, n, rstd, dy, dresidual, dweight, dpost, dgate,
        partials, floats, y_stride, stride, gate_stride, out_type, stream_type, weight_type, post_type, gate_type, gate_kind, T, H,
        scale, eps, unit_offset))


def _norm_shape(residual):
    T, H = residual.shape
    if not 1 <= H <= MAX_NORM_COLS or T > _INT_MAX:
        raise ValueError(f"rows of 1 to {MAX_NORM_COLS} columns, not {H}")
    return T, H


def _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, stats):
    index = residual.get_device()
    r = _float_rows(residual, "residual", index)
    T, H = _norm_shape(residual)
    if y is None:
        raise TypeError("y [T, H] float32 or bfloat16 expected")
    b = _float_rows(y, "y", index, residual.shape)
    w, p, g = _norm_weight(weight, "weight", H, index), _norm_weight(post, "post", H, index), _norm_gate(gate, T, H, index)
    h = residual.new_empty((T, H))
    n = None if weight is None else y.new_empty((T, H))
    rstd = h.new_empty((2, T), dtype=torch.float32) if stats else None
    _norm_launch("d3_add_norm", index, b, r, w, p, g, T, H, b[2], scale, eps, unit_offset, 0, 0, h.data_ptr(), _at(n), _at(rstd))
    return h, n, rstd


class _Saved(tuple):
    """add_norm_forward's (rstd, residual) with what residual's version was (None: not known)."""
    version = None


def _version(t):
    """(A view's version counts writes to its whole base: those to other layers' rows of one buffer, say.)"""
    return None if t.is_inference() or t._is_view() else t._version


def add_norm_forward(y, residual, weight, *, post=None, gate=None, scale=1.0, eps=1e-6, unit_offset=False):
    """add_norm's (h, n) and what add_norm_backward needs beside them: (rstd [2, T] float32, residual); autograd does not see it.
    The residual stream is kept, not copied: a bfloat16 one has to stay as it is until add_norm_backward has read it (one that torch
    knows to have changed is refused there); a float32 one is not read again."""
    with torch.no_grad():
        h, n, rstd = _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, True)
        saved = _Saved((rstd, residual))
        saved.version = _version(residual)
        return h, n, saved


def add_norm_backward(dh, dn, y, h, saved, weight, *, post=None, gate=None, scale=1.0, unit_offset=False,
                      needs=(True, True, True, True, True)):
    """(dy, dresidual, dweight, dpost, dgate) of add_norm for the gradients dh and dn of its outputs (either may be None: zero),
    with y, residual (a bfloat16 one), weight, post, gate, scale and unit_offset as they went in and h and `saved` as
    add_norm_forward returned them. Each gradient has its input's type and shape; None where the input is absent or `needs` says
    so. Float32 inside; of a bfloat16 stream h is not read but made again from y and `saved`'s residual, since its rounding would
    show in the gradients. Sums over the rows (dweight, dpost, a gate per channel) are the same bits from call to call."""
    with torch.no_grad():
        if y is None:
            raise TypeError("y [T, H] float32 or bfloat16 expected")
        rstd, residual = saved
        if dn is not None and h.dtype is torch.bfloat16 and isinstance(saved, _Saved) and saved.version != _version(residual):
            raise RuntimeError("add_norm_backward: residual was changed in place after add_norm_forward, which a bfloat16 stream's "
                               "gradients read again")
        return _add_norm_backward(dh, dn, y, h, rstd, residual, weight, post, gate, scale, unit_offset, needs, None)


def _add_norm_backward(dh, dn, y, h, rstd, residual, weight, post, gate, scale, unit_offset, needs, out_dtype):
    index = h.get_device()
    if y is not None and h.dtype is torch.bfloat16:
        if residual.dtype is not h.dtype or residual.shape != h.shape:
            raise ValueError("saved (rstd, residual) of add_norm_forward expected")
        r = _float_rows(residual, "residual", index)
    else:
        r = _float_rows(h, "h", index)
    T, H = _norm_shape(h)
    b = (None, 0, _TYPES[out_dtype]) if y is None else _float_rows(y, "y", index, h.shape)
    out_dtype = out_dtype if y is None else y.dtype
    w, p, g = _norm_weight(weight, "weight", H, index), _norm_weight(post, "post", H, index), _norm_gate(gate, T, H, index)
    if dh is None and dn is None:
        raise ValueError("dh or dn expected")
    if weight is None and dn is not None:
        raise ValueError("dn goes with weight")
    if rstd is None or rstd.dtype is not torch.float32 or rstd.shape != (2, T) or not rstd.is_contiguous() or \
            rstd.get_device() != index:
        raise ValueError(f"rstd [2, {T}] float32 of add_norm_forward expected")
    if dh is not None:
        if dh.dtype is not h.dtype or dh.shape != (T, H) or dh.get_device() != index:
            raise ValueError("dh of h's type and shape, on its device, expected")
        dh = dh.contiguous()
    if dn is not None:
        if dn.dtype is not out_dtype or dn.shape != (T, H) or dn.get_device() != index:
            raise ValueError("dn of n's type and shape, on its device, expected")
        dn = dn.contiguous()
    if not any(needs):
        return (None,) * 5
    new = h.new_empty
    dy = new((T, H), dtype=out_dtype) if y is not None and needs[0] else None
    dresidual = new((T, H)) if needs[1] else None
    dweight = new((H,), dtype=weight.dtype) if weight is not None and needs[2] else None
    dpost = new((H,), dtype=post.dtype) if post is not None and needs[3] else None
    dgate = new(gate.shape, dtype=gate.dtype) if gate is not None and needs[4] else None
    parts = (dweight is not None) + (dpost is not None) + (dgate is not None and g[2] == 2)
    floats = parts * _lib.lib().d3_add_norm_partials(T, H)
    partials = new((floats,), dtype=torch.float32) if parts else None
    _norm_launch("d3_add_norm_backward", index, b, r, w, p, g, T, H, b[2], scale, 0.0, unit_offset, _at(dh), _at(dn), r[0].data_ptr(), 0,
                 rstd.data_ptr(), _at(dy), _at(dresidual), _at(dweight), _at(dpost), _at(dgate), _at(partials), floats)
    return dy, dresidual, dweight, dpost, dgate


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, post, gate, scale, eps, unit_offset):
        h, n, rstd = _add_norm(y, residual, weight, post, gate, scale, eps, unit_offset, True)
        # (a float32 stream needs h, a bfloat16 one residual: the other is not kept alive)
        ctx.save_for_backward(y, residual if residual.dtype is torch.bfloat16 else h, rstd, weight, post, gate)
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
        grads = _add_norm_backward(dh, dn, y, h, rstd, h, weight, post, gate, *ctx.options, ctx.needs_input_grad[:5], None)
        return grads + (None,) * 3


def add_norm(y, residual, weight, *, post=None, gate=None, scale=1.0, eps=1e-6, unit_offset=False):
    """The end of one block and the start of the next, in one pass: (h, n) with h = residual + scale * gate * v, in residual's
    type, and n = h / rms(h) * weight, in y's type; v is the block's output y, or y / rms(y) * post with `post` (a norm after the
    block as well). y and residual [T, H], float32 or bfloat16 each; weight and post [H]; gate a value per row [T, 1], per
    channel [H] or per element [T, H]. rms(z) = sqrt(mean(z^2) + eps); with unit_offset weight and post are read as 1 + w.
    weight None: n is None. Float32 inside, h and n each rounded once (n comes from h before its rounding). Differentiable."""
    _no_tangent("add_norm", y, residual, weight, post, gate)
    if torch.is_grad_enabled() and _any_grad(y, residual, weight, post, gate):
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
        _no_capture("norm")
        x, rstd, weight = ctx.saved_tensors
        unit_offset, dtype = ctx.options
        return _norm_backward(dn, x, rstd, weight, unit_offset, dtype, ctx.needs_input_grad[:2]) + (None,) * 3


def _norm(x, weight, eps, unit_offset, dtype, stats):
    if weight is None:
        raise ValueError("weight [H] expected")
    index = x.get_device()
    r = _float_rows(x, "x", index)
    T, H = _norm_shape(x)
    n = x.new_empty((T, H), dtype=dtype)
    rstd = n.new_empty((2, T), dtype=torch.float32) if stats else None
    _norm_launch("d3_add_norm", index, (None, 0, 0), r, _norm_weight(weight, "weight", H, index), (None, 0), (None, 0, 0, 0), T, H,
                 _TYPES[dtype], 1.0, eps, unit_offset, n=n.data_ptr(), rstd=_at(rstd))
    return n, rstd


def _norm_backward(dn, x, rstd, weight, unit_offset, dtype, needs):
    _, dx, dweight, _, _ = _add_norm_backward(None, dn, None, x, rstd, None, weight, None, None, 1.0, unit_offset,
                                              (False, *needs, False, False), dtype)
    return dx, dweight


def _norm_type(x, dtype):
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _TYPES or x.dtype not in _TYPES:
        raise TypeError("float32 or bfloat16 expected")
    return dtype


def norm_forward(x, weight, *, eps=1e-6, unit_offset=False, dtype=None):
    """norm's n and what norm_backward needs beside x: rstd [2, T] float32 (its second row is add_norm's); autograd does not see it."""
    with torch.no_grad():
        return _norm(x, weight, eps, unit_offset, _norm_type(x, dtype), True)


def norm_backward(dn, x, saved, weight, *, unit_offset=False, needs=(True, True)):
    """(dx, dweight) of norm for the gradient dn of its output, with x, weight and unit_offset as they went in and `saved` as
    norm_forward returned it, each of its input's type; None where `needs` says so. dweight is the same bits from call to call."""
    with torch.no_grad():
        if dn is None or weight is None or dn.dtype not in _TYPES:
            raise ValueError("dn [T, H] float32 or bfloat16, and weight, expected")
        return _norm_backward(dn, x, saved, weight, unit_offset, dn.dtype, needs)


def norm(x, weight, *, eps=1e-6, unit_offset=False, dtype=None):
    """x / rms(x) * weight of rows x [T, H] (float32 or bfloat16), in `dtype` (x's without it): the norm before a model's first
    block; add_norm makes the others. Differentiable."""
    dtype = _norm_type(x, dtype)
    _no_tangent("norm", x, weight)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)):
        return _Norm.apply(x, weight, eps, unit_offset, dtype)
    return _norm(x, weight, eps, unit_offset, dtype, False)[0]


# ------------------------------------------------------------------------------------------------------- the whole block
def gate_weight(shared_gate):
    """A shared expert's gate [H] bfloat16 as sparse_block reads it, laid out once: [8, H], zeros below."""
    if shared_gate.dim() != 1 or shared_gate.dtype is not torch.bfloat16:
        raise TypeError("shared_gate [H] bfloat16 expected")
    out = shared_gate.new_zeros((8, shared_gate.numel()))
    out[0] = shared_gate
    return out


def sparse_block(n, h, router, gate_up, down, topk, *, shared=None, shared_gate=None, shared_lora=(None, None), ids=None,
                 next_weight=None, scale=1.0, eps=1e-6, unit_offset=False):
    """A block's expert half on unquantized weights, from its normalized rows n [T, H] bfloat16 and the residual stream h [T, H] to
    the next block's: (h, n) as add_norm returns them with `next_weight` (n None without it). router [E, H] gives the logits (E a
    multiple of 8), kernels.route the experts, kernels.bf16_layer the routed layer on banks gate_up [E * 2I, H] and down [E * H, I].
    shared = (gate_up, down): the shared expert, gated_ffn with `shared_lora` = (gate_up_lora, down_lora) of the rows' adapters
    `ids`; it enters times sigmoid(n . gate) where shared_gate (gate_weight's) is given. The routed and the shared output are each
    added to the stream, times `scale`, and rounded to its type. Any number of rows; nothing waits on the host. No backward pass."""
    loras = [t for lora in shared_lora for t in lora or ()]
    tensors = (n, h, router, gate_up, down, shared_gate, next_weight, *(shared or ()), *loras)
    _no_tangent("sparse_block", *tensors)
    if torch.is_grad_enabled() and _any_grad(*tensors):
        raise RuntimeError("sparse_block has no backward pass: call it under torch.no_grad()")
    if shared is None and (shared_gate is not None or ids is not None or tuple(shared_lora) != (None, None)):
        raise ValueError("shared_gate, shared_lora and ids go with shared")
    if shared_gate is not None and shared_gate.dim() != 2:
        raise ValueError("shared_gate as gate_weight lays it out expected")
    options = {"scale": scale, "eps": eps, "unit_offset": unit_offset}
    logits = linear(n, router)
    if n.shape[0] == 0:
        return add_norm(n, h, next_weight, **options)
    experts, weights = kernels.route(logits, topk)
    routed = kernels.bf16_layer(n, experts, weights, gate_up, down, router.shape[0])
    if shared is None:
        return add_norm(routed, h, next_weight, **options)
    y = gated_ffn(n, *shared, gate_up_lora=shared_lora[0], down_lora=shared_lora[1], ids=ids)
    gate = None if shared_gate is None else torch.sigmoid(linear(n, shared_gate)[:, :1])
    h, _ = add_norm(routed, h, None, scale=scale)
    return add_norm(y, h, next_weight, gate=gate, **options)
