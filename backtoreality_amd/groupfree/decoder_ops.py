"""The operators of a transformer decoder layer for float32, bfloat16 and float16, with gradients:

    layer_norm(x, weight, bias, residual=, eps=)           csrc/layer_norm.hip
    linear(x, weight, bias, activation=, residual=)        csrc/linear.hip
    cross_attention(query, key, value, key_lengths=, key_padding_mask=, scale=)
                                                           csrc/cross_attention.hip

The reference's decoder layer (detection/GroupFree3D/models/transformer.py:36-76) is these three.
`fused_decoder` runs it whole for float32 at the detector's own sizes; these are for what that call
does not cover -- 16-bit types, padded keys, key / value heads shared by several query heads, widths
and strides of any kind -- and `TransformerDecoderLayer` is built on them there.

All three take CUDA (HIP) tensors of one type on one device, enqueue on that device's current stream
without synchronising, and raise RuntimeError for anything else.  Rows are read where they are when
the last axis is contiguous, whatever the other strides; otherwise the tensor is copied first.
Workspaces come from torch's allocator per call, so calls may be captured into HIP graphs and made
from several streams.  (As for any operator here: torch's engine cannot capture a backward pass while
an eager graph of the same leaves is alive.)  First derivatives in backward mode only: a second
derivative, a forward-mode one and torch.func's transforms are refused.
"""
import ctypes

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from ..pointnet2 import _ext

_call, _lib = _ext._call, _ext._lib
_addressof = ctypes.addressof
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # BTR_F32, BTR_BF16, BTR_F16
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2}                      # BTR_ACT_*
_MAX_ROWS = 2 ** 30
# (the checks below are written out, without helpers that format or build tuples on the way: a call
# of a decoder's size is bound by the host: 17.4 -> 11.6 us without gradients, 20.6 -> 17.5 with)


def _refuse(message, *args):
    raise RuntimeError(message % args)


def _check_one(name, key, t, ref):
    if not isinstance(t, torch.Tensor) or t.device != ref.device:
        _refuse("%s: %s is not on %s", name, key, ref.device)
    if t.dtype != ref.dtype:
        _refuse("%s: %s is %s, expected %s", name, key, t.dtype, ref.dtype)


def _check_ref(name, t):
    if not isinstance(t, torch.Tensor):
        _refuse("%s: expected a tensor", name)
    if not t.is_cuda:
        _refuse("%s: CPU not supported", name)
    if t.dtype not in _DTYPES:
        _refuse("%s: %s not supported", name, t.dtype)


# (the handle without a Stream object around it: one microsecond a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _ext._stream


_tracing = torch._C._get_tracing_state


def transformed():
    """Is this call differentiated in forward mode, transformed (torch.func), traced or compiled?  The
    operators refuse most of that; a caller that has elementary torch operations to offer takes those."""
    return (forward_ad._current_level >= 0 or _tracing() is not None or
            torch._C._functorch.peek_interpreter_stack() is not None or torch.compiler.is_compiling())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _launch(t, fn, *args):
    """fn(*args, stream) on the device of t, on its current stream."""
    dev = t.get_device()
    if dev == torch.cuda.current_device():
        _call(fn, *args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            _call(fn, *args, _raw_stream(dev))


def _rows(t):
    """(tensor, row stride): the rows of t (its last axis) at one stride, copied if they are not."""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, width
    if t.dim() > 1 and (t.stride(-1) == 1 or width == 1):
        # leading axes of size 1 have no stride; the others must fold into one
        dims = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
        if not dims:
            return t, width
        if all(dims[i][1] == dims[i + 1][0] * dims[i + 1][1] for i in range(len(dims) - 1)) and \
                dims[-1][1] >= width:
            return t, dims[-1][1]
    return t.contiguous(), width


def _workspace(nbytes, device):
    return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None


def _wants_grad(*tensors):
    # Without gradients the autograd node around the call is left out -- but not where the node is what
    # refuses a forward-mode derivative (a dual tensor need not require a gradient; without the node its
    # tangent would be lost without a word), or what torch.jit.trace records (it does not see the kernel
    # write the result).
    if forward_ad._current_level >= 0 or _tracing() is not None:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# --------------------------------------------------------------------------------- layer norm
def _layer_norm_forward(x, weight, bias, residual, eps, keep):
    width = x.shape[-1]
    rows = x.numel() // width
    xr, ldx = _rows(x)
    rr, ldr = (None, 0) if residual is None else _rows(residual)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if keep else None
    _launch(x, _lib.btr_layer_norm_fwd, _DTYPES[x.dtype], rows, width, xr.data_ptr(), ldx, _ptr(rr),
            ldr, _ptr(w), _ptr(b), eps, y.data_ptr(), _ptr(stats))
    return y, xr, rr, w, stats, (rows, width, ldx, ldr)


class _LayerNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, xr, rr, w, stats, ctx.layout = _layer_norm_forward(x, weight, bias, residual, eps, True)
        ctx.save_for_backward(xr, rr, w, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, residual, weight, stats = ctx.saved_tensors
        rows, width, ldx, ldr = ctx.layout
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        gr, ldg = _rows(dy)
        dev, dtype = x.device, x.dtype
        dx = torch.empty(dy.shape, dtype=dtype, device=dev)
        dw = torch.empty((width,), dtype=dtype, device=dev) if need_w else None
        db = torch.empty((width,), dtype=dtype, device=dev) if need_b else None
        nbytes = _lib.btr_layer_norm_bwd_workspace_bytes(rows, width) if need_w or need_b else 0
        ws = _workspace(nbytes, dev)
        _launch(x, _lib.btr_layer_norm_bwd, _DTYPES[dtype], rows, width, x.data_ptr(), ldx,
                _ptr(residual), ldr, gr.data_ptr(), ldg, _ptr(weight), stats.data_ptr(),
                dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), nbytes)
        return dx if need_x else None, dw, db, dx if need_r else None, None


def layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5):
    """Layer norm over the last axis of `x + residual` (residual: the shape of x, or None), times
    `weight` plus `bias` (its width, or None).  Statistics in float32 over the unrounded sum."""
    _check_ref("layer_norm", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        _refuse("layer_norm: shape %s", tuple(x.shape))
    for key, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_one("layer_norm", key, t, x)
            if t.dim() != 1 or t.shape[0] != x.shape[-1]:
                _refuse("layer_norm: %s of shape %s for width %d", key, tuple(t.shape), x.shape[-1])
    if residual is not None:
        _check_one("layer_norm", "residual", residual, x)
        if residual.shape != x.shape:
            _refuse("layer_norm: residual of shape %s for %s", tuple(residual.shape), tuple(x.shape))
    eps = float(eps)
    if not eps >= 0:
        _refuse("layer_norm: eps %s", eps)
    if _wants_grad(x, weight, bias, residual):
        return _LayerNorm.apply(x, weight, bias, residual, eps)
    return _layer_norm_forward(x, weight, bias, residual, eps, False)[0]


# ------------------------------------------------------------------------------------- linear
def _linear_forward(x, weight, bias, residual, act, keep):
    n, k = weight.shape
    m = x.numel() // k
    xr, ldx = _rows(x)
    wr, ldw = _rows(weight)
    rr, ldr = (None, 0) if residual is None else _rows(residual)
    b = None if bias is None else bias.contiguous()
    dev = x.device
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    kept, slope = None, None          # kept: what dz is made of in the backward
    if act and keep:
        if act == 1 and residual is None:
            kept = y                    # on where y > 0 or NaN: a z that rounds to 0 is off
        else:
            kept = slope = torch.empty((m, n), dtype=x.dtype, device=dev)
    p = _ext.Linear(_DTYPES[x.dtype], m, n, k, act, xr.data_ptr(), wr.data_ptr(), _ptr(b), _ptr(rr),
                    ldx, ldw, ldr)
    addr = _addressof(p)
    nbytes = _lib.btr_linear_fwd_workspace_bytes(addr)
    ws = _workspace(nbytes, dev)
    _launch(x, _lib.btr_linear_fwd, addr, y.data_ptr(), _ptr(slope), _ptr(ws), nbytes)
    return y, xr, wr, kept, (m, n, k, act, ldx, ldw, x.shape)


class _Linear(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, xr, wr, kept, ctx.layout = _linear_forward(x, weight, bias, residual, act,
                                                      any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(xr, wr, kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, kept = ctx.saved_tensors
        m, n, k, act, ldx, ldw, shape = ctx.layout
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dev, dtype = x.device, x.dtype
        dx = torch.empty(shape, dtype=dtype, device=dev) if need_x else None
        dw = torch.empty((n, k), dtype=dtype, device=dev) if need_w else None
        db = torch.empty((n,), dtype=dtype, device=dev) if need_b else None
        if need_x or need_w or need_b:
            gr, ldg = _rows(dy)
            p = _ext.Linear(_DTYPES[dtype], m, n, k, act, x.data_ptr(), weight.data_ptr(), None, None,
                            ldx, ldw, 0)
            addr = _addressof(p)
            nbytes = _lib.btr_linear_bwd_workspace_bytes(addr, gr.data_ptr(), ldg)
            ws = _workspace(nbytes, dev)
            _launch(x, _lib.btr_linear_bwd, addr, _ptr(kept), gr.data_ptr(), ldg, _ptr(dx), _ptr(dw),
                    _ptr(db), _ptr(ws), nbytes)
        return dx, dw, db, dy if need_r else None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual: x (..., k), weight (n, k), bias (n) or None, activation
    None / "relu" / "gelu" (the erf form), residual (..., n) or None.  Sums, activation and residual
    in float32, rounded once.

    Gradients: the gradient of the sum, dy act', enters the two products in the type of x; bfloat16 and
    float16 layers keep GELU's slope in 16 bits (2^-16, small ones of the negative tail 2^-10 of
    themselves, 0 below 2^-30).  ReLU is on where its rounded result is positive or NaN.  float32 rows
    run as sums of three bfloat16 terms, exact to the 24th bit (elements below 2^-108 keep fewer), without
    the three smallest of their nine products; an infinite element makes the sums it enters NaN."""
    _check_ref("linear", x)
    _check_one("linear", "weight", weight, x)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        _refuse("linear: activation should be None/relu/gelu, not %s", activation)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        _refuse("linear: x of shape %s for a weight of shape %s", tuple(x.shape), tuple(weight.shape))
    n, k = weight.shape
    if bias is not None:
        _check_one("linear", "bias", bias, x)
        if bias.dim() != 1 or bias.shape[0] != n:
            _refuse("linear: bias of shape %s for %d outputs", tuple(bias.shape), n)
    if residual is not None:
        _check_one("linear", "residual", residual, x)
        if residual.shape != x.shape[:-1] + (n,):
            _refuse("linear: residual of shape %s for an output of shape %s", tuple(residual.shape),
                    tuple(x.shape[:-1]) + (n,))
    if x.numel() // k > _MAX_ROWS:
        _refuse("linear: %d rows", x.numel() // k)
    if _wants_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act)
    return _linear_forward(x, weight, bias, residual, act, False)[0]


# ---------------------------------------------------------------------------- cross-attention
def _describe(q, k, v, lengths, mask, scale):
    b, lq, h, d = q.shape
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    return _ext.CrossAttention(
        _DTYPES[q.dtype], b, lq, k.shape[1], h, k.shape[2], d, q.data_ptr(), k.data_ptr(),
        v.data_ptr(), qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], _ptr(lengths),
        _ptr(mask), 0 if mask is None else mask.stride(0), scale)


def _last_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _cross_attention_forward(q, k, v, lengths, mask, scale, keep):
    q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
    dev = q.device
    p = _describe(q, k, v, lengths, mask, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((p.b * p.h * p.lq,), dtype=torch.float32, device=dev) if keep else None
    addr = _addressof(p)
    nbytes = _lib.btr_cross_attention_fwd_workspace_bytes(addr)
    ws = _workspace(nbytes, dev)
    _launch(q, _lib.btr_cross_attention_fwd, addr, out.data_ptr(), _ptr(lse), _ptr(ws), nbytes)
    return out, q, k, v, lse


class _CrossAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        out, q, k, v, lse = _cross_attention_forward(q, k, v, lengths, mask, scale, True)
        ctx.save_for_backward(q, k, v, lengths, mask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lengths, mask, out, lse = ctx.saved_tensors
        dev, dtype = q.device, q.dtype
        dout = dout.contiguous()
        p = _describe(q, k, v, lengths, mask, ctx.scale)
        dq = torch.empty(q.shape, dtype=dtype, device=dev)
        dk = torch.empty(k.shape, dtype=dtype, device=dev)
        dv = torch.empty(v.shape, dtype=dtype, device=dev)
        addr = _addressof(p)
        nbytes = _lib.btr_cross_attention_bwd_workspace_bytes(addr, dout.data_ptr())
        ws = _workspace(nbytes, dev)
        _launch(q, _lib.btr_cross_attention_bwd, addr, out.data_ptr(), lse.data_ptr(),
                dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), nbytes)
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
                None, None, None)


def cross_attention(query, key, value, key_lengths=None, key_padding_mask=None, scale=None):
    """softmax(scale query key^T) value per head.

    query (B, Lq, H, D), key and value (B, Lk, Hk, D), H a multiple of Hk, at most 128 times it
    (query head i reads key head i // (H // Hk)), D <= 128; result (B, Lq, H, D).  Of batch entry b
    the keys from key_lengths[b] (int32 (B), on the device) on and those where key_padding_mask (bool
    (B, Lk)) is True take no part, whatever they hold; a query left without keys gets zeros, and gives
    none of its gradient to anybody.  scale: D ** -0.5 by default, positive.

    Scores, softmax statistics and sums in float32.  For bfloat16 and float16 the probabilities (and in
    the backward the scores' gradients) enter the products in 16 bits, half a step off each, and the
    backward's rowsum(dout out) takes the rounded result."""
    _check_ref("cross_attention", query)
    _check_one("cross_attention", "key", key, query)
    _check_one("cross_attention", "value", value, query)
    if query.dim() != 4 or key.dim() != 4 or value.dim() != 4:
        _refuse("cross_attention: expected (batch, length, head, width) tensors")
    B, _, H, D = query.shape
    kB, Lk, Hk, kD = key.shape
    if key.shape != value.shape or kB != B or kD != D:
        _refuse("cross_attention: query %s, key %s, value %s", tuple(query.shape), tuple(key.shape),
                tuple(value.shape))
    if Hk < 1 or H < 1 or H % Hk or H // Hk > 128:
        _refuse("cross_attention: %d heads on %d key heads", H, Hk)
    if not 1 <= D <= 128:
        _refuse("cross_attention: head width %d (1 .. 128)", D)
    if key_lengths is not None:
        if not isinstance(key_lengths, torch.Tensor) or key_lengths.dtype != torch.int32 or \
                tuple(key_lengths.shape) != (B,) or key_lengths.device != query.device:
            _refuse("cross_attention: key_lengths should be int32 of shape (%d,) on %s", B,
                    query.device)
        key_lengths = key_lengths.contiguous()
    if key_padding_mask is not None:
        if not isinstance(key_padding_mask, torch.Tensor) or \
                key_padding_mask.dtype != torch.bool or \
                tuple(key_padding_mask.shape) != (B, Lk) or key_padding_mask.device != query.device:
            _refuse("cross_attention: key_padding_mask should be bool of shape (%d, %d) on %s", B, Lk,
                    query.device)
        key_padding_mask = _last_contiguous(key_padding_mask)
    scale = float(D) ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        _refuse("cross_attention: scale %s", scale)
    if _wants_grad(query, key, value):
        return _CrossAttention.apply(query, key, value, key_lengths, key_padding_mask, scale)
    return _cross_attention_forward(query, key, value, key_lengths, key_padding_mask, scale, False)[0]
