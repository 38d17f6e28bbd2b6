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
from several streams.  First derivatives only.
"""
import ctypes

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ..pointnet2 import _ext

_call, _lib, _on, _stream = _ext._call, _ext._lib, _ext._on, _ext._stream
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # BTR_F32, BTR_BF16, BTR_F16
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2}                      # BTR_ACT_*
_INT_MAX = 2 ** 30


def _ptr(t):
    return None if t is None else t.data_ptr()


def _require(cond, message, *args):
    if not cond:
        raise RuntimeError(message % args)


def _check(name, ref, **tensors):
    """All on the device and of the type of `ref`."""
    _require(isinstance(ref, torch.Tensor), "%s: expected a tensor", name)
    _require(ref.is_cuda, "%s: CPU not supported", name)
    _require(ref.dtype in _DTYPES, "%s: %s not supported", name, ref.dtype)
    for key, t in tensors.items():
        if t is None:
            continue
        _require(isinstance(t, torch.Tensor) and t.device == ref.device,
                 "%s: %s is not on %s", name, key, ref.device)
        _require(t.dtype == ref.dtype, "%s: %s is %s, expected %s", name, key, t.dtype, ref.dtype)


def _rows(t):
    """(tensor, row stride): the rows of t (its last axis) at one stride, copied if they are not."""
    width = t.shape[-1]
    if t.dim() == 1:
        return t.contiguous(), width
    if t.stride(-1) == 1 or width == 1:
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


# --------------------------------------------------------------------------------- layer norm
class _LayerNorm(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        width = x.shape[-1]
        rows = x.numel() // width
        xr, ldx = _rows(x)
        rr, ldr = (None, 0) if residual is None else _rows(residual)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = None
        if any(ctx.needs_input_grad):
            stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
        with _on(x) as dev:
            _call(_lib.btr_layer_norm_fwd, _DTYPES[x.dtype], rows, width, _ptr(xr), ldx, _ptr(rr),
                  ldr, _ptr(w), _ptr(b), eps, _ptr(y), _ptr(stats), _stream(dev))
        ctx.save_for_backward(xr, rr, w, stats)
        ctx.layout = (rows, width, ldx, ldr)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, residual, weight, stats = ctx.saved_tensors
        rows, width, ldx, ldr = ctx.layout
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        gr, ldg = _rows(dy)
        dev = x.device
        dx = torch.empty(dy.shape, dtype=x.dtype, device=dev)
        dw = torch.empty((width,), dtype=x.dtype, device=dev) if need_w else None
        db = torch.empty((width,), dtype=x.dtype, device=dev) if need_b else None
        nbytes = _lib.btr_layer_norm_bwd_workspace_bytes(rows, width) if need_w or need_b else 0
        ws = _workspace(nbytes, dev)
        with _on(x) as d:
            _call(_lib.btr_layer_norm_bwd, _DTYPES[x.dtype], rows, width, _ptr(x), ldx,
                  _ptr(residual), ldr, _ptr(gr), ldg, _ptr(weight), _ptr(stats), _ptr(dx),
                  _ptr(dw), _ptr(db), _ptr(ws), nbytes, _stream(d))
        return dx if need_x else None, dw, db, dx if need_r else None, None


def layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5):
    """Layer norm over the last axis of `x + residual` (residual: the shape of x, or None), times
    `weight` plus `bias` (its width, or None).  Statistics in float32 over the unrounded sum."""
    _check("layer_norm", x, weight=weight, bias=bias, residual=residual)
    _require(x.dim() >= 1 and x.shape[-1] >= 1, "layer_norm: shape %s", tuple(x.shape))
    width = x.shape[-1]
    for key, t in (("weight", weight), ("bias", bias)):
        _require(t is None or tuple(t.shape) == (width,), "layer_norm: %s of shape %s for width %d",
                 key, None if t is None else tuple(t.shape), width)
    _require(residual is None or residual.shape == x.shape,
             "layer_norm: residual of shape %s for %s",
             None if residual is None else tuple(residual.shape), tuple(x.shape))
    _require(eps >= 0, "layer_norm: eps %s", eps)
    return _LayerNorm.apply(x, weight, bias, residual, float(eps))


# ------------------------------------------------------------------------------------- linear
class _Linear(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        n, k = weight.shape
        m = x.numel() // k
        xr, ldx = _rows(x)
        wr, ldw = _rows(weight)
        rr, ldr = (None, 0) if residual is None else _rows(residual)
        b = None if bias is None else bias.contiguous()
        dev = x.device
        y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
        keep, slope = None, None      # keep: what dz is made of in the backward
        if act and any(ctx.needs_input_grad[:3]):
            if act == _ACTIVATIONS["relu"] and residual is None:
                keep = y                                          # y > 0 exactly where z > 0
            else:
                keep = slope = torch.empty((m, n), dtype=x.dtype, device=dev)
        p = _ext.Linear(_DTYPES[x.dtype], m, n, k, act, xr.data_ptr(), wr.data_ptr(), _ptr(b),
                        _ptr(rr), ldx, ldw, ldr)
        addr = ctypes.addressof(p)
        nbytes = _lib.btr_linear_fwd_workspace_bytes(addr)
        ws = _workspace(nbytes, dev)
        with _on(x) as d:
            _call(_lib.btr_linear_fwd, addr, y.data_ptr(), _ptr(slope), _ptr(ws), nbytes, _stream(d))
        ctx.save_for_backward(xr, wr, keep)
        ctx.layout = (m, n, k, act, ldx, ldw, x.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, keep = ctx.saved_tensors
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
            addr = ctypes.addressof(p)
            nbytes = _lib.btr_linear_bwd_workspace_bytes(addr, gr.data_ptr(), ldg)
            ws = _workspace(nbytes, dev)
            with _on(x) as d:
                _call(_lib.btr_linear_bwd, addr, _ptr(keep), gr.data_ptr(), ldg, _ptr(dx), _ptr(dw),
                      _ptr(db), _ptr(ws), nbytes, _stream(d))
        return dx, dw, db, dy if need_r else None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual: x (..., k), weight (n, k), bias (n) or None, activation
    None / "relu" / "gelu" (the erf form), residual (..., n) or None.  One kernel forward; sums,
    activation and residual in float32, rounded once."""
    _check("linear", x, weight=weight, bias=bias, residual=residual)
    _require(activation in _ACTIVATIONS, "linear: activation should be None/relu/gelu, not %s",
             activation)
    _require(weight.dim() == 2 and x.dim() >= 1 and min(weight.shape) >= 1 and
             x.shape[-1] == weight.shape[1], "linear: x of shape %s for a weight of shape %s",
             tuple(x.shape), tuple(weight.shape))
    n, k = weight.shape
    _require(bias is None or tuple(bias.shape) == (n,), "linear: bias of shape %s for %d outputs",
             None if bias is None else tuple(bias.shape), n)
    _require(residual is None or residual.shape == x.shape[:-1] + (n,),
             "linear: residual of shape %s for an output of shape %s",
             None if residual is None else tuple(residual.shape), tuple(x.shape[:-1]) + (n,))
    _require(x.numel() // k <= _INT_MAX, "linear: %d rows", x.numel() // k)
    return _Linear.apply(x, weight, bias, residual, _ACTIVATIONS[activation])


# ---------------------------------------------------------------------------- cross-attention
def _describe(q, k, v, lengths, mask, scale):
    p = _ext.CrossAttention()
    p.dtype = _DTYPES[q.dtype]
    p.b, p.lq, p.h, p.d = q.shape
    p.lk, p.hk = k.shape[1], k.shape[2]
    p.q, p.k, p.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    p.q_sb, p.q_sl, p.q_sh = q.stride()[:3]
    p.k_sb, p.k_sl, p.k_sh = k.stride()[:3]
    p.v_sb, p.v_sl, p.v_sh = v.stride()[:3]
    p.lengths = _ptr(lengths)
    p.mask = _ptr(mask)
    p.mask_sb = 0 if mask is None else mask.stride(0)
    p.scale = scale
    return p


def _last_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _CrossAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
        dev = q.device
        p = _describe(q, k, v, lengths, mask, scale)
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = None
        if any(ctx.needs_input_grad):
            lse = torch.empty((p.b * p.h * p.lq,), dtype=torch.float32, device=dev)
        addr = ctypes.addressof(p)
        nbytes = _lib.btr_cross_attention_fwd_workspace_bytes(addr)
        ws = _workspace(nbytes, dev)
        with _on(q) as d:
            _call(_lib.btr_cross_attention_fwd, addr, _ptr(out), _ptr(lse), _ptr(ws), nbytes,
                  _stream(d))
        ctx.save_for_backward(q, k, v, lengths, mask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lengths, mask, out, lse = ctx.saved_tensors
        dev = q.device
        dout = dout.contiguous()
        p = _describe(q, k, v, lengths, mask, ctx.scale)
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk = torch.empty(k.shape, dtype=q.dtype, device=dev)
        dv = torch.empty(v.shape, dtype=q.dtype, device=dev)
        addr = ctypes.addressof(p)
        nbytes = _lib.btr_cross_attention_bwd_workspace_bytes(addr)
        ws = _workspace(nbytes, dev)
        with _on(q) as d:
            _call(_lib.btr_cross_attention_bwd, addr, _ptr(out), _ptr(lse), _ptr(dout), _ptr(dq),
                  _ptr(dk), _ptr(dv), _ptr(ws), nbytes, _stream(d))
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
                None, None, None)


def cross_attention(query, key, value, key_lengths=None, key_padding_mask=None, scale=None):
    """softmax(scale query key^T) value per head.

    query (B, Lq, H, D), key and value (B, Lk, Hk, D), H a multiple of Hk (query head i reads key
    head i // (H // Hk)), D <= 128; result (B, Lq, H, D).  Of batch entry b the keys from
    key_lengths[b] (int32 (B), on the device) on and those where key_padding_mask (bool (B, Lk)) is
    True take no part, whatever they hold; a query left without keys gets zeros, and gives none of
    its gradient to anybody.  scale: D ** -0.5 by default, positive."""
    _check("cross_attention", query, key=key, value=value)
    _require(query.dim() == 4 and key.dim() == 4 and value.dim() == 4,
             "cross_attention: expected (batch, length, head, width) tensors")
    B, _, H, D = query.shape
    Lk, Hk = key.shape[1], key.shape[2]
    _require(key.shape == value.shape and key.shape[0] == B and key.shape[3] == D,
             "cross_attention: query %s, key %s, value %s", tuple(query.shape), tuple(key.shape),
             tuple(value.shape))
    _require(Hk >= 1 and H >= 1 and H % Hk == 0, "cross_attention: %d heads on %d key heads", H, Hk)
    _require(1 <= D <= 128, "cross_attention: head width %d (1 .. 128)", D)
    for name, t, dtype, shape in (("key_lengths", key_lengths, torch.int32, (B,)),
                                  ("key_padding_mask", key_padding_mask, torch.bool, (B, Lk))):
        if t is not None:
            _require(t.dtype == dtype and tuple(t.shape) == shape and t.device == query.device,
                     "cross_attention: %s should be %s of shape %s on %s", name, dtype, shape,
                     query.device)
    if key_lengths is not None:
        key_lengths = key_lengths.contiguous()
    if key_padding_mask is not None:
        key_padding_mask = _last_contiguous(key_padding_mask)
    scale = float(D) ** -0.5 if scale is None else float(scale)
    _require(0.0 < scale < float("inf"), "cross_attention: scale %s", scale)
    return _CrossAttention.apply(query, key, value, key_lengths, key_padding_mask, scale)
