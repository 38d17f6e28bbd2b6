"""The decoder layer of GroupFree3D (detection/GroupFree3D/models/transformer.py:11-76):
post-norm self-attention over the query points, cross-attention onto the seed points, FFN;
position embeddings are added to queries and keys AND to the values (the reference passes
the position-augmented tensors as `value`).  `torch.nn.MultiheadAttention` is the module the
reference vendors a copy of (models/multi_head_attention.py), same parameter names; on the
GPU the whole layer is one library call (groupfree/fused_decoder.py -> csrc/decoder.hip); the
op-by-op form below (attention core through groupfree/fused_attention.py) is the CPU path and
what `BTR_FUSED_DECODER=0` selects.  Layers in bfloat16 / float16 and keys with padding
(`key_padding_mask`) run on the operators of groupfree/decoder_ops.py where those do what the modules
would (`_ops_covered`)."""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from . import decoder_ops, fused_attention, fused_decoder

_ACTIVATIONS = {F.relu: "relu", F.gelu: "gelu"}


def _own_call(m, kind, dtype):
    """Is calling `m` what its class does with its parameters, and nothing else?  Exactly a `kind` (a
    subclass, a wrapper or a parametrised module has a forward of its own) without hooks (weight_norm
    and pruning make their weight in one), its parameters plain tensors of the layer's type."""
    return (type(m) is kind and "forward" not in m.__dict__ and
            not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or
                 m._backward_pre_hooks) and
            all(p is None or (p.dtype == dtype and type(p) is nn.Parameter)
                for p in m._parameters.values()))


def _mha_covered(mha, dtype):
    """Packed projections of one width, nothing appended to the keys, and no dropout on the attention
    weights in this call.  (The output projection is read, never called, by the stock module too.)"""
    return (_own_call(mha, nn.MultiheadAttention, dtype) and mha._qkv_same_embed_dim and
            mha.bias_k is None and mha.bias_v is None and not mha.add_zero_attn and
            not getattr(mha, "batch_first", False) and mha.head_dim <= 128 and
            (mha.dropout == 0 or not mha.training) and mha.out_proj.weight.dtype == dtype and
            (mha.out_proj.bias is None or mha.out_proj.bias.dtype == dtype))


def _norm_covered(n, width, dtype):
    return _own_call(n, nn.LayerNorm, dtype) and tuple(n.normalized_shape) == (width,)


def _stock_attention(mha, query, key, key_padding_mask=None):
    """mha(query, key, value=key)[0].  Attention that torch would do in bfloat16 on the GPU -- the
    layer's type, or autocast's -- is done in float32 and rounded once: torch multiplies its batches of
    matrices by transposed views, and such a product of bfloat16 has faulted this GPU in the library's
    kernel.  The module is called as it is (its own forward, hooks), on float32 copies of its
    parameters."""
    bf16 = torch.bfloat16
    in_bf16 = query.is_cuda and (torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda")
                                 else query.dtype) == bf16
    if not in_bf16:
        return mha(query, key, value=key, key_padding_mask=key_padding_mask)[0]
    q = query.float()
    k = q if key is query else key.float()
    params = {name: p.float() for name, p in mha.named_parameters()}
    with torch.autocast("cuda", enabled=False):
        out = torch.func.functional_call(mha, params, (q, k), {
            "value": k, "key_padding_mask": key_padding_mask})[0]
    return out.to(bf16)


class TransformerDecoderLayer(nn.Module):
    def __init__(self, d_model, nhead, dim_feedforward=2048, dropout=0.1, activation="relu",
                 self_posembed=None, cross_posembed=None):
        super().__init__()
        self.self_attn = nn.MultiheadAttention(d_model, nhead, dropout=dropout)
        self.multihead_attn = nn.MultiheadAttention(d_model, nhead, dropout=dropout)
        self.linear1 = nn.Linear(d_model, dim_feedforward)
        self.dropout = nn.Dropout(dropout)
        self.linear2 = nn.Linear(dim_feedforward, d_model)
        self.norm1 = nn.LayerNorm(d_model)
        self.norm2 = nn.LayerNorm(d_model)
        self.norm3 = nn.LayerNorm(d_model)
        self.dropout1 = nn.Dropout(dropout)
        self.dropout2 = nn.Dropout(dropout)
        self.dropout3 = nn.Dropout(dropout)
        if activation not in ("relu", "gelu", "glu"):
            raise RuntimeError("activation should be relu/gelu, not %s." % activation)
        self.activation = getattr(F, activation)
        self.self_posembed = self_posembed
        self.cross_posembed = cross_posembed

    def _ops_covered(self, query, key, key_padding_mask):
        """Does groupfree/decoder_ops.py run this call?  Padded keys and 16-bit layers, of one type
        throughout and without autocast, which chooses types module by module, and only modules that
        are what they look like (_own_call), called as they are (not in forward mode, torch.func or a
        trace); float32 without padding has the whole-layer call, and BTR_FUSED_DECODER=0 has the
        modules (second derivatives need them)."""
        dtype = query.dtype
        if not (query.is_cuda and dtype in (torch.float32, torch.bfloat16, torch.float16) and
                (key_padding_mask is not None or dtype != torch.float32) and key.dtype == dtype and
                self.activation in _ACTIVATIONS and not torch.is_autocast_enabled("cuda") and
                fused_decoder.enabled() and not decoder_ops.transformed() and
                not _has_any_global_hook()):
            return False
        width = query.shape[1]
        return (all(_norm_covered(n, width, dtype) for n in (self.norm1, self.norm2, self.norm3)) and
                _own_call(self.linear1, nn.Linear, dtype) and
                _own_call(self.linear2, nn.Linear, dtype) and
                _mha_covered(self.self_attn, dtype) and _mha_covered(self.multihead_attn, dtype))

    def _forward_ops(self, query, key, q_pos, k_pos, key_padding_mask):
        """The layer on (B, P, C) rows: every projection one kernel with its bias (and activation),
        every residual addition inside its norm."""
        def norm(n, branch, x):
            return decoder_ops.layer_norm(branch, n.weight, n.bias, residual=x, eps=n.eps)

        def attend(mha, rows_q, rows_k, mask=None):
            heads, width = mha.num_heads, mha.head_dim
            W, b = mha.in_proj_weight, mha.in_proj_bias
            E = mha.embed_dim
            if rows_k is None:
                q, k, v = decoder_ops.linear(rows_q, W, b).unflatten(2, (3, heads, width)).unbind(2)
            else:
                q = decoder_ops.linear(rows_q, W[:E], None if b is None else b[:E])
                q = q.unflatten(2, (heads, width))
                k, v = decoder_ops.linear(rows_k, W[E:], None if b is None else b[E:]).unflatten(
                    2, (2, heads, width)).unbind(2)
            out = decoder_ops.cross_attention(q, k, v, key_padding_mask=mask)
            return decoder_ops.linear(out.flatten(2), mha.out_proj.weight, mha.out_proj.bias)

        x, memory = query.transpose(1, 2).contiguous(), key.transpose(1, 2)
        pos = None if q_pos is None else q_pos.transpose(1, 2)
        qp = x if pos is None else x + pos
        x = norm(self.norm1, self.dropout1(attend(self.self_attn, qp, None)), x)
        qp = x if pos is None else x + pos
        kp = memory if k_pos is None else memory + k_pos.transpose(1, 2)
        x = norm(self.norm2, self.dropout2(attend(self.multihead_attn, qp, kp, key_padding_mask)), x)
        h = decoder_ops.linear(x, self.linear1.weight, self.linear1.bias,
                               activation=_ACTIVATIONS[self.activation])
        f = decoder_ops.linear(self.dropout(h), self.linear2.weight, self.linear2.bias)
        return norm(self.norm3, self.dropout3(f), x).transpose(1, 2)

    def forward(self, query, key, query_pos, key_pos, key_padding_mask=None):
        """query (B,C,Pq), key (B,C,Pk), query_pos (B,Pq,3|6), key_pos (B,Pk,3) -> (B,C,Pq).
        key_padding_mask (B,Pk) bool or None: True marks keys that take no part, as in
        `nn.MultiheadAttention`; every scene needs a key that is not padding unless the layer runs on
        the library's operators, where a scene without keys gets a cross-attention of zero."""
        q_pos = self.self_posembed(query_pos) if self.self_posembed is not None else None
        k_pos = self.cross_posembed(key_pos) if self.cross_posembed is not None else None
        if self._ops_covered(query, key, key_padding_mask):
            return self._forward_ops(query, key, q_pos, k_pos, key_padding_mask)
        # the whole layer as one library call (csrc/decoder.hip) when it covers the configuration
        out = None
        if key_padding_mask is None:
            out = fused_decoder.layer_forward(self, query, key, q_pos, k_pos)
        if out is not None:
            return out
        q_pos = q_pos.permute(2, 0, 1) if q_pos is not None else None
        k_pos = k_pos.permute(2, 0, 1) if k_pos is not None else None
        query = query.permute(2, 0, 1)
        key = key.permute(2, 0, 1)

        # attention core: the fused kernels (csrc/attention.hip) when they cover the call, else
        # the stock module (CPU, BTR_FUSED_ATTENTION=0)
        qp = query if q_pos is None else query + q_pos
        att = fused_attention.mha_forward(self.self_attn, qp, qp)
        if att is None:
            att = _stock_attention(self.self_attn, qp, qp)
        query = self.norm1(query + self.dropout1(att))

        qp = query if q_pos is None else query + q_pos
        kp = key if k_pos is None else key + k_pos
        att = None
        if key_padding_mask is None:
            att = fused_attention.mha_forward(self.multihead_attn, qp, kp)
        if att is None:
            att = _stock_attention(self.multihead_attn, qp, kp, key_padding_mask)
        query = self.norm2(query + self.dropout2(att))

        ffn = self.linear2(self.dropout(self.activation(self.linear1(query))))
        query = self.norm3(query + self.dropout3(ffn))
        return query.permute(1, 2, 0)
