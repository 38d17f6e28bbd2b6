"""Which path a TransformerDecoderLayer call takes (groupfree/transformer.py, fused_attention.py,
fused_decoder.py): host decisions, looked at without a GPU through tensors that say they are on one."""
import pytest
import torch

from backtoreality_amd.groupfree import fused_attention, fused_decoder
from backtoreality_amd.groupfree.transformer import TransformerDecoderLayer


class OnGpu(torch.Tensor):
    is_cuda = True


def _on_gpu(*shape, dtype=torch.float32):
    return torch.randn(shape).to(dtype).as_subclass(OnGpu)


@pytest.fixture
def autocast():
    """CUDA autocast to bfloat16, which torch.autocast turns off where there is no GPU."""
    torch.set_autocast_dtype("cuda", torch.bfloat16)
    yield lambda on: torch.set_autocast_enabled("cuda", on)
    torch.set_autocast_enabled("cuda", False)
    torch.set_autocast_dtype("cuda", torch.float16)


# -------------------------------------------------- the float32 kernels get nothing but float32
def test_fused_attention_covers_float32_throughout_only(autocast):
    """The projections' results are what the kernels read, four bytes an element."""
    mha = torch.nn.MultiheadAttention(64, 2)
    q, k = _on_gpu(5, 2, 64), _on_gpu(9, 2, 64)
    assert fused_attention._covered(mha, q, k)
    autocast(True)
    assert not fused_attention._covered(mha, q, k)
    autocast(False)
    assert not fused_attention._covered(mha, q, _on_gpu(9, 2, 64, dtype=torch.bfloat16))
    assert not fused_attention._covered(torch.nn.MultiheadAttention(64, 2).bfloat16(), q, k)
    mha.out_proj.half()
    assert not fused_attention._covered(mha, q, k)


def test_fused_attention_core_refuses_16_bit_projections():
    for q, kv in ((torch.zeros(4, 2, 192, dtype=torch.bfloat16), None),
                  (torch.zeros(4, 2, 64), torch.zeros(6, 2, 128, dtype=torch.float16))):
        with pytest.raises(RuntimeError, match="float32"):
            fused_attention._AttentionCore.apply(q, kv, 2, 0.0, 0)


def test_fused_decoder_covers_float32_parameters_only():
    query, key = _on_gpu(2, 64, 5), _on_gpu(2, 64, 9)
    assert fused_decoder.covered(TransformerDecoderLayer(64, 2, 128, 0.0), query, key, None, None)
    for name in ("linear1", "norm2", "self_attn", "multihead_attn"):
        layer = TransformerDecoderLayer(64, 2, 128, 0.0)
        getattr(layer, name).bfloat16()
        assert not fused_decoder.covered(layer, query, key, None, None), name


def test_decoder_stack_refuses_a_converted_detector():
    """The checks kept with a detector are not made again: parameters of another type are seen where
    their pointers are."""
    import types
    from backtoreality_amd.groupfree import fused_stack
    params = [torch.zeros(4), None, torch.zeros(4, dtype=torch.bfloat16)]
    det, ent = types.SimpleNamespace(num_decoder_layers=0), types.SimpleNamespace(ptrs=None, d=None)
    with pytest.raises(RuntimeError, match="float32"):
        fused_stack._set_pointers(ent, det, [], params, [])


# ------------------------------------------------------- torch's attention in bfloat16 on the GPU
class NoBfloat16Batches(torch.utils._python_dispatch.TorchDispatchMode):
    """Batched products of bfloat16, by any name, are an error; counts the others."""

    def __init__(self):
        super().__init__()
        self.batches = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if any(n in func.name() for n in ("bmm", "attention")):
            self.batches += 1
            assert not any(isinstance(a, torch.Tensor) and a.dtype == torch.bfloat16 for a in args), func
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("how", ["layer", "autocast"])
def test_bfloat16_attention_of_the_modules_runs_in_float32(how, masked, autocast, monkeypatch):
    """Dropout on the attention weights, autocast: the module's attention, forward and backward, without
    a batched product of bfloat16."""
    torch.manual_seed(0)
    layer = TransformerDecoderLayer(32, 4, 64, 0.1).train()
    dtype = torch.float32
    if how == "layer":
        layer, dtype = layer.bfloat16(), torch.bfloat16
    query, key = (_on_gpu(2, 32, n, dtype=dtype).requires_grad_(True) for n in (5, 9))
    mask = torch.zeros((2, 9), dtype=torch.bool)
    mask[:, 6:] = True
    autocast(how == "autocast")
    monkeypatch.setenv("BTR_FUSED_DECODER", "0")     # (the whole-layer call takes float32 as it is)
    with NoBfloat16Batches() as seen:
        out = layer(query, key, None, None, key_padding_mask=mask if masked else None)
        assert out.dtype == dtype
        out.sum().backward()
    assert seen.batches >= 8
    assert all(p.grad is not None and p.grad.dtype == p.dtype for p in layer.parameters())
    assert query.grad is not None and key.grad is not None


def test_bfloat16_attention_keeps_the_module_and_its_result():
    """The module's own forward and hooks; the float32 result rounded once."""
    torch.manual_seed(1)
    from backtoreality_amd.groupfree.transformer import _stock_attention
    mha = torch.nn.MultiheadAttention(32, 4).bfloat16()
    seen = []
    mha.register_forward_hook(lambda m, args, out: seen.append(args[0].dtype))
    q, k = _on_gpu(5, 2, 32, dtype=torch.bfloat16), _on_gpu(7, 2, 32, dtype=torch.bfloat16)
    mask = torch.zeros((2, 7), dtype=torch.bool)
    mask[1, 3:] = True
    got = _stock_attention(mha, q, k, mask)
    assert seen == [torch.float32] and got.dtype == torch.bfloat16
    assert all(p.dtype == torch.bfloat16 for p in mha.parameters())
    wide = torch.nn.MultiheadAttention(32, 4).double()
    wide.load_state_dict(mha.state_dict())
    q64, k64 = (t.as_subclass(torch.Tensor).double() for t in (q, k))
    want = wide(q64, k64, k64, key_padding_mask=mask)[0]
    # float32 sums of some 32 terms, then half a step of bfloat16
    off = (got.as_subclass(torch.Tensor).double() - want).abs()
    assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all())


# ----------------------------------------------- the operators replace nothing but the stock modules
def _covered(layer, dtype=torch.bfloat16, mask=True):
    mask = torch.zeros((2, 9), dtype=torch.bool) if mask else None
    return layer._ops_covered(_on_gpu(2, 32, 5, dtype=dtype), _on_gpu(2, 32, 9, dtype=dtype), mask)


def _plain_layer(dtype=torch.bfloat16):
    return TransformerDecoderLayer(32, 4, 64, 0.0).to(dtype)


class AddingLinear(torch.nn.Linear):
    def forward(self, x):
        return super().forward(x) + 100


def test_operators_take_the_stock_modules():
    for dtype in (torch.bfloat16, torch.float16):
        assert _covered(_plain_layer(dtype), dtype) and _covered(_plain_layer(dtype), dtype, mask=False)
    assert _covered(_plain_layer(torch.float32), torch.float32)
    assert not _covered(_plain_layer(torch.float32), torch.float32, mask=False)
    layer = _plain_layer()
    layer.norm2 = torch.nn.LayerNorm(32, elementwise_affine=False)
    layer.linear1 = torch.nn.Linear(32, 64, bias=False).bfloat16()
    assert _covered(layer)


def _hooked(register):
    return lambda m: getattr(m, register)(lambda *a: None)


@pytest.mark.parametrize("change", [
    _hooked("register_forward_hook"), _hooked("register_forward_pre_hook"),
    _hooked("register_full_backward_hook"), _hooked("register_full_backward_pre_hook"),
    lambda m: setattr(m, "forward", lambda *a, **k: None),
], ids=["hook", "pre", "backward", "backward_pre", "forward"])
@pytest.mark.parametrize("name", ["linear1", "linear2", "norm1", "norm2", "norm3", "self_attn",
                                  "multihead_attn"])
def test_operators_leave_changed_modules_alone(name, change):
    layer = _plain_layer()
    change(getattr(layer, name))
    assert not _covered(layer) and not _covered(layer, mask=False)


@pytest.mark.parametrize("name,make", [
    ("linear1", lambda: AddingLinear(32, 64)),
    ("linear2", lambda: torch.nn.Sequential(torch.nn.Linear(64, 32))),
    ("linear1", lambda: torch.nn.utils.parametrizations.weight_norm(torch.nn.Linear(32, 64))),
    ("linear2", lambda: torch.nn.utils.prune.l1_unstructured(torch.nn.Linear(64, 32), "weight", 0.5)),
    ("linear1", lambda: torch.nn.utils.spectral_norm(torch.nn.Linear(32, 64))),
    ("norm1", torch.nn.Identity), ("norm3", lambda: torch.nn.RMSNorm(32)),
    ("norm2", lambda: torch.nn.LayerNorm((5, 32))),
    ("self_attn", lambda: type("Own", (torch.nn.MultiheadAttention,), {})(32, 4)),
])
def test_operators_leave_other_modules_alone(name, make):
    import torch.nn.utils.prune  # noqa: F401
    layer = _plain_layer()
    setattr(layer, name, make().bfloat16())
    assert not _covered(layer) and not _covered(layer, mask=False)


def test_operators_stay_out_of_global_hooks():
    layer = _plain_layer()
    handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        assert not _covered(layer)
    finally:
        handle.remove()
    assert _covered(layer)


# ------------------------------------------------------------------ what the operators cannot derive
def test_operators_stay_out_of_transformed_calls(monkeypatch):
    """Forward mode, torch.func, tracing: the modules, whose operations torch knows; and by the switch."""
    import torch.autograd.forward_ad as forward_ad
    layer = _plain_layer()
    assert _covered(layer)
    with forward_ad.dual_level():
        assert not _covered(layer)
    seen = []

    def look(x):
        seen.append(_covered(layer))
        return x * 2
    torch.func.vmap(look, randomness="same")(torch.ones(3))
    torch.jit.trace(look, torch.ones(3), check_trace=False)
    assert seen == [False, False] and _covered(layer)
    monkeypatch.setenv("BTR_FUSED_DECODER", "0")
    assert not _covered(layer)


@pytest.fixture
def calls_on_the_cpu(monkeypatch):
    """The operators with their kernels left out: results of zeros."""
    from backtoreality_amd.groupfree import decoder_ops
    real = torch.empty
    monkeypatch.setattr(decoder_ops, "_launch", lambda *a: None)
    monkeypatch.setattr(decoder_ops, "_check_ref", lambda *a: None)
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: real(*a, **kw).zero_())
    return {"layer_norm": lambda x: decoder_ops.layer_norm(x),
            "linear": lambda x: decoder_ops.linear(x, torch.ones(3, 8)),
            "cross_attention": lambda x: decoder_ops.cross_attention(*[x.view(1, 4, 1, 8)] * 3)}


@pytest.mark.parametrize("name", ["layer_norm", "linear", "cross_attention"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(calls_on_the_cpu, name, grad):
    """A dual tensor without requires_grad: an error, not a result without its tangent."""
    import torch.autograd.forward_ad as forward_ad
    fn, x = calls_on_the_cpu[name], torch.randn(4, 8)
    with torch.set_grad_enabled(grad):
        assert not fn(x).requires_grad
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="jvp"):
                fn(forward_ad.make_dual(x, torch.ones_like(x)))
            assert not fn(x).any()               # no dual among its inputs: an ordinary call
        with pytest.raises(RuntimeError):
            torch.func.jvp(fn, (x,), (x,))


@pytest.mark.parametrize("name", ["layer_norm", "linear", "cross_attention"])
@pytest.mark.parametrize("grad", [True, False])
def test_a_trace_records_the_call(calls_on_the_cpu, name, grad):
    """... and not the allocation of its result as the result."""
    with torch.set_grad_enabled(grad):
        graph = torch.jit.trace(calls_on_the_cpu[name], torch.randn(4, 8), check_trace=False).graph
    kinds = [n.kind() for n in graph.nodes()]
    assert "prim::PythonOp" in kinds and "aten::empty" not in kinds, kinds


def test_lengths_and_masks_that_are_no_tensors_are_refused(calls_on_the_cpu):
    from backtoreality_amd.groupfree import decoder_ops
    x = torch.randn(1, 4, 1, 8)
    for kw in (dict(key_lengths=[4]), dict(key_padding_mask=[[False] * 4])):
        with pytest.raises(RuntimeError, match="should be"):
            decoder_ops.cross_attention(x, x, x, **kw)
