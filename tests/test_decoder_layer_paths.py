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
