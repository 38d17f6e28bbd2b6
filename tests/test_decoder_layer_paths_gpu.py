"""TransformerDecoderLayer calls that the operators of groupfree/decoder_ops.py do not take: through the
layer's modules."""
import copy

import pytest
import torch

from backtoreality_amd.groupfree.transformer import TransformerDecoderLayer

pytestmark = pytest.mark.gpu


def _inputs(cuda, dtype, E=64):
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)
    mask = torch.rand((2, 90), generator=gen, device="cuda") < 0.3
    return r(2, E, 40), r(2, E, 90), mask, r(2, E, 40)


def _layer(cuda, dtype, dropout=0.0, activation="gelu"):
    torch.manual_seed(4)
    return TransformerDecoderLayer(64, 2, 128, dropout, activation).to(cuda).to(dtype)


def _near_float64(layer, q, k, mask, out, grads, dy, step):
    """Eight roundings forward and as many back, amplified a few times, root mean square."""
    cpu = copy.deepcopy(layer).cpu().double()
    q64, k64 = (t.detach().cpu().double().requires_grad_(True) for t in (q, k))
    want = cpu(q64, k64, None, None, key_padding_mask=None if mask is None else mask.cpu())
    grads64 = torch.autograd.grad(want, [q64, k64] + list(cpu.parameters()), dy.cpu().double())
    for a, b in zip([out] + list(grads), [want] + list(grads64)):
        a, b = a.detach().cpu().double(), b.detach()
        assert float((a - b).pow(2).mean().sqrt()) <= 60 * step * float(b.pow(2).mean().sqrt()) + 1e-9


@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("weights", [torch.float32, torch.bfloat16], ids=str)
def test_decoder_layer_under_bfloat16_autocast(cuda, weights, masked):
    """Float32 and bfloat16 layers, with and without padding: attention in float32, everything else in
    the types autocast chooses."""
    layer = _layer(cuda, weights)
    q, k, mask, dy = _inputs(cuda, weights)
    q, k = q.requires_grad_(True), k.requires_grad_(True)
    mask = mask if masked else None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = layer(q, k, None, None, key_padding_mask=mask)
    grads = torch.autograd.grad(out, [q, k] + list(layer.parameters()), dy.to(out.dtype))
    _near_float64(layer, q, k, mask, out, grads, dy, 2.0 ** -8)


@pytest.mark.parametrize("masked", [True, False])
def test_bfloat16_layer_trains_with_dropout(cuda, masked):
    """Dropout on the attention weights, the layer's default: finite, the same again under the same
    seed, and without the dropout near float64."""
    layer = _layer(cuda, torch.bfloat16, dropout=0.1, activation="relu").train()
    q, k, mask, dy = _inputs(cuda, torch.bfloat16)
    q, k = q.requires_grad_(True), k.requires_grad_(True)
    mask = mask if masked else None
    runs = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        out = layer(q, k, None, None, key_padding_mask=mask)
        assert out.dtype == torch.bfloat16
        runs.append([out] + list(torch.autograd.grad(out, [q, k] + list(layer.parameters()), dy)))
        assert all(bool(torch.isfinite(t).all()) for t in runs[-1])
    assert torch.equal(runs[0][0], runs[1][0])
    assert not torch.equal(runs[0][0], runs[2][0])
    for m in layer.modules():       # the attention's own dropout alone, next to nothing: the modules' path
        if isinstance(m, torch.nn.Dropout):
            m.p = 0.0
    layer.self_attn.dropout = layer.multihead_attn.dropout = 1e-7
    out = layer(q, k, None, None, key_padding_mask=mask)
    grads = torch.autograd.grad(out, [q, k] + list(layer.parameters()), dy)
    _near_float64(layer.eval(), q, k, mask, out, grads, dy, 2.0 ** -8)


def test_a_trace_of_the_operators_runs(cuda):
    """torch.jit.trace without gradients: the traced function computes, on other inputs too."""
    from backtoreality_amd.groupfree import decoder_ops
    w, b = torch.randn(24, 16, device=cuda), torch.randn(24, device=cuda)
    x = torch.randn(5, 16, device=cuda)
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: decoder_ops.layer_norm(decoder_ops.linear(t, w, b, "relu")), x,
                                 check_trace=False)
        for _ in range(2):
            assert torch.equal(traced(x), decoder_ops.layer_norm(decoder_ops.linear(x, w, b, "relu")))
            x = torch.randn(5, 16, device=cuda)
