"""groupfree/decoder_ops.py at the ends of its types' ranges, against float64: values of very different
sizes in one call, tails, signs of zero, elements next to the type's largest (decoder_ops_common.py has
the forms and their bounds)."""
import pytest
import torch

import decoder_ops_common as ref
from backtoreality_amd.groupfree import decoder_ops as ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)


def _leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def _attention_grads(q, k, v, dy, scale, lengths=None, mask=None):
    leaves = [_leaf(q), _leaf(k), _leaf(v)]
    out = ops.cross_attention(*leaves, key_lengths=lengths, key_padding_mask=mask, scale=scale)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, dy))


# --------------------------------------------------------------------- float16 attention gradients
@pytest.mark.parametrize("Lq,Lk,H,Hk,D", [(40, 16, 2, 1, 64), (3, 2, 1, 1, 64), (150, 300, 4, 2, 128),
                                          (5, 5000, 2, 1, 40)])
@pytest.mark.parametrize("pad", [False, True])
def test_float16_key_gradients_with_values_of_different_sizes(cuda, Lq, Lk, H, Hk, D, pad):
    """Keys whose values are 1, 2^-2 .. 2^-14 of the others' or nothing at all, dout along the result:
    dS of a small value's key is as large as the others' (its D comes from them).  The bound of dk is
    each term's rounding; a term that the type's smallest steps touch is 2^-39 of its key's largest
    at most, far below that one's half step."""
    gen = _gen(100 + Lk)
    B = 2
    q = _randn(gen, (B, Lq, H, D), torch.float16)
    k = _randn(gen, (B, Lk, Hk, D), torch.float16, 0.2)
    size = torch.pow(2.0, -2.0 * (torch.arange(Lk, device=cuda) % 9 - 1).clamp(min=0).float())
    size[torch.arange(Lk, device=cuda) % 9 == 8] = 0.0
    v = (_randn(gen, (B, Lk, Hk, D), torch.float32, 0.2, 1.0) * size[None, :, None, None]).half()
    dy = _randn(gen, (B, Lq, H, D), torch.float16, 0.2, 1.0)
    mask = None
    if pad:                       # what is padded has values beyond all others, and takes no part
        mask = torch.zeros((B, Lk), dtype=torch.bool, device=cuda)
        mask[:, 1::7] = True
        v = v.masked_fill(mask[:, :, None, None], 6e4)
    got = _attention_grads(q, k, v, dy, D ** -0.5, mask=mask)
    want = ref.cross_attention(q, k, v, None, mask, D ** -0.5, dy)
    for t, (name, value, bound) in zip(got, want):
        ref.close(name, t, value, bound)


@pytest.mark.parametrize("Lq,Lk,H,Hk,D", [(40, 24, 2, 1, 64), (2, 2, 1, 1, 8), (200, 130, 4, 2, 128),
                                          (7, 5000, 2, 1, 40)])
@pytest.mark.parametrize("size,even", [(256.0, True), (2e3, True), (1e2, False), (1e4, False)])
def test_float16_gradients_with_large_values(cuda, Lq, Lk, H, Hk, D, size, even):
    """|v| of 10^2 to 10^4, a gradient that makes dq and dk fit: even -- a key's value is +-size in
    every column, dout the same, so that no term of dP cancels -- or random."""
    gen = _gen(200 + Lk)
    B = 2
    q = _randn(gen, (B, Lq, H, D), torch.float16, 2.0 ** -5)
    k = _randn(gen, (B, Lk, Hk, D), torch.float16, 2.0 ** -5)
    if even:
        sign = (torch.rand((B, Lk, Hk, 1), generator=gen, device=cuda) < 0.5).float() * 2 - 1
        v = (sign * size).expand(B, Lk, Hk, D).half().contiguous()
        dy = torch.full((B, Lq, H, D), 0.01, device=cuda, dtype=torch.float16)
    else:
        v, dy = _randn(gen, (B, Lk, Hk, D), torch.float16, size), _randn(gen, (B, Lq, H, D), torch.float16, 0.01)
    want = ref.cross_attention(q, k, v, None, None, D ** -0.5, dy)
    assert all(float(value.abs().max()) < 3e4 for _, value, _ in want[1:])
    for t, (name, value, bound) in zip(_attention_grads(q, k, v, dy, D ** -0.5), want):
        ref.close(name, t, value, bound)


# -------------------------------------------------------------------------------------- activations
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("cols", [1, 70])        # straight from the long operand, and in tiles
def test_relu_with_and_without_a_residual_agree_on_what_is_on(cuda, dtype, cols):
    """NaN of either sign lets the gradient through, as torch's ReLU does; what counts as positive does
    not depend on a residual: a z that the type rounds to zero is off."""
    nan = torch.tensor([0x7fc0, 0xffc0 - 0x10000], dtype=torch.int16, device=cuda).view(torch.bfloat16)
    far = float("inf") if dtype != torch.float32 else 2.0      # (infinite float32: NaN, as documented)
    z = torch.cat([torch.tensor([1.0, -1.0, 0.0, -0.0, far, -far], device=cuda), nan.float()]).to(dtype)
    on = torch.tensor([1, 0, 0, 0, 1, 0, 1, 1], device=cuda, dtype=dtype)
    x = _leaf(z.repeat(40)[:, None])
    w, b = torch.ones((cols, 1), device=cuda, dtype=dtype), _leaf(torch.zeros(cols, device=cuda, dtype=dtype))
    small = 2.0 ** -13
    grads = []
    for residual in (None, torch.zeros((320, cols), device=cuda, dtype=dtype)):
        y = ops.linear(x, w, b, activation="relu", residual=residual)
        dx, db = torch.autograd.grad(y, [x, b], torch.ones_like(y))
        assert torch.equal(dx[:, 0], on.repeat(40) * cols)
        assert bool((db == 40 * on.sum()).all())
        # two factors of 2^-13: 2^-26, which float16 rounds to zero and the others keep
        t = _leaf(torch.full((320, 1), small, device=cuda, dtype=dtype))
        y = ops.linear(t, torch.full((cols, 1), small, device=cuda, dtype=dtype), activation="relu",
                       residual=residual)
        grads.append(torch.autograd.grad(y, [t], torch.ones_like(y))[0])
    assert torch.equal(grads[0], grads[1])
    assert bool((grads[0] == 0).all()) == (dtype == torch.float16)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("cols", [1, 70])
def test_gelu_gradient_in_the_tail(cuda, dtype, cols):
    """z in [-6, -4], slopes from 7e-4 to 4e-8: relative to each.  One term per row (W one column's
    unit): the slope's own arithmetic 2^-14 and, for 16 bits, its code's half step 2^-10, dz's rounding
    and the result's."""
    n = 1000
    z = torch.linspace(-6.0, -4.0, n, device=cuda).to(dtype)
    x = _leaf(z[:, None])
    w = torch.zeros((cols, 1), device=cuda, dtype=dtype)
    w[cols // 2] = 1
    dy = torch.full((n, cols), 2.0 ** 14, device=cuda, dtype=dtype)
    # (the other columns' z is 0: their slope of a half meets a weight of 0)
    (dx,) = torch.autograd.grad(ops.linear(x, w, activation="gelu"), [x], dy)
    want = ref.linear(x, w, None, "gelu", None, dy)[1][1]
    u = ref.half_step(dtype)
    rel = 2.0 ** -14 if dtype == torch.float32 else 2.0 ** -14 + 2.0 ** -10 + 2 * u
    ref.close("dx", dx, want, rel * want.abs() + ref.tiny(dtype))
    # beyond: exactly nothing
    x = _leaf(torch.tensor([[-20.0], [-40.0], [-300.0]], device=cuda, dtype=dtype))
    (dx,) = torch.autograd.grad(ops.linear(x, w, activation="gelu"), [x], dy[:3])
    assert not dx.any()


@pytest.mark.parametrize("m,k,n", [(100, 48, 96), (700, 130, 65), (5, 33, 7)])
@pytest.mark.parametrize("size,ws,xs", [(2.0 ** -13, 2.0 ** 9, 2.0 ** 9), (2.0 ** -20, 2.0 ** 13, 2.0 ** 13)])
def test_float16_gelu_gradients_use_their_range(cuda, m, k, n, size, ws, xs):
    """A small dy on slopes of 2^-5 and less: dz below float16's smallest normal value, weights and
    inputs that bring dx and dW back into the range.  Each term: the slope's relative error (2^-10 of its
    code, 2^-12 of its arithmetic and of z's sum), dz's rounding; the sums in float32."""
    gen = _gen(300 + m)
    f16, u = torch.float16, ref.half_step(torch.float16)
    # z is the bias: x's one column of inputs meets a column of zeros
    x, w = torch.zeros((m, k), device=cuda, dtype=f16), _randn(gen, (n, k), f16, ws)
    x[:, 0], w[:, 0] = _randn(gen, (m,), f16, xs), 0
    bias = -(torch.rand((n,), generator=gen, device=cuda) * 1.5 + 2.5).half()
    x, w, bias = _leaf(x), _leaf(w), _leaf(bias)
    dy = _randn(gen, (m, n), f16, size)
    y = ops.linear(x, w, bias, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, [x, w, bias], dy)
    z = x.double() @ w.double().t() + bias.double()
    cdf = torch.special.erfc(-z / 2 ** 0.5) / 2
    dz = dy.double() * (cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5)
    rel = u + 2.0 ** -10 + 2.0 ** -11
    e = rel * dz.abs()
    for name, got, want, bound in (("dx", dx, dz @ w.double(), e @ w.double().abs()),
                                   ("dw", dw, dz.t() @ x.double(), e.t() @ x.double().abs()),
                                   ("db", db, dz.sum(0), e.sum(0))):
        ref.close(name, got, want, 1.01 * bound + u * want.abs() + ref.tiny(f16))


# --------------------------------------------------------------------------- float32's largest elements
@pytest.mark.parametrize("m,k,n", [(3, 40, 50), (200, 40, 200), (300, 700, 20), (130, 64, 70)])
def test_float32_elements_above_the_largest_bfloat16(cuda, m, k, n):
    """Finite operands between bfloat16's largest value and float32's, small ones against them: every
    product finite and as exact as any other."""
    gen = _gen(400 + m)
    f32, top = torch.float32, torch.finfo(torch.float32).max
    big = torch.tensor([top, -top, top * (1 - 2.0 ** -9 + 2.0 ** -12), -top * (1 - 2.0 ** -12)], device=cuda)

    def sprinkle(t, every):
        t = t.clone()
        at = torch.arange(0, t.numel(), every, device=cuda)
        t.view(-1)[at] = big[torch.arange(len(at), device=cuda) % 4]
        return t
    x = _leaf(sprinkle(_randn(gen, (m, k), f32), 7 * k + 1))       # one of a row at most
    w = _leaf(_randn(gen, (n, k), f32, 2.0 ** -10))
    dy = _randn(gen, (m, n), f32, 2.0 ** -20)
    y = ops.linear(x, w)
    want = ref.linear(x, w, None, None, None, dy)
    for t, (name, value, bound) in zip([y] + list(torch.autograd.grad(y, [x, w], dy)), want):
        ref.close(name, t.detach(), value, bound)
    # ... in the weight
    x, w = _leaf(_randn(gen, (m, k), f32, 2.0 ** -10)), _leaf(sprinkle(_randn(gen, (n, k), f32), 7 * k + 1))
    y = ops.linear(x, w)
    want = ref.linear(x, w, None, None, None, dy)
    for t, (name, value, bound) in zip([y] + list(torch.autograd.grad(y, [x, w], dy)), want):
        ref.close(name, t.detach(), value, bound)
    # ... and in dy
    w, dy = _leaf(_randn(gen, (n, k), f32, 2.0 ** -10)), sprinkle(_randn(gen, (m, n), f32), 7 * n + 1)
    want = ref.linear(x, w, None, None, None, dy)[1:]
    for t, (name, value, bound) in zip(torch.autograd.grad(ops.linear(x, w), [x, w], dy), want):
        ref.close(name, t, value, bound)


# ------------------------------------------------------------------------- more than a grid has threads
def test_linear_of_more_rows_than_one_launch_has_room_for(cuda):
    """2^27 rows and a few, one input, one output: a power of two times each."""
    m = 2 ** 27 + 5
    x = torch.arange(m, device=cuda, dtype=torch.int32).remainder_(1021).float()[:, None]
    w, b = torch.full((1, 1), 0.5, device=cuda), torch.full((1,), 3.0, device=cuda)
    r = x.flip(0)
    y = ops.linear(x, w, b, residual=r)
    assert torch.equal(y, 0.5 * x + 3.0 + r)


def test_layer_norm_of_a_very_wide_row(cuda):
    """2^26 columns: their parameter gradients are more than one grid of 32 columns a workgroup."""
    n = 2 ** 26
    x = (torch.arange(n, device=cuda, dtype=torch.int32).remainder_(5).float() - 2).half()[None]
    w, b = _leaf(torch.ones(n, device=cuda, dtype=torch.float16)), _leaf(torch.zeros(n, device=cuda, dtype=torch.float16))
    dy = x.flip(1).contiguous()
    dw, db = torch.autograd.grad(ops.layer_norm(x, w, b), [w, b], dy)
    assert torch.equal(db, dy[0])
    xh = x.double() * (2.0 + 1e-5) ** -0.5       # (mean within 2^-24 of 0, mean square of 2)
    off = (dw.double() - (dy.double() * xh)[0]).abs()
    assert float(off.max()) <= 3 * 2.0 ** -11 + 1e-4
