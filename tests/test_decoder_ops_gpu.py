"""groupfree/decoder_ops.py (csrc/layer_norm.hip, linear.hip, cross_attention.hip) against float64,
element by element, within what the kernels' roundings can change (decoder_ops_common.py)."""
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


def _all_close(got, want):
    for (name, value, bound), t in zip(want, got):
        ref.close(name, t.detach(), value, bound)
    assert len(got) == len(want)


# ---------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("rows,width", [
    (1, 1), (1, 288), (5, 7), (1024, 288), (33, 256), (130, 511), (9, 513), (257, 1024), (3, 1025),
    (70, 2047), (18, 4095), (5, 8192), (3, 8193), (2, 20001), (2500, 64), (4099, 1100),
])
def test_layer_norm(cuda, rows, width, dtype):
    gen = _gen(rows * 10007 + width)
    x, r = (_leaf(_randn(gen, (rows, width), dtype, 2.0, 0.5)) for _ in range(2))
    w, b = _leaf(_randn(gen, (width,), dtype, 0.2, 1.0)), _leaf(_randn(gen, (width,), dtype))
    dy = _randn(gen, (rows, width), dtype)
    y = ops.layer_norm(x, w, b, residual=r)
    dx, dr, dw, db = torch.autograd.grad(y, [x, r, w, b], dy)
    assert torch.equal(dx, dr)
    want = ref.layer_norm(x, w, b, r, 1e-5, dy)
    _all_close([y, dx, dw, db], want)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("width", [96, 1155, 9001])
def test_layer_norm_without_parameters_and_on_slices(cuda, width, dtype):
    gen = _gen(width)
    base = _randn(gen, (3, 11, width + 5), dtype)
    x = _leaf(base[:, :, 3:3 + width])                           # rows at odd addresses
    dy = _randn(gen, (3, 11, width + 1), dtype)[:, :, 1:]
    y = ops.layer_norm(x, eps=1e-3)
    (dx,) = torch.autograd.grad(y, [x], dy)
    _all_close([y, dx], ref.layer_norm(x, None, None, None, 1e-3, dy)[:2])
    xt = _leaf(_randn(gen, (width, 11), dtype).t())              # the last axis not contiguous
    y = ops.layer_norm(xt)
    _all_close([y], ref.layer_norm(xt, None, None, None, 1e-5))


def test_layer_norm_of_a_large_offset_keeps_the_deviations(cuda):
    """Rows far from zero: the sum of squared deviations, not a difference of squares."""
    gen = _gen(1)
    x = _randn(gen, (64, 384), torch.float32, 0.01, 1000.0)
    _all_close([ops.layer_norm(x)], ref.layer_norm(x, None, None, None, 1e-5))


def test_layer_norm_of_nothing(cuda):
    x = torch.empty((0, 40), device=cuda, requires_grad=True)
    w = torch.ones(40, device=cuda, requires_grad=True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert y.shape == (0, 40) and dx.shape == (0, 40) and torch.equal(dw, torch.zeros_like(dw))


# ------------------------------------------------------------------------------------- linear
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 288, 864), (3, 17, 5), (64, 64, 64), (65, 63, 129), (16, 1000, 40), (17, 2048, 288),
    (200, 36, 2048), (1024, 288, 288), (129, 775, 301), (48, 4096, 96), (2, 5000, 3), (700, 9, 700),
    (2048, 512, 2304), (1000, 3375, 23), (333, 300, 16), (41, 1111, 64), (33, 600, 47), (64, 1030, 500),
    (31, 2048, 129), (4097, 40, 32), (300, 2049, 31),
])
@pytest.mark.parametrize("act,bias,residual", [(None, True, False), ("relu", True, True),
                                               ("relu", False, False), ("gelu", True, True)])
def test_linear(cuda, m, k, n, act, bias, residual, dtype):
    gen = _gen(m * 31 + k * 7 + n)
    x = _leaf(_randn(gen, (m, k), dtype))
    w = _leaf(_randn(gen, (n, k), dtype, k ** -0.5))
    b = _leaf(_randn(gen, (n,), dtype, 0.3)) if bias else None
    r = _leaf(_randn(gen, (m, n), dtype)) if residual else None
    dy = _randn(gen, (m, n), dtype)
    y = ops.linear(x, w, b, activation=act, residual=r)
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    _all_close([y] + list(grads), ref.linear(x, w, b, act, r, dy))


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_linear_on_slices(cuda, dtype):
    """Odd row strides and addresses of every operand, a (batch, length, width) input, a transposed
    weight."""
    gen = _gen(5)
    x = _leaf(_randn(gen, (4, 37, 83), dtype)[:, :, 2:81])
    w = _leaf(_randn(gen, (53, 90), dtype, 0.1)[:, 7:86])
    r = _leaf(_randn(gen, (4, 37, 60), dtype)[:, :, 1:54])
    dy = _randn(gen, (4, 37, 55), dtype)[:, :, 2:]
    y = ops.linear(x, w, residual=r, activation="gelu")
    _all_close([y] + list(torch.autograd.grad(y, [x, w, r], dy)),
               ref.linear(x, w, None, "gelu", r, dy))
    wt = _leaf(_randn(gen, (79, 53), dtype, 0.1).t())
    y = ops.linear(x, wt)
    _all_close([y] + list(torch.autograd.grad(y, [x, wt], dy)), ref.linear(x, wt, None, None, None, dy))


def test_linear_gradient_of_a_broadcast_output(cuda):
    """dy of stride zero, as sum() gives it."""
    gen = _gen(6)
    x, w = _leaf(_randn(gen, (33, 20), torch.float32)), _leaf(_randn(gen, (12, 20), torch.float32))
    ops.linear(x, w).sum().backward()
    want = ref.linear(x, w, None, None, None, torch.ones(33, 12, device=cuda))
    _all_close([x.grad, w.grad], want[1:])


def test_linear_of_nothing(cuda):
    x = torch.empty((0, 40), device=cuda, requires_grad=True)
    w, b = torch.ones((9, 40), device=cuda, requires_grad=True), torch.ones(9, device=cuda, requires_grad=True)
    y = ops.linear(x, w, b, activation="gelu")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert y.shape == (0, 9) and dx.shape == (0, 40)
    assert torch.equal(dw, torch.zeros_like(dw)) and torch.equal(db, torch.zeros_like(db))


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_linear_activations_at_the_ends(cuda, dtype):
    """The identity product hands z through: far tails, signed zeros, infinities."""
    z = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 3.0, -3.0, 9.0, -9.0, 40.0, -40.0, 1000.0, -1000.0],
                     device=cuda).to(dtype)
    one = torch.ones((1, 1), device=cuda, dtype=dtype)
    for act in ("relu", "gelu"):
        x = _leaf(z[:, None])
        y = ops.linear(x, one, activation=act)
        (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
        want = ref.linear(x, one, None, act, None, torch.ones_like(y))
        _all_close([y, dx], want[:2])
    if dtype != torch.float32:
        y = ops.linear(torch.tensor([[float("inf")], [float("-inf")], [float("nan")]], device=cuda,
                                    dtype=dtype), one, activation="gelu")[:, 0].tolist()
        assert y[0] == float("inf") and y[1] == 0.0 and y[2] != y[2]


# ---------------------------------------------------------------------------- cross-attention
def _attend(gen, B, Lq, Lk, H, Hk, D, dtype, lengths=None, mask=None, scale=None, train=True):
    q = _randn(gen, (B, Lq, H, D), dtype)
    kv = _randn(gen, (B, Lk, 2, Hk, D), dtype)
    k, v = kv[:, :, 0], kv[:, :, 1]
    if train:
        q, k, v = _leaf(q), _leaf(k), _leaf(v)
    out = ops.cross_attention(q, k, v, key_lengths=lengths, key_padding_mask=mask, scale=scale)
    s = D ** -0.5 if scale is None else scale
    if not train:
        _all_close([out], ref.cross_attention(q, k, v, lengths, mask, s))
        return
    dy = _randn(gen, (B, Lq, H, D), dtype)
    grads = torch.autograd.grad(out, [q, k, v], dy)
    _all_close([out] + list(grads), ref.cross_attention(q, k, v, lengths, mask, s, dy))


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [
    (1, 1, 1, 1, 1, 1), (2, 1, 77, 4, 2, 16), (1, 3, 2, 2, 1, 5), (4, 256, 256, 8, 8, 36),
    (2, 33, 1024, 8, 8, 36), (1, 32, 129, 3, 3, 64), (2, 31, 64, 6, 2, 32), (3, 65, 63, 4, 4, 80),
    (1, 130, 513, 4, 1, 96), (2, 128, 200, 2, 2, 128), (1, 7, 3001, 4, 2, 128), (1, 500, 40, 4, 2, 127),
    (1, 1, 5000, 8, 1, 72), (1, 1100, 300, 2, 1, 24), (8, 200, 260, 8, 4, 40), (1, 17, 1, 2, 2, 33),
])
def test_cross_attention(cuda, B, Lq, Lk, H, Hk, D, dtype):
    _attend(_gen(B + 3 * Lq + 5 * Lk + H + D), B, Lq, Lk, H, Hk, D, dtype)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
@pytest.mark.parametrize("Lq,H,Hk,D", [(1, 8, 2, 64), (40, 4, 4, 36), (200, 4, 2, 128)])
@pytest.mark.parametrize("pad", ["lengths", "mask", "both"])
def test_cross_attention_padding(cuda, Lq, H, Hk, D, pad, dtype):
    """Lengths of nothing, one, a tile's edge and everything; scattered masks that leave a batch
    entry one key, or none; padded rows that hold NaN and infinities."""
    gen = _gen(Lq + D)
    B, Lk = 6, 640
    lengths = mask = None
    if pad != "mask":
        lengths = torch.tensor([0, 1, 128, 639, 640, 301], dtype=torch.int32, device=cuda)
    if pad != "lengths":
        mask = torch.rand((B, Lk), generator=gen, device=cuda) < 0.4
        mask[2] = True
        mask[3] = True
        mask[3, 517] = False
        mask[4, :256] = True
    live = ref.live_keys(torch.empty((B, Lk)).to(cuda), lengths, mask)
    q = _randn(gen, (B, Lq, H, D), dtype)
    kv = _randn(gen, (B, Lk, 2, Hk, D), dtype)
    dy = _randn(gen, (B, Lq, H, D), dtype)
    results = []
    for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        t = kv.masked_fill(~live[:, :, None, None, None], fill)
        leaves = [_leaf(q), _leaf(t[:, :, 0]), _leaf(t[:, :, 1])]
        out = ops.cross_attention(*leaves, key_lengths=lengths, key_padding_mask=mask)
        results.append([out.detach()] + list(torch.autograd.grad(out, leaves, dy)))
    for other in results[1:]:          # what padding holds changes nothing
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    _all_close(results[0], ref.cross_attention(q, kv[:, :, 0], kv[:, :, 1], lengths, mask, D ** -0.5, dy))
    out, dq, dk, dv = results[0]
    empty = ~live.any(1)
    assert bool(empty.any()) and not out[empty].any() and not dq[empty].any()
    dead = ~live[:, :, None, None].expand_as(dk)
    assert not dk[dead].any() and not dv[dead].any()


@pytest.mark.parametrize("Lq,Lk,H,Hk,D", [(65, 4096, 2, 2, 64), (200, 9, 4, 2, 40), (7, 20000, 4, 1, 128)])
@pytest.mark.parametrize("size,qs,ks", [(2.0 ** -12, 2.0 ** -6, 2.0 ** 6), (2.0 ** -12, 2.0 ** 6, 2.0 ** -6),
                                        (1.0, 1.0, 1.0), (2.0 ** 12, 2.0 ** -12, 2.0 ** -12)])
def test_cross_attention_float16_backward_uses_its_range(cuda, Lq, Lk, H, Hk, D, size, qs, ks):
    """Even rows of many keys with a small gradient -- P and dS below float16's smallest normal value
    -- and rows of few keys with a large one, dS beyond its largest; q and k of sizes that bring dq or
    dk back into the type's range."""
    gen = _gen(Lk)
    q = _leaf(_randn(gen, (2, Lq, H, D), torch.float16, qs))
    k = _leaf(_randn(gen, (2, Lk, Hk, D), torch.float16, ks))
    v = _leaf(_randn(gen, (2, Lk, Hk, D), torch.float16, 8.0))
    dy = _randn(gen, (2, Lq, H, D), torch.float16, size)
    scale = 0.3 / D ** 0.5
    out = ops.cross_attention(q, k, v, scale=scale)
    grads = torch.autograd.grad(out, [q, k, v], dy)
    want = ref.cross_attention(q, k, v, None, None, scale, dy)
    _all_close([out] + list(grads), want)
    # as a whole: what three roundings (P or dS, D of a rounded out, the result) leave, and the
    # result's own smallest steps
    for got, (name, value, _) in zip(grads, want[1:]):
        far = (got.double() - value).norm() / (value.norm() + value.numel() ** 0.5 * 2.0 ** -14)
        assert torch.isfinite(got).all() and far <= 3 * ref.half_step(torch.float16), (name, float(far))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_cross_attention_lengths_out_of_range_are_clamped(cuda, dtype):
    gen = _gen(3)
    q, k = _randn(gen, (3, 5, 2, 32), dtype), _randn(gen, (3, 50, 2, 32), dtype)
    a = ops.cross_attention(q, k, k, key_lengths=torch.tensor([-7, 2 ** 31 - 1, 50], dtype=torch.int32, device=cuda))
    b = ops.cross_attention(q, k, k, key_lengths=torch.tensor([0, 50, 50], dtype=torch.int32, device=cuda))
    assert torch.equal(a, b) and not a[0].any()


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_cross_attention_strides(cuda, dtype):
    """Queries and keys out of wider buffers at odd addresses, (length, batch) order, expanded heads
    and batches, a last axis that is not contiguous, a strided mask."""
    gen = _gen(8)
    B, Lq, Lk, H, D = 2, 19, 150, 4, 44
    q = _randn(gen, (Lq, B, H * D + 3), dtype)[:, :, 3:].unflatten(2, (H, D)).transpose(0, 1)
    k = _randn(gen, (Lk, B, H, D + 1), dtype)[..., 1:].transpose(0, 1)
    v = _randn(gen, (B, Lk, D, H), dtype).transpose(2, 3)
    mask = (torch.rand((Lk, B), generator=gen, device=cuda) < 0.3).t()
    dy = _randn(gen, (B, Lq, D, H), dtype).transpose(2, 3)
    leaves = [_leaf(t) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, key_padding_mask=mask, scale=0.3)
    _all_close([out] + list(torch.autograd.grad(out, leaves, dy)),
               ref.cross_attention(q, k, v, None, mask, 0.3, dy))
    one = _leaf(_randn(gen, (1, Lk, 1, D), dtype))               # one set of keys for everybody
    shared = one.expand(B, Lk, H, D)
    out = ops.cross_attention(leaves[0], shared, shared)
    (g,) = torch.autograd.grad(out, [one], dy)
    want = ref.cross_attention(q, shared.detach(), shared.detach(), None, None, D ** -0.5, dy)
    total = (want[2][1] + want[3][1]).sum((0, 2), keepdim=True)
    # the sums over batch and heads are torch's, of rounded values: a rounding at each of 8 + 1
    bound = (want[2][2] + want[3][2]).sum((0, 2), keepdim=True) + 2 * B * H * ref.half_step(dtype) * (
        want[2][1].abs() + want[3][1].abs()).sum((0, 2), keepdim=True)
    ref.close("shared", g, total, bound)


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_cross_attention_sharp_and_flat_rows(cuda, dtype):
    """Scores of hundreds (one key takes everything, the maximum moves late) and all equal ones."""
    gen = _gen(9)
    q, k = _randn(gen, (1, 40, 2, 64), dtype, 8.0), _randn(gen, (1, 700, 2, 64), dtype, 2.0)
    k[:, 650] = q[:, 7]
    v = _randn(gen, (1, 700, 2, 64), dtype)
    dy = _randn(gen, (1, 40, 2, 64), dtype)
    for a, b in ((q, k), (torch.zeros_like(q), k)):
        leaves = [_leaf(t) for t in (a, b, v)]
        out = ops.cross_attention(*leaves, scale=1.0)
        _all_close([out] + list(torch.autograd.grad(out, leaves, dy)),
                   ref.cross_attention(a, b, v, None, None, 1.0, dy))


def test_cross_attention_nan_queries_stay_nan(cuda):
    for Lq, Lk in ((1, 4000), (1, 60), (200, 300)):
        q = torch.ones((1, Lq, 1, 32), device=cuda, dtype=torch.bfloat16)
        q[:, 0] = float("nan")
        k = torch.ones((1, Lk, 1, 32), device=cuda, dtype=torch.bfloat16)
        out = ops.cross_attention(q, k, k)
        assert bool(out[:, 0].isnan().all()) and bool((out[:, 1:] == 1).all())


def test_cross_attention_of_nothing(cuda):
    q = torch.randn((2, 3, 4, 16), device=cuda, requires_grad=True)
    none = torch.empty((2, 0, 4, 16), device=cuda, requires_grad=True)
    out = ops.cross_attention(q, none, none)
    dq, dk = torch.autograd.grad(out, [q, none], torch.ones_like(out))
    assert not out.any() and not dq.any() and dk.shape == none.shape
    k = torch.randn((2, 9, 4, 16), device=cuda, requires_grad=True)
    q0 = torch.empty((2, 0, 4, 16), device=cuda, requires_grad=True)
    out = ops.cross_attention(q0, k, k)
    dq, dk = torch.autograd.grad(out, [q0, k], torch.ones_like(out))
    assert out.shape == q0.shape and dq.shape == q0.shape and not dk.any()


def test_gradients_against_differences(cuda):
    """Directional derivatives of the forwards themselves, float32: central differences of step e
    are off by e^2 / 6 of the third derivative and by rounding / e."""
    gen = _gen(11)
    f32 = torch.float32
    mask = torch.rand((2, 70), generator=gen, device=cuda) < 0.3
    cases = [
        (lambda x, w, b, r: ops.layer_norm(x, w, b, residual=r),
         [(6, 40), (40,), (40,), (6, 40)]),
        (lambda x, w, b, r: ops.linear(x, w, b, activation="gelu", residual=r),
         [(9, 30), (21, 30), (21,), (9, 21)]),
        (lambda q, k, v: ops.cross_attention(q, k, v, key_padding_mask=mask),
         [(2, 9, 4, 20), (2, 70, 2, 20), (2, 70, 2, 20)]),
    ]
    for fn, shapes in cases:
        xs = [_leaf(_randn(gen, s, f32)) for s in shapes]
        ds = [_randn(gen, s, f32) for s in shapes]
        out = fn(*xs)
        w = _randn(gen, out.shape, f32)
        analytic = sum(float((g.double() * d.double()).sum())
                       for g, d in zip(torch.autograd.grad(out, xs, w), ds))
        e = 2.0 ** -8
        up, down = (float((fn(*[x.detach() + t * d for x, d in zip(xs, ds)]).double() * w.double()).sum())
                    for t in (e, -e))
        size = float((out.detach().double().abs() * w.double().abs()).sum())
        assert abs((up - down) / (2 * e) - analytic) <= 1e-3 * size, (analytic, (up - down) / (2 * e))


# -------------------------------------------------------------------- how a program calls them
def _three(gen, dtype, cuda):
    """A run of the three as a decoder layer uses them: inputs and a function of them."""
    B, Lq, Lk, H, D = 2, 50, 300, 4, 32
    E = H * D
    shapes = dict(x=(B, Lq, E), mem=(B, Lk, E), wq=(E, E), wkv=(2 * E, E), wo=(E, E), bo=(E,),
                  g1=(E,), b1=(E,), w1=(3 * E, E), c1=(3 * E,), w2=(E, 3 * E), c2=(E,))
    t = {n: _leaf(_randn(gen, s, dtype, 0.08 if len(s) == 2 else 1.0)) for n, s in shapes.items()}
    lengths = torch.tensor([211, 300], dtype=torch.int32, device=cuda)

    def run(t):
        q = ops.linear(t["x"], t["wq"]).unflatten(2, (H, D))
        kv = ops.linear(t["mem"], t["wkv"]).unflatten(2, (2, H, D))
        a = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], key_lengths=lengths).flatten(2)
        h = ops.layer_norm(ops.linear(a, t["wo"], t["bo"], residual=t["x"]), t["g1"], t["b1"])
        f = ops.linear(h, t["w1"], t["c1"], activation="gelu")
        return ops.layer_norm(ops.linear(f, t["w2"], t["c2"]), t["g1"], t["b1"], residual=h)
    return t, run


def _plain_three(t, run_dtype=torch.float64):
    import torch.nn.functional as nnf
    t = {n: v.detach().to(run_dtype).requires_grad_(True) for n, v in t.items()}
    B, Lq, E = t["x"].shape
    H, D = 4, 32
    q = (t["x"] @ t["wq"].t()).unflatten(2, (H, D)).transpose(1, 2)
    kv = (t["mem"] @ t["wkv"].t()).unflatten(2, (2, H, D))
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    s = q @ k.transpose(-1, -2) * D ** -0.5
    gone = torch.arange(s.shape[-1], device=s.device)[None] >= torch.tensor([211, 300], device=s.device)[:, None]
    a = (torch.softmax(s.masked_fill(gone[:, None, None], float("-inf")), -1) @ v).transpose(1, 2).flatten(2)
    h = nnf.layer_norm(a @ t["wo"].t() + t["bo"] + t["x"], (E,), t["g1"], t["b1"])
    f = nnf.gelu(h @ t["w1"].t() + t["c1"])
    return t, nnf.layer_norm(f @ t["w2"].t() + t["c2"] + h, (E,), t["g1"], t["b1"])


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_a_run_of_the_three(cuda, dtype):
    """Nine calls in a row.  Each rounds its result and, going back, its gradients; each rounding
    reaches the end changed in size by the operators between, which here (norms of unit rows,
    products of weights of norm about one) is a factor of a few: 30 half steps, root mean square,
    against the float64 run; float32 sums carry up to a few hundred f."""
    t, run = _three(_gen(12), dtype, cuda)
    out = run(t)
    dy = _randn(_gen(13), out.shape, dtype)
    grads = torch.autograd.grad(out, list(t.values()), dy)
    t64, want = _plain_three(t)
    grads64 = torch.autograd.grad(want, list(t64.values()), dy.double())
    for name, a, b in zip(["out"] + list(t), [out] + list(grads), [want] + list(grads64)):
        err = float((a.double() - b).pow(2).mean().sqrt() / b.pow(2).mean().sqrt())
        assert err <= 30 * max(ref.half_step(dtype), 2.0 ** -24), (name, err)


def test_same_results_every_time_and_on_another_stream(cuda):
    t, run = _three(_gen(14), torch.bfloat16, cuda)
    dy = _randn(_gen(15), (2, 50, 128), torch.bfloat16)

    def once():
        out = run(t)
        return [out] + list(torch.autograd.grad(out, list(t.values()), dy))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_forward_and_backward_replay(cuda):
    """One graph with the whole run and its gradients, replayed on new inputs with eager work
    between, every replay against the eager result."""
    t, run = _three(_gen(16), torch.float16, cuda)
    dy = _randn(_gen(17), (2, 50, 128), torch.float16)

    def once():
        out = run(t)
        return [out] + list(torch.autograd.grad(out, list(t.values()), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for i in range(4):
        with torch.no_grad():
            t["x"].copy_(_randn(_gen(20 + i), t["x"].shape, torch.float16))
            t["mem"].copy_(_randn(_gen(30 + i), t["mem"].shape, torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        for a, b in zip(got, once()):
            assert torch.equal(a, b)


def test_only_the_gradients_asked_for(cuda):
    gen = _gen(18)
    x, w, b = (_randn(gen, s, torch.float32) for s in ((20, 16), (8, 16), (8,)))
    full = [_leaf(t) for t in (x, w, b)]
    want = torch.autograd.grad(ops.linear(*full, activation="gelu").sum(), full)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        ops.linear(*some, activation="gelu").sum().backward()
        for j in range(3):
            assert (some[j].grad is None) == (j != i)
        assert torch.equal(some[i].grad, want[i])
    with torch.no_grad():
        assert not ops.linear(*full).requires_grad


def test_double_backward_is_refused(cuda):
    x = torch.randn((4, 8), device=cuda, requires_grad=True)
    (g,) = torch.autograd.grad(ops.layer_norm(x).pow(2).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


# ------------------------------------------------------------------------ the decoder layer on them
def _layer(cuda, dtype, activation="relu", E=96, heads=4, posembed=True):
    import torch.nn as nn
    from backtoreality_amd.groupfree.transformer import TransformerDecoderLayer
    torch.manual_seed(3)

    class Position(nn.Module):        # (B, P, 3) -> (B, E, P)
        def __init__(self):
            super().__init__()
            self.map = nn.Linear(3, E)

        def forward(self, xyz):
            return self.map(xyz).transpose(1, 2)
    layer = TransformerDecoderLayer(E, heads, 4 * E, 0.0, activation,
                                    self_posembed=Position() if posembed else None,
                                    cross_posembed=Position() if posembed else None)
    with torch.no_grad():
        for p in layer.parameters():
            if p.dim() == 1:
                p.add_(torch.randn(p.shape) * 0.1)
    return layer.to(cuda).to(dtype)


def _layer_inputs(cuda, dtype, E=96):
    gen = _gen(21)
    B, Pq, Pk = 3, 70, 260
    mask = torch.rand((B, Pk), generator=gen, device=cuda) < 0.3
    mask[1, 100:] = True
    return (_randn(gen, (B, E, Pq), dtype), _randn(gen, (B, E, Pk), dtype),
            _randn(gen, (B, Pq, 3), dtype), _randn(gen, (B, Pk, 3), dtype), mask,
            _randn(gen, (B, E, Pq), dtype))


@pytest.mark.parametrize("activation", ["relu", "gelu"])
@pytest.mark.parametrize("masked", [True, False])
@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_decoder_layer_on_the_operators(cuda, dtype, masked, activation, monkeypatch):
    """TransformerDecoderLayer in every type, with and without padded keys, against the stock modules
    in float64 on the CPU: output, input gradients and parameter gradients, root mean square.  Eight
    roundings forward and as many back reach each result, amplified a few times: 60 half steps
    (ReLU's switches next to zero included), as in the run of the three above."""
    import copy
    from backtoreality_amd.groupfree import decoder_ops
    layer = _layer(cuda, dtype, activation)
    q, k, qpos, kpos, mask, dy = _layer_inputs(cuda, dtype)
    if not masked:
        mask = None
    calls = []
    real = decoder_ops.cross_attention
    monkeypatch.setattr(decoder_ops, "cross_attention",
                        lambda *a, **kw: calls.append(1) or real(*a, **kw))
    q, k = _leaf(q), _leaf(k)
    out = layer(q, k, qpos, kpos, key_padding_mask=mask)
    # (unpadded float32 has the whole-layer call)
    assert len(calls) == (0 if dtype == torch.float32 and not masked else 2)
    params = list(layer.parameters())
    grads = torch.autograd.grad(out, [q, k] + params, dy)
    cpu = copy.deepcopy(layer).cpu().double()
    q64, k64 = (t.detach().cpu().double().requires_grad_(True) for t in (q, k))
    want = cpu(q64, k64, qpos.cpu().double(), kpos.cpu().double(),
               key_padding_mask=None if mask is None else mask.cpu())
    grads64 = torch.autograd.grad(want, [q64, k64] + list(cpu.parameters()), dy.cpu().double())
    names = ["out", "query", "key"] + [n for n, _ in layer.named_parameters()]
    step = max(ref.half_step(dtype), 2.0 ** -22)
    for name, a, b in zip(names, [out] + list(grads), [want] + list(grads64)):
        err = float((a.detach().cpu().double() - b.detach()).pow(2).mean().sqrt())
        assert err <= 60 * step * float(b.detach().pow(2).mean().sqrt()) + 1e-9, (name, err)


def test_decoder_layer_ignores_what_padding_holds(cuda):
    layer = _layer(cuda, torch.bfloat16)
    q, k, qpos, kpos, mask, _ = _layer_inputs(cuda, torch.bfloat16)
    mask[2] = True                                            # a scene without keys
    with torch.no_grad():
        a = layer(q, k, qpos, kpos, key_padding_mask=mask)
        b = layer(q, k.masked_fill(mask[:, None], float("nan")), qpos, kpos, key_padding_mask=mask)
    assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


def test_decoder_layer_with_attention_dropout_keeps_the_stock_core(cuda, monkeypatch):
    """Dropout on the attention weights is not the operator's: a padded training call goes through
    nn.MultiheadAttention, the same layer in eval mode through the operators."""
    from backtoreality_amd.groupfree import decoder_ops
    layer = _layer(cuda, torch.float32)
    layer.self_attn.dropout = layer.multihead_attn.dropout = 0.1
    q, k, qpos, kpos, mask, _ = _layer_inputs(cuda, torch.float32)
    calls = []
    real = decoder_ops.cross_attention
    monkeypatch.setattr(decoder_ops, "cross_attention",
                        lambda *a, **kw: calls.append(1) or real(*a, **kw))
    layer.train()
    layer(q, k, qpos, kpos, key_padding_mask=mask)
    assert not calls
    layer.eval()
    layer(q, k, qpos, kpos, key_padding_mask=mask)
    assert len(calls) == 2


def test_decoder_layer_of_several_types_stays_with_the_stock_modules(cuda):
    """Under autocast, and with norms of another type, types are chosen module by module: not the
    operators' calls.  (The choice only: the stock modules' attention multiplies batches of bfloat16 by
    a transposed view, which has faulted the GPU in torch's library call.)"""
    layer = _layer(cuda, torch.bfloat16).eval()
    q, k, _, _, mask, _ = _layer_inputs(cuda, torch.bfloat16)
    assert layer._ops_covered(q, k, mask) and layer._ops_covered(q, k, None)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert not layer._ops_covered(q, k, mask) and not layer._ops_covered(q, k, None)
    layer.norm3.float()
    assert not layer._ops_covered(q, k, mask)


# ------------------------------------------------------------------------------------- the edges
def test_refusals(cuda):
    """Wrong types, shapes and devices: RuntimeError, nothing launched."""
    f = lambda *s, dtype=torch.float32: torch.zeros(s, device=cuda, dtype=dtype)
    x, w = f(4, 8), f(3, 8)
    q, k = f(2, 3, 4, 16), f(2, 5, 2, 16)
    bad = [
        lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, f(7)),
        lambda: ops.layer_norm(x, f(8, dtype=torch.bfloat16)), lambda: ops.layer_norm(x, f(8).cpu()),
        lambda: ops.layer_norm(x, residual=f(4, 7)), lambda: ops.layer_norm(x, eps=-1.0),
        lambda: ops.layer_norm(f(4, 0)), lambda: ops.layer_norm(f()), lambda: ops.layer_norm(x, f(1, 8)),
        lambda: ops.linear(x, f(3, 7)), lambda: ops.linear(x, f(8)), lambda: ops.linear(x, w.half()),
        lambda: ops.linear(x, w, f(4)), lambda: ops.linear(x, w, activation="glu"),
        lambda: ops.linear(x, w, residual=f(3, 4)), lambda: ops.linear(x, w, residual=f(4, 3).cpu()),
        lambda: ops.linear(x, f(0, 8)), lambda: ops.linear(x.long(), w),
        lambda: ops.cross_attention(q, k, f(2, 6, 2, 16)), lambda: ops.cross_attention(q[0], k, k),
        lambda: ops.cross_attention(q, f(2, 5, 3, 16), f(2, 5, 3, 16)),
        lambda: ops.cross_attention(q, f(1, 5, 2, 16), f(1, 5, 2, 16)),
        lambda: ops.cross_attention(f(1, 1, 1, 129), f(1, 1, 1, 129), f(1, 1, 1, 129)),
        lambda: ops.cross_attention(f(1, 1, 258, 8), f(1, 1, 2, 8), f(1, 1, 2, 8)),
        lambda: ops.cross_attention(q, k.half(), k.half()),
        lambda: ops.cross_attention(q, k, k, key_lengths=torch.zeros(2, device=cuda, dtype=torch.int64)),
        lambda: ops.cross_attention(q, k, k, key_lengths=torch.zeros(2, dtype=torch.int32)),
        lambda: ops.cross_attention(q, k, k, key_lengths=torch.zeros(3, device=cuda, dtype=torch.int32)),
        lambda: ops.cross_attention(q, k, k, key_padding_mask=f(2, 5)),
        lambda: ops.cross_attention(q, k, k, key_padding_mask=f(2, 4).bool()),
        lambda: ops.cross_attention(q, k, k, scale=0.0),
        lambda: ops.cross_attention(q, k, k, scale=float("nan")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("call %d was not refused" % i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_offsets_beyond_32_bits(cuda, dtype):
    """Rows so far apart that the last ones start behind element 2^31: the same bits as from a compact
    copy."""
    apart, n, D = 1 << 16, 34000, 64
    wide = torch.empty((n, apart), device=cuda, dtype=dtype)      # (only the columns below are touched)
    gen = _gen(31)
    kv = _randn(gen, (n, 2 * D), dtype)
    wide[:, :2 * D] = kv
    q, dy = _randn(gen, (1, 40, 1, D), dtype), _randn(gen, (1, 40, 1, D), dtype)
    lengths = torch.tensor([n - 3], dtype=torch.int32, device=cuda)
    res = []
    for src in (wide[:, :2 * D], kv):
        k, v = (_leaf(src[:, i * D:(i + 1) * D][None, :, None]) for i in (0, 1))
        out = ops.cross_attention(q, k, v, key_lengths=lengths)
        res.append([out] + list(torch.autograd.grad(out, [k, v], dy)))
        one = ops.cross_attention(q[:, :1], k.detach(), v.detach(), key_lengths=lengths)
        x, w = _leaf(src), _leaf(_randn(_gen(32), (24, 2 * D), dtype))
        y = ops.linear(x, w, activation="relu")
        res[-1] += [one, y] + list(torch.autograd.grad(y, [x, w], torch.ones_like(y)))
        y = ops.layer_norm(x)
        res[-1] += [y, torch.autograd.grad(y, [x], src)[0]]
    for i, (a, b) in enumerate(zip(*res)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("dtype", ref.DTYPES, ids=str)
def test_one_tensor_in_several_places(cuda, dtype):
    """The same leaf as input and residual, as query, key and value, as input and weight: gradients
    add up."""
    gen = _gen(33)
    x = _leaf(_randn(gen, (24, 24), dtype))
    dy = _randn(gen, (24, 24), dtype)
    u = ref.half_step(dtype)
    two = lambda want, i, j: (want[i][1] + want[j][1], want[i][2] + want[j][2] + 2 * u * (
        want[i][1].abs() + want[j][1].abs()))                     # torch adds the rounded two
    y = ops.layer_norm(x, residual=x)
    (g,) = torch.autograd.grad(y, [x], dy)
    ref.close("norm", g, *two(ref.layer_norm(x, None, None, x, 1e-5, dy), 1, 1))
    y = ops.linear(x, x)
    (g,) = torch.autograd.grad(y, [x], dy)
    ref.close("linear", g, *two(ref.linear(x, x, None, None, None, dy), 1, 2))
    s = _leaf(_randn(gen, (2, 40, 3, 16), dtype))
    dy = _randn(gen, (2, 40, 3, 16), dtype)
    out = ops.cross_attention(s, s, s)
    (g,) = torch.autograd.grad(out, [s], dy)
    want = ref.cross_attention(s, s, s, None, None, 0.25, dy)
    total = sum(w[1] for w in want[1:])
    ref.close("attention", g, total, sum(w[2] for w in want[1:]) + 4 * u * sum(w[1].abs() for w in want[1:]))


def test_gradients_beside_a_living_graph_of_the_same_leaves(cuda):
    """Two forwards of the same leaves alive at once, taken back in either order."""
    t, run = _three(_gen(34), torch.bfloat16, cuda)
    dy = _randn(_gen(35), (2, 50, 128), torch.bfloat16)
    a, b = run(t), run(t)
    gb = torch.autograd.grad(b, list(t.values()), dy)
    ga = torch.autograd.grad(a, list(t.values()), dy)
    for x, y in zip(ga, gb):
        assert torch.equal(x, y)


def test_a_result_changed_in_place_is_noticed(cuda):
    """ReLU's backward reads the result: autograd refuses if it was overwritten."""
    x, w = torch.randn((8, 8), device=cuda, requires_grad=True), torch.randn((8, 8), device=cuda)
    y = ops.linear(x, w, activation="relu")
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
