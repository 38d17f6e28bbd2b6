"""The decoder operators of `backtoreality_amd.groupfree.decoder_ops`, timed one pass at a time.

Three operators that a transformer decoder layer is made of:

    layer_norm       y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias,  s = x [+ residual]
    linear           y = act(x weight^T + bias) [+ residual],  act = identity, ReLU or GELU (erf)
    cross_attention  softmax(scale q k^T) v per head onto keys of another length, some of them
                     padding; several query heads may share one key / value head

each forward only ("infer") or forward with every gradient ("train").  With `own` false `run`
computes them from elementary torch operations in float32, rounded once at the end; with `own`
true it calls the library's operators.  `exact` evaluates the definitions and the gradients'
closed forms in float64.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5


# ------------------------------------------------------------------------------------- cases
def listed():
    """The timed cases; 288 channels, 8 heads of 36, 2048 hidden, 4 scenes of 256 queries and 1024
    seed points are GroupFree3D's decoder, the others are generic transformer sizes."""
    return [
        # one decoder layer's post-attention norm in its training step: the smallest call
        dict(name="norm_decoder_f32", op="norm", rows=1024, width=288, dtype="f32", residual=True,
             strided=False, train=True),
        # a long batch of wide tokens: as much as the memory carries
        dict(name="norm_tokens_bf16", op="norm", rows=32768, width=2048, dtype="bf16",
             residual=True, strided=False, train=True),
        # inference on a slice of a wider buffer, odd width: no row starts on an aligned address
        dict(name="norm_odd_f16", op="norm", rows=5003, width=1155, dtype="f16", residual=False,
             strided=True, train=False),
        # one token through an output projection while answering: the weight's bytes are the time
        dict(name="linear_token_bf16", op="linear", rows=1, inner=4096, outer=4096, dtype="bf16",
             act="none", bias=True, residual=True, train=False),
        # the decoder's first feed-forward product, training in float32
        dict(name="linear_decoder_f32", op="linear", rows=1024, inner=288, outer=2048,
             dtype="f32", act="relu", bias=True, residual=False, train=True),
        # a feed-forward product over a long batch: matrix cores
        dict(name="linear_tokens_bf16", op="linear", rows=16384, inner=1024, outer=4096,
             dtype="bf16", act="gelu", bias=True, residual=False, train=True),
        # nothing a multiple of anything
        dict(name="linear_odd_f16", op="linear", rows=1999, inner=775, outer=1301, dtype="f16",
             act="relu", bias=True, residual=True, train=True),
        # decoder cross-attention onto padded seed points, training in float32
        dict(name="attend_decoder_f32", op="attend", batch=4, queries=256, keys=1024, heads=8,
             kv_heads=8, dim=36, dtype="f32", pad="mask", train=True),
        # one new token against long encoder states of several lengths
        dict(name="attend_token_bf16", op="attend", batch=8, queries=1, keys=32768, heads=32,
             kv_heads=8, dim=128, dtype="bf16", pad="lengths", train=False),
        # a training batch of ragged encoder states
        dict(name="attend_batch_bf16", op="attend", batch=4, queries=2048, keys=4096, heads=16,
             kv_heads=16, dim=64, dtype="bf16", pad="lengths", train=True),
        # odd lengths, shared heads, scattered padding and one batch entry with no key left
        dict(name="attend_odd_f16", op="attend", batch=3, queries=333, keys=1777, heads=12,
             kv_heads=4, dim=80, dtype="f16", pad="empty", train=True),
        # a long document read by a long prompt: the largest
        dict(name="attend_long_bf16", op="attend", batch=2, queries=4096, keys=16384, heads=16,
             kv_heads=4, dim=128, dtype="bf16", pad="none", train=False),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["norm", "linear", "attend", "attend"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    if op == "norm":
        return dict(op=op, rows=_spread(rng, 1, 32768), width=_spread(rng, 17, 8192), dtype=dtype,
                    residual=rng.random() < 0.5, strided=rng.random() < 0.3, train=train)
    if op == "linear":
        return dict(op=op, rows=_spread(rng, 1, 16384), inner=_spread(rng, 17, 8192),
                    outer=_spread(rng, 17, 8192), dtype=dtype,
                    act=rng.choice(["none", "relu", "gelu"]), bias=rng.random() < 0.8,
                    residual=rng.random() < 0.5, train=train)
    kv_heads = rng.choice([1, 2, 4, 8])
    return dict(op=op, batch=rng.choice([1, 2, 3, 4, 8]),
                queries=1 if rng.random() < 0.2 else _spread(rng, 2, 4096),
                keys=_spread(rng, 1, 32768), heads=kv_heads * rng.choice([1, 1, 2, 4]),
                kv_heads=kv_heads, dim=rng.choice([16, 32, 36, 40, 64, 72, 80, 96, 128]),
                dtype=dtype, pad=rng.choice(["none", "lengths", "mask", "empty"]), train=train)


def draw(rng):
    """One more case of the same ranges, no larger than the largest listed one."""
    while True:
        case = _draw_once(rng)
        if work(case)["flops"] <= (2e11 if case["dtype"] == "f32" else 4e11) and \
                work(case)["bytes"] <= 1e9 and \
                (case["op"] != "attend" or
                 case["batch"] * case["heads"] * case["queries"] * case["keys"] <= 6e8):
            return case


def _key_counts(case):
    """Keys left of every batch entry, in an order that the seed shuffles."""
    b, n = case["batch"], case["keys"]
    if case["pad"] == "lengths":       # from a quarter to all of them
        return [max(1, n - (3 * n * i) // (4 * max(b - 1, 1))) for i in range(b)]
    if case["pad"] == "mask":          # an eighth is padding
        return [n - n // 8] * b
    if case["pad"] == "empty":         # the same, and one entry with none
        return [n - n // 8] * (b - 1) + [0]
    return [n] * b


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    train = case["train"]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        moved = rows * width * (2 + case["residual"])       # x, residual, y
        if train:
            moved += rows * width * 2 + 2 * width           # dy, the one gradient of x + residual
        return {"bytes": size * (moved + 2 * width), "flops": rows * width * (20 if train else 8)}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        once = m * k + n * k + n * case["bias"]
        moved = once + m * n * (1 + case["residual"])
        if train:
            moved += once + m * n                           # dx, dweight, dbias; dy
        return {"bytes": size * moved, "flops": 2 * m * n * k * (3 if train else 1)}
    q_elems = case["batch"] * case["queries"] * case["heads"] * case["dim"]
    kv_row = 2 * case["kv_heads"] * case["dim"]
    left = sum(_key_counts(case))
    moved = 2 * q_elems + left * kv_row                     # q, out, k and v
    if train:                                               # dout, dq; dk and dv whole
        moved += 2 * q_elems + case["batch"] * case["keys"] * kv_row
    pairs = case["queries"] * left * case["heads"] * case["dim"]
    return {"bytes": size * moved, "flops": pairs * (14 if train else 4)}


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype, train = _TYPES[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale + shift).to(dtype)

    state = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # hidden states: a spread of two around an offset
        x = normal(rows, width + 5 if case["strided"] else width, scale=2.0, shift=0.5)
        state["x"] = x[:, 3:3 + width] if case["strided"] else x
        state["residual"] = normal(rows, width) if case["residual"] else None
        state["weight"] = normal(width, scale=0.2, shift=1.0)
        state["bias"] = normal(width, scale=0.2)
        leaves, shape = ["x", "residual", "weight", "bias"], (rows, width)
    elif case["op"] == "linear":
        m, k, n = case["rows"], case["inner"], case["outer"]
        state["x"] = normal(m, k)
        state["weight"] = normal(n, k, scale=k ** -0.5)
        state["bias"] = normal(n, scale=0.2) if case["bias"] else None
        state["residual"] = normal(m, n) if case["residual"] else None
        leaves, shape = ["x", "weight", "bias", "residual"], (m, n)
    else:
        b, lq, lk, d = case["batch"], case["queries"], case["keys"], case["dim"]
        state["query"] = normal(b, lq, case["heads"], d)
        kv = normal(b, lk, 2, case["kv_heads"], d)          # one packed projection
        state["key"], state["value"] = kv[:, :, 0], kv[:, :, 1]
        counts = torch.tensor(_key_counts(case), device=dev)
        counts = counts[torch.randperm(b, generator=gen, device=dev)]
        state["lengths"] = state["mask"] = None
        if case["pad"] == "lengths":
            state["lengths"] = counts.to(torch.int32)
        elif case["pad"] != "none":                         # True: padding
            order = torch.rand((b, lk), generator=gen, device=dev).argsort(1).argsort(1)
            state["mask"] = order >= counts[:, None]
        leaves, shape = ["query", "key", "value"], (b, lq, case["heads"], d)
    leaves = [name for name in leaves if state[name] is not None]
    state["leaves"] = leaves if train else None
    if train:
        state["grad"] = normal(*shape)
        for name in leaves:
            state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------- plain
def _plain_norm(st):
    s = st["x"].float()
    if st["residual"] is not None:
        s = s + st["residual"].float()
    c = s - s.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    return (c * r * st["weight"].float() + st["bias"].float()).to(st["x"].dtype)


def _plain_linear(st):
    act = st["case"]["act"]
    z = st["x"].float() @ st["weight"].float().t()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    if act == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "gelu":
        z = z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if st["residual"] is not None:
        z = z + st["residual"].float()
    return z.to(st["x"].dtype)


def _plain_attend(st):
    q, k, v = st["query"], st["key"], st["value"]
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    g = h // hk
    # query heads that share a key head are rows of one product
    qs = q.float().view(b, lq, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * lq, d)
    ks = k.float().permute(0, 2, 3, 1).contiguous()
    vs = v.float().permute(0, 2, 1, 3).contiguous()
    s = (qs @ ks) * d ** -0.5
    gone = st["mask"]
    if st["lengths"] is not None:
        gone = torch.arange(lk, device=q.device)[None] >= st["lengths"][:, None]
    if gone is not None:
        s = s.masked_fill(gone[:, None, None, :], float("-inf"))
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = (p @ vs).view(b, hk, g, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)
    return out.to(q.dtype)


# ------------------------------------------------------------------------------------- own
def _own_norm(st):
    from backtoreality_amd.groupfree import decoder_ops
    return decoder_ops.layer_norm(st["x"], st["weight"], st["bias"], residual=st["residual"],
                                  eps=_EPS)


def _own_linear(st):
    from backtoreality_amd.groupfree import decoder_ops
    act = st["case"]["act"]
    return decoder_ops.linear(st["x"], st["weight"], st["bias"],
                              activation=None if act == "none" else act, residual=st["residual"])


def _own_attend(st):
    from backtoreality_amd.groupfree import decoder_ops
    return decoder_ops.cross_attention(st["query"], st["key"], st["value"],
                                       key_lengths=st["lengths"], key_padding_mask=st["mask"])


def run(state):
    """One pass: [y], or [y, a gradient for every input] of a training case."""
    forms = {"norm": (_plain_norm, _own_norm), "linear": (_plain_linear, _own_linear),
             "attend": (_plain_attend, _own_attend)}
    y = forms[state["case"]["op"]][own](state)
    if state["leaves"] is None:
        return [y]
    grads = torch.autograd.grad(y, [state[name] for name in state["leaves"]], state["grad"])
    return [y.detach()] + list(grads)


# ------------------------------------------------------------------------------------- exact
def _exact_norm(st, dy):
    x = st["x"].double()
    s = x if st["residual"] is None else x + st["residual"].double()
    n = s.shape[1]
    var, mean = torch.var_mean(s, 1, unbiased=False, keepdim=True)
    inv = (var + _EPS) ** -0.5
    xhat = (s - mean) * inv
    w = st["weight"].double()
    y = xhat * w + st["bias"].double()
    if dy is None:
        return [y]
    t = dy * w
    dx = inv * (t - t.sum(1, keepdim=True) / n - xhat * ((t * xhat).sum(1, keepdim=True) / n))
    return [y, dx] + ([dx] if st["residual"] is not None else []) + [(dy * xhat).sum(0), dy.sum(0)]


def _exact_linear(st, dy):
    act = st["case"]["act"]
    x, w = st["x"].double(), st["weight"].double()
    z = torch.mm(x, w.t())
    if st["bias"] is not None:
        z += st["bias"].double()
    if act == "relu":
        a, slope = z.clamp(min=0), (z > 0).double()
    elif act == "gelu":
        cdf = torch.special.erfc(-z / math.sqrt(2)) / 2
        a, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        a, slope = z, torch.ones_like(z)
    y = a if st["residual"] is None else a + st["residual"].double()
    if dy is None:
        return [y]
    dz = dy * slope
    out = [y, torch.mm(dz, w), torch.mm(dz.t(), x)]
    if st["bias"] is not None:
        out.append(dz.sum(0))
    if st["residual"] is not None:
        out.append(dy)
    return out


def _exact_attend(st, dy):
    q, k, v = st["query"], st["key"], st["value"]
    b, lq, h, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d)
    y = torch.zeros((b, lq, h, d), dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(y), None, None
    if dy is not None:
        dk = torch.zeros((b, lk, hk, d), dtype=torch.float64, device=q.device)
        dv = torch.zeros_like(dk)
    for i in range(b):
        if st["lengths"] is not None:
            live = torch.arange(int(st["lengths"][i]), device=q.device)
        elif st["mask"] is not None:
            live = torch.nonzero(~st["mask"][i]).flatten()
        else:
            live = torch.arange(lk, device=q.device)
        if live.numel() == 0:
            continue
        for j in range(h):                     # only the keys that are left take part
            g = j // (h // hk)
            qm = q[i, :, j].double()
            km, vm = k[i, live, g].double(), v[i, live, g].double()
            p = torch.softmax(scale * (qm @ km.t()), dim=1)
            y[i, :, j] = p @ vm
            if dy is None:
                continue
            g_out = dy[i, :, j]
            dv[i, live, g] = dv[i, live, g] + p.t() @ g_out
            ds = p * (g_out @ vm.t() - (g_out * y[i, :, j]).sum(1, keepdim=True)) * scale
            dq[i, :, j] = ds @ km
            dk[i, live, g] = dk[i, live, g] + ds.t() @ qm
    return [y] if dy is None else [y, dq, dk, dv]


def exact(case, seed):
    """What `run` returns, from the definitions and the gradients' closed forms in float64."""
    st = prepare(case, seed)
    dy = st["grad"].double() if case["train"] else None
    with torch.no_grad():
        form = {"norm": _exact_norm, "linear": _exact_linear, "attend": _exact_attend}[case["op"]]
        return form(st, dy)
