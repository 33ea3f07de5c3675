"""Timed cases of what surrounds the packed products of a decoder: the norm in front of them, the gated feed-forward
block, the head's loss, and the gradients through frozen codes.

A packed matrix is two-byte codes into 8-wide centroids (a second plane of codes, two bytes or one, adds a second
centroid) and a scale for each row; its activations come rotated (a permutation, signs and a Hadamard transform in
blocks).  Sizes are those of the 2048-wide model of the benchmark (6144 inside its feed-forward block at 4 bits a
weight, 151,936 tokens at 2) and other, odd ones.

A case is a dict.  ``kind``
"norm": ``tokens``, ``n``, ``dtype``, ``residual`` (added first), ``zero`` (weights hold their distance from 1), ``hb`` (rotation's
block, 0: none), ``bits`` (16, or 8: whole numbers under a scale for each row), ``grad`` (the backward pass instead);
"gated": ``tokens``, ``n``, ``rows``, ``dtype``, ``stages`` (1: 16-bit codes, 2: two planes of them, 3: 16- and 8-bit codes), ``act``,
``bits`` (of the activation rows), ``grad`` (forward and backward), ``scales`` (with the row scales' gradients);
"product": the backward pass of a packed product, ``tokens``, ``n``, ``rows``, ``dtype``, ``stages``, ``scales``;
"loss": ``tokens``, ``n``, ``rows`` (the vocabulary), ``dtype``, ``stages``, ``grad`` (forward and backward), ``scales``.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HIDDEN, INNER, VOCAB = 2048, 6144, 151936
EPS = 1e-6
IGNORE = -100

def _norm(tokens, n, dtype, residual=True, zero=False, hb=0, bits=16, grad=False, **more):
    return dict(more, kind="norm", tokens=tokens, n=n, dtype=dtype, residual=residual, zero=zero, hb=hb, bits=bits, grad=grad)

def _gated(tokens, n, rows, dtype, stages=1, act="silu", bits=16, grad=False, scales=False, **more):
    return dict(more, kind="gated", tokens=tokens, n=n, rows=rows, dtype=dtype, stages=stages, act=act, bits=bits,
                grad=grad, scales=scales)

def _product(tokens, n, rows, dtype, stages=1, scales=False, **more):
    return dict(more, kind="product", tokens=tokens, n=n, rows=rows, dtype=dtype, stages=stages, scales=scales)

def _loss(tokens, n, rows, dtype, stages=1, grad=False, scales=False, **more):
    return dict(more, kind="loss", tokens=tokens, n=n, rows=rows, dtype=dtype, stages=stages, grad=grad, scales=scales)

def listed():
    return [
        # one decoded token in front of its projections: latency
        _norm(1, HIDDEN, "bf16", hb=HIDDEN, name="norm_t1"),
        # a prompt's chunk, rotated and handed on in 8 bits
        _norm(1000, HIDDEN, "fp16", zero=True, hb=HIDDEN, bits=8, name="norm_t1000_8bit"),
        # a batch of prompts through a layer's norm, not rotated
        _norm(16384, HIDDEN, "bf16", name="norm_t16384"),
        # a training step's norm inside the feed-forward block, rotated in three blocks
        _norm(8192, INNER, "bf16", hb=2048, grad=True, name="norm_t8192_grad"),
        # one decoded token through the feed-forward block
        _gated(1, HIDDEN, INNER, "bf16", stages=2, name="gated_t1"),
        # a prompt of odd length through a shared expert of odd width, its rows in 8 bits
        _gated(333, HIDDEN, 1000, "fp16", bits=8, name="gated_t333_8bit"),
        # a training step of the feed-forward block
        _gated(4096, HIDDEN, INNER, "bf16", stages=2, grad=True, name="gated_t4096_grad"),
        # adapters tuned on one short document: the gradient through the o projection
        _product(200, HIDDEN, HIDDEN, "fp16", name="product_t200_grad"),
        # a training step through the down projection, its row scales tuned too
        _product(4096, INNER, HIDDEN, "bf16", stages=2, scales=True, name="product_t4096_grad"),
        # the log-likelihood of one given token
        _loss(1, HIDDEN, VOCAB, "fp16", name="loss_t1"),
        # scoring the continuations of a question over a vocabulary of odd size
        _loss(96, HIDDEN, 50257, "bf16", name="loss_t96"),
        # a training step's loss, the head's row scales tuned too
        _loss(4096, HIDDEN, VOCAB, "bf16", grad=True, scales=True, name="loss_t4096_grad"),
    ]

def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

def draw(rng):
    dtype = rng.choice(["fp16", "bf16"])
    kind = rng.choice(["norm", "gated", "product", "loss"])
    n = 64 * _log_int(rng, 4, 32)
    stages = rng.choice([1, 1, 2, 3])
    if kind == "norm":
        n = rng.choice([64 * _log_int(rng, 1, 128), _log_int(rng, 100, 8192)])
        hb = 0 if n % 64 or rng.random() < 0.4 else min(2048, n & -n)
        grad = rng.random() < 0.4
        return _norm(_log_int(rng, 1, max(1, 16384 * HIDDEN // n)), n, rng.choice([dtype, "fp32"]) if grad else dtype,
                     rng.random() < 0.7, rng.random() < 0.4, hb, 16 if grad else rng.choice([16, 16, 8]), grad)
    grad = rng.random() < 0.5
    scales = grad and rng.random() < 0.5
    if kind == "gated":
        return _gated(_log_int(rng, 1, 4096), n, _log_int(rng, 64, INNER), dtype, stages, rng.choice(["silu", "gelu_tanh"]),
                      16 if grad else rng.choice([16, 16, 8]), grad, scales)
    if kind == "product":
        return _product(_log_int(rng, 1, 4096), rng.choice([n, 3 * n]), _log_int(rng, 64, HIDDEN), dtype, stages, scales or rng.random() < 0.3)
    return _loss(_log_int(rng, 1, 4096), n, _log_int(rng, 1000, VOCAB // (2 if stages > 1 else 1)), dtype, stages, grad, scales)

# ------------------------------------------------------------------ inputs
def _matrix(case, g, rows):
    """one packed matrix: its planes of codes and its row scales"""
    groups = case["n"] // 8
    i0 = torch.randint(-32768, 32768, (rows, groups), generator=g, device=DEV, dtype=torch.int32).to(torch.int16)
    i1 = None
    if case["stages"] == 2:
        i1 = torch.randint(-32768, 32768, (rows, groups), generator=g, device=DEV, dtype=torch.int32).to(torch.int16)
    elif case["stages"] == 3:
        i1 = torch.randint(0, 256, (rows, groups), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    # scales that bring a row's product with unit activations near the size it has in a trained model
    scale = (torch.rand(rows, generator=g, device=DEV) + 0.5) * math.sqrt(8.0 / case["n"])
    return i0, i1, scale.to(torch.float32 if case.get("scales") else torch.bfloat16)

def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1009 + 41)
    T, n, dt = case["tokens"], case["n"], TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["kind"] == "norm":
        weight = randn(n) * 0.1 + (0.0 if case["zero"] else 1.0)
        # a residual stream has some channels far larger than the others
        wide = 1.0 + 20.0 * (torch.rand(n, generator=g, device=DEV) < 0.01)
        inp = {"x": randn(T, n).to(dt), "weight": weight.to(dt), "residual": None}
        if case["residual"]:
            inp["residual"] = (randn(T, n) * wide).to(dt)
        if case["grad"]:
            inp = {"h": (randn(T, n) * wide).to(dt), "weight": weight.to(dt), "dy": (randn(T, n) * 1e-3).to(dt),
                   "dh": (randn(T, n) * 1e-3).to(dt) if case["residual"] else None}
        if case["hb"]:
            inp["perm"] = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
            inp["sign"] = (torch.randint(0, 2, (n,), generator=g, device=DEV) * 2 - 1).to(torch.int8)
            H = torch.ones(1, 1, device=DEV)
            while H.shape[0] < case["hb"]:
                H = torch.cat([torch.cat([H, H], 1), torch.cat([H, -H], 1)], 0)
            inp["H"] = H
        return inp
    inp = {"cb0": (randn(65536, 8) * 8.0 ** -0.5).to(torch.float16), "cb1": None}
    if case["stages"] > 1:  # the second stage holds what the first leaves
        inp["cb1"] = (randn(65536 if case["stages"] == 2 else 256, 8) * 0.1).to(torch.float16)
    inp["x"], inp["x_scale"] = randn(T, n).to(dt), None
    if case.get("bits") == 8:
        top = inp["x"].float().abs().amax(1)
        inp["x_scale"] = top / 127.0
        inp["x"] = torch.round(inp["x"].float() / inp["x_scale"][:, None]).to(torch.int8)
    if case["kind"] == "gated":
        inp["gate"], inp["up"] = _matrix(case, g, case["rows"]), _matrix(case, g, case["rows"])
        if case["grad"]:
            inp["dact"] = (randn(T, case["rows"]) * 1e-3).to(dt)
    elif case["kind"] == "product":
        inp["matrix"] = _matrix(case, g, case["rows"])
        inp["dy"] = (randn(T, case["rows"]) * 1e-3).to(dt)
    else:
        inp["matrix"] = _matrix(case, g, case["rows"])
        inp["x"] = (inp["x"].float() * 2.5).to(dt)
        # tokens by a power law; the prompt's own tokens, a quarter, are not trained on
        inp["targets"] = (case["rows"] ** torch.rand(T, generator=g, device=DEV, dtype=torch.float64)).long() - 1
        if case["grad"]:
            skip = torch.rand(T, generator=g, device=DEV) < 0.25
            inp["targets"] = torch.where(skip, torch.full_like(inp["targets"], IGNORE), inp["targets"])
            inp["dloss"] = (~skip).float() / (~skip).sum().clamp(min=1)
    return inp

def prepare(case, seed):
    return dict(case=case, inp=_inputs(case, seed))

# ------------------------------------------------------- the operators' plain forms
def _plain_weights(inp, matrix):
    """[rows, n] without the row scales, in 32 bits"""
    i0, i1, _ = matrix
    w = inp["cb0"].float()[i0.long() & 0xFFFF]
    if i1 is not None:
        w = w + inp["cb1"].float()[i1.long() & (0xFF if i1.dtype == torch.uint8 else 0xFFFF)]
    return w.view(i0.shape[0], -1)

def _plain_rotate(inp, y):
    H = inp["H"]
    y = y[:, inp["perm"].long()] * inp["sign"].float()
    return (y.view(-1, H.shape[0]) @ H).view(y.shape) * H.shape[0] ** -0.5

def _plain_norm(case, inp):
    dt = inp["x"].dtype
    h = inp["x"].float()
    if inp["residual"] is not None:
        h = h + inp["residual"].float()
    w = inp["weight"].float() + (1.0 if case["zero"] else 0.0)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w
    if case["hb"]:
        y = _plain_rotate(inp, y)
    h = h.to(dt)
    if case["bits"] == 16:
        return {"y": y.to(dt), "h": h}
    scale = y.abs().amax(-1, keepdim=True) / 127.0
    q = torch.where(scale > 0, torch.round(y / scale), 0.0)
    return {"y": (q * scale).to(dt), "scale": scale.view(-1), "h": h}

def _plain_norm_grad(case, inp):
    h, dy = inp["h"].float(), inp["dy"].float()
    if case["hb"]:
        H = inp["H"]
        g = (dy.view(-1, H.shape[0]) @ H).view(dy.shape) * (H.shape[0] ** -0.5 * inp["sign"].float())
        dy = torch.empty_like(g).index_copy_(1, inp["perm"].long(), g)
    w = inp["weight"].float() + (1.0 if case["zero"] else 0.0)
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    dw = (dy * h * r).sum(0)
    g = dy * w
    dx = r * g - h * (r * r * r * (g * h).mean(-1, keepdim=True))
    if inp["dh"] is not None:
        dx = dx + inp["dh"].float()
    return {"dx": dx.to(inp["h"].dtype), "dweight": dw}

def _plain_rows(inp):
    x = inp["x"].float()
    return x if inp["x_scale"] is None else x * inp["x_scale"][:, None]

def _plain_act(case, g):
    """the activation and its derivative"""
    if case["act"] == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)

def _plain_gated(case, inp):
    x = _plain_rows(inp)
    wg, wu = _plain_weights(inp, inp["gate"]), _plain_weights(inp, inp["up"])
    sg, su = inp["gate"][2].float(), inp["up"][2].float()
    rg, ru = x @ wg.t(), x @ wu.t()
    a, da = _plain_act(case, rg * sg)
    out_dt = TYPES[case["dtype"]]
    out = {"act": (a * (ru * su)).to(out_dt)}
    if case["grad"]:
        d = inp["dact"].float()
        dg, du = d * (ru * su) * da, d * a
        out["dx"] = ((dg * sg) @ wg + (du * su) @ wu).to(out_dt)
        if case["scales"]:
            out["dgate"], out["dup"] = (dg * rg).sum(0), (du * ru).sum(0)
    return out

def _plain_product(case, inp):
    w, s, dy = _plain_weights(inp, inp["matrix"]), inp["matrix"][2].float(), inp["dy"].float()
    out = {"dx": ((dy * s) @ w).to(inp["x"].dtype)}
    if case["scales"]:
        out["dscale"] = (dy * (inp["x"].float() @ w.t())).sum(0)
    return out

def _plain_loss(case, inp):
    x, t, s = inp["x"].float(), inp["targets"], inp["matrix"][2].float()
    w = _plain_weights(inp, inp["matrix"])
    raw = x @ w.t()
    logits = raw * s
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).view(-1)
    at = t.clamp(min=0).view(-1, 1)
    used = t != IGNORE
    out = {"loss": torch.where(used, lse - logits.gather(1, at).view(-1), 0.0), "lse": lse}
    if case["grad"]:
        d = (e / total).scatter_add_(1, at, torch.full_like(lse, -1.0).view(-1, 1))
        d = d * torch.where(used, inp["dloss"], 0.0).view(-1, 1)
        out["dx"] = ((d * s) @ w).to(inp["x"].dtype)
        if case["scales"]:
            out["dscale"] = (d * raw).sum(0)
    return out

# ------------------------------------------------------- the framework's calls
def _rotation(case, inp):
    return dict(perm=inp["perm"], sign=inp["sign"], hb=case["hb"]) if case["hb"] else {}

def _own_norm(case, inp):
    from compressai_amd import kernels as K

    y, h, scale = K.vq_add_rms_norm(inp["x"], inp["weight"], inp["residual"], eps=EPS, zero_centred=case["zero"],
                                    out_dtype=torch.int8 if case["bits"] == 8 else None, **_rotation(case, inp))
    if case["bits"] == 16:
        return {"y": y, "h": h}
    return {"y": (y * scale[:, None]).to(inp["x"].dtype), "scale": scale, "h": h}

def _own_norm_grad(case, inp):
    from compressai_amd import kernels as K

    dx, dweight = K.vq_add_rms_norm_backward(inp["dy"], inp["h"], inp["weight"], inp["dh"], eps=EPS,
                                             zero_centred=case["zero"], **_rotation(case, inp))
    return {"dx": dx, "dweight": dweight}

def _own_gated(case, inp):
    from compressai_amd import kernels as K

    args = (inp["gate"], inp["up"], inp["cb0"], inp["cb1"], case["n"])
    out = {"act": K.vq_gated_rows(inp["x"], *args, activation=case["act"], x_scale=inp["x_scale"],
                                  out_dtype=TYPES[case["dtype"]])}
    if case["grad"]:
        out["dx"], dgate, dup = K.vq_gated_rows_backward(inp["dact"], inp["x"], *args, activation=case["act"],
                                                         scale_grad=case["scales"])
        if case["scales"]:
            out["dgate"], out["dup"] = dgate, dup
    return out

def _own_product(case, inp):
    from compressai_amd import kernels as K

    i0, i1, scale = inp["matrix"]
    dx, dscale = K.vq_gemm_backward(inp["dy"], inp["x"], i0, i1, inp["cb0"], inp["cb1"], scale, case["rows"], case["n"],
                                    scale_grad=case["scales"])
    return {"dx": dx, "dscale": dscale} if case["scales"] else {"dx": dx}

def _own_loss(case, inp):
    from compressai_amd import kernels as K

    i0, i1, scale = inp["matrix"]
    args = (i0, i1, inp["cb0"], inp["cb1"], scale, case["rows"], case["n"])
    loss, lse = K.vq_head_loss(inp["x"], inp["targets"], *args, ignore_index=IGNORE)
    out = {"loss": loss, "lse": lse}
    if case["grad"]:
        out["dx"], dscale = K.vq_head_loss_backward(inp["x"], inp["targets"], lse, inp["dloss"], *args,
                                                    ignore_index=IGNORE, scale_grad=case["scales"])
        if case["scales"]:
            out["dscale"] = dscale
    return out

def run(state):
    case, inp = state["case"], state["inp"]
    kind = case["kind"] + ("_grad" if case["kind"] == "norm" and case["grad"] else "")
    if own:
        return {"norm": _own_norm, "norm_grad": _own_norm_grad, "gated": _own_gated, "product": _own_product,
                "loss": _own_loss}[kind](case, inp)
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "gated": _plain_gated, "product": _plain_product,
            "loss": _plain_loss}[kind](case, inp)

# ------------------------------------------------- what a pass cannot do without
def work(case):
    T, n = case["tokens"], case["n"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        stages = case["hb"].bit_length() - 1 if case["hb"] else 0
        if case["grad"]:
            return {"bytes": T * n * size * (3 + case["residual"]) + n * (size + 4), "flops": T * n * (10 + stages)}
        moved = T * n * (size * (1 + case["residual"] + (1 if case["residual"] else 0)) + case["bits"] // 8) + n * size
        return {"bytes": moved + (T * 4 if case["bits"] == 8 else 0), "flops": T * n * (6 + stages)}
    rows = case["rows"] * (2 if case["kind"] == "gated" else 1)
    codes = rows * (n // 8) * {1: 2, 2: 4, 3: 3}[case["stages"]] + rows * (4 if case["scales"] else 2)
    books = 65536 * 16 * (2 if case["stages"] == 2 else 1)
    moved = codes + books + T * n * (1 if case.get("bits") == 8 else 2)
    product = 2 * T * rows * n
    if case["kind"] == "product":
        return {"bytes": moved * (1 if case["scales"] else 0) + (0 if case["scales"] else codes + books) + T * rows * 2
                + T * n * 2 + case["scales"] * rows * 4, "flops": product * (2 if case["scales"] else 1)}
    passes = 2 if case["grad"] else 1
    if case["kind"] == "gated":
        return {"bytes": moved + T * case["rows"] * 2 * passes + case["grad"] * T * n * 2 + case["scales"] * rows * 4,
                "flops": product * passes}
    return {"bytes": moved + T * 16 + case["grad"] * T * n * 2 + case["scales"] * rows * 4, "flops": product * passes}

# --------------------------------------------- from the definitions, in 64 bits
def _exact_matrix(inp, matrix):
    """[rows, n], row scales included, and the scales"""
    i0, i1, s = matrix
    w = torch.index_select(inp["cb0"].double(), 0, (i0.to(torch.int64).reshape(-1) + 65536) % 65536)
    if i1 is not None:
        w += torch.index_select(inp["cb1"].double(), 0, (i1.to(torch.int64).reshape(-1) + 65536) % 65536)
    return w.reshape(i0.shape[0], -1) * s.double()[:, None], s.double()

def _exact_hadamard(v, hb):
    """the transform along the last axis, by sums and differences of halves"""
    v, step = v.reshape(-1, hb), 1
    while step < hb:
        a = v.reshape(-1, hb // (2 * step), 2, step)
        v = torch.stack([a[:, :, 0] + a[:, :, 1], a[:, :, 0] - a[:, :, 1]], dim=2).reshape(-1, hb)
        step *= 2
    return v / math.sqrt(hb)

def _exact_norm(case, inp):
    h = inp["x"].double()
    if case["residual"]:
        h = h + inp["residual"].double()
    gain = inp["weight"].double() + float(case["zero"])
    y = h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["n"] + EPS) * gain
    if case["hb"]:
        y = _exact_hadamard(y.index_select(1, inp["perm"].long()) * inp["sign"].double(), case["hb"]).reshape(h.shape)
    if case["bits"] == 16:
        return {"y": y, "h": h}
    step = y.abs().max(1, keepdim=True).values / 127
    return {"y": torch.where(step > 0, torch.round(y / step) * step, 0.0), "scale": step.reshape(-1), "h": h}

def _exact_norm_grad(case, inp):
    h = inp["h"].double()
    up = inp["dy"].double()
    if case["hb"]:  # the transform is its own inverse
        back = _exact_hadamard(up, case["hb"]).reshape(h.shape) * inp["sign"].double()
        up = back.index_select(1, torch.argsort(inp["perm"].long()))
    gain = inp["weight"].double() + float(case["zero"])
    rms = torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["n"] + EPS)
    unit = h / rms
    dx = (up * gain - unit * (up * gain * unit).sum(1, keepdim=True) / case["n"]) / rms
    if case["residual"]:
        dx = dx + inp["dh"].double()
    return {"dx": dx, "dweight": (up * unit).sum(0)}

def _exact_gated(case, inp):
    x = inp["x"].double()
    if inp["x_scale"] is not None:
        x = x * inp["x_scale"].double()[:, None]
    (wg, sg), (wu, su) = _exact_matrix(inp, inp["gate"]), _exact_matrix(inp, inp["up"])
    g, u = x @ wg.t(), x @ wu.t()
    if case["act"] == "silu":
        gate = torch.sigmoid(g)
        a, slope = g * gate, gate + g * gate * torch.sigmoid(-g)
    else:
        # 0.5 (1 + tanh z) is the logistic function of 2 z
        z = math.sqrt(8.0 / math.pi) * (g + 0.044715 * g.pow(3))
        gate = torch.sigmoid(z)
        a, slope = g * gate, gate + g * gate * torch.sigmoid(-z) * math.sqrt(8.0 / math.pi) * (1 + 0.134145 * g.pow(2))
    out = {"act": a * u}
    if case["grad"]:
        d = inp["dact"].double()
        dg, du = d * u * slope, d * a
        out["dx"] = dg @ wg + du @ wu
        if case["scales"]:
            out["dgate"], out["dup"] = (dg * g).sum(0) / sg, (du * u).sum(0) / su
    return out

def _exact_product(case, inp):
    w, s = _exact_matrix(inp, inp["matrix"])
    dy = inp["dy"].double()
    out = {"dx": dy @ w}
    if case["scales"]:
        out["dscale"] = ((dy.t() @ inp["x"].double()) * w).sum(1) / s
    return out

def _exact_loss(case, inp):
    x, t = inp["x"].double(), inp["targets"]
    w, s = _exact_matrix(inp, inp["matrix"])
    logits = x @ w.t()
    lse = torch.logsumexp(logits, 1)
    used = t >= 0
    pick = (x * w[t.clamp(min=0)]).sum(1)
    out = {"loss": torch.where(used, lse - pick, 0.0), "lse": lse}
    if case["grad"]:
        d = torch.exp(logits - lse[:, None])
        d[torch.arange(len(t), device=DEV)[used], t[used]] -= 1.0
        d *= torch.where(used, inp["dloss"].double(), 0.0)[:, None]
        out["dx"] = d @ w
        if case["scales"]:
            out["dscale"] = (d * logits).sum(0) / s
    return out

def exact(case, seed):
    inp = _inputs(case, seed)
    if case["kind"] == "norm":
        return (_exact_norm_grad if case["grad"] else _exact_norm)(case, inp)
    return {"gated": _exact_gated, "product": _exact_product, "loss": _exact_loss}[case["kind"]](case, inp)
