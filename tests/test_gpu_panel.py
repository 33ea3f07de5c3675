"""The gated block, the head's loss and the gradients through packed matrices
(vq2_gated_rows, vq2_head_loss, vq2_gemm_backward and the backward passes) on
the GPU against the formulas in 64 bits.

Tolerances, from the arithmetic that include/vq2_amd.h and the source state.
A product of K terms takes K / 32 steps of the matrix core (twice as many
where weights are held in two parts), each rounding the running sum a few
times: it is off by at most (K / 4) 2^-24 of the sum of its terms' magnitudes,
M = sum |x_k w_k|, to which the second part's own rounding adds 2^-22 of them.
A weight that is rounded to fp16 once (results in bf16) is off by 2^-11 of
itself: 2^-11 M.  Rounding a result adds half a step.  A gradient is rounded to fp16 between
its two products: 2^-11 of each term (and 2^-25 of the largest scale's), so
2^-11 of the sum of the terms' magnitudes.  exp and log are good to 2^-20 of
their results over these ranges (__expf: a rounded product with log2 e, so
|x| 2^-23 more).
"""
import math

import pytest
import torch

from compressai_amd import kernels as K, synth
from compressai_amd.graph import DecodeStepGraph

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
E = 2.0 ** -24


def half(t, ref):
    return ref.abs() * {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[t] + (
        2.0 ** -25 if t == torch.float16 else 0.0)


class Mat:
    """a packed matrix, on the host, and its weights in 64 bits (no scales)"""

    def __init__(self, seed, rows, n, stages, cb, sdt="bf16"):
        self.i0 = synth.indices16(seed, (rows, n // 8))
        self.i1 = None if stages == 1 else synth.indices16(seed + 1, (rows, n // 8)) if stages == 2 else synth.indices8(seed + 1, (rows, n // 8))
        self.scale = synth.scales(seed + 2, rows, DT[sdt]) * (8 / n) ** 0.5
        self.cb0, self.cb1 = cb[0], cb[1] if stages == 2 else cb[2] if stages == 3 else None
        w = self.cb0.double()[self.i0.long() & 0xFFFF]
        if stages > 1:
            w = w + self.cb1.double()[self.i1.long() & (0xFFFF if stages == 2 else 0xFF)]
        self.w = w.reshape(rows, n)
        self.s = self.scale.double()
        self.exact = stages == 1 and self.cb0.dtype != torch.float32

    def on(self, dev):
        to = lambda t: None if t is None else t.to(dev)
        return to(self.i0), to(self.i1), to(self.cb0), to(self.cb1), to(self.scale)


_CB = {}


def books(dtype):
    if dtype not in _CB:
        _CB[dtype] = [synth.codebook(1, dtype=DT[dtype]), (synth.codebook(2) * 0.3).to(DT[dtype]),
                      (synth.codebook(3, rows=256) * 0.3).to(DT[dtype])]
    return _CB[dtype]


def rows_of(seed, T, n, dtype):
    """(device rows, x_scale, the values in 64 bits)"""
    x = synth.activations(seed, (T, n), torch.float32)
    if dtype in DT:
        x = x.to(DT[dtype])
        return x, None, x.double()
    if dtype == "int8":
        s = x.abs().amax(-1) / 127
        q = torch.round(x / s[:, None]).to(torch.int8)
    else:
        s = x.abs().amax(-1) / 448
        q = (x / s[:, None]).to(torch.float8_e4m3fn)
    return q, s, q.float().double() * s.double()[:, None]


def product_err(x64, m, rounded):
    """bound of a raw product's error (before its scale)"""
    mag = x64.abs() @ m.w.abs().t()
    return mag * (x64.shape[1] / 4 * E + 2.0 ** -22 + (2.0 ** -11 if rounded and not m.exact else 0))


def act64(a, g):
    if a == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


SIZES = [(1, 1, 64), (2, 16, 64), (16, 17, 128), (63, 100, 192), (64, 256, 320), (65, 257, 64), (127, 40, 256), (128, 300, 128),
         (129, 15, 512), (300, 513, 192), (0, 32, 64), (5, 1000, 2048)]
KINDS = [("fp16", 1, "fp16", "bf16"), ("bf16", 1, "fp16", "fp32"), ("bf16", 2, "fp16", "fp16"), ("fp16", 2, "fp16", "bf16"),
         ("bf16", 3, "bf16", "bf16"), ("fp16", 1, "fp32", "fp16"), ("bf16", 1, "bf16", "bf16"), ("fp16", 3, "fp16", "fp32")]


# ------------------------------------------------------------- gated block
@pytest.mark.parametrize("T,rows,n", SIZES)
@pytest.mark.parametrize("xdt,stages,cdt,sdt", KINDS + [("int8", 1, "fp16", "bf16"), ("e4m3", 2, "fp16", "fp16")])
def test_gated(dev, T, rows, n, xdt, stages, cdt, sdt):
    act = "silu" if (T + stages) % 2 else "gelu_tanh"
    x, xs, x64 = rows_of(T + 1, T, n, xdt)
    g, u = Mat(10 + rows, rows, n, stages, books(cdt), sdt), Mat(50 + rows, rows, n, stages, books(cdt), sdt)
    dg, du = g.on(dev), u.on(dev)
    for odt in (DT[xdt] if xdt in DT else torch.bfloat16, torch.float32):
        y = K.vq_gated_rows(x.to(dev), (dg[0], dg[1], dg[4]), (du[0], du[1], du[4]), dg[2], dg[3], n, 1.25, activation=act,
                            x_scale=None if xs is None else xs.to(dev), out_dtype=odt)
        assert y.shape == (T, rows) and y.dtype == odt
        gv, uv = (x64 @ m.w.t() * m.s * 1.25 for m in (g, u))
        eg, eu = (product_err(x64, m, odt == torch.bfloat16) * m.s * 1.25 + 4 * E * v.abs() for m, v in ((g, gv), (u, uv)))
        f, df = act64(act, gv)
        # |f'| <= 1.13; f itself is good to |g| 2^-22 and 2^-20 of it
        tol = (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * gv.abs()) * (uv.abs() + eu) + f.abs() * eu
        off = (y.cpu().double() - f * uv).abs() - tol - half(odt, f * uv)
        assert off.numel() == 0 or off.max() <= 0, float(off.max())


@pytest.mark.parametrize("T,rows,n", SIZES)
@pytest.mark.parametrize("xdt,stages,cdt,sdt", KINDS)
def test_gated_backward(dev, T, rows, n, xdt, stages, cdt, sdt):
    act = "silu" if (T + stages) % 2 else "gelu_tanh"
    x, _, x64 = rows_of(T + 2, T, n, xdt)
    d = (synth.activations(3 + T, (T, rows), torch.float32) * 1e-3).to(DT[xdt])
    g, u = Mat(20 + rows, rows, n, stages, books(cdt), sdt), Mat(60 + rows, rows, n, stages, books(cdt), sdt)
    dg, du = g.on(dev), u.on(dev)
    args = (d.to(dev), x.to(dev), (dg[0], dg[1], dg[4]), (du[0], du[1], du[4]), dg[2], dg[3], n, 1.25)
    dx, sg, su = K.vq_gated_rows_backward(*args, activation=act, scale_grad=True)
    dx1, none, none2 = K.vq_gated_rows_backward(*args, activation=act)
    assert none is None and none2 is None and dx.dtype == x.dtype and dx.shape == x.shape
    rg, ru = (x64 @ m.w.t() * 1.25 for m in (g, u))
    gv, uv, d64 = rg * g.s, ru * u.s, d.double()
    f, df = act64(act, gv)
    tg, tu = d64 * uv * df, d64 * f
    want = (tg * g.s * 1.25) @ g.w + (tu * u.s * 1.25) @ u.w
    for got, rounded in ((dx, False), (dx1, x.dtype == torch.bfloat16)):
        eg, eu = (product_err(x64, m, rounded) * m.s * 1.25 + 4 * E * v.abs() for m, v in ((g, gv), (u, uv)))
        # |f''| <= 1.2 (silu 0.5, gelu 1.13)
        etg = d64.abs() * (eu * (df.abs() + 1.2 * eg) + uv.abs() * (1.2 * eg + 2.0 ** -19 * (1 + gv.abs())))
        etu = d64.abs() * (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * gv.abs())
        # rounded to fp16 between the products: 2^-11 of a term, and 2^-25 under the
        # row's power of two, at most 2^6 of its largest upstream value
        floor = 2.0 ** -19 * d64.abs().amax(-1, keepdim=True) if rows else 0
        top = torch.maximum(g.s.max(), u.s.max())
        pg, pu = (t.abs() * 2.0 ** -11 * m.s + floor * top * 2 for t, m in ((tg, g), (tu, u)))
        w11 = 2.0 ** -11 if x.dtype == torch.bfloat16 and not g.exact else 0.0
        rel = (2 * rows / 4) * E + 2.0 ** -22 + w11
        tol = 1.25 * ((etg * g.s + pg + rel * (tg * g.s).abs()) @ g.w.abs() + (etu * u.s + pu + rel * (tu * u.s).abs()) @ u.w.abs())
        off = (got.cpu().double() - want).abs() - tol - half(x.dtype, want)
        assert off.numel() == 0 or off.max() <= 0, float(off.max())
    eg, eu = (product_err(x64, m, False) * m.s * 1.25 + 4 * E * v.abs() for m, v in ((g, gv), (u, uv)))
    etg = d64.abs() * (eu * (df.abs() + 1.2 * eg) + uv.abs() * (1.2 * eg + 2.0 ** -19 * (1 + gv.abs())))
    etu = d64.abs() * (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * gv.abs())
    for got, t, e, r, er, m in ((sg, tg, etg, rg, eg, g), (su, tu, etu, ru, eu, u)):
        want = (t * r).sum(0)
        tol = (e * r.abs() + (t.abs() + e) * er / m.s + (T + 8) * E * (t * r).abs()).sum(0) + 1e-30
        assert ((got.cpu().double() - want).abs() <= tol).all()


# ------------------------------------------------------ gradient of a product
@pytest.mark.parametrize("T,rows,n", SIZES)
@pytest.mark.parametrize("xdt,stages,cdt,sdt", KINDS)
def test_gemm_backward(dev, T, rows, n, xdt, stages, cdt, sdt):
    x, _, x64 = rows_of(T + 3, T, n, xdt)
    ddt = torch.float32 if stages == 3 else DT[xdt]
    d = (synth.activations(4 + T, (T, rows), torch.float32) * 1e-4).to(ddt)
    m = Mat(30 + rows, rows, n, stages, books(cdt), sdt)
    i0, i1, cb0, cb1, sc = m.on(dev)
    dx, ds = K.vq_gemm_backward(d.to(dev), x.to(dev), i0, i1, cb0, cb1, sc, rows, n, 0.5, scale_grad=True)
    dx2, none = K.vq_gemm_backward(d.to(dev), None, i0, i1, cb0, cb1, sc, rows, n, 0.5, dx_dtype=x.dtype)
    assert none is None and torch.equal(dx, dx2)
    d64 = d.double()
    t = d64 * m.s * 0.5
    want = t @ m.w
    # the row's largest value lies in [2^14, 2^15) before its scale: what fp16 cannot hold is below 2^-39 of it
    p = t.abs() * 2.0 ** -11 + 2.0 ** -38 * d64.abs().amax(-1, keepdim=True) * m.s.max() if rows and T else t.abs()
    w11 = 2.0 ** -11 if x.dtype == torch.bfloat16 and not m.exact else 0.0
    tol = (p + (rows / 4 * E + 2.0 ** -22 + w11) * t.abs()) @ m.w.abs()
    off = (dx.cpu().double() - want).abs() - tol - half(dx.dtype, want)
    assert off.numel() == 0 or off.max() <= 0, float(off.max())
    raw = x64 @ m.w.t()
    want = 0.5 * (d64 * raw).sum(0)
    tol = 0.5 * (d64.abs() * product_err(x64, m, False) + (T + 8) * E * (d64 * raw).abs()).sum(0) + 1e-30
    assert ((ds.cpu().double() - want).abs() <= tol).all()


# ---------------------------------------------------------------- head's loss
def loss64(x64, m, t, rs, ignore):
    z = x64 @ m.w.t() * m.s * rs
    lse = torch.logsumexp(z, -1) if z.numel() else z.sum(-1)
    used = t != ignore
    pick = z.gather(1, t.clamp(0, m.w.shape[0] - 1)[:, None]).view(-1) if z.numel() else lse
    return z, lse, torch.where(used, lse - pick, 0.0), used


@pytest.mark.parametrize("T,rows,n", SIZES + [(3, 16385, 64), (70, 20000, 64)])
@pytest.mark.parametrize("xdt,stages,cdt,sdt", KINDS + [("int8", 1, "fp16", "bf16"), ("e4m3", 3, "fp16", "fp16")])
def test_head_loss(dev, T, rows, n, xdt, stages, cdt, sdt):
    x, xs, x64 = rows_of(T + 5, T, n, xdt)
    m = Mat(40 + rows, rows, n, stages, books(cdt), sdt)
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(T))
    if T > 2:
        t[0], t[1], t[T // 2] = rows - 1, 0, -7
    loss, lse = K.vq_head_loss(x.to(dev), t.to(dev), i0, i1, cb0, cb1, sc, rows, n, 2.0, ignore_index=-7,
                               x_scale=None if xs is None else xs.to(dev))
    z, lse64, want, used = loss64(x64, m, t, 2.0, -7)
    ez = product_err(x64, m, False) * m.s * 2.0 + 4 * E * z.abs()
    # the sum of exponentials: each off by 2^-20 and the distance's 2^-23, sums of at most `rows` of them in a tree of short runs
    e_lse = ez.amax(-1) + 2.0 ** -19 + 4 * E * lse64.abs() if rows else lse64
    assert ((lse.cpu().double() - lse64).abs() <= e_lse).all()
    assert ((loss.cpu().double() - want).abs() <= torch.where(used, 2 * e_lse + 2 * E * (want.abs() + lse64.abs()), 0.0)).all()


@pytest.mark.parametrize("T,rows,n", SIZES + [(130, 20000, 64)])
@pytest.mark.parametrize("xdt,stages,cdt,sdt", KINDS)
def test_head_loss_backward(dev, T, rows, n, xdt, stages, cdt, sdt):
    x, _, x64 = rows_of(T + 6, T, n, xdt)
    m = Mat(45 + rows, rows, n, stages, books(cdt), sdt)
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(T + 1))
    if T > 2:
        t[0], t[1], t[T // 2] = rows - 1, 0, -100
    dl = synth.activations(T, T, torch.float32) * 1e-2
    args = (x.to(dev), t.to(dev))
    rest = (i0, i1, cb0, cb1, sc, rows, n, 2.0)
    _, lse = K.vq_head_loss(*args, *rest)
    dx, ds = K.vq_head_loss_backward(*args, lse, dl.to(dev), *rest, scale_grad=True)
    dx2, none = K.vq_head_loss_backward(*args, lse, dl.to(dev), *rest)
    assert none is None and dx.shape == x.shape and dx.dtype == x.dtype and torch.equal(dx, dx2)
    z, lse64, _, used = loss64(x64, m, t, 2.0, -100)
    p = torch.exp(z - lse64[:, None])
    if T:
        p[torch.arange(T)[used], t[used]] -= 1
        p[~used] = 0
    up = torch.where(used, dl.double(), 0.0)[:, None]
    ez = product_err(x64, m, False) * m.s * 2.0 + 4 * E * z.abs()
    elog = ez + (ez.amax(-1, keepdim=True) if rows else 0) + 2.0 ** -19 + 4 * E * (lse64.abs()[:, None] + z.abs())
    ep = torch.exp(z - lse64[:, None]) * (elog + 2.0 ** -20)
    want = up * ((p * m.s * 2.0) @ m.w)
    w11 = 2.0 ** -11 if x.dtype == torch.bfloat16 and not m.exact else 0.0
    # fp16 of p s / 2^e 2^14: 2^-11 of it, and 2^-25 2^-14 of the largest scale
    tp = p.abs() * m.s * 2.0 * (2.0 ** -11 + rows / 4 * E + 2.0 ** -22 + w11) + ep * m.s * 2.0 + 2.0 ** -38 * 2 * m.s.max()
    tol = up.abs() * (tp @ m.w.abs()) + 4 * E * want.abs()
    off = (dx.cpu().double() - want).abs() - tol - half(x.dtype, want)
    assert off.numel() == 0 or off.max() <= 0, float(off.max())
    raw = x64 @ m.w.t() * 2.0
    wds = (up * p * raw).sum(0)
    eds = (up.abs() * (ep * raw.abs() + (p.abs() + ep) * ez / m.s + (T + 8) * E * (p * raw).abs())).sum(0) + 1e-30
    assert ((ds.cpu().double() - wds).abs() <= eds).all()
    assert T <= 2 or (dx[T // 2] == 0).all()


def test_loss_gradient_against_differences(dev):
    """(L(x + d) - L(x - d)) / 2 step, L = sum of dloss * loss in 64 bits; the step's second order and the rounding to
    bf16 of the gradient, 2^-9 of each term"""
    T, rows, n = 6, 300, 128
    x, _, x64 = rows_of(77, T, n, "bf16")
    m = Mat(78, rows, n, 1, books("fp16"), "fp32")
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(79))
    dl, d = synth.activations(80, T, torch.float32), synth.activations(81, (T, n), torch.float32).double()
    _, lse = K.vq_head_loss(x.to(dev), t.to(dev), i0, i1, cb0, cb1, sc, rows, n)
    dx, ds = K.vq_head_loss_backward(x.to(dev), t.to(dev), lse, dl.to(dev), i0, i1, cb0, cb1, sc, rows, n, scale_grad=True)
    L = lambda xx: (dl.double() * loss64(xx, m, t, 1.0, -100)[2]).sum()
    num = (L(x64 + 1e-5 * d) - L(x64 - 1e-5 * d)) / 2e-5
    ana = dx.cpu().double() * d
    assert abs(num - ana.sum()) <= 2.0 ** -8 * ana.abs().sum()
    base, v = m.s, synth.activations(82, rows, torch.float32).double() * 1e-5
    m.s = base + v
    up = L(x64)
    m.s = base - v
    num, ana = (up - L(x64)) / 2, ds.cpu().double() * v
    assert abs(num - ana.sum()) <= 1e-4 * ana.abs().sum()


def test_loss_targets(dev):
    """targets outside the vocabulary give NaN, in their own rows alone; those of
    ignore_index give zeros whatever their row holds"""
    T, rows, n = 9, 40, 64
    x, _, _ = rows_of(90, T, n, "bf16")
    m = Mat(91, rows, n, 1, books("fp16"))
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.tensor([3, rows, -1, -100, 2 ** 40, 5, -100, rows - 1, -2 ** 62])
    x[6] = math.nan
    x[5] = math.inf
    one = torch.ones(T, device=dev)
    rest = (i0, i1, cb0, cb1, sc, rows, n)
    loss, lse = K.vq_head_loss(x.to(dev), t.to(dev), *rest)
    assert torch.isnan(loss.cpu()).tolist() == [False, True, True, False, True, True, False, False, True]
    assert loss[3] == 0 and loss[6] == 0
    dx, ds = K.vq_head_loss_backward(x.to(dev), t.to(dev), lse, one, *rest, scale_grad=True)
    bad = torch.isnan(dx.cpu()).all(-1)
    assert bad.tolist() == [False, True, True, False, True, True, False, False, True]
    assert (dx[3] == 0).all() and (dx[6] == 0).all() and torch.isnan(ds).all()
    t = torch.tensor([3, -100, 4, -100, 5, -100, -100, rows - 1, 0])
    dx, ds = K.vq_head_loss_backward(x.to(dev), t.to(dev), lse, one, *rest, scale_grad=True)
    assert torch.isfinite(ds).all() and torch.isfinite(dx).all()


def test_large_logits(dev):
    """logits some 1000 apart, and rows whose values span fp16's range and bf16's"""
    T, rows, n = 20, 1000, 64
    m = Mat(95, rows, n, 1, books("fp16"), "fp32")
    i0, i1, cb0, cb1, sc = m.on(dev)
    x = synth.activations(96, (T, n), torch.float32) * torch.logspace(-20, 3, T)[:, None]
    x = x.to(torch.bfloat16)
    t = torch.randint(0, rows, (T,), generator=synth.gen(97))
    loss, lse = K.vq_head_loss(x.to(dev), t.to(dev), i0, i1, cb0, cb1, sc, rows, n)
    z, lse64, want, _ = loss64(x.double(), m, t, 1.0, -100)
    ez = (product_err(x.double(), m, False) * m.s + 4 * E * z.abs()).amax(-1)
    assert ((lse.cpu().double() - lse64).abs() <= ez + 2.0 ** -19 + 4 * E * lse64.abs()).all()
    assert ((loss.cpu().double() - want).abs() <= 2 * ez + 2.0 ** -18 + 8 * E * (lse64.abs() + z.abs().amax(-1))).all()
    dx, _ = K.vq_head_loss_backward(x.to(dev), t.to(dev), lse, torch.ones(T, device=dev), i0, i1, cb0, cb1, sc, rows, n)
    assert torch.isfinite(dx).all()


def test_more_tokens_than_a_chunk(dev):
    """8192 tokens are taken at a time: every entry equals its own calls on the parts, sums of scales to their order"""
    T, rows, n = 8192 + 133, 48, 64
    m, u = Mat(98, rows, n, 1, books("fp16"), "fp32"), Mat(99, rows, n, 1, books("fp16"), "fp32")
    i0, i1, cb0, cb1, sc = m.on(dev)
    gate, up = (i0, i1, sc), (u.i0.to(dev), None, u.scale.to(dev))
    x, _, x64 = rows_of(100, T, n, "bf16")
    x = x.to(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(101)).to(dev)
    d = synth.activations(102, (T, rows), torch.bfloat16).to(dev)
    dl = torch.rand(T, generator=synth.gen(103)).to(dev)
    rest = (i0, i1, cb0, cb1, sc, rows, n)
    cut = [slice(0, 8192), slice(8192, T)]

    def all_of(sl):
        loss, lse = K.vq_head_loss(x[sl], t[sl], *rest)
        return (loss, lse, K.vq_gated_rows(x[sl], gate, up, cb0, cb1, n),
                *K.vq_head_loss_backward(x[sl], t[sl], lse, dl[sl], *rest, scale_grad=True),
                *K.vq_gated_rows_backward(d[sl], x[sl], gate, up, cb0, cb1, n, scale_grad=True),
                *K.vq_gemm_backward(d[sl], x[sl], *rest, scale_grad=True))

    whole, parts = all_of(slice(0, T)), [all_of(s) for s in cut]
    for k, w in enumerate(whole):
        a, b = parts[0][k], parts[1][k]
        if w.shape[0] == T:
            assert torch.equal(w, torch.cat([a, b])), k
        else:
            assert torch.equal(w, a + b), k


def test_graph_streams_and_runs(dev):
    """norm, block, product and loss with their gradients as a step: captured and replayed, on another stream, two at once"""
    T, n, inner, vocab = 37, 256, 192, 1000
    cb = books("fp16")
    g, u, dn, hd = Mat(110, inner, n, 2, cb), Mat(113, inner, n, 2, cb), Mat(116, n, inner, 2, cb), Mat(119, vocab, n, 1, cb)
    gd, ud, dd, hh = (m.on(dev) for m in (g, u, dn, hd))
    w = torch.ones(n, device=dev, dtype=torch.bfloat16)
    t = torch.randint(0, vocab, (T,), generator=synth.gen(120)).to(dev)
    dl = torch.full((T,), 1 / T, device=dev)

    def step(x, res):
        y, h, _ = K.vq_add_rms_norm(x, w, res, hb=256)
        gate, up = (gd[0], gd[1], gd[4]), (ud[0], ud[1], ud[4])
        act = K.vq_gated_rows(y, gate, up, gd[2], gd[3], n)
        ar = K.vq_rht(act, hb=64)
        o = K.vq_rows_gemm(ar, [(dd[0], dd[1], dd[4], n)], dd[2], dd[3], inner, hb=0, act_dtype=torch.bfloat16,
                           out_dtype=torch.bfloat16)[0]
        y2, h2, _ = K.vq_add_rms_norm(o, w, h, hb=256)
        rest = (hh[0], hh[1], hh[2], hh[3], hh[4], vocab, n)
        loss, lse = K.vq_head_loss(y2, t, *rest)
        dy2, dsh = K.vq_head_loss_backward(y2, t, lse, dl, *rest, scale_grad=True)
        dh2, dw2 = K.vq_add_rms_norm_backward(dy2, h2, w, hb=256)
        dar, dsd = K.vq_gemm_backward(dh2, ar, dd[0], dd[1], dd[2], dd[3], dd[4], n, inner, scale_grad=True)
        dact = K.vq_rht(dar, hb=64, inverse=True)
        dy, dsg, dsu = K.vq_gated_rows_backward(dact, y, gate, up, gd[2], gd[3], n, scale_grad=True)
        dx, dw = K.vq_add_rms_norm_backward(dy, h, w, dh2, hb=256)
        return loss, lse, dx, dw, dw2, dsh, dsd, dsg, dsu

    mk = lambda k: synth.activations(k, (T, n), torch.bfloat16).to(dev)
    graphs = [DecodeStepGraph(step, [mk(1), mk(2)]) for _ in range(2)]
    for k in range(4):
        a, b = mk(10 + k), mk(20 + k)
        want = step(a, b)
        torch.cuda.synchronize()
        got = graphs[k % 2](a, b)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        torch.ones(1 << 22, device=dev).sum().item()
    ins = [(mk(30), mk(31)), (mk(32), mk(33))]
    want = [step(*i) for i in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = step(*ins[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def _views(t, off, dev):
    """the tensor at an address that is only aligned to its elements"""
    buf = torch.empty(t.numel() + off, dtype=t.dtype, device=dev)
    v = buf[off:].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("T", [1, 5, 100, 300])
@pytest.mark.parametrize("stages", [1, 2, 3])
def test_planes_and_rows_at_any_address(dev, T, stages):
    """planes, scales and upstream rows aligned to their elements alone, and rows no multiple of 4: the aligned call's
    results up to the order of sums (2^-20 of the largest).  Few aligned tokens go through a kernel that multiplies the stages one by
    one, unaligned ones through panels, whose weights of two stages are rounded to fp16 for the block's bf16 result (2^-11 of
    each): its g and u are then 2^-11 of M apart, M the sum of their terms' magnitudes, and f(g) u |f'| <= 1.13 times that by
    |u|, and |f| times it"""
    n, rows = 128, 203
    cb = books("fp16")
    a, b = Mat(300, rows, n, stages, cb), Mat(303, rows, n, stages, cb)
    x = rows_of(T, T, n, "bf16")[0].to(dev)
    d = (synth.activations(5, (T, rows), torch.float32) * 1e-2).to(torch.bfloat16)
    t = torch.randint(0, rows, (T,), generator=synth.gen(T)).to(dev)
    dl = torch.ones(T, device=dev)

    def all_of(put, dy):
        (a0, a1, c0, c1, sa), (b0, b1, _, _, sb) = ((put(m.i0), None if m.i1 is None else put(m.i1), m.cb0.to(dev),
                                                    None if m.cb1 is None else m.cb1.to(dev), put(m.scale)) for m in (a, b))
        gate, up, head = (a0, a1, sa), (b0, b1, sb), (a0, a1, c0, c1, sa, rows, n)
        loss, lse = K.vq_head_loss(x, t, *head)
        return (loss, lse, K.vq_gated_rows(x, gate, up, c0, c1, n), *K.vq_head_loss_backward(x, t, lse, dl, *head, scale_grad=True),
                *K.vq_gated_rows_backward(dy, x, gate, up, c0, c1, n, scale_grad=True), *K.vq_gemm_backward(dy, x, *head, scale_grad=True))

    want = all_of(lambda v: v.to(dev), d.to(dev))
    got = all_of(lambda v: _views(v, 1, dev), _views(d, 1, dev))
    for k, (p, q) in enumerate(zip(got, want)):
        step = 0 if p.dtype == torch.float32 else 2.0 ** -7  # (a sum near a border may round the other way)
        tol = step * q.double().abs() + 2.0 ** -20 * q.double().abs().max()
        if k == 2 and stages > 1:
            x64 = x.double().cpu()
            g, v = x64 @ a.w.t() * a.s, x64 @ b.w.t() * b.s
            eg, ev = (2.0 ** -11 * (x64.abs() @ w.w.abs().t()) * w.s for w in (a, b))
            tol = tol + (1.13 * eg * (v.abs() + ev) + act64("silu", g)[0].abs() * ev).to(dev)
        assert ((p.double() - q.double()).abs() <= tol).all(), k


LARGE = [  # sizes that fill the device: wave tiles of 128 rows, several pieces of a matrix, one and more slices
    ("loss", 1100, 17000, 64), ("loss", 2500, 40000, 64), ("gated", 2050, 4100, 64), ("gated", 300, 9000, 64),
    ("product", 2048, 100, 4096), ("product", 2048, 600, 4096), ("product", 4100, 300, 2048), ("product", 130, 40000, 64)]


@pytest.mark.parametrize("kind,T,rows,n", LARGE)
@pytest.mark.parametrize("stages", [1, 2])
def test_large(dev, kind, T, rows, n, stages):
    """as the tests above, the 64-bit side on the GPU"""
    x, _, _ = rows_of(T + 9, T, n, "bf16")
    x = x.to(dev)
    x64 = x.double()
    cb = books("fp16")
    m, u = Mat(400 + rows, rows, n, stages, cb, "fp32"), Mat(403 + rows, rows, n, stages, cb, "fp32")
    for k in (m, u):
        k.w, k.s = k.w.to(dev), k.s.to(dev)
    i0, i1, cb0, cb1, sc = m.on(dev)
    head = (i0, i1, cb0, cb1, sc, rows, n)
    gen = torch.Generator(device=dev).manual_seed(T)
    if kind == "loss":
        t = torch.randint(0, rows, (T,), generator=gen, device=dev)
        t[::3] = -100
        dl = torch.rand(T, generator=gen, device=dev)
        loss, lse = K.vq_head_loss(x, t, *head)
        dx, ds = K.vq_head_loss_backward(x, t, lse, dl, *head, scale_grad=True)
        z, lse64, want, used = loss64(x64, m, t, 1.0, -100)
        ez = product_err(x64, m, False) * m.s + 4 * E * z.abs()
        el = ez.amax(-1) + 2.0 ** -19 + 4 * E * lse64.abs()
        assert ((lse.double() - lse64).abs() <= el).all()
        assert ((loss.double() - want).abs() <= torch.where(used, 2 * el + 2 * E * (want.abs() + lse64.abs()), 0.0)).all()
        p = torch.exp(z - lse64[:, None])
        ep = p * (ez + el[:, None] + 2.0 ** -18 + 4 * E * z.abs())
        p[torch.arange(T, device=dev)[used], t[used]] -= 1
        p[~used] = 0
        up = torch.where(used, dl.double(), 0.0)[:, None]
        want = up * ((p * m.s) @ m.w)
        tp = p.abs() * m.s * (2.0 ** -11 + rows / 4 * E + 2.0 ** -22 + (0 if m.exact else 2.0 ** -11)) + ep * m.s + 2.0 ** -38 * m.s.max()
        assert ((dx.double() - want).abs() <= up.abs() * (tp @ m.w.abs()) + half(x.dtype, want) + 4 * E * want.abs()).all()
        raw = z / m.s
        eds = (up.abs() * (ep * raw.abs() + (p.abs() + ep) * ez / m.s + (T + 8) * E * (p * raw).abs())).sum(0) + 1e-30
        assert ((ds.double() - (up * p * raw).sum(0)).abs() <= eds).all()
        return
    d = (torch.randn(T, rows, generator=gen, device=dev) * 1e-3).to(torch.bfloat16)
    d64 = d.double()
    if kind == "product":
        dx, ds = K.vq_gemm_backward(d, x, *head, scale_grad=True)
        t = d64 * m.s
        w11 = 0.0 if m.exact else 2.0 ** -11
        tol = (t.abs() * (2.0 ** -11 + rows / 4 * E + 2.0 ** -22 + w11) + 2.0 ** -38 * d64.abs().amax(-1, keepdim=True) * m.s.max()) @ m.w.abs()
        assert ((dx.double() - t @ m.w).abs() <= tol + half(x.dtype, t @ m.w)).all()
        raw = x64 @ m.w.t()
        tol = (d64.abs() * product_err(x64, m, False) + (T + 8) * E * (d64 * raw).abs()).sum(0) + 1e-30
        assert ((ds.double() - (d64 * raw).sum(0)).abs() <= tol).all()
        return
    gate, up = (i0, i1, sc), (u.i0.to(dev), None if u.i1 is None else u.i1.to(dev), u.scale.to(dev))
    y = K.vq_gated_rows(x, gate, up, cb0, cb1, n)
    dx, _, _ = K.vq_gated_rows_backward(d, x, gate, up, cb0, cb1, n)
    g64, u64 = (x64 @ k.w.t() * k.s for k in (m, u))
    eg, eu = (product_err(x64, k, True) * k.s + 4 * E * v.abs() for k, v in ((m, g64), (u, u64)))
    f, df = act64("silu", g64)
    tol = (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * g64.abs()) * (u64.abs() + eu) + f.abs() * eu
    assert ((y.double() - f * u64).abs() <= tol + half(y.dtype, f * u64)).all()
    tg, tu = d64 * u64 * df, d64 * f
    want = (tg * m.s) @ m.w + (tu * u.s) @ u.w
    etg = d64.abs() * (eu * (df.abs() + 1.2 * eg) + u64.abs() * (1.2 * eg + 2.0 ** -19 * (1 + g64.abs())))
    etu = d64.abs() * (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * g64.abs())
    floor = 2.0 ** -18 * d64.abs().amax(-1, keepdim=True) * max(m.s.max(), u.s.max())
    rel = 2.0 ** -11 * (1 if m.exact else 2) + 2 * rows / 4 * E + 2.0 ** -22
    tol = ((etg + rel * tg.abs()) * m.s + floor) @ m.w.abs() + ((etu + rel * tu.abs()) * u.s + floor) @ u.w.abs()
    assert ((dx.double() - want).abs() <= tol + half(x.dtype, want)).all()


def test_small_values(dev):
    """rows, upstream rows and scales far below and above 1: powers of two scale results and nothing else"""
    T, rows, n = 40, 96, 128
    m, u = Mat(500, rows, n, 1, books("fp16"), "fp32"), Mat(503, rows, n, 1, books("fp16"), "fp32")
    x = rows_of(7, T, n, "bf16")[0].to(dev)
    d = synth.activations(8, (T, rows), torch.bfloat16).to(dev)
    i0, _, cb0, _, sc = m.on(dev)
    base = K.vq_gemm_backward(d, x, i0, None, cb0, None, sc, rows, n, scale_grad=True)
    for e, f in ((-60, 0), (60, 0), (0, -50), (0, 50), (-40, 30)):
        got = K.vq_gemm_backward(d * 2.0 ** e, x, i0, None, cb0, None, sc * 2.0 ** f, rows, n, scale_grad=True)
        assert torch.equal(got[0].double(), base[0].double() * 2.0 ** (e + f))
        assert torch.equal(got[1].double(), base[1].double() * 2.0 ** e)
    # fp16 rows below fp16's normal numbers
    tiny = (x.float() * 2.0 ** -18).half()
    y = K.vq_gated_rows(tiny, (i0, None, sc * 2.0 ** 18), (u.i0.to(dev), None, u.scale.to(dev) * 2.0 ** 18), cb0, None, n, out_dtype=torch.float32)
    x64 = tiny.double().cpu() * 2.0 ** 18
    g, v = x64 @ m.w.t() * m.s, x64 @ u.w.t() * u.s
    want = act64("silu", g)[0] * v
    eg, eu = product_err(x64, m, False) * m.s, product_err(x64, u, False) * u.s
    tol = (1.13 * eg + 2.0 ** -20 * g.abs()) * (v.abs() + eu) + act64("silu", g)[0].abs() * eu + 2.0 ** -22 * want.abs()
    assert ((y.cpu().double() - want).abs() <= tol).all()
    one = K.vq_gated_rows(tiny[:1], (i0, None, sc * 2.0 ** 18), (u.i0.to(dev), None, u.scale.to(dev) * 2.0 ** 18), cb0, None, n,
                          out_dtype=torch.float32)
    assert ((one.cpu().double() - want[:1]).abs() <= tol[:1]).all()


def test_gradient_of_tiny_rows_and_scales(dev):
    """upstream rows and scales whose powers of two together leave fp32's range:
    the gradient of the same rows at ordinary size, times both, as far as bf16
    holds it (steps of 2^-133 at its smallest)"""
    T, rows, n = 20, 96, 128
    m = Mat(530, rows, n, 1, books("fp16"), "fp32")
    d = synth.activations(15, (T, rows), torch.bfloat16).to(dev)
    i0, _, cb0, _, sc = m.on(dev)
    base = K.vq_gemm_backward(d, None, i0, None, cb0, None, sc, rows, n)[0].double()
    for e, f in ((-64, -64), (-70, -58), (64, -64), (-90, 60), (60, 60)):
        got = K.vq_gemm_backward(d * 2.0 ** e, None, i0, None, cb0, None, sc * 2.0 ** f, rows, n)[0].double()
        want = base * 2.0 ** (e + f)
        assert torch.isfinite(got).all() and ((got - want).abs() <= 2.0 ** -133).logical_or(got == want).all()


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("stages", [1, 3])
@pytest.mark.parametrize("xf,sf,df", [(0, 0, 0), (-20, 0, 0), (0, -20, 0), (-30, -30, 30), (0, 14, 0), (10, 14, -40), (40, -36, -60)])
def test_gated_backward_of_any_activations(dev, act, stages, xf, sf, df):
    """The panel between the products is fp16 (steps of 2^-24 at its smallest)
    under powers of two that bring a token's largest upstream value into [2^14,
    2^15), and a bound B = 1.13 n max|x| max|w| max|s| of the activations to 1:
    each of its factors is rounded up to a power of two, so by at most 2 (the
    codebooks' as often as there are stages, the scales' twice: once more in
    front of the second product).  That is half a step of 2^-25 2^-14 2^6 (2^7)
    max|dy| B max|s| of a term."""
    T, rows, n = 40, 96, 192
    b = books("fp16")
    g, u = Mat(520, rows, n, stages, b, "fp32"), Mat(523, rows, n, stages, b, "fp32")
    for m in (g, u):
        m.scale = m.scale * 2.0 ** sf
        m.s = m.scale.double()
    x = (rows_of(13, T, n, "bf16")[0].float() * 2.0 ** xf).bfloat16()
    d = (synth.activations(14, (T, rows), torch.float32) * 2.0 ** df).bfloat16()
    x64, d64 = x.double(), d.double()
    dg, du = g.on(dev), u.on(dev)
    dx, _, _ = K.vq_gated_rows_backward(d.to(dev), x.to(dev), (dg[0], dg[1], dg[4]), (du[0], du[1], du[4]), dg[2], dg[3], n, activation=act)
    gv, uv = (x64 @ m.w.t() * m.s for m in (g, u))
    f, dv = act64(act, gv)
    tg, tu = d64 * uv * dv, d64 * f
    want = (tg * g.s) @ g.w + (tu * u.s) @ u.w
    eg, eu = (product_err(x64, m, True) * m.s + 4 * E * v.abs() for m, v in ((g, gv), (u, uv)))
    # f' moves by at most 1.2 a unit, and lies in [-0.13, 1.13]
    edf = torch.clamp(1.2 * eg, max=1.3) + 2.0 ** -19
    etg = d64.abs() * (eu * (dv.abs() + edf) + uv.abs() * edf)
    etu = d64.abs() * (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * gv.abs())
    wmax = b[0].double().abs().max() + (b[2].double().abs().max() if stages == 3 else 0)
    top = torch.maximum(g.s.max(), u.s.max())
    floor = 2.0 ** (-33 if stages == 1 else -32) * d64.abs().amax(-1, keepdim=True) * 1.13 * n * x64.abs().amax(-1, keepdim=True) * wmax * top * top
    w11 = 2.0 ** -11 if stages > 1 else 0.0
    rel = (2 * rows / 4) * E + 2.0 ** -22 + w11 + 2.0 ** -11
    tol = (etg * g.s + floor + rel * (tg * g.s).abs()) @ g.w.abs() + (etu * u.s + floor + rel * (tu * u.s).abs()) @ u.w.abs()
    off = (dx.cpu().double() - want).abs() - tol - half(torch.bfloat16, want) - 2.0 ** -133
    assert off.max() <= 0, float(off.max())


def test_nan_and_infinity_stay_in_their_rows(dev):
    T, rows, n = 150, 64, 64
    m, u = Mat(510, rows, n, 1, books("fp16")), Mat(513, rows, n, 1, books("fp16"))
    i0, _, cb0, _, sc = m.on(dev)
    gate, up = (i0, None, sc), (u.i0.to(dev), None, u.scale.to(dev))
    x = rows_of(11, T, n, "bf16")[0].to(dev)
    d = synth.activations(12, (T, rows), torch.bfloat16).to(dev)
    bx, bd = x.clone(), d.clone()
    bx[3, 5], bx[70, 0], bd[9, 1], bd[140, 63] = math.nan, math.inf, math.nan, -math.inf
    hit = torch.zeros(T, dtype=torch.bool, device=dev)
    hit[[3, 70, 9, 140]] = True
    for few in (T, 20):
        a, b = K.vq_gated_rows(x[:few], gate, up, cb0, None, n), K.vq_gated_rows(bx[:few], gate, up, cb0, None, n)
        keep = ~hit[:few]
        assert torch.equal(a[keep], b[keep]) and not torch.isfinite(b[3]).all()
    for f in (lambda p, q: K.vq_gated_rows_backward(q, p, gate, up, cb0, None, n)[0],
              lambda p, q: K.vq_gemm_backward(q, p, i0, None, cb0, None, sc, rows, n)[0]):
        a, b = f(x, d), f(bx, bd)
        assert torch.equal(a[~hit], b[~hit])
        assert not torch.isfinite(b[9]).any() and not torch.isfinite(b[140]).all()


def test_refusals(dev):
    n, rows, T = 64, 32, 4
    m = Mat(130, rows, n, 1, books("fp16"))
    i0, i1, cb0, cb1, sc = m.on(dev)
    x = torch.zeros(T, n, device=dev, dtype=torch.bfloat16)
    t = torch.zeros(T, device=dev, dtype=torch.int64)
    lse = torch.zeros(T, device=dev)
    d = torch.zeros(T, rows, device=dev, dtype=torch.bfloat16)
    head = (i0, i1, cb0, cb1, sc, rows, n)
    gate = (i0, i1, sc)
    bad = [
        (lambda: K.vq_head_loss(x.float(), t, *head), "dtype"),
        (lambda: K.vq_head_loss(x, t.int(), *head), "targets"),
        (lambda: K.vq_head_loss(x, t[:2], *head), "targets"),
        (lambda: K.vq_head_loss(x, t, *head, x_scale=lse), "8-bit"),
        (lambda: K.vq_head_loss(x.to(torch.int8), t, *head), "x_scale"),
        (lambda: K.vq_head_loss(x.to(torch.int8), t, *head, x_scale=lse[:2]), "x_scale"),
        (lambda: K.vq_head_loss(x, t, i0[:8], i1, cb0, cb1, sc, rows, n), "codes"),
        (lambda: K.vq_head_loss(x, t, i0, i1, cb0, cb1, sc[:8], rows, n), "scale"),
        (lambda: K.vq_head_loss(x[:, :32], t, *head), "last dim"),
        (lambda: K.vq_head_loss(x.cpu(), t, *head), "GPU"),
        (lambda: K.vq_head_loss_backward(x, t, lse[:1], lse, *head), "lse"),
        (lambda: K.vq_head_loss_backward(x, t, lse, lse.half(), *head), "dloss"),
        (lambda: K.vq_head_loss_backward(x.to(torch.int8), t, lse, lse, *head), "dtype"),
        (lambda: K.vq_gated_rows(x, gate, gate, cb0, cb1, n, activation="relu"), "activation"),
        (lambda: K.vq_gated_rows(x, gate, (i0[:16], None, sc[:16]), cb0, cb1, n), "rows"),
        (lambda: K.vq_gated_rows(x, gate, (i0, None, sc.float()), cb0, cb1, n), "scales"),
        (lambda: K.vq_gated_rows(x.t(), gate, gate, cb0, cb1, n), "last dim"),
        (lambda: K.vq_gated_rows_backward(d[:2], x, gate, gate, cb0, cb1, n), "dact"),
        (lambda: K.vq_gemm_backward(d, None, *head, scale_grad=True), "needs xr"),
        (lambda: K.vq_gemm_backward(d, x[:2], *head), "different rows"),
        (lambda: K.vq_gemm_backward(d, None, *head, dx_dtype=torch.float32), "fp16 or bf16"),
        (lambda: K.vq_gemm_backward(d[:, :8], None, *head), "last dim"),
    ]
    for call, match in bad:
        with pytest.raises(K.Vq2Error, match=match):
            call()
    # a width that the products do not take
    w = Mat(131, rows, 72, 1, books("fp16"))
    a0, a1, c0, c1, s = w.on(dev)
    with pytest.raises(K.Vq2Error, match="multiple of 64"):
        K.vq_head_loss(torch.zeros(T, 72, device=dev, dtype=torch.bfloat16), t, a0, a1, c0, c1, s, rows, 72)
    buf = torch.zeros(T * n + 4, device=dev, dtype=torch.bfloat16)
    with pytest.raises(K.Vq2Error, match="16-byte"):
        K.vq_head_loss(buf[1:T * n + 1].view(T, n), t, *head)
