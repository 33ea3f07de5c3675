"""Few tokens through packed matrices (the gated block and the head's loss,
whose centroids are gathered straight into the matrix cores' operands) and
wide rows, where the common sizes do not reach."""
import math

import pytest
import torch

from compressai_amd import kernels as K, synth
import test_gpu_panel as base
from test_gpu_panel import E, Mat, act64, books, half, loss64, product_err, rows_of

pytestmark = pytest.mark.gpu


def moved(t, dev, off=1):
    """the tensor at an address that is only aligned to its elements"""
    if t is None:
        return None
    buf = torch.empty(t.numel() + off, dtype=t.dtype, device=dev)
    return buf[off:].view(t.shape).copy_(t)


@pytest.mark.parametrize("T", [1, 4, 5, 17, 64, 96, 128, 300])
@pytest.mark.parametrize("stages,cdt", [(1, "fp16"), (2, "bf16"), (3, "fp16")])
def test_planes_at_any_address_give_the_same(dev, T, stages, cdt):
    n, rows = 192, 203
    a, b = Mat(600, rows, n, stages, books(cdt)), Mat(603, rows, n, stages, books(cdt))
    x = rows_of(T, T, n, "bf16")[0].to(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(T)).to(dev)
    out = []
    for put in (lambda v: None if v is None else v.to(dev), lambda v: moved(v, dev), lambda v: moved(v, dev, 5)):
        (i0, i1, c0, c1, s), (j0, j1, _, _, u) = ((put(m.i0), put(m.i1), m.cb0.to(dev), None if m.cb1 is None else m.cb1.to(dev),
                                                  put(m.scale)) for m in (a, b))
        out.append((K.vq_gated_rows(x, (i0, i1, s), (j0, j1, u), c0, c1, n), *K.vq_head_loss(x, t, i0, i1, c0, c1, s, rows, n)))
    for got in out[1:]:
        assert all(torch.equal(p, q) for p, q in zip(got, out[0]))


@pytest.mark.parametrize("T", [3, 40, 300])
def test_silu_far_below_zero(dev, T):
    """gates down to -87, where the sigmoid is still a normal number, times an up product large enough to show them; an
    infinite gate gives 0.  Of the result: e of the gate (exp), 2^-20 + 90 2^-23 of __expf and the reciprocal's 2^-23"""
    n, rows = 64, 160
    a, b = Mat(610, rows, n, 1, books("fp16"), "fp32"), Mat(613, rows, n, 1, books("fp16"), "fp32")
    x, _, x64 = rows_of(T, T, n, "bf16")
    a.scale = a.scale * 30.0
    b.scale = b.scale * 2.0 ** 100
    a.s, b.s = a.scale.double(), b.scale.double()
    i0, _, c0, _, s = a.on(dev)
    j0, _, _, _, u = b.on(dev)
    y = K.vq_gated_rows(x.to(dev), (i0, None, s), (j0, None, u), c0, None, n, out_dtype=torch.float32).cpu().double()
    g, v = x64 @ a.w.t() * a.s, x64 @ b.w.t() * b.s
    want = torch.nn.functional.silu(g) * v
    eg, ev = product_err(x64, a, False) * a.s + 4 * E * g.abs(), product_err(x64, b, False) * b.s + 4 * E * v.abs()
    far = (g < -60) & (g > -87)
    assert far.sum() > 3 and ((g < -80) & far).any()
    tol = want.abs() * (2 * eg + 2.0 ** -20 + 90 * 2.0 ** -23 + 2.0 ** -22) + want.abs() / v.abs() * ev * 1.01
    assert ((y - want).abs() <= tol)[far].all()
    assert torch.isfinite(y).all()
    s[7] = -math.inf
    y = K.vq_gated_rows(x.to(dev), (i0, None, s), (j0, None, u), c0, None, n, out_dtype=torch.float32).cpu()
    assert (y[:, 7][g[:, 7] > 0] == 0).all()


# --------------------------------- waves with rows of their own (1024 pairs of row tiles and more, over 64 tokens a block)
def loss_of(dev, T, rows, stages, cdt):
    """sizes of test_gpu_panel.test_head_loss, the 64-bit side on the GPU"""
    n = 64
    x, _, x64 = rows_of(T + 7, T, n, "bf16")
    m = Mat(620 + T, rows, n, stages, books(cdt), "fp32")
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.randint(0, rows, (T,), generator=synth.gen(T + 2))
    t[0], t[1], t[2], t[3], t[T - 1] = rows - 1, 0, -7, rows, -1
    loss, lse = K.vq_head_loss(x.to(dev), t.to(dev), i0, i1, cb0, cb1, sc, rows, n, 2.0, ignore_index=-7)
    m.w, m.s, x64, t = m.w.to(dev), m.s.to(dev), x64.to(dev), t.to(dev)
    z, lse64, want, used = loss64(x64, m, t, 2.0, -7)
    ez = product_err(x64, m, False) * m.s * 2.0 + 4 * E * z.abs()
    e_lse = ez.amax(-1) + 2.0 ** -19 + 4 * E * lse64.abs()
    assert ((lse.double() - lse64).abs() <= e_lse).all()
    bad = (t >= rows) | (t == -1)
    assert torch.equal(torch.isnan(loss), bad) and (loss[t == -7] == 0).all()
    tol = torch.where(used, 2 * e_lse + 2 * E * (want.abs() + lse64.abs()), 0.0)
    assert ((loss.double() - want).abs() <= tol)[~bad].all()


@pytest.mark.parametrize("T,rows", [(65, 32769), (96, 50257), (97, 32769), (128, 50257), (192, 32753), (200, 32769),
                                    (96, 100003), (128, 100003)])
@pytest.mark.parametrize("stages", [1, 2, 3])
@pytest.mark.parametrize("cdt", ["fp16", "bf16"])
def test_loss_of_many_rows(dev, T, rows, stages, cdt):
    """the last workgroup has waves without rows; above 65536 rows a wave has several pairs of tiles"""
    loss_of(dev, T, rows, stages, cdt)


@pytest.mark.parametrize("T,rows", [(65, 16385), (70, 17001), (96, 16369), (128, 17001)])
@pytest.mark.parametrize("stages", [1, 2, 3])
@pytest.mark.parametrize("cdt", ["fp16", "bf16"])
def test_gated_of_many_rows(dev, T, rows, stages, cdt):
    n = 64
    act = "silu" if stages % 2 else "gelu_tanh"
    x, _, x64 = rows_of(T + 8, T, n, "bf16")
    g, u = Mat(630, rows, n, stages, books(cdt), "fp32"), Mat(633, rows, n, stages, books(cdt), "fp32")
    i0, i1, cb0, cb1, s = g.on(dev)
    j0, j1, _, _, t = u.on(dev)
    y = K.vq_gated_rows(x.to(dev), (i0, i1, s), (j0, j1, t), cb0, cb1, n, 1.25, activation=act, out_dtype=torch.float32)
    for m in (g, u):
        m.w, m.s = m.w.to(dev), m.s.to(dev)
    x64 = x64.to(dev)
    gv, uv = (x64 @ m.w.t() * m.s * 1.25 for m in (g, u))
    eg, eu = (product_err(x64, m, False) * m.s * 1.25 + 4 * E * v.abs() for m, v in ((g, gv), (u, uv)))
    f, _ = act64(act, gv)
    tol = (1.13 * eg + 2.0 ** -20 * f.abs() + 2.0 ** -22 * gv.abs()) * (uv.abs() + eu) + f.abs() * eu
    assert ((y.double() - f * uv).abs() <= tol + half(torch.float32, f * uv)).all()


# ------------------------------------ rows that do not stay in registers while they are packed (more than 4096 values)
@pytest.mark.parametrize("T,rows,n", [(1, 40, 4160), (5, 33, 6144), (70, 20, 32768), (130, 40, 4160)])
@pytest.mark.parametrize("xdt,stages,cdt,sdt", [*base.KINDS[:4], ("int8", 1, "fp16", "bf16"), ("e4m3", 2, "fp16", "fp16")])
def test_wide_rows(dev, T, rows, n, xdt, stages, cdt, sdt):
    """every entry at these widths, by the checks of the narrower ones"""
    kind = (dev, T, rows, n, xdt, stages, cdt, sdt)
    base.test_gated(*kind)
    base.test_head_loss(*kind)
    if xdt in base.DT:
        base.test_gated_backward(*kind)
        base.test_gemm_backward(*kind)
        base.test_head_loss_backward(*kind)


def test_ignored_rows_of_any_content(dev):
    """NaN and infinities in tokens that do not count, in rows packed by two readings"""
    T, rows, n = 9, 40, 6144
    x = rows_of(640, T, n, "bf16")[0]
    m = Mat(641, rows, n, 1, books("fp16"))
    i0, i1, cb0, cb1, sc = m.on(dev)
    t = torch.tensor([3, -100, 4, -100, 5, -100, 0, rows - 1, -100])
    clean = x.clone()
    x[1], x[3, 7], x[5, n - 1], x[8, 4097] = math.nan, math.inf, -math.inf, math.nan
    clean[t == -100] = 0
    one = torch.ones(T, device=dev)
    rest = (i0, i1, cb0, cb1, sc, rows, n)
    out = []
    for v in (x, clean):
        loss, lse = K.vq_head_loss(v.to(dev), t.to(dev), *rest)
        dx, ds = K.vq_head_loss_backward(v.to(dev), t.to(dev), lse, one, *rest, scale_grad=True)
        out.append((loss, dx, ds))
    assert all(torch.equal(p, q) for p, q in zip(*out))
    assert (out[0][1][t == -100] == 0).all() and (out[0][0][t == -100] == 0).all()
