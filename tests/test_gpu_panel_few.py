"""Few tokens through packed matrices (the gated block and the head's loss,
whose centroids are gathered straight into the matrix cores' operands) and
wide rows, where the common sizes do not reach."""
import math

import pytest
import torch

from compressai_amd import kernels as K, synth
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
