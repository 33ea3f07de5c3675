"""vq2_add_rms_norm and its backward pass on the GPU against the formulas in 64 bits.

Tolerances.  A row's sum of squares is a tree of fp32 additions, at most 32
of them in a thread and 8 above: its square root is off by at most 20 * 2^-24
of itself; with the additions, multiplications and conversions around it a
value u = h r w is within 32 * 2^-24 of itself (its h = x + residual is an
fp32 sum, off by 2^-24 of |x| + |residual|).  A stage of the transform adds
two values: after log2(hb) stages and the scale a value is off by at most
(log2(hb) + 34) * 2^-24 of the block's norm (scale sqrt(hb) = 1).  Rounding to 16
bits adds half a step, 2^-8 (bf16) or 2^-11 (fp16) of the value, and for fp16
below 2^-14 2^-25.
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
    """half a step of type t at ref"""
    return ref.abs() * {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[t] + (
        2.0 ** -25 if t == torch.float16 else 0.0)


def hadamard(v, hb):
    step, x = 1, v.reshape(-1, hb)
    while step < hb:
        a = x.reshape(-1, hb // (2 * step), 2, step)
        x = torch.stack([a[:, :, 0] + a[:, :, 1], a[:, :, 0] - a[:, :, 1]], 2).reshape(-1, hb)
        step *= 2
    return (x * hb ** -0.5).reshape(v.shape)


def case(seed, T, n, dtype, residual, hb, wdt="fp32", zero=False):
    g = synth.gen(seed)
    x = torch.randn(T, n, generator=g).to(DT[dtype])
    r = (torch.randn(T, n, generator=g) * 3).to(DT[dtype]) if residual else None
    w = (torch.randn(n, generator=g) * 0.2 + (0 if zero else 1)).to(DT[wdt])
    rot = {}
    if hb:
        rot = dict(perm=torch.randperm(n, generator=g).to(torch.int32), sign=synth.signs(seed + 1, n), hb=hb)
    return x, r, w, rot


def on(dev, rot):
    return {k: v.to(dev) if torch.is_tensor(v) else v for k, v in rot.items()}


def forward64(x, r, w, rot, eps, zero):
    """(h, y, size of a block's norm at each value)"""
    h = x.double() + (0 if r is None else r.double())
    u = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps) * (w.double() + (1 if zero else 0))
    if not rot:
        return h, u, torch.zeros_like(u)
    n, hb = h.shape[-1], rot["hb"]
    v = u if rot.get("perm") is None else u[:, rot["perm"].long()]
    if rot.get("sign") is not None:
        v = v * rot["sign"].double()
    size = v.reshape(-1, n // hb, hb).norm(dim=-1, keepdim=True).expand(-1, -1, hb).reshape(u.shape)
    return h, hadamard(v, hb), size


def err32(ref, size, hb):
    return 34 * E * ref.abs() + (math.log2(hb) + 34 if hb else 0) * E * size


SHAPES = [(1, 1, 0), (3, 7, 0), (5, 63, 0), (2, 64, 64), (9, 100, 0), (4, 192, 64), (6, 512, 512), (5, 513, 0), (7, 640, 128),
          (3, 1024, 1024), (2, 1000, 0), (4, 1536, 512), (1, 2048, 2048), (33, 2048, 0), (2, 2049, 0), (3, 2944, 128),
          (2, 4096, 4096), (3, 6144, 2048), (2, 6144, 0), (2, 8192, 8192), (2, 8192, 1024), (2, 8191, 0), (0, 64, 0)]


@pytest.mark.parametrize("T,n,hb", SHAPES)
@pytest.mark.parametrize("dtype,residual,odt", [("bf16", True, None), ("fp16", False, None), ("fp32", True, "bf16"),
                                                ("bf16", True, "fp32"), ("fp16", True, "fp16")])
def test_forward(dev, T, n, hb, dtype, residual, odt):
    x, r, w, rot = case(100 + n + T, T, n, dtype, residual, hb, "bf16" if dtype == "bf16" else "fp32", zero=residual)
    y, h, s = K.vq_add_rms_norm(x.to(dev), w.to(dev), None if r is None else r.to(dev), eps=1e-5, zero_centred=residual,
                                out_dtype=DT[odt] if odt else None, **on(dev, rot))
    assert s is None and y.dtype == DT[odt or dtype] and h.dtype == DT[dtype] and y.shape == x.shape
    h64, y64, size = forward64(x, r, w, rot, 1e-5, residual)
    mag = x.double().abs() + (0 if r is None else r.double().abs())
    assert ((h.cpu().double() - h64).abs() <= half(DT[dtype], h64) + E * mag).all()
    # (a value that the residual cancels is off by its addends' roundings, not its own)
    gain = (w.double() + (1 if residual else 0)).abs()
    scale = 1 / torch.sqrt(h64.pow(2).mean(-1, keepdim=True) + 1e-5)
    add = E * mag * scale * gain
    if hb:
        add = add.reshape(-1, n // hb, hb).norm(dim=-1, keepdim=True).expand(-1, -1, hb).reshape(add.shape) * math.sqrt(hb)
    tol = half(y.dtype, y64) + err32(y64, size, hb) + add
    off = (y.cpu().double() - y64).abs() - tol
    assert off.numel() == 0 or off.max() <= 0, float(off.max())


@pytest.mark.parametrize("T,n,hb", [(1, 64, 64), (5, 100, 0), (3, 801, 0), (4, 2048, 2048), (2, 6144, 2048), (9, 512, 256)])
@pytest.mark.parametrize("odt", [torch.int8, torch.float8_e4m3fn])
def test_8bit(dev, T, n, hb, odt):
    """y_scale is the largest magnitude / 127 (448); a value is off by half a
    step of the 8 bits, and by what fp32 is off."""
    x, r, w, rot = case(300 + n, T, n, "fp16", True, hb)
    y, h, s = K.vq_add_rms_norm(x.to(dev), w.to(dev), r.to(dev), out_dtype=odt, **on(dev, rot))
    assert y.dtype == odt and s.dtype == torch.float32 and s.shape == (T,)
    _, y64, size = forward64(x, r, w, rot, 1e-6, False)
    tol32 = err32(y64, size, hb) + 4 * E * y64.norm(dim=-1, keepdim=True)
    top = 127.0 if odt == torch.int8 else 448.0
    s64 = y64.abs().amax(-1) / top
    sc = s.cpu().double()
    assert ((sc - s64).abs() <= tol32.amax(-1) / top + 2 * E * s64).all()
    got = y.cpu().to(torch.float64 if odt == torch.int8 else torch.float32).double() * sc[:, None]
    # fp8: half a step is 2^-4 of the value, and 2^-10 of the scale below 2^-6
    step = 0.5 * sc[:, None] if odt == torch.int8 else torch.maximum(2.0 ** -4 * y64.abs(), 2.0 ** -10 * sc[:, None])
    assert ((got - y64).abs() <= step * (1 + 2.0 ** -20) + 2 * tol32).all()
    if odt == torch.int8:
        assert int(y.cpu().int().abs().max()) == 127


@pytest.mark.parametrize("hb", [0, 64])
@pytest.mark.parametrize("odt", [torch.int8, torch.float8_e4m3fn])
def test_8bit_of_tiny_rows(dev, hb, odt):
    """rows whose largest magnitude has a scale below 2^-126: that is their
    scale, and half a step of it (e4m3: half a step of a value, 2^-10 of the
    scale among its smallest numbers) is what y is off by, but for fp32's own
    subnormal steps before"""
    x = synth.activations(3, (5, 128), torch.float32) * 2.0 ** -134
    x[4] = 0
    y, _, sc = K.vq_add_rms_norm(x.to(dev), torch.ones(128, device=dev), out_dtype=odt, hb=hb, eps=1e-6)
    u = x.double() * 1e-6 ** -0.5
    if hb:
        h = torch.ones(1, 1, dtype=torch.float64)
        while h.shape[0] < hb:
            h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
        u = (u.view(5, 2, hb) @ h * hb ** -0.5).reshape(5, 128)
    assert (sc[:4].cpu() == 2.0 ** -126).all() and sc[4] == 0
    got = y.cpu().float().double() * sc.cpu().double()[:, None]
    step = 2.0 ** -127 if odt == torch.int8 else torch.maximum(2.0 ** -4 * u.abs(), torch.tensor(2.0 ** -136, dtype=torch.float64))
    # 128 values of up to 2^-149 of rounding each, and 2^-20 of the value
    assert ((got - u).abs() <= step + 2.0 ** -141 + 2.0 ** -20 * u.abs()).all()
    assert (y[4].float() == 0).all()


def test_8bit_odd_rows(dev):
    """a row of zeros has scale 0 and gives zeros; a NaN or an infinity shows in the row's scale, not in others"""
    x = torch.randn(4, 128, generator=synth.gen(5))
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    w = torch.ones(128)
    for kw in (dict(), dict(hb=128)):
        y, _, s = K.vq_add_rms_norm(x.to(dev), w.to(dev), out_dtype=torch.int8, eps=0.0 if not kw else 1e-6, **kw)
        s = s.cpu()
        assert math.isfinite(s[0]) and s[0] > 0 and math.isnan(s[2]) and not math.isfinite(s[3])
        if kw:
            assert s[1] == 0 and (y.cpu()[1] == 0).all()
        else:  # 0 / 0, as the formula has it
            assert math.isnan(s[1])


def backward64(dy, h, w, dh, rot, eps, zero):
    h, g = h.double(), dy.double()
    n = h.shape[-1]
    size = torch.zeros_like(g)
    if rot:
        hb = rot["hb"]
        size = g.reshape(-1, n // hb, hb).norm(dim=-1, keepdim=True).expand(-1, -1, hb).reshape(g.shape)
        g = hadamard(g, hb)
        if rot.get("sign") is not None:
            g = g * rot["sign"].double()
        if rot.get("perm") is not None:
            inv = torch.argsort(rot["perm"].long())
            g, size = g[:, inv], size[:, inv]
    gain = w.double() + (1 if zero else 0)
    r = 1 / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    dx = r * g * gain - h * r ** 3 * (g * gain * h).mean(-1, keepdim=True)
    if dh is not None:
        dx = dx + dh.double()
    return dx, (g * h * r).sum(0), g, r, gain, size


@pytest.mark.parametrize("T,n,hb", SHAPES)
@pytest.mark.parametrize("dtype,with_dh,ddt", [("bf16", True, "bf16"), ("fp32", False, "fp32"), ("fp16", True, "fp32")])
def test_backward(dev, T, n, hb, dtype, with_dh, ddt):
    h, dh, w, rot = case(500 + n + T, T, n, dtype, with_dh, hb, "fp32", zero=with_dh)
    dy = (torch.randn(T, n, generator=synth.gen(7 + n)) * 0.3).to(DT[ddt])
    dx, dw = K.vq_add_rms_norm_backward(dy.to(dev), h.to(dev), w.to(dev), None if dh is None else dh.to(dev), eps=1e-5,
                                        zero_centred=with_dh, **on(dev, rot))
    assert dx.dtype == DT[dtype] and dw.dtype == torch.float32
    dx64, dw64, g, r, gain, size = backward64(dy, h, w, dh, rot, 1e-5, with_dh)
    # g is off by the transform's error; the mean is a sum of n products,
    # each and their sums off by 48 * 2^-24 of their magnitudes
    eg = E * (g.abs() + (math.log2(hb) + 4 if hb else 0) * size)
    hh = h.double().abs()
    mean = (g.abs() * gain.abs() * hh).mean(-1, keepdim=True)
    emean = (eg * gain.abs() * hh).mean(-1, keepdim=True) + 80 * E * mean
    tol = r * gain.abs() * (eg + 40 * E * g.abs()) + hh * r ** 3 * emean + 4 * E * dx64.abs()
    if dh is not None:
        tol = tol + 2 * E * dh.double().abs()
    off = (dx.cpu().double() - dx64).abs() - tol - half(DT[dtype], dx64)
    assert off.numel() == 0 or off.max() <= 0, float(off.max())
    # rows are added one by one in a workgroup, then its sums: at most T of them
    tw = ((eg + (40 + T) * E * g.abs()) * hh * r).sum(0) + 1e-30
    assert ((dw.cpu().double() - dw64).abs() <= tw).all()


@pytest.mark.parametrize("hb", [0, 64])
def test_backward_against_differences(dev, hb):
    """(L(h + d) - L(h - d)) / 2 with L = sum(dy * y(h)) in 64 bits"""
    T, n = 3, 192
    h, _, w, rot = case(900, T, n, "fp32", False, hb)
    dy, d = torch.randn(2, T, n, generator=synth.gen(901)).double()
    dx, dw = K.vq_add_rms_norm_backward(dy.float().to(dev), h.to(dev), w.to(dev), **on(dev, rot))
    f = lambda hh, ww: (dy.float().double() * forward64(hh, None, ww, rot, 1e-6, False)[1]).sum()
    step = 1e-5
    num = (f(h.double() + step * d, w.double()) - f(h.double() - step * d, w.double())) / (2 * step)
    ana = (dx.cpu().double() * d).sum()
    # second differences: step^2; fp32: n values' roundings
    assert abs(num - ana) <= 1e-4 * (dx.cpu().double().abs() * d.abs()).sum()
    num = (f(h.double(), w.double() + step * d[0]) - f(h.double(), w.double() - step * d[0])) / (2 * step)
    assert abs(num - (dw.cpu().double() * d[0]).sum()) <= 1e-4 * (dw.cpu().double().abs() * d[0].abs()).sum()


def test_many_rows(dev):
    """more rows than a launch has workgroups, by the first and last of them and the sums"""
    T, n = 20001, 256
    x, r, w, rot = case(40, T, n, "bf16", True, 256, "bf16")
    y, h, _ = K.vq_add_rms_norm(x.to(dev), w.to(dev), r.to(dev), **on(dev, rot))
    _, y64, size = forward64(x, r, w, rot, 1e-6, False)
    mag = (x.double().abs() + r.double().abs()).norm(dim=-1, keepdim=True)
    off = (y.cpu().double() - y64).abs() - half(torch.bfloat16, y64) - err32(y64, size, 256) - 8 * E * mag
    assert off.max() <= 0
    a = K.vq_add_rms_norm_backward(y, h, w.to(dev), **on(dev, rot))
    b = K.vq_add_rms_norm_backward(y, h, w.to(dev), **on(dev, rot))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # a fixed order
    _, dw64, g, rr, _, sz = backward64(y.cpu(), h.cpu(), w, None, rot, 1e-6, False)
    tw = ((T + 60) * E * (g.abs() + sz) * h.cpu().double().abs() * rr).sum(0)
    assert ((a[1].cpu().double() - dw64).abs() <= tw).all()


def test_in_place_and_layouts(dev):
    x, r, w, rot = case(41, 6, 512, "bf16", True, 512, "bf16")
    x, r, w, rot = x.to(dev), r.to(dev), w.to(dev), on(dev, rot)
    y, h, _ = K.vq_add_rms_norm(x, w, r, **rot)
    r2 = r.clone()
    y2, h2, _ = K.vq_add_rms_norm(x, w, r2, h=r2, **rot)
    assert h2 is r2 and torch.equal(h, r2) and torch.equal(y, y2)
    # three dims, and rows that start between 16-byte borders (not rotated)
    y3, h3, _ = K.vq_add_rms_norm(x.view(2, 3, 512), w, r.view(2, 3, 512), **rot)
    assert torch.equal(y3.view(6, 512), y) and torch.equal(h3.view(6, 512), h)
    buf = torch.empty(6 * 512 + 1, dtype=x.dtype, device=dev)
    odd = buf[1:].view(6, 512)
    odd.copy_(x)
    a, ha, _ = K.vq_add_rms_norm(odd, w, r)
    b, hb_, _ = K.vq_add_rms_norm(x, w, r)
    assert torch.equal(ha, hb_)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * b.float().abs().max()  # a step apart at most
    # the tables alone: no permutation, no signs
    z, _, _ = K.vq_add_rms_norm(x, w, r, hb=512, out_dtype=torch.float32)
    u, _, _ = K.vq_add_rms_norm(x, w, r, out_dtype=torch.float32)
    v = K.vq_rht(u, hb=512)
    assert (z - v).abs().max() <= 64 * E * u.norm(dim=-1).max()
    # the same rotation as the products' own
    z, _, _ = K.vq_add_rms_norm(x, w, r, out_dtype=torch.float32, **rot)
    v = K.vq_rht(u, rot["perm"], rot["sign"], 512)
    assert (z - v).abs().max() <= 64 * E * u.norm(dim=-1).max()


def test_graph_and_streams(dev):
    x, r, w, rot = (t if not torch.is_tensor(t) else t.to(dev) for t in case(42, 5, 2048, "bf16", True, 2048, "bf16"))
    rot = on(dev, rot)

    def step(x, r):
        y, h, _ = K.vq_add_rms_norm(x, w, r, **rot)
        return (y, h, *K.vq_add_rms_norm_backward(y, h, w, h, **rot))

    g = DecodeStepGraph(step, [x, r])
    for k in range(4):
        xk = torch.randn(5, 2048, generator=synth.gen(50 + k)).to(torch.bfloat16).to(dev)
        want = step(xk, r)
        torch.cuda.synchronize()
        for a, b in zip(g(xk, r), want):
            assert torch.equal(a, b)
        torch.zeros(1 << 20, device=dev).add_(1).sum().item()
    side = torch.cuda.Stream()
    want = step(x, r)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(dev):
    x = torch.zeros(2, 128, device=dev, dtype=torch.bfloat16)
    w = torch.ones(128, device=dev)
    bad = [
        (dict(x=x, weight=w[:64]), "expected 128"),
        (dict(x=x, weight=w, residual=x[:1]), "residual"),
        (dict(x=x, weight=w, residual=x.float()), "residual"),
        (dict(x=x, weight=w, h=x), "without a residual"),
        (dict(x=x, weight=w, perm=torch.arange(128, device=dev, dtype=torch.int32)), "block hb"),
        (dict(x=x, weight=w, hb=48), "power of two"),
        (dict(x=x, weight=w, hb=256), "power of two"),
        (dict(x=x, weight=w, hb=32), "power of two"),
        (dict(x=x, weight=w, hb=64, perm=torch.arange(64, device=dev, dtype=torch.int32)), "perm"),
        (dict(x=x, weight=w, eps=-1.0), "eps"),
        (dict(x=x.t(), weight=w[:2]), "contiguous"),
        (dict(x=x, weight=w.cpu()), "GPU"),
        (dict(x=torch.zeros(1, 8193, device=dev), weight=torch.zeros(8193, device=dev)), "8193"),
        (dict(x=x.to(torch.int32), weight=w, out_dtype=torch.bfloat16), "dtype"),
    ]
    for kw, match in bad:
        with pytest.raises(K.Vq2Error, match=match):
            K.vq_add_rms_norm(**kw)
    with pytest.raises(K.Vq2Error, match="dy"):
        K.vq_add_rms_norm_backward(x[:1], x, w)
    with pytest.raises(K.Vq2Error, match="dh"):
        K.vq_add_rms_norm_backward(x, x, w, x.float())
