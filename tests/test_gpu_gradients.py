"""Gradients through packed layers where a type, a size or a mode is out of the
ordinary, against torch's autograd in 64 bits on the dequantized matrices."""
import pytest
import torch

from compressai_amd import kernels as K, synth, tuning as T
from compressai_amd.runtime import PackedLinear, PackedLMHead, PackedMLP, PackedProjections

pytestmark = pytest.mark.gpu
H, I, V = 256, 512, 600


def books(dev, dtype=torch.float16):
    return {"16": synth.codebook(1).to(dev, dtype), "16_16": (synth.codebook(2) * 0.3).to(dev, dtype)}


def lin(seed, out, n, tag, cbs, cfg=(16,), gain=1.0, **kw):
    m = synth.vq_matrix(seed, out, n, bpw=2 if len(cfg) == 1 else 4)
    idx = [m["idx0"]] + ([m["idx1"]] if len(cfg) == 2 else [])
    return PackedLinear((out, n), cfg, tag, idx, m["scale"].float() * (gain * (8 / n) ** 0.5), cbs, cbs["16"].device, **kw)


def weight64(m):
    w = m._cbs[0]["16"].double()[m.idx0.long() & 0xFFFF]
    if len(m.cfg) == 2:
        w = w + m._cbs[0]["16_16"].double()[m.idx1.long() & 0xFFFF]
    return w.reshape(m.out, m.n)


def rot64(rot):
    n, hb = rot.n, rot.hb
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < hb:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    m = torch.block_diag(*[h * hb ** -0.5] * (n // hb)).to(rot.perm.device)
    return lambda x: (x[:, rot.perm] * rot.sign.double()) @ m


def linear64(m, x, scale=None):
    return rot64(m.rot)(x) @ (weight64(m) * (m.scale.detach().double() if scale is None else scale)[:, None]).t()


def close(got, want, rel):
    """the difference's norm over the norm"""
    err = (got.double() - want).norm() / want.norm()
    assert err <= rel, float(err)


@pytest.mark.parametrize("rows", [1, 5])
def test_mlp_result_type_under_grad(dev, rows):
    """the block's result leaves in the type that is asked for, with a gradient as without: fp32 results of 16-bit rows
    beyond fp16's range, in steps finer than the rows' type.  Roundings to the rows' type: x rotated, act, act rotated,
    each as often again for what it does to the values it meets"""
    cbs = books(dev)
    mlp = PackedMLP(lin(10, I, H, "mlp.in", cbs), lin(20, I, H, "mlp.in", cbs), lin(30, H, I, "mlp.down", cbs, gain=2.0 ** 20))
    for dtype in (torch.float16, torch.bfloat16):
        x = synth.activations(rows, (rows, H), dtype).to(dev)
        want = x.double()
        r = [linear64(m, want) for m in (mlp.gate, mlp.up)]
        want = linear64(mlp.down, torch.nn.functional.silu(r[0]) * r[1])
        with torch.no_grad():
            plain = mlp(x, out_dtype=torch.float32)
        y = mlp(x.requires_grad_(), out_dtype=torch.float32)
        for v in (plain, y):
            assert v.dtype == torch.float32 and torch.isfinite(v).all() and v.abs().max() > 2.0 ** 16
            assert (v != v.to(dtype).float()).any()
            close(v, want, 6 * torch.finfo(dtype).eps / 2)
        # (in fp16, too, the gradient of 2^20 W comes back in range)
        (y * 2.0 ** -20).sum().backward()
        assert torch.isfinite(x.grad).all() and x.grad.abs().max() > 0
