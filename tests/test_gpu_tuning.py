"""Gradients through packed layers (compressai_amd.tuning, PackedMLP,
PackedLMHead.loss) against torch's autograd in 64 bits on the dequantized
matrices, with the same rounding of rotated rows; and a training step of a small
model built from them."""
import pytest
import torch

from compressai_amd import kernels as K, synth, tuning as T
from compressai_amd.graph import DecodeStepGraph
from compressai_amd.runtime import PackedLinear, PackedLMHead, PackedMLP
from compressai_amd.rot import get_rot

pytestmark = pytest.mark.gpu
H, I, V = 256, 512, 600


def _lin(seed, out, n, tag, dev, cfg=(16,), **kw):
    cbs = _lin.cbs
    if not cbs:
        cbs.update({"16": synth.codebook(1).to(dev), "16_16": (synth.codebook(2) * 0.3).to(torch.float16).to(dev)})
    m = synth.vq_matrix(seed, out, n, bpw=2 if len(cfg) == 1 else 4)
    idx = [m["idx0"]] + ([m["idx1"]] if len(cfg) == 2 else [])
    return PackedLinear((out, n), cfg, tag, idx, m["scale"] * (8 / n) ** 0.5, cbs, dev, **kw)


_lin.cbs = {}


def _weight64(lin):
    w = _lin.cbs["16"].double()[lin.idx0.long() & 0xFFFF]
    if len(lin.cfg) == 2:
        w = w + _lin.cbs["16_16"].double()[lin.idx1.long() & 0xFFFF]
    return w.reshape(lin.out, lin.n)


def _rot64(rot):
    n, hb = rot.n, rot.hb
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < hb:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    m = torch.block_diag(*[h * hb ** -0.5] * (n // hb)).to(rot.perm.device)
    return lambda x: (x[:, rot.perm] * rot.sign.double()) @ m


def _close(got, want, rel):
    """difference's norm over the norm: rel by the roundings named at the call"""
    err = (got.double() - want).norm() / want.norm()
    assert err <= rel, float(err)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T_", [1, 5, 150])
def test_mlp(dev, dtype, activation, T_):
    """forward and gradients; half a step of the type, at most, at each of x
    rotated, act, act rotated, y (forward) and dy, d act rotated, d act, dx
    rotated, dx (backward): 10 of them, and as many again for what their
    errors do to the values that meet them"""
    half = torch.finfo(dtype).eps / 2
    gate, up = _lin(10, I, H, "mlp.in", dev, (16, 16)), _lin(20, I, H, "mlp.in", dev, (16, 16))
    down = _lin(30, H, I, "mlp.down", dev, (16, 16))
    mlp = PackedMLP(gate, up, down, activation)
    for m in (gate, up, down):
        m.scale = m.scale.float().requires_grad_()
    x = synth.activations(T_, (T_, H), dtype).to(dev).requires_grad_()
    dy = synth.activations(T_ + 1, (T_, H), dtype).to(dev)
    y = mlp(x)
    y.backward(dy)
    x64 = x.detach().double().requires_grad_()
    s64 = [m.scale.detach().double().requires_grad_() for m in (gate, up, down)]
    f = torch.nn.functional.silu if activation == "silu" else lambda v: torch.nn.functional.gelu(v, approximate="tanh")
    r1, r2 = _rot64(gate.rot), _rot64(down.rot)
    xr = r1(x64)
    act = f(xr @ (_weight64(gate) * s64[0][:, None]).t()) * (xr @ (_weight64(up) * s64[1][:, None]).t())
    want = r2(act) @ (_weight64(down) * s64[2][:, None]).t()
    want.backward(dy.double())
    _close(y, want, 20 * half)
    _close(x.grad, x64.grad, 20 * half)
    for m, s in zip((gate, up, down), s64):
        assert m.scale.grad.dtype == torch.float32
        _close(m.scale.grad, s.grad, 20 * half)
    with torch.no_grad():
        _close(mlp(x), want, 20 * half)  # (one row: the sorted layout where it is)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_head_loss(dev, dtype):
    half = torch.finfo(torch.float16 if dtype == torch.float32 else dtype).eps / 2
    lin = _lin(40, V, H, "head", dev)
    lin.scale = lin.scale.float().requires_grad_()
    head = PackedLMHead(lin)
    x = synth.activations(41, (3, 20, H), dtype).to(dev).requires_grad_()
    t = torch.randint(0, V, (3, 20), generator=synth.gen(42)).to(dev)
    t[0, :7] = -100
    loss = head.loss(x, t)
    assert loss.shape == (60,) and loss.dtype == torch.float32 and (loss[:7] == 0).all()
    (loss.sum() / 53).backward()
    x64 = x.detach().double().requires_grad_()
    s64 = lin.scale.detach().double().requires_grad_()
    z = _rot64(lin.rot)(x64.reshape(-1, H)) @ (_weight64(lin) * s64[:, None]).t()
    want = torch.nn.functional.cross_entropy(z, t.reshape(-1), ignore_index=-100, reduction="none")
    (want.sum() / 53).backward()
    # roundings: x rotated (in the logits, and so in every probability), dx rotated, dx
    _close(loss, want, 20 * half)
    _close(x.grad, x64.grad, 20 * half)
    _close(lin.scale.grad, s64.grad, 20 * half)
    with torch.no_grad():
        assert torch.equal(head.loss(x, t), loss)


def test_norm(dev):
    rot = get_rot("mlp.in", H, dev)
    x, r = (synth.activations(k, (7, H), torch.bfloat16).to(dev).requires_grad_() for k in (50, 51))
    w = (synth.activations(52, H, torch.float32) * 0.1 + 1).to(dev).requires_grad_()
    dy, dh = (synth.activations(k, (7, H), torch.bfloat16).to(dev) for k in (53, 54))
    y, h = T.add_rms_norm(x, w, r, rot=rot)
    torch.autograd.backward([y, h], [dy, dh])
    a, b, c = (v.detach().double().requires_grad_() for v in (x, r, w))
    h64 = a + b
    y64 = _rot64(rot)(h64 / torch.sqrt(h64.pow(2).mean(-1, keepdim=True) + 1e-6) * c)
    torch.autograd.backward([y64, h64], [dy.double(), dh.double()])
    half = 2.0 ** -8
    for got, want in ((y, y64), (h, h64), (x.grad, a.grad), (r.grad, b.grad), (w.grad, c.grad)):
        _close(got, want, 4 * half)  # (the backward pass starts from the rounded h)
    assert torch.equal(x.grad, r.grad)
    # h alone, and the norm without a residual
    x.grad = None
    y, h = T.add_rms_norm(x, w, r)
    h.backward(dh)
    assert torch.equal(x.grad, dh)
    x.grad = None
    y, h = T.add_rms_norm(x, w)
    assert h is x
    y.backward(dy)
    z = x.detach().double().requires_grad_()
    (z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + 1e-6) * c.detach()).backward(dy.double())
    _close(x.grad, z.grad, 2 * half)


def test_refusals(dev):
    gate, up = _lin(10, I, H, "mlp.in", dev), _lin(20, I, H, "mlp.in", dev)
    down = _lin(30, H, I, "mlp.down", dev)
    with pytest.raises(K.Vq2Error, match="share shape"):
        PackedMLP(gate, _lin(20, I, H, "other", dev), down)
    with pytest.raises(K.Vq2Error, match="takes"):
        PackedMLP(gate, up, gate)
    with pytest.raises(K.Vq2Error, match="activation"):
        PackedMLP(gate, up, down, "relu")
    with pytest.raises(K.Vq2Error, match="float16"):
        T.linear(gate, torch.zeros(2, H, device=dev))
    big = _lin(60, 4096, 2048, "big", dev)
    big.release_planes()
    with pytest.raises(K.Vq2Error, match="released"):
        PackedLMHead(big).loss(torch.zeros(2, 2048, device=dev, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(K.Vq2Error, match="released"):
        T.linear(big, torch.zeros(2, 2048, device=dev, dtype=torch.bfloat16))


def test_training_step(dev):
    """a model of an embedding, two blocks and a head: a step's gradients are
    there, finite and the same on a second run, and small steps along them go down
    as the gradient says: the loss changes by -step |g|^2 up to second order and
    bf16's rounding"""
    torch.manual_seed(0)
    blocks = [(torch.ones(H, device=dev), PackedMLP(_lin(70 + 10 * k, I, H, "mlp.in", dev), _lin(71 + 10 * k, I, H, "mlp.in", dev),
                                                      _lin(72 + 10 * k, H, I, "mlp.down", dev))) for k in range(2)]
    head = PackedLMHead(_lin(95, V, H, "head", dev))
    emb = torch.randn(V, H, generator=synth.gen(1)).to(dev)
    params = [emb] + [w for w, _ in blocks]
    for b in blocks:
        for m in (b[1].gate, b[1].up, b[1].down):
            m.scale = m.scale.float()
            params.append(m.scale)
    for p in params:
        p.requires_grad_()
    tok = torch.randint(0, V, (64,), generator=synth.gen(2)).to(dev)

    def loss():
        h, x = None, emb[tok[:-1]].to(torch.bfloat16)
        for w, mlp in blocks:
            y, h = T.add_rms_norm(x, w, h if h is not None else torch.zeros_like(x))
            x = mlp(y)
        y, _ = T.add_rms_norm(x, torch.ones(H, device=dev), h)
        return head.loss(y, tok[1:]).mean()

    a = torch.autograd.grad(loss(), params)
    b = torch.autograd.grad(loss(), params)
    # (index_put of the embedding's gradient adds in any order)
    for k, (p, q) in enumerate(zip(a, b)):
        assert torch.isfinite(p).all() and p.abs().max() > 0
        assert k == 0 or torch.equal(p, q)


@pytest.mark.parametrize("rows", [1, 40])
def test_captured_step(dev, rows):
    """a block and the head's loss, forward and backward, captured: every replay
    gives the eager result, also with eager steps of the same layers in between"""
    gate, up = _lin(110, I, H, "mlp.in", dev), _lin(111, I, H, "mlp.in", dev)
    mlp = PackedMLP(gate, up, _lin(112, H, I, "mlp.down", dev))
    head = PackedLMHead(_lin(113, V, H, "head", dev))
    gate.scale, up.scale = gate.scale.float(), up.scale.float()
    w = torch.ones(H, device=dev)

    def step(x, r, tok, up_):
        leaves = [t.detach().requires_grad_() for t in (x, w, gate.scale)]
        gate.scale, keep = leaves[2], gate.scale
        y, h = T.add_rms_norm(leaves[0], leaves[1], r)
        z, _ = T.add_rms_norm(mlp(y), leaves[1], h)
        loss = head.loss(z, tok)
        gate.scale = keep
        return [loss.detach(), *torch.autograd.grad(loss, leaves, up_)]

    def inputs(k):
        return (synth.activations(120 + k, (rows, H), torch.bfloat16).to(dev), synth.activations(130 + k, (rows, H), torch.bfloat16).to(dev),
                torch.randint(0, V, (rows,), generator=synth.gen(140 + k)).to(dev),
                synth.activations(150 + k, (rows,), torch.float32).to(dev))

    graph = DecodeStepGraph(step, inputs(0))
    for k in range(4):
        a = inputs(k)
        got = [t.clone() for t in graph(*a)]
        want = step(*a)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert all(torch.isfinite(p).all() for p in got)
