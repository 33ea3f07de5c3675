"""vq2_sample on the GPU against the fp64 oracle: tokens exactly, log
probabilities to the rounding of their fp32 result plus that of the total,
a sum of V whole numbers of 2^-42, each off by at most half of one, over a
largest weight of 1: |lp| 2^-24 + V 2^-43 + 2^-40 for the 64-bit logarithms."""
import numpy as np
import pytest
import torch

from compressai_amd import kernels as K, synth
from compressai_amd.graph import DecodeStepGraph
from oracle import selection as S

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _logits(seed, B, V, dtype="fp32", steep=None):
    """A power law over tokens, steep or flat, with noise."""
    g = synth.gen(seed)
    s = torch.rand(B, 1, generator=g) * 1.8 + 0.7 if steep is None else steep
    x = 16.0 - s * (torch.rand(B, V, generator=g) * V + 2.0).log() + 0.4 * torch.randn(B, V, generator=g)
    return x.to(DT[dtype])


def _check(got, logits, u, **kw):
    idx, lp = (t.cpu().numpy() for t in got)
    host = lambda v: v.cpu().double().numpy() if torch.is_tensor(v) else np.float32(v).astype(np.float64)
    ref_idx, ref_lp = S.sample(logits.float().cpu().numpy(), host(u), **{k: host(v) for k, v in kw.items()})
    assert idx.dtype == np.int64 and lp.dtype == np.float32
    assert np.array_equal(idx, ref_idx)
    live = ref_idx >= 0
    assert np.isnan(lp[~live]).all()
    tol = np.abs(ref_lp[live]) * 2.0 ** -24 + logits.shape[-1] * 2.0 ** -43 + 2.0 ** -40
    off = np.abs(lp[live] - ref_lp[live]) > tol
    assert not off.any(), (lp[live][off][:5], ref_lp[live][off][:5])


SETTINGS = [
    dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=50, top_p=0.9, temperature=0.7),
    dict(top_p=0.95), dict(top_p=0.3, temperature=1.4), dict(min_p=0.05), dict(top_p=0.9, min_p=0.02, temperature=1.1),
    dict(top_k=700, top_p=0.99, min_p=0.001), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0),
    dict(top_k=3000, temperature=2.0), dict(top_p=0.9999), dict(temperature=1e-6), dict(temperature=50.0, top_p=0.5),
]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("B,V,dtype", [
    (1, 5000, "fp32"), (3, 1, "bf16"), (2, 7, "fp32"), (4, 4099, "bf16"), (9, 1000, "fp16"), (2, 32000, "bf16"), (5, 64, "fp32")])
def test_settings(dev, B, V, dtype, kw):
    x = _logits(8000 + V, B, V, dtype)
    u = torch.rand(B, generator=synth.gen(8001 + B))
    _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9, temperature=0.7), dict(top_p=0.95), dict(top_p=0.9, min_p=0.01),
                                dict(top_k=1000), dict(top_k=100000, top_p=0.8)], ids=str)
@pytest.mark.parametrize("dtype,steep", [("fp32", 1.2), ("bf16", 1.2), ("fp32", 0.1), ("bf16", 0.1), ("fp16", 2.5)])
def test_whole_vocabulary(dev, dtype, steep, kw):
    """Peaked rows and rows nearly flat, whose kept sets are long."""
    x = _logits(8100, 2, 151936, dtype, steep)
    u = torch.tensor([0.137, 0.861])
    _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


@pytest.mark.parametrize("B", [1, 2, 31, 257, 700])
def test_row_counts_and_settings_by_row(dev, B):
    V = 1500
    g = synth.gen(8200 + B)
    x = _logits(8201, B, V, "bf16")
    x[:, V - 40:] = -float("inf")
    pick = lambda lo, hi, off: torch.where(torch.rand(B, generator=g) < 0.4, torch.tensor(off), torch.rand(B, generator=g) * (hi - lo) + lo)
    kw = dict(temperature=pick(0.4, 1.5, 0.0), top_k=pick(1, 200, 0.0).to(torch.int32), top_p=pick(0.3, 0.99, 1.0),
              min_p=pick(0.01, 0.2, 0.0))
    u = torch.rand(B, generator=g)
    _check(K.vq_sample(x.to(dev), u.to(dev), **{k: v.to(dev) for k, v in kw.items()}), x, u, **kw)
    # one setting by row beside common ones
    _check(K.vq_sample(x.to(dev), u.to(dev), top_k=kw["top_k"].to(dev), top_p=0.9), x, u, top_k=kw["top_k"], top_p=0.9)


def test_settings_outside_their_range_by_row(dev):
    """On the device nothing can refuse them: each acts as the nearest inside."""
    x = _logits(8250, 8, 900)
    u = torch.rand(8, generator=synth.gen(8251))
    nan = float("nan")
    f = lambda *v: torch.tensor(v, device=dev)
    got = K.vq_sample(x.to(dev), u.to(dev), temperature=f(-1.0, nan, 1, 1, 1, 1, 1, 1), top_p=f(1, 1, -2.0, nan, 7.0, 1, 1, 1),
                      min_p=f(0, 0, 0, 0, 0, -1.0, 3.0, nan), top_k=torch.tensor([0, 0, 0, 0, 0, 0, 0, -5], dtype=torch.int32, device=dev))
    _check(got, x, u, temperature=torch.tensor([0.0, 0, 1, 1, 1, 1, 1, 1]), top_p=torch.tensor([1.0, 1, 0, 1, 1, 1, 1, 1]),
           min_p=torch.tensor([0.0, 0, 0, 0, 0, 0, 1, 1]))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=5), dict(top_k=1), dict(top_p=0.5), dict(top_k=700, top_p=0.25), dict(min_p=0.5),
                                dict(top_p=0.999), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("V", [7, 1023, 20000, 70001])
def test_ties(dev, V, kw):
    """Rows of one value, of two, of zeros of both signs: the lower columns
    stay, and the draw of an even row is floor(u n).  Weights are 1 or
    exp(-1) (rounded the same by any summation of so few values)."""
    x = torch.zeros(5, V)
    x[1, ::3] = 1.0
    x[2, 1::2] = -0.0
    x[3] = torch.finfo(torch.float32).min
    x[4, : V // 2] = -1.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999])
    _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


def test_absent_columns(dev):
    inf, nan = float("inf"), float("nan")
    V = 3001
    x = _logits(8300, 12, V)
    x[0] = -inf
    x[1] = nan
    x[2, :-1] = -inf
    x[3, 1:] = nan
    x[4, 100] = inf
    x[5, ::7] = inf
    x[6, ::2] = -inf
    x[7, ::3] = nan
    x[8, 5:] = torch.finfo(torch.float32).min
    x[9, : V - 1] = -inf
    x[10] = inf
    x[11, 17] = nan
    u = torch.rand(12, generator=synth.gen(8301))
    for kw in (dict(), dict(top_k=20), dict(top_p=0.8), dict(min_p=0.1, temperature=0.5), dict(temperature=0.0), dict(top_k=2000, top_p=0.9)):
        _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


def test_borders_of_u(dev):
    x = _logits(8400, 6, 2000)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, 2.0, 2.0 ** -60])
    for kw in (dict(), dict(top_k=30), dict(top_p=0.9), dict(min_p=0.1)):
        _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


def test_frequencies(dev):
    """Evenly spaced numbers draw each kept token as often as its weight
    says, to one draw."""
    n, V = 4096, 50
    x = _logits(8500, 1, V)
    u = (torch.arange(n) + 0.5) / n
    for kw in (dict(), dict(temperature=0.6), dict(top_k=9), dict(top_p=0.8)):
        idx, lp = K.vq_sample(x.expand(n, V).contiguous().to(dev), u.to(dev), **kw)
        kept = S.sample_row(x[0].numpy(), 0.5, **kw)[2]
        share = np.bincount(idx.cpu().numpy(), minlength=V) / n
        assert np.abs(share - kept / kept.sum()).max() <= 1.0 / n + 1e-12
        assert np.allclose(np.exp(lp.cpu().numpy()), (kept / kept.sum())[idx.cpu().numpy()], rtol=1e-5)


def test_strides(dev):
    B, V = 5, 4001
    for dtype in DT:
        wide = _logits(8600, 2 * B, V + 300, dtype).to(dev)
        u = torch.rand(B, generator=synth.gen(8601))
        for view in (wide[::2, 3:3 + V], wide[:B, 1:V + 1], wide[:B, :V]):
            for kw in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.9)):
                _check(K.vq_sample(view, u.to(dev), **kw), view, u, **kw)
    x = _logits(8602, 6, 100)
    assert torch.equal(K.vq_sample(x.view(2, 3, 100).to(dev), torch.full((6,), 0.5, device=dev))[0],
                       K.vq_sample(x.to(dev), torch.full((6,), 0.5, device=dev))[0])
    idx, lp = K.vq_sample(wide[:0, :V], torch.zeros(0, device=dev))
    assert idx.shape == (0,) and lp.shape == (0,)


def test_refusals(dev):
    x, u = torch.zeros(4, 64, device=dev), torch.zeros(4, device=dev)
    f = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt, device=dev)
    for b in (dict(u=f(3)), dict(u=f(4, torch.float64)), dict(u=u.cpu()), dict(temperature=-1.0), dict(top_p=-0.1),
              dict(min_p=1.1), dict(top_k=-2), dict(temperature=f(3)), dict(top_k=f(4)), dict(top_k=f(4, torch.int64)),
              dict(top_p=f(8)[::2]), dict(min_p=f(4).cpu()), dict(logits=x.to(torch.int32)), dict(logits=x.t()),
              dict(logits=x[:, ::2]), dict(logits=x[:1].expand(4, 64)), dict(logits=x[:, :0]),
              dict(temperature=float("nan"))):
        with pytest.raises(K.Vq2Error):
            K.vq_sample(**dict(dict(logits=x, u=u), **b))


@pytest.mark.parametrize("B,V", [(1, 151936), (40, 9000)])
def test_streams_graphs_and_repeats(dev, B, V):
    """Another stream, two streams at once, a captured graph replayed among
    eager calls: the same results, bit for bit."""
    xs = [_logits(8700 + i, B, V, "bf16").to(dev) for i in range(3)]
    u = torch.rand(B, generator=synth.gen(8710)).to(dev)
    for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95)):
        refs = [K.vq_sample(x, u, **kw) for x in xs]
        torch.cuda.synchronize(dev)
        sides = [torch.cuda.Stream(dev) for _ in xs]
        got = []
        for _ in range(4):
            for x, s in zip(xs, sides):
                with torch.cuda.stream(s):
                    got.append(K.vq_sample(x, u, **kw))
        torch.cuda.synchronize(dev)
        for i, g in enumerate(got):
            assert torch.equal(g[0], refs[i % 3][0]) and torch.equal(g[1], refs[i % 3][1])
        steps = [DecodeStepGraph(lambda x: K.vq_sample(x, u, **kw), [xs[0]]) for _ in range(2)]
        for i in (0, 1, 2, 2, 0, 1):
            for step in steps:
                g = step(xs[i])
                torch.cuda.synchronize(dev)
                assert torch.equal(g[0], refs[i][0]) and torch.equal(g[1], refs[i][1])
            K.vq_sample(xs[1], u, **kw)


def test_head_sample(dev):
    """PackedLMHead.sample draws from the head's fp32 logits, at every batch
    size the head has a path for."""
    from compressai_amd.runtime import PackedLinear, PackedLMHead

    rows, n = 4000, 512
    m = synth.vq_matrix(8800, rows, n, bpw=2)
    lin = PackedLinear((rows, n), (16,), "head", [m["idx0"]], m["scale"], {"16": synth.codebook(8801).to(dev)}, dev)
    head = PackedLMHead(lin)
    for B in (1, 2, 4, 9):
        h = synth.activations(8810 + B, (B, n)).to(dev)
        u = torch.rand(B, generator=synth.gen(8811)).to(dev)
        logits = lin(h, out_dtype=torch.float32)
        for kw in (dict(), dict(temperature=0.7, top_k=50, top_p=0.9), dict(temperature=torch.full((B,), 0.5, device=dev), min_p=0.1)):
            got = head.sample(h, u, **kw)
            _check(got, logits, u, **kw)
        assert torch.equal(head.sample(h, u, temperature=0.0)[0], logits.argmax(-1))


@pytest.mark.parametrize("temperature", [1e-3, 1e-9, 1e-30, 1e-44, 1e6, 1e30, float("inf")])
@pytest.mark.parametrize("dtype", list(DT))
def test_extreme_temperatures(dev, dtype, temperature):
    """Differences of logits times 1 / temperature leave the range of 64-bit
    weights (one entry counts) or vanish in it (all count alike); logits near
    one another, near zero and huge.  (An infinite
    temperature counts as the largest finite one.  Beside an infinite logit
    every finite one weighs nothing, however high the temperature.)"""
    g = synth.gen(8900)
    x = torch.randn(8, 5000, generator=g)
    x[1] = 16.0 + 1e-6 * x[1]
    x[2] *= 1e-20
    x[3] *= 1e4
    x[4, ::2] = -float("inf")
    x[5, 4000] = float("inf")
    x[6] = -60000.0
    x = x.to(DT[dtype])
    u = torch.rand(8, generator=g)
    t = torch.tensor(min(temperature, torch.finfo(torch.float32).max), dtype=torch.float32)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.7), dict(min_p=0.2), dict(top_k=4000, top_p=0.5, min_p=0.01)):
        _check(K.vq_sample(x.to(dev), u.to(dev), temperature=temperature, **kw), x, u, temperature=t, **kw)


@pytest.mark.parametrize("order", ["descending", "ascending"])
@pytest.mark.parametrize("kw", [dict(top_k=50), dict(top_p=0.95), dict(min_p=0.001), dict(top_k=2500), dict()], ids=str)
def test_sorted_vocabularies(dev, order, kw):
    """Vocabularies sorted by frequency: the likely tokens stand side by
    side, in the first or the last slice of the row alone."""
    x, _ = torch.sort(_logits(8950, 3, 100003, "fp32", 1.3), dim=-1, descending=order == "descending")
    u = torch.tensor([0.01, 0.5, 0.99])
    _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


def test_offsets_past_32_bits(dev):
    """Rows more than 2^31 elements apart."""
    stride, V = (1 << 31) + 8, 3000
    buf = torch.empty(stride + V + 1, dtype=torch.bfloat16, device=dev)
    x = _logits(8960, 2, V, "bf16")
    view = buf.as_strided((2, V), (stride, 1), 1)
    view.copy_(x.to(dev))
    u = torch.tensor([0.3, 0.7])
    for kw in (dict(), dict(top_k=40), dict(top_p=0.9)):
        _check(K.vq_sample(view, u.to(dev), **kw), x, u, **kw)


def test_many_rows(dev):
    """Rows in the last places of the grid."""
    B, V = 65535, 24
    x = _logits(8970, B, V, "bf16")
    u = torch.rand(B, generator=synth.gen(8971))
    for kw in (dict(), dict(top_k=5), dict(top_p=0.8)):
        idx, lp = K.vq_sample(x.to(dev), u.to(dev), **kw)
        pick = torch.randint(0, B, (300,), generator=synth.gen(8972))
        pick[:2] = torch.tensor([0, B - 1])
        _check((idx.cpu()[pick], lp.cpu()[pick]), x[pick], u[pick], **kw)
    with pytest.raises(K.Vq2Error, match="rows"):
        K.vq_sample(torch.zeros(65536, 4, device=dev), torch.zeros(65536, device=dev))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=30, top_p=0.9), dict(top_p=0.9)], ids=str)
def test_native_and_python_entries_agree(dev, kw, monkeypatch):
    """The native twin and the Python entry: the same launches; a call that the
    twin declines (numpy settings) is the Python entry's."""
    from compressai_amd import _lib

    x = _logits(8980, 4, 7001, "fp16").to(dev)
    u = torch.rand(4, generator=synth.gen(8981)).to(dev)
    native = _lib.host().sample(x, u, *[kw.get(k, d) for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))])
    assert native is not None
    got = K.vq_sample(x, u, **{k: np.float32(v) if k == "top_p" else v for k, v in kw.items()})
    assert all(torch.equal(a, b) for a, b in zip(native, got))
    assert _lib.host().sample(x, u, np.float32(1.0), 0, 1.0, 0.0) is None
    assert all(torch.equal(a, b) for a, b in zip(K.vq_sample(x, u, temperature=np.float32(1.0)), K.vq_sample(x, u)))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=5000, top_p=0.7),
                                dict(temperature=0.0), dict(temperature=3e38)], ids=str)
def test_infinite_logits(dev, dtype, kw):
    """+inf next to the type's largest finite logit, several of them, rows of
    nothing else, and longer than the lists hold."""
    V = 20000
    x = torch.randn(6, V, generator=synth.gen(9000)).to(DT[dtype])
    big = torch.finfo(DT[dtype]).max
    x[0, 3], x[0, 9] = big, float("inf")
    x[1, [5, 700, 19999]] = float("inf")
    x[2, :10] = big
    x[3] = float("inf")
    x[4, ::2] = float("inf")
    x[5] = -float("inf")
    x[5, 77] = float("inf")
    for at in (0.0, 0.4, 0.999):
        u = torch.full((6,), at)
        _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.9999), dict(min_p=1e-9)], ids=str)
def test_units_without_weight(dev, dtype, kw):
    """u = 0 is the first column with a weight: what is ahead of it lies more
    than 64-bit weights hold below the maximum (e^-6000 in total)."""
    V = 30000
    x = torch.full((3, V), -6000.0)
    x[0, 20000:] = 0.0
    x[1, 29999] = 0.0
    x[2, 15000:] = 1.0
    x = x.to(DT[dtype])
    u = torch.zeros(3)
    _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)
    assert K.vq_sample(x.to(dev), u.to(dev), **kw)[0].tolist() == [20000, 29999, 15000]


def test_u_of_nan_is_zero(dev):
    x = _logits(9100, 2, 5000, "fp32").to(dev)
    for kw in (dict(), dict(top_k=20), dict(top_p=0.9)):
        got = K.vq_sample(x, torch.tensor([float("nan"), 0.5], device=dev), **kw)
        ref = K.vq_sample(x, torch.tensor([0.0, 0.5], device=dev), **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("top_k", [50, 5000])
def test_long_ties_under_every_border(dev, top_k):
    """Rows whose border lies among more ties than the list holds, one slice's
    ties, and ties behind a few larger logits."""
    V = 30011
    x = torch.zeros(4, V)
    x[1, ::2] = 1.0
    x[2, 9000:16000] = 2.0
    x[3, ::1000] = 3.0
    u = torch.tensor([0.2, 0.5, 0.8, 0.97])
    for dtype in DT.values():
        for kw in (dict(top_k=top_k), dict(top_p=0.7), dict(top_k=top_k, top_p=0.5), dict(top_k=top_k, top_p=0.5, min_p=0.3),
                   dict(top_p=0.999, temperature=4.0)):
            _check(K.vq_sample(x.to(dtype).to(dev), u.to(dev), **kw), x.to(dtype), u, **kw)


def test_calls_side_by_side(dev):
    """Two streams with a call each, again and again, and two graphs replayed in
    turn with eager calls between: every result is the one of a call alone."""
    a, b = _logits(9200, 3, 151936, "bf16", 0.1).to(dev), _logits(9201, 40, 9000, "fp32").to(dev)
    ua, ub = torch.rand(3, generator=synth.gen(9202)).to(dev), torch.rand(40, generator=synth.gen(9203)).to(dev)
    calls = [lambda: K.vq_sample(a, ua, top_p=0.95), lambda: K.vq_sample(b, ub, top_k=700, top_p=0.9)]
    ref = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(10):
        for i, (c, st) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(st):
                got[i].append(c())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(c())
    for _ in range(4):
        for i in (0, 1):
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
            got[1 - i].append(calls[1 - i]())
            got[i].append([o.clone() for o in outs[i]])
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert torch.equal(g[0], ref[i][0]) and torch.equal(g[1], ref[i][1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("scale", [1e-36, 1e-37, 1e-39, 1e-43])
@pytest.mark.parametrize("V", [5000, 5120])
def test_logits_a_tiny_way_apart(dev, dtype, scale, V):
    """Rows whose logits lie so close that their range has no reciprocal of 32
    bits, subnormal ones among them (5120 columns fill every group of the
    row): every entry weighs 1, and the order is still the logits'."""
    x = (torch.rand(4, V, generator=synth.gen(9300)).double() * scale).to(DT[dtype])
    x[1] = 2 * scale + x[1]
    u = torch.tensor([0.05, 0.4, 0.75, 0.999])
    for kw in (dict(top_k=3), dict(top_k=20), dict(top_k=300), dict(top_k=20, top_p=0.5), dict(top_p=0.6), dict(min_p=0.5),
               dict(top_k=4000, top_p=0.9), dict()):
        _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)


@pytest.mark.parametrize("orders", [850, 905, 950, 995, 1005])
@pytest.mark.parametrize("dtype", list(DT))
def test_logits_one_step_apart_a_range_of_weights_apart(dev, dtype, orders):
    """Temperatures at which neighbouring logits of the type differ by about
    as many binary orders as a sum of 64-bit weights can hold, in rows that
    ascend under each lane: all but the maxima weigh nothing."""
    B, V = 64, 151936
    step = 16.0 * torch.finfo(DT[dtype]).eps
    col = torch.arange(V)
    rows = []
    for r in range(4):
        rise = (col // (256 * (r + 1))) % 4 if r < 3 else torch.randint(0, 4, (V,), generator=synth.gen(9310))
        rows.append(16.0 + step * rise)
    x = torch.stack(rows).to(DT[dtype])
    u = torch.tensor([0.1, 0.45, 0.7, 0.95])
    t = float(np.float32(step * np.log2(np.e) / orders))
    logits, us = x.to(dev).repeat(B // 4, 1), u.to(dev).repeat(B // 4)
    for kw in (dict(), dict(top_p=0.5)):
        idx, lp = K.vq_sample(logits, us, temperature=t, **kw)
        assert torch.equal(idx, idx[:4].repeat(B // 4)) and torch.equal(lp, lp[:4].repeat(B // 4))
        _check((idx[:4], lp[:4]), x, u, temperature=t, **kw)


def _check_long(got, logits, u, rows, **kw):
    """_check for picked rows of a long vocabulary, whose draw and logprob are
    the sorted arrays' (settings are held in 32 bits)."""
    idx, lp = (t.cpu() for t in got)
    kw = {k: v if k == "top_k" else float(np.float32(v)) for k, v in kw.items()}
    for r in rows:
        ref_idx, ref_lp = S.sample_long_row(logits[r].float().cpu().numpy(), float(u[r]), **kw)
        assert int(idx[r]) == ref_idx, r
        assert abs(float(lp[r]) - ref_lp) <= abs(ref_lp) * 2.0 ** -24 + logits.shape[-1] * 2.0 ** -43 + 2.0 ** -40, r


def _long_logits(dev, B, V, dtype, steep):
    """_logits made on the device."""
    g = torch.Generator(device=dev).manual_seed(9400 + V % 1000)
    rank = torch.rand(B, V, generator=g, device=dev) * V + 2.0
    return (16.0 - steep * rank.log() + 0.4 * steep * torch.randn(B, V, generator=g, device=dev)).to(DT[dtype])


LONG = [dict(), dict(top_p=0.9, min_p=0.01), dict(top_k=50, top_p=0.9, temperature=0.7), dict(min_p=0.3), dict(top_k=700),
        dict(top_k=20000), dict(top_k=20000, top_p=0.5, min_p=0.02)]


@pytest.mark.parametrize("kw", LONG, ids=str)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("steep", [1.3, 0.1])
def test_large_batches_of_a_whole_vocabulary(dev, dtype, steep, kw):
    """256 rows cut into units that a wave reads in many steps (19 over fp32, 10
    over bf16), peaked and nearly flat."""
    B, V = 256, 151936
    x = _long_logits(dev, B, V, dtype, steep)
    u = torch.rand(B, generator=synth.gen(9401))
    rows = [0, 101, 255]
    u[101], u[255] = 1.0 - 2.0 ** -24, 0.0
    _check_long(K.vq_sample(x, u.to(dev), **kw), x, u, rows, **kw)


@pytest.mark.parametrize("kw", LONG, ids=str)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,steep", [(1 << 21, 1.3), ((1 << 21) - 3, 0.1)])
def test_the_longest_vocabulary(dev, V, steep, dtype, kw):
    """Rows of as many units and slices as there can be."""
    x = _long_logits(dev, 3, V, dtype, steep)
    u = torch.tensor([0.0, 0.5, 1.0 - 2.0 ** -24])
    _check_long(K.vq_sample(x, u.to(dev), **kw), x, u, range(3), **kw)
    one = K.vq_sample(x[1:2], u[1:2].to(dev), **kw)
    _check_long(one, x[1:2], u[1:2], [0], **kw)


@pytest.mark.parametrize("V", [1, 2, 3])
@pytest.mark.parametrize("top_k", [1, 2, 3, 9])
def test_a_top_k_of_the_whole_row(dev, V, top_k):
    """top_k at the number of columns, one column's among them, beside the
    other settings, common and by row."""
    x = torch.tensor([[0.5, 2.0, 1.0], [float("nan"), 0.0, -1.0]])[:, :V].contiguous()
    u = torch.tensor([0.3, 0.8])
    for kw in (dict(), dict(top_p=0.5), dict(min_p=0.5), dict(top_p=0.0, min_p=1.0), dict(temperature=0.0), dict(temperature=1e-4, top_p=0.9)):
        kw = dict(kw, top_k=top_k)
        _check(K.vq_sample(x.to(dev), u.to(dev), **kw), x, u, **kw)
        by_row = {k: torch.full((2,), v, dtype=torch.int32 if k == "top_k" else torch.float32) for k, v in kw.items()}
        _check(K.vq_sample(x.to(dev), u.to(dev), **{k: v.to(dev) for k, v in by_row.items()}), x, u, **by_row)
