"""vq2_router_select on the GPU against the fp64 oracle: expert ids exactly,
weights to one rounding.

Weights are computed in 64 bits and rounded once to fp32, half a step, 2^-24 of
the value; the 64-bit arithmetic before it (an exponential, a sum of up to
1024 of them, a quotient) is off by less than 2^-40, so rtol is 2^-24 (1 +
2^-10); below 2^-126 fp32's steps are 2^-149 whatever the value, half of one
2^-150.  The shared expert's weight is sigmoid(d) of an fp32 sum d of n products: each
product is exact to 2^-24 and passes at most n / 16 + 8 additions, so d is off
by at most (n / 16 + 9) 2^-24 sum |g h|, the sigmoid by a quarter of that, plus
8 half steps of its own exponential, sum and quotient."""
import numpy as np
import pytest
import torch

from compressai_amd import kernels as K, synth
from compressai_amd.graph import DecodeStepGraph
from oracle import selection as S

pytestmark = pytest.mark.gpu
RTOL = 2.0 ** -24 * (1 + 2.0 ** -10)
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _logits(seed, T, E, dtype, spread=1.7):
    return (torch.randn(T, E, generator=synth.gen(seed)) * spread).to(DT[dtype])


def _check(got, logits, k, **kw):
    ids, w = (t.cpu().numpy() for t in got)
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].cpu().double().numpy()
    kw["scale"] = float(np.float32(kw.get("scale", 1.0)))
    ref_ids, ref_w = S.router_select(logits.float().cpu().numpy(), k, **kw)
    assert ids.shape[1] >= k and ids.dtype == np.int32 and w.dtype == np.float32
    assert np.array_equal(ids[:, :k], ref_ids)
    off = np.abs(w[:, :k] - ref_w) > np.maximum(RTOL * np.abs(ref_w), 2.0 ** -150)
    assert not off.any(), (w[:, :k][off][:5], ref_w[off][:5])


FORMS = [
    dict(), dict(renormalise=False, scale=16.0), dict(scoring="sigmoid"), dict(scoring="sigmoid", renormalise=False),
    dict(scoring="sigmoid", bias=0.05, scale=2.5), dict(bias=0.002), dict(scoring="sigmoid", bias=0.0),
]


def _run(dev, seed, T, E, k, dtype, form, **more):
    kw = dict(form, **more)
    lg = _logits(seed, T, E, dtype).to(dev)
    if kw.get("bias") is not None:
        kw["bias"] = (torch.randn(E, generator=synth.gen(seed + 1)) * kw["bias"]).to(dev)
    _check(K.vq_router_select(lg, k, **kw), lg, k, **kw)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("T,E,k,dtype", [
    (1, 256, 8, "fp32"), (5, 64, 6, "bf16"), (3, 1, 1, "fp16"), (67, 160, 6, "fp32"), (130, 257, 12, "bf16"),
    (9, 512, 10, "fp16"), (2, 1024, 32, "fp32"), (17, 37, 32, "fp16"), (64, 8, 8, "bf16"), (33, 100, 16, "fp16"), (4, 700, 1, "bf16")])
def test_forms(dev, T, E, k, dtype, form):
    _run(dev, 7000 + E + T, T, E, k, dtype, form)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("E,G,keep,k,dtype", [
    (256, 8, 4, 8, "bf16"), (160, 8, 3, 6, "fp32"), (64, 64, 6, 6, "fp32"), (48, 3, 1, 16, "fp16"), (512, 16, 16, 10, "bf16"),
    (1024, 4, 2, 32, "bf16"), (63, 9, 2, 3, "fp32"), (72, 8, 1, 9, "fp16"), (1024, 64, 5, 20, "fp32"), (96, 2, 1, 4, "bf16"),
    (384, 12, 2, 7, "fp32"), (128, 32, 3, 12, "bf16"), (16, 16, 5, 5, "fp32"), (8, 2, 1, 3, "bf16"), (510, 15, 4, 12, "fp32"),
    (500, 5, 4, 11, "fp16"), (33, 11, 9, 12, "bf16")])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_groups(dev, E, G, keep, k, dtype, form, group_score):
    _run(dev, 7100 + E + G, 37, E, k, dtype, form, n_groups=G, topk_groups=keep, group_score=group_score)


@pytest.mark.parametrize("T", [1, 2, 3, 4, 7, 15, 16, 17, 63, 1000])
@pytest.mark.parametrize("E", [48, 256])
def test_token_counts(dev, T, E):
    _run(dev, 7200 + T, T, E, 8, "fp32", dict(scoring="sigmoid", bias=0.05), n_groups=8, topk_groups=3, group_score="top2")


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("E,G", [(256, 1), (256, 8), (100, 5), (600, 1)])
def test_ties_go_to_the_lower_id(dev, E, G, form):
    """Logits of a handful of values, zeros of both signs among them, and one
    bias for all: nearly every choice is a tie."""
    lg = (torch.randint(-2, 3, (40, E), generator=synth.gen(7300)) * 0.5).float()
    lg[lg == 0] *= torch.where(torch.rand(int((lg == 0).sum()), generator=synth.gen(7301)) < 0.5, -1.0, 1.0)
    lg[0] = 0.25
    kw = dict(form)
    if kw.get("bias") is not None:
        kw["bias"] = torch.full((E,), 0.125, device=dev)
    for gs in ("max", "top2"):
        more = dict(n_groups=G, topk_groups=max(1, G // 2), group_score=gs, **kw)
        _check(K.vq_router_select(lg.to(dev), 9, **more), lg, 9, **more)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("G", [1, 8])
def test_masked_experts(dev, G, form):
    """-inf and NaN logits and biases, whole groups, whole tokens; the
    type's lowest value is an ordinary logit."""
    E, k = 128, 12
    lg = _logits(7400, 24, E, "fp32")
    lg[0] = -float("inf")
    lg[1] = float("nan")
    lg[2, 5:] = -float("inf")
    lg[3, 16:] = torch.finfo(torch.float32).min
    lg[4] = torch.finfo(torch.float32).min
    lg[5:12][torch.rand(7, E, generator=synth.gen(7401)) < 0.8] = -float("inf")
    lg[12:20][torch.rand(8, E, generator=synth.gen(7402)) < 0.5] = float("nan")
    lg[20, 40] = float("inf")
    kw = dict(form)
    if kw.get("bias") is not None:
        kw["bias"] = torch.randn(E, generator=synth.gen(7403)) * kw["bias"]
        kw["bias"][7] = -float("inf")
        kw["bias"][9] = float("nan")
        kw["bias"] = kw["bias"].to(dev)
    for gs in ("max", "top2"):
        more = dict(n_groups=G, topk_groups=max(1, G // 4), group_score=gs, **kw)
        _check(K.vq_router_select(lg.to(dev), k, **more), lg, k, **more)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("form", [dict(), dict(scoring="sigmoid"), dict(scoring="sigmoid", renormalise=False)], ids=str)
def test_large_logits(dev, dtype, form):
    """Scores that round to 0 or 1 still choose by their logits."""
    lg = _logits(7500, 20, 256, dtype, spread=60.0)
    for G in (1, 8):
        more = dict(form, n_groups=G, topk_groups=max(1, G // 2))
        _check(K.vq_router_select(lg.to(dev), 8, **more), lg, 8, **more)


@pytest.mark.parametrize("hidden", [8, 100, 2048, 5000])
@pytest.mark.parametrize("h_dtype,g_dtype", [("fp16", "fp16"), ("bf16", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("T,E", [(1, 256), (13, 40), (6, 600)])
def test_shared_expert(dev, T, E, hidden, h_dtype, g_dtype):
    lg = _logits(7600, T, E, "bf16").to(dev)
    h = torch.randn(T, hidden, generator=synth.gen(7601)).to(DT[h_dtype])
    gate = (torch.randn(hidden, generator=synth.gen(7602)) * 0.05).to(DT[g_dtype])
    ids, w = K.vq_router_select(lg, 4, scoring="sigmoid", h=h.to(dev), shared_gate=gate.to(dev), shared_id=E)
    _check((ids, w), lg, 4, scoring="sigmoid")
    assert ids.shape == (T, 5) and (ids[:, 4] == E).all()
    hd, gd = h.double().numpy(), gate.double().numpy()
    ref = 1.0 / (1.0 + np.exp(-(hd @ gd)))
    tol = (hidden / 16 + 9) * 2.0 ** -24 * (np.abs(hd) @ np.abs(gd)) / 4 + 8 * 2.0 ** -24 * ref
    assert (np.abs(w[:, 4].cpu().numpy() - ref) <= tol).all()
    ids, w = K.vq_router_select(lg, 4, shared_id=7)  # no gate: weight 1
    _check((ids, w), lg, 4)
    assert (ids[:, 4] == 7).all() and (w[:, 4] == 1.0).all()


def test_strides_outputs_and_offsets(dev):
    """Rows of a wider matrix at odd offsets; given outputs, and nothing
    written beside them."""
    T, E, k = 21, 96, 5
    for dtype in DT:
        wide = _logits(7700, T + 2, 3 * E + 1, dtype).to(dev)
        for view in (wide[1:T + 1, 7:7 + E], wide[::2, E + 2:2 * E + 2], wide[:1, 1:E + 1]):
            n = view.shape[0]
            buf_i = torch.full((n * k + 16,), 77, dtype=torch.int32, device=dev)
            buf_w = torch.full((n * k + 16,), 0.5, device=dev)
            ids, w = buf_i[8:8 + n * k].view(n, k), buf_w[8:8 + n * k].view(n, k)
            got = K.vq_router_select(view, k, scoring="sigmoid", ids=ids, w=w)
            assert got[0] is ids and got[1] is w
            _check(got, view, k, scoring="sigmoid")
            for b, v in ((buf_i, 77), (buf_w, 0.5)):
                assert (b[:8] == v).all() and (b[8 + n * k:] == v).all()
    ids, w = K.vq_router_select(wide[:0, :E], k)
    assert ids.shape == (0, k) and w.shape == (0, k)
    assert K.vq_router_select(wide.reshape(-1)[:2 * 4 * E].view(2, 4, E), k)[0].shape == (8, k)


def test_refusals(dev):
    lg = torch.zeros(4, 64, device=dev)
    ok = dict(logits=lg, k=4)
    bad = [dict(k=0), dict(k=33), dict(k=65), dict(n_groups=3), dict(n_groups=4, topk_groups=5), dict(n_groups=32, topk_groups=1),
           dict(bias=torch.zeros(63, device=dev)), dict(bias=torch.zeros(64, device=dev, dtype=torch.float16)),
           dict(bias=torch.zeros(64)), dict(bias=torch.zeros(128, device=dev)[::2]), dict(logits=lg.to(torch.int32)),
           dict(logits=lg.t()[:, :3]), dict(logits=lg.double()), dict(shared_id=64, shared_gate=torch.zeros(8, device=dev)),
           dict(shared_id=64, shared_gate=torch.zeros(8, device=dev), h=torch.zeros(4, 7, device=dev)),
           dict(ids=torch.zeros(4, 5, dtype=torch.int32, device=dev)), dict(ids=torch.zeros(4, 4, device=dev)),
           dict(w=torch.zeros(4, 4, dtype=torch.float16, device=dev)), dict(logits=torch.zeros(4, 1025, device=dev)),
           dict(scale=float("nan"))]
    for b in bad:
        with pytest.raises(K.Vq2Error):
            K.vq_router_select(**dict(ok, **b))


def test_streams_graphs_and_repeats(dev):
    T, E, k = 50, 256, 8
    kw = dict(scoring="sigmoid", n_groups=8, topk_groups=4, group_score="top2", scale=2.5)
    bias = (torch.randn(E, generator=synth.gen(7801)) * 0.05).to(dev)
    a, b = (_logits(s, T, E, "bf16").to(dev) for s in (7802, 7803))
    refs = [K.vq_router_select(x, k, bias=bias, **kw) for x in (a, b)]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = K.vq_router_select(a, k, bias=bias, **kw)
    torch.cuda.synchronize(dev)
    assert all(torch.equal(x, y) for x, y in zip(got, refs[0]))
    step = DecodeStepGraph(lambda x: K.vq_router_select(x, k, bias=bias, **kw), [a])
    for i in (0, 1, 1, 0, 1):
        got = step((a, b)[i])
        torch.cuda.synchronize(dev)
        assert all(torch.equal(x, y) for x, y in zip(got, refs[i]))
        K.vq_router_select(b, k, bias=bias, **kw)


def test_agrees_with_the_softmax_router(dev):
    """The form vq_router_topk has: the same experts, weights to that entry's
    fp32 arithmetic."""
    lg = _logits(7900, 300, 256, "fp32").to(dev)
    ids, w = K.vq_router_select(lg, 8)
    ref_ids, ref_w = K.vq_router_topk(lg, 8)
    assert torch.equal(ids, ref_ids)
    assert torch.allclose(w, ref_w, rtol=1e-5, atol=0)


@pytest.mark.parametrize("E,k,G", [(256, 8, 1), (256, 8, 8), (64, 6, 1), (512, 12, 16), (40, 2, 5), (700, 5, 7)])
@pytest.mark.parametrize("bias", [False, True])
def test_choices_a_rounding_apart(dev, E, k, G, bias):
    """Logits that differ in their last bits: which expert is chosen shows in
    the eighth digit of its choice."""
    g = synth.gen(7950 + E)
    lg = 1.0 + torch.randint(0, 40, (50, E), generator=g).float() * 2.0 ** -23
    lg[25:, ::3] = 0.5
    kw = dict(scoring="sigmoid", n_groups=G, topk_groups=max(1, G // 2), group_score="top2",
              bias=torch.randint(0, 3, (E,), generator=g).float().to(dev) * 2.0 ** -20 if bias else None)
    _check(K.vq_router_select(lg.to(dev), k, **kw), lg, k, **kw)
    lg16 = (1.0 + torch.randint(0, 4, (50, E), generator=g).float() / 128).to(torch.bfloat16)
    _check(K.vq_router_select(lg16.to(dev), k, **kw), lg16, k, **kw)


def test_offsets_past_32_bits(dev):
    """Tokens' logits more than 2^31 elements apart."""
    stride, E = (1 << 31) + 8, 96
    buf = torch.empty(stride + E + 1, dtype=torch.bfloat16, device=dev)
    lg = _logits(7960, 2, E, "bf16")
    view = buf.as_strided((2, E), (stride, 1), 1)
    view.copy_(lg.to(dev))
    for k in (5, 20):
        _check(K.vq_router_select(view, k, scoring="sigmoid"), lg, k, scoring="sigmoid")


def test_many_tokens(dev):
    T, E = 300001, 24
    lg = _logits(7970, T, E, "bf16").to(dev)
    bias = (torch.randn(E, generator=synth.gen(7971)) * 0.05).to(dev)
    ids, w = K.vq_router_select(lg, 3, scoring="sigmoid", bias=bias)
    pick = torch.randint(0, T, (400,), generator=synth.gen(7972))
    pick[:2] = torch.tensor([0, T - 1])
    _check((ids.cpu()[pick], w.cpu()[pick]), lg.cpu()[pick], 3, scoring="sigmoid", bias=bias)


def test_native_and_python_entries_agree(dev):
    """Given outputs take the Python entry, the same launch."""
    lg = _logits(7980, 90, 256, "fp32").to(dev)
    h, gate = synth.activations(7981, (90, 512)).to(dev), synth.activations(7982, 512).to(dev)
    for kw in (dict(), dict(scoring="sigmoid", n_groups=8, topk_groups=2, scale=2.0), dict(h=h, shared_gate=gate, shared_id=256)):
        slots = 9 if "h" in kw else 8
        ref = K.vq_router_select(lg, 8, **kw)
        got = K.vq_router_select(lg, 8, ids=torch.empty(90, slots, dtype=torch.int32, device=dev), **kw)
        assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.parametrize("E,k,G", [(64, 6, 1), (256, 8, 8), (512, 12, 1), (100, 20, 5), (1024, 32, 1)])
@pytest.mark.parametrize("bias", [0.0, 0.125, -3.0])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_choices_that_differ_in_their_last_bits(dev, E, k, G, bias, dtype):
    """Sigmoids close to 1 under one bias for all (a balance bias that has not
    moved yet): choices differ from the 43rd bit on and are still in order."""
    lg = (27.0 + 9.0 * torch.rand(30, E, generator=synth.gen(7995))).to(DT[dtype])
    for gs in ("max", "top2"):
        more = dict(scoring="sigmoid", bias=torch.full((E,), bias, device=dev), n_groups=G, topk_groups=max(1, G // 2), group_score=gs)
        _check(K.vq_router_select(lg.to(dev), k, **more), lg, k, **more)


@pytest.mark.parametrize("E,k,G", [(16, 12, 1), (24, 10, 2), (100, 20, 1), (700, 5, 7)])
@pytest.mark.parametrize("low,high", [(-708.0, -690.0), (-709.7, -699.0), (-745.0, -700.0)])
@pytest.mark.parametrize("form", [dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=0.0), dict(bias=0.0)], ids=str)
def test_scores_near_the_end_of_64_bits(dev, E, k, G, low, high, form):
    """Sigmoids and softmax terms of e^-690 and below are in order and weighed
    against each other, down to the steps of 2^-1074 that 64 bits end in; a
    sigmoid is 0 from -709.78 on.  (Softmax: one expert far above, which its
    bias keeps from being chosen.)"""
    lg = low + (high - low) * torch.rand(24, E, generator=synth.gen(7990))
    if low < -740.0 and "scoring" in form:
        lg[:, ::2] += 9.0
    kw = dict(form)
    if "bias" in kw:
        kw["bias"] = torch.zeros(E)
    if "scoring" not in kw:
        lg[:, E // 2] = 0.0
        kw["bias"][E // 2] = -2.0
    kw["bias"] = kw["bias"].to(dev) if "bias" in kw else None
    more = dict(n_groups=G, topk_groups=max(1, G // 2), **kw)
    _check(K.vq_router_select(lg.to(dev), k, **more), lg, k, **more)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("E,k,G", [(256, 8, 1), (160, 6, 8), (700, 20, 1)])
def test_a_token_does_not_depend_on_the_others(dev, E, k, G, form):
    """The same logits alone, among a few and among many: the same bits."""
    lg = _logits(7999, 700, E, "fp32").to(dev)
    kw = dict(form, n_groups=G, topk_groups=max(1, G // 2))
    if kw.get("bias") is not None:
        kw["bias"] = (torch.randn(E, generator=synth.gen(8000)) * kw["bias"]).to(dev)
    ids, w = K.vq_router_select(lg, k, **kw)
    for a, b in ((0, 1), (3, 9), (500, 700), (699, 700)):
        part = K.vq_router_select(lg[a:b], k, **kw)
        assert torch.equal(part[0], ids[a:b]) and torch.equal(part[1], w[a:b])
