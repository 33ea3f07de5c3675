"""MoE layers that route by vq_router_select, and a decoded token's whole way:
layer, head and draw in one captured step."""
import numpy as np
import pytest
import torch

from compressai_amd import kernels as K, synth
from compressai_amd.graph import DecodeStepGraph
from compressai_amd.moe import MoELayer
from compressai_amd.runtime import PackedLinear, PackedLMHead
from oracle import selection as S, vq2_oracle as O

pytestmark = pytest.mark.gpu
E, H, I = 16, 512, 128


def _pools(dev):
    return (synth.indices16(8900, (E + 1, 2 * I, H // 8)).to(dev), synth.scales(8901, (E + 1, 2 * I)).to(dev),
            synth.indices16(8902, (E + 1, H, I // 8)).to(dev), synth.scales(8903, (E + 1, H)).to(dev),
            synth.codebook(8904).to(dev))


def _layer(dev, gate=True, **kw):
    g = (synth.activations(8905, H) * 0.02).to(dev) if gate else None
    return MoELayer(*_pools(dev), g, top_k=4, **kw)


FORMS = [
    (True, dict(scoring="sigmoid")),
    (True, dict(scoring="sigmoid", router_bias=True, n_groups=4, topk_groups=2, group_score="top2", routed_scale=2.5)),
    (False, dict(n_groups=2, topk_groups=1, renormalise=False, routed_scale=16.0)),
    (False, dict()),
]


@pytest.mark.parametrize("gate,form", FORMS, ids=str)
@pytest.mark.parametrize("T,sorted_layout", [(1, None), (3, None), (3, False), (400, None)])
def test_layer_against_the_oracle(dev, gate, form, T, sorted_layout):
    """The layer's own bar, 1e-3 of its largest value, and bit for bit the
    experts given the routed ids and weights."""
    kw = dict(form)
    if kw.get("router_bias"):
        kw["router_bias"] = (torch.randn(E, generator=synth.gen(8906)) * 0.1).to(dev)
    layer = _layer(dev, gate, sorted_layout=sorted_layout, **kw)
    h = synth.activations(8907, (T, H)).to(dev)
    lg = synth.activations(8908, (T, E), dtype=torch.float32).to(dev)
    out = layer(h, lg)
    ids, w = layer.route(h, lg)
    assert torch.equal(out, layer.experts_mod.experts(h, ids, w))
    form64 = {("bias" if k == "router_bias" else "scale" if k == "routed_scale" else k): v for k, v in kw.items()}
    if "bias" in form64:
        form64["bias"] = form64["bias"].cpu().numpy()
    ref_ids, ref_w = S.router_select(lg.cpu().numpy(), 4, **form64)
    sw = np.ones((T, 1))
    if gate:
        sw = 1.0 / (1.0 + np.exp(-(h.double().cpu().numpy() @ layer.shared_gate.double().cpu().numpy())))[:, None]
    gu, gus, dn, dns, cb = (t.cpu() for t in _pools(dev))
    rh, ri = layer.experts_mod.rot_h, layer.experts_mod.rot_i
    n = min(T, 6)
    ref = O.moe_experts(h[:n].cpu(), np.concatenate([ref_ids, np.full((T, 1), E)], 1)[:n], np.concatenate([ref_w, sw], 1)[:n],
                        lambda e: (gu[e].numpy(), None, gus[e], dn[e].numpy(), None, dns[e]), cb, None,
                        rh.perm.cpu().numpy(), rh.sign.float().cpu().numpy(), ri.perm.cpu().numpy(), ri.sign.float().cpu().numpy())
    assert O.max_rel_err(out[:n].cpu().numpy(), ref) < 1e-3


def test_default_layer_keeps_its_router(dev):
    layer = _layer(dev)
    assert layer.router_form is None and _layer(dev, n_groups=4, topk_groups=4).router_form is None
    with pytest.raises(K.Vq2Error):
        _layer(dev, scoring="sigmoid")(synth.activations(8909, (1, H)).to(dev), torch.zeros(1, E - 1, device=dev))
    with pytest.raises(K.Vq2Error):
        _layer(dev, scoring="tanh")(synth.activations(8909, (1, H)).to(dev), torch.zeros(1, E, device=dev))


@pytest.mark.parametrize("T", [1, 5])
def test_layer_head_and_draw_in_one_captured_step(dev, T):
    layer = _layer(dev, scoring="sigmoid", n_groups=4, topk_groups=2, group_score="top2", routed_scale=2.5,
                   router_bias=(torch.randn(E, generator=synth.gen(8910)) * 0.1).to(dev))
    V = 6000
    m = synth.vq_matrix(8911, V, H, bpw=2)
    head = PackedLMHead(PackedLinear((V, H), (16,), "head", [m["idx0"]], m["scale"], {"16": layer.experts_mod.cb16}, dev))
    router = (torch.randn(H, E, generator=synth.gen(8912)) * H ** -0.5).to(dev)
    settings = dict(temperature=torch.full((T,), 0.8, device=dev), top_k=50, top_p=0.9, min_p=0.01)

    def step(h, u):
        x = h.float()
        x = x + layer(h, x @ router)
        x = x / x.norm(dim=-1, keepdim=True) * H ** 0.5
        return head.sample(x.to(torch.float16), u, **settings)

    hs = [synth.activations(8920 + i, (T, H)).to(dev) for i in range(4)]
    us = [torch.rand(T, generator=synth.gen(8930 + i)).to(dev) for i in range(4)]
    refs = [step(h, u) for h, u in zip(hs, us)]
    graph = DecodeStepGraph(step, [hs[0], us[0]])
    for i in (0, 1, 2, 3, 3, 1, 0):
        got = graph(hs[i], us[i])
        torch.cuda.synchronize(dev)
        assert torch.equal(got[0], refs[i][0]) and torch.equal(got[1], refs[i][1]), i
        step(hs[2], us[2])
    assert len({int(r[0][0]) for r in refs}) > 1
