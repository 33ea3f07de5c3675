"""Which entry a sorted MoE module calls (on the CPU, the entries replaced by
recorders): the grouped kernel takes no call that it, or the router in front
of it, refuses and the one-pair kernels take, and none that those refuse."""
import re

import pytest
import torch

from compressai_amd import _lib, kernels as K, synth
from compressai_amd.moe import MoELayer

E, H, I = 65, 64, 64


@pytest.fixture
def calls(monkeypatch):
    """Names of the expert entries called, in order; their results are zeros."""
    names = []

    def moe_rows(h, ids, w, *a, **kw):
        names.append("rows")
        return torch.zeros(h.reshape(-1, H).shape)

    def sorted_moe(h, *a, logits=None, **kw):
        names.append("sorted")
        out = torch.zeros(h.reshape(-1, H).shape)
        return out if logits is None else (out, None, None)

    def router(logits, k, *a, **kw):
        T = logits.shape[0]
        return torch.zeros(T, k + 1, dtype=torch.int32), torch.zeros(T, k + 1)

    monkeypatch.setattr(K, "vq_moe_rows", moe_rows)
    monkeypatch.setattr(K, "vq_sorted_moe", sorted_moe)
    monkeypatch.setattr(K, "vq_router_topk", router)
    return names


def _layer(top_k):
    gu, dn = synth.indices16(8620, (E, 2 * I, H // 8)), synth.indices16(8621, (E, H, I // 8))
    return MoELayer(gu, synth.scales(8622, (E, 2 * I)), dn, synth.scales(8623, (E, H)), synth.codebook(8624),
                    torch.zeros(H), top_k=top_k, sorted_layout=True)


@pytest.mark.parametrize("top_k,entry", [(8, "rows"), (32, "rows"), (33, "sorted"), (64, "sorted")])
def test_top_k_of_the_router_in_front_of_the_grouped_kernel(calls, top_k, entry):
    """The router entry takes VQ2_ROUTER_MAX_TOPK experts a token, the one
    built into the one-pair launch 64: layers above stay there for any T."""
    limit = int(re.search(r"#define VQ2_ROUTER_MAX_TOPK (\d+)", _lib.HEADER_PATH.read_text()).group(1))
    assert limit == K.ROUTER_MAX_TOPK and (entry == "rows") == (top_k <= limit)
    layer = _layer(top_k)
    T = 12000 // (top_k + 1)
    assert K.moe_rows_faster(T * (top_k + 1), E, H, I)
    layer(torch.zeros(1, H), torch.zeros(1, E - 1))
    layer(torch.zeros(T, H), torch.zeros(T, E - 1))
    assert calls == ["sorted", entry]


@pytest.mark.parametrize("columns,entry", [(E - 1, "rows"), (E, "rows"), (E + 1, "sorted"), (7, "sorted")])
def test_logits_the_one_pair_launch_refuses_are_left_to_it(calls, columns, entry):
    """Logits of more columns than the pool has entries, or fewer than top_k:
    refused for few tokens, so for many as well."""
    T = 1500
    layer = _layer(8)
    assert K.moe_rows_faster(T * 9, E, H, I)
    layer(torch.zeros(T, H), torch.zeros(T, columns))
    assert calls == [entry]


def test_token_count_of_activations_with_more_dims(calls):
    """experts() flattens h: the grouped kernel's token limit counts tokens,
    whatever the first dimension holds."""
    m = _layer(1).experts_mod
    T = K.MOE_ROWS_MAX_TOKENS + 1
    for h, entry in ((torch.zeros(T // 2, 2, H), "sorted"), (torch.zeros(T - 1, 1, H), "rows"),
                     (torch.zeros(2, T // 2, H), "sorted")):
        n = h.numel() // H
        m.experts(h, torch.zeros(n, 1, dtype=torch.int32), torch.zeros(n, 1))
        assert calls[-1] == entry, h.shape


def _routed(top_k=4, **kw):
    gu, dn = synth.indices16(8620, (E, 2 * I, H // 8)), synth.indices16(8621, (E, H, I // 8))
    return MoELayer(gu, synth.scales(8622, (E, 2 * I)), dn, synth.scales(8623, (E, H)), synth.codebook(8624),
                    torch.zeros(H), top_k=top_k, sorted_layout=False, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(scoring="sigmoid", router_bias=torch.zeros(E)), "bias"), (dict(router_bias=torch.zeros(E - 1).half()), "bias"),
    (dict(router_bias=torch.zeros(2 * E - 2)[::2]), "bias"), (dict(router_bias=torch.zeros(E - 1, device="meta")), "router_bias"),
    (dict(n_groups=8, topk_groups=0), "topk_groups"), (dict(n_groups=8, topk_groups=9), "topk_groups"),
    (dict(n_groups=32, topk_groups=1), "topk_groups"), (dict(scoring="sigmoid", top_k=33), "k=33"),
    (dict(scoring="sigmoid", top_k=0), "k=0"), (dict(routed_scale=float("nan")), "scale")])
def test_router_forms_are_checked_when_the_layer_is_made(kw, msg):
    with pytest.raises(K.Vq2Error, match=msg):
        _routed(**kw)
    assert _routed(scoring="sigmoid", router_bias=torch.zeros(E - 1), n_groups=8, topk_groups=2).router_form is not None


@pytest.mark.parametrize("n_routed", [E, E + 3])
def test_a_shared_expert_outside_the_pool_is_refused(n_routed):
    """The built-in router refuses it at the call; a router in front of the
    experts hands them ids, and an id outside the pool computes NaN."""
    with pytest.raises(K.Vq2Error, match="pool"):
        _routed(scoring="sigmoid", n_routed=n_routed)
    assert _routed(scoring="sigmoid", n_routed=E - 5).n_routed == E - 5
