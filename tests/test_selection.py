"""The selections of a decoded token without a GPU: the oracle against closed
forms and counts, and what vq2_router_select, vq2_sample and their Python
entries refuse (on the host, before any launch)."""
import numpy as np
import pytest
import torch

from compressai_amd import _lib, kernels as K
from oracle import selection as S, vq2_oracle as O


# ------------------------------------------------------------------- oracle
def test_router_oracle_is_the_softmax_router_without_extras():
    lg = np.random.default_rng(1).normal(size=(7, 33))
    ids, w = S.router_select(lg, 5)
    ref_ids, ref_w = O.router_topk(lg, 5)
    assert np.array_equal(ids, ref_ids)
    assert np.allclose(w, ref_w, rtol=1e-12, atol=0)


def test_router_oracle_closed_forms():
    # two groups of two, sigmoid 0.5 each: bias decides the choice, not the weight
    ids, w = S.router_select(np.zeros((1, 4)), 2, "sigmoid", bias=[0.0, 0.0, 0.3, 0.1], n_groups=2, topk_groups=1,
                             group_score="top2", renormalise=False, scale=3.0)
    assert ids.tolist() == [[2, 3]] and np.allclose(w, 1.5)
    # the best single expert against the best pair
    c = np.log(np.array([[0.6, 0.001, 0.4, 0.39]]))
    assert S.router_select(c, 1, n_groups=2, topk_groups=1, group_score="max")[0].tolist() == [[0]]
    assert S.router_select(c, 1, n_groups=2, topk_groups=1, group_score="top2")[0].tolist() == [[2]]
    # ties to the lower id; masked experts last with weight 0; a token without experts
    assert S.router_select(np.zeros((1, 6)), 3)[0].tolist() == [[0, 1, 2]]
    ids, w = S.router_select([[-np.inf, 1.0, np.nan, 1.0]], 3)
    assert ids.tolist() == [[1, 3, 0]] and np.allclose(w, [[0.5, 0.5, 0.0]])
    ids, w = S.router_select(np.full((1, 4), -np.inf), 2, "sigmoid")
    assert ids.tolist() == [[0, 1]] and (w == 0).all()


def test_sample_oracle_frequencies_and_filters():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    us = (np.arange(1000) + 0.5) / 1000
    count = np.bincount([S.sample_row(x, u)[0] for u in us], minlength=4)
    assert np.abs(count / 1000 - [0.1, 0.4, 0.2, 0.3]).max() <= 1e-3
    assert S.sample_row(x, 0.0)[0] == 0 and S.sample_row(x, 1.0)[0] == 3
    kept = lambda **kw: np.flatnonzero(S.sample_row(x, 0.5, **kw)[2]).tolist()
    assert kept(top_k=2) == [1, 3] and kept(top_k=9) == [0, 1, 2, 3]
    assert kept(top_p=0.45) == [1, 3] and kept(top_p=0.35) == [1] and kept(top_p=0.0) == [1]
    assert kept(min_p=0.6) == [1, 3] and kept(min_p=1.0) == [1]
    assert kept(top_k=3, top_p=0.8) == [1, 2, 3]
    assert kept(top_k=3, top_p=0.7) == [1, 3]  # of the 0.9 that top-k kept
    assert S.sample_row(x, 0.9, temperature=0.0)[:2] == (1, 0.0)
    assert S.sample_row([0.0] * 4, 0.5, top_k=3)[0] == 1  # ties: the first three columns
    assert S.sample_row([-np.inf, np.nan], 0.5)[0] == -1
    assert S.sample_row([np.inf, 1.0, np.inf], 0.6)[:2] == (2, np.log(0.5))


@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.6), dict(top_k=9), dict(top_p=0.7), dict(top_p=0.0), dict(min_p=0.2),
                                dict(top_k=40, top_p=0.8, min_p=0.05, temperature=1.3), dict(top_k=1000)], ids=str)
def test_sample_oracle_of_long_rows_is_the_other_one(kw):
    g = np.random.default_rng(2)
    for n in (1, 2, 50, 301):
        x = np.round(g.normal(size=n) * 2, 1)  # (ties among them)
        for u in (0.0, 0.3, 0.8, 1.0):
            token, lp = S.sample_long_row(x, u, **kw)
            ref_token, ref_lp, _ = S.sample_row(x, u, **kw)
            assert token == ref_token and abs(lp - ref_lp) < 1e-12


# ----------------------------------------------------------------- refusals
def _err(code):
    assert code != _lib.OK
    return _lib.load().vq2_last_error().decode()


def _select(**kw):
    a = dict(logits=16, dt=0, stride=64, tokens=1, E=64, k=4, scoring=0, bias=None, groups=1, keep=1, gs=0, renorm=1,
             scale=1.0, h=None, h_dt=0, hidden=0, gate=None, g_dt=0, shared=-1, ids=16, w=16, stream=None)
    a.update(kw)
    return _lib.load().vq2_router_select(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=-1), "token count"), (dict(E=0), "n_experts"), (dict(E=1025, stride=1025), "n_experts"),
    (dict(k=0), "k=0"), (dict(k=33), "k=33"), (dict(k=5, E=4, stride=4), "k=5"), (dict(scoring=2), "scoring"),
    (dict(groups=0), "n_groups"), (dict(groups=5), "n_groups"), (dict(E=130, stride=130, groups=65), "n_groups"),
    (dict(groups=4, keep=0), "topk_groups"), (dict(groups=4, keep=5), "topk_groups"),
    (dict(groups=32, keep=1), "topk_groups"), (dict(gs=2), "group_score"), (dict(scale=float("nan")), "scale"),
    (dict(shared=1 << 31), "shared_id"), (dict(logits=None), "NULL"), (dict(ids=None), "NULL"), (dict(w=None), "NULL"),
    (dict(dt=3), "dtype"), (dict(tokens=2, stride=63), "l_stride"), (dict(shared=64, gate=16), "needs h"),
    (dict(shared=64, gate=16, h=16, hidden=8, h_dt=9), "dtype")])
def test_router_select_refuses(kw, msg):
    assert msg in _err(_select(**kw))


def test_router_select_of_no_tokens():
    assert _select(tokens=0, logits=None, ids=None, w=None) == _lib.OK


def _sample(**kw):
    a = dict(logits=16, dt=0, stride=64, rows=1, vocab=64, u=16, t=1.0, t_rows=None, k=0, k_rows=None, p=1.0, p_rows=None,
             m=0.0, m_rows=None, idx=16, lp=16, ws=None, nbytes=0, stream=None)
    a.update(kw)
    return _lib.load().vq2_sample(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=-1), "row count"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 21) + 1, stride=1 << 22), "vocab"),
    (dict(rows=65536), "rows"), (dict(t=-0.5), "temperature"), (dict(t=float("nan")), "temperature"),
    (dict(p=-0.1), "top_p"), (dict(p=float("nan")), "top_p"), (dict(m=-0.1), "min_p"), (dict(m=1.5), "min_p"),
    (dict(m=float("nan")), "min_p"), (dict(k=-1), "top_k"), (dict(logits=None), "NULL"), (dict(u=None), "NULL"),
    (dict(idx=None), "NULL"), (dict(lp=None), "NULL"), (dict(dt=7), "dtype"), (dict(rows=2, stride=63), "l_stride"),
    (dict(idx=12), "aligned"), (dict(logits=18), "aligned"), (dict(logits=17, dt=2), "aligned")])
def test_sample_refuses(kw, msg):
    assert msg in _err(_sample(**kw))


def test_sample_workspace_is_checked():
    L = _lib.load()
    assert _sample(rows=0, logits=None, u=None, idx=None, lp=None) == _lib.OK
    assert L.vq2_sample_workspace(0, 100) == 0 and L.vq2_sample_workspace(1, 0) == 0
    assert L.vq2_sample_workspace(1, (1 << 21) + 1) == 0 and L.vq2_sample_workspace(65536, 100) == 0
    need = L.vq2_sample_workspace(1, 151936)
    if need:
        assert "workspace" in _err(_sample(vocab=151936, ws=256, nbytes=need - 1))
        assert "aligned" in _err(_sample(vocab=151936, ws=128, nbytes=need))


def test_python_entries_refuse():
    x = torch.zeros(2, 16)
    with pytest.raises(K.Vq2Error, match="GPU tensors"):
        K.vq_router_select(x, 2)
    with pytest.raises(K.Vq2Error, match="GPU tensors"):
        K.vq_sample(x, torch.zeros(2))
    with pytest.raises(K.Vq2Error, match="scoring"):
        K.vq_router_select(x, 2, scoring="relu")
    with pytest.raises(K.Vq2Error, match="group_score"):
        K.vq_router_select(x, 2, group_score="mean")


def test_rows_of_any_stride():
    x = torch.zeros(5, 40)
    assert K._rows2d(x, "x")[1] == 40 and K._rows2d(x[:, 3:9], "x")[1] == 40 and K._rows2d(x[::2], "x")[1] == 80
    assert K._rows2d(x[1:2, 3:9], "x")[1] == 6 and K._rows2d(x.view(5, 2, 20), "x")[0].shape == (10, 20)
    assert K._rows2d(torch.zeros(16), "x")[0].shape == (1, 16)
    for bad in (x[:, ::2], x.t(), x[:1].expand(5, 40), torch.zeros(2, 0), torch.tensor(1.0), x[:, 3:9].unsqueeze(0)):
        with pytest.raises(K.Vq2Error):
            K._rows2d(bad, "x")


@pytest.mark.parametrize("kw", [dict(logits=18), dict(logits=17, dt=1), dict(logits=17, dt=2)])
def test_router_select_refuses_logits_between_elements(kw):
    assert "aligned" in _err(_select(**kw))


@pytest.mark.parametrize("scale", [float("inf"), -float("inf")])
def test_router_select_refuses_an_infinite_scale(scale):
    """A masked expert's weight, 0, would be 0 times infinity."""
    assert "scale" in _err(_select(scale=scale))
