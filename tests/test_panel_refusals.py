"""What the norm's and the panels' C entries refuse on the host, before any
HIP call (the pointers are never dereferenced)."""
import ctypes

import pytest

from compressai_amd import _lib


def _err(status):
    assert status == _lib.ERR_ARG
    return _lib.load().vq2_last_error().decode()


P = 4096  # an aligned address


def _norm(**kw):
    a = dict(x=P, x_dt=2, residual=P, rows=2, n=128, weight=P, w_dt=2, zero=0, eps=1e-6, perm=None, sign=None, hb=0, sc=1.0,
             y=P, y_dt=2, y_scale=None, h=P)
    a.update(kw)
    return _lib.load().vq2_add_rms_norm(*a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(rows=-1), "rows=-1"), (dict(n=0), "n=0"), (dict(n=8193), "n=8193"), (dict(x_dt=3), "dtype"), (dict(y_dt=7), "y dtype"),
    (dict(eps=float("nan")), "eps"), (dict(weight=None), "weight"), (dict(h=None), "h must"), (dict(x=None), "NULL"),
    (dict(y_dt=3), "y_scale"), (dict(y_scale=P), "y_scale"), (dict(perm=P), "without hb"), (dict(hb=32), "power of two"),
    (dict(hb=96, n=192), "power of two"), (dict(hb=128, n=192), "power of two"), (dict(hb=-64), "power of two"), (dict(hb=128, x=P + 2), "16-byte"),
    (dict(x=P + 1), "aligned"), (dict(weight=P + 1), "aligned"), (dict(hb=64, perm=P + 2), "aligned")])
def test_norm(kw, match):
    assert match in _err(_norm(**kw))


def test_norm_empty_and_workspace():
    L = _lib.load()
    assert _norm(rows=0) == _lib.OK
    assert L.vq2_add_rms_norm_backward_workspace(5, 100) > 0
    for rows, n in ((-1, 8), (3, 0), (3, 8193), (0, 8)):
        assert L.vq2_add_rms_norm_backward_workspace(rows, n) == 0
    back = lambda dy=P, dw=P, ws=P, size=1 << 30, rows=2: L.vq2_add_rms_norm_backward(
        dy, 2, P, 2, None, rows, 128, P, 2, 0, 1e-6, None, None, 0, 1.0, P, dw, ws, size, None)
    assert "NULL" in _err(back(dy=None))
    assert "workspace" in _err(back(ws=None)) and "workspace" in _err(back(size=8)) and "256-byte" in _err(back(ws=P + 16))
    assert back(rows=0, dw=None) == _lib.OK


def _loss(**kw):
    a = dict(x=P, x_dt=2, x_scale=None, tokens=3, targets=P, ignore=-100, i0=P, i1=None, s2=0, cb0=P, cb1=None, cb_dt=1, scale=P,
             s_dt=2, rows=100, n=128, rs=1.0, loss=P, lse=P, ws=P, size=1 << 40)
    a.update(kw)
    return _lib.load().vq2_head_loss(*a.values(), None)


@pytest.mark.parametrize("kw,match", [
    (dict(tokens=-1), "tokens"), (dict(rows=0), "out_rows"), (dict(rows=(1 << 22) + 1), "out_rows"), (dict(n=96), "multiple of 64"),
    (dict(n=0), "multiple of 64"), (dict(n=32832), "multiple of 64"), (dict(cb0=None), "cb0"), (dict(s2=2), "cb1"),
    (dict(s2=2, cb1=P), "idx1"), (dict(i1=P), "idx1"), (dict(s2=9), "s2_kind"), (dict(s_dt=5), "scale dtype"), (dict(i0=None), "NULL"),
    (dict(i0=P + 1), "aligned"), (dict(x=None), "x is NULL"), (dict(x_dt=0), "fp16 or bf16"), (dict(x_dt=3), "x_scale"),
    (dict(x_scale=P), "x_scale"), (dict(x=P + 8), "16-byte"), (dict(size=100), "workspace"), (dict(ws=None), "workspace"),
    (dict(ws=P + 64), "256-byte"), (dict(targets=None), "NULL"), (dict(loss=None), "NULL"), (dict(targets=P + 4), "aligned")])
def test_head_loss(kw, match):
    assert match in _err(_loss(**kw))


def test_head_loss_empty():
    assert _loss(tokens=0, x=None, targets=None, loss=None, lse=None, ws=None, size=0) == _lib.OK
    L = _lib.load()
    assert L.vq2_head_loss_workspace(0, 100, 128, 0, 1) == 0 and L.vq2_head_loss_workspace(4, 100, 100, 0, 1) == 0
    assert L.vq2_head_loss_backward_workspace(4, 100, 128, 0, 1, 2, 1) > L.vq2_head_loss_backward_workspace(4, 100, 128, 0, 1, 2, 0) > 0


def _segs(r0=64, r1=64, i1=None):
    s = (_lib.Seg * 2)()
    s[0] = _lib.Seg(P, i1, P, None, r0, r0)
    s[1] = _lib.Seg(P, i1, P, None, r1, r1)
    return s


def test_gated_and_product():
    L = _lib.load()
    g = lambda segs=None, act=0, y_dt=2, y=P, x_dt=2, s2=0: L.vq2_gated_rows(
        P, x_dt, None, 3, segs if segs is not None else _segs(), s2, P, None, 1, 2, 128, 1.0, act, y, y_dt, P, 1 << 40, None)
    assert "up 32" in _err(g(_segs(64, 32)))
    assert "activation 9" in _err(g(act=9))
    assert "y dtype" in _err(g(y_dt=4))
    assert "y is NULL" in _err(g(y=None))
    assert "x_scale" in _err(g(x_dt=4))
    assert "idx1" in _err(g(_segs(i1=P)))
    assert "mats" in _err(L.vq2_gated_rows(P, 2, None, 3, None, 0, P, None, 1, 2, 128, 1.0, 0, P, 2, P, 1 << 40, None))
    b = lambda dx_dt=2, dg=P, du=P, x_dt=2, dy=P: L.vq2_gated_rows_backward(
        dy, 2, P, x_dt, 3, _segs(), 0, P, None, 1, 2, 128, 1.0, 0, P, dx_dt, dg, du, P, 1 << 40, None)
    assert "fp16 or bf16" in _err(b(dx_dt=0))
    assert "both or neither" in _err(b(du=None))
    assert "fp16 or bf16" in _err(b(x_dt=3))
    assert "dy or dx" in _err(b(dy=None))
    p = lambda dx_dt=2, x=P, ds=P, dy_dt=0: L.vq2_gemm_backward(dy_dt and P, dy_dt, x, 2, 3, P, None, 0, P, None, 1, P, 2, 100, 128, 1.0, P,
                                                                dx_dt, ds, P, 1 << 40, None)
    assert "fp16 or bf16" in _err(p(dx_dt=0))
    assert "x is NULL" in _err(p(x=None))
    assert "dy dtype" in _err(p(dy_dt=3))
    assert "dy or dx" in _err(p())


def test_fp32_gradients_have_a_name_of_their_own():
    """dx in fp32 is for its range: the plain type is refused, the name for it is taken (up to the next check)"""
    L = _lib.load()
    assert _lib.DT_F32_RANGE == 5
    call = lambda dx_dt, size=1 << 40: L.vq2_gemm_backward(P, 2, None, 2, 3, P, None, 0, P, None, 1, P, 2, 100, 128, 1.0, P, dx_dt, None, P,
                                                           size, None)
    assert "F32_RANGE" in _err(call(0)) and "fp16 or bf16" in _err(call(3))
    need = L.vq2_gemm_backward_workspace(3, 100, 128, 0, 1, _lib.DT_F32_RANGE, 0)
    assert need > 0 and "workspace" in _err(call(_lib.DT_F32_RANGE, need - 256))
    # two parts of a weight, as for fp16, where its stages' sum has more bits
    for entry, sizes in (("head_loss", (3, 100, 128, 2, 1)), ("gated_rows", (3, 100, 128, 2, 1)), ("gemm", (3, 100, 128, 2, 1))):
        ws = getattr(L, f"vq2_{entry}_backward_workspace")
        assert ws(*sizes, _lib.DT_F32_RANGE, 0) == ws(*sizes, 1, 0) > ws(*sizes, 2, 0) > 0


def test_few_tokens_keep_no_weights():
    """the workspace of calls that gather centroids as they go holds no dequantized rows: tokens, sums and no more"""
    L = _lib.load()
    for s2, cb in ((0, 1), (1, 1), (2, 2)):
        assert L.vq2_head_loss_workspace(1, 151936, 2048, s2, cb) < 8 << 20
        assert L.vq2_head_loss_workspace(64, 151936, 2048, s2, cb) < 8 << 20
        assert L.vq2_gated_rows_workspace(1, 6144, 2048, s2, cb, 2) < 2 << 20
    # where weights are kept they are there: 4096 tokens read 32768 rows of them at a time
    assert L.vq2_head_loss_workspace(4096, 151936, 2048, 0, 1) > 32768 * 2048 * 2
