"""Gradients through packed layers, for tuning around frozen codes.

What a packed model learns without touching its codes: the norms' weights, the
row scales (make ``PackedLinear.scale`` a leaf: ``lin.scale.requires_grad_()``, in
fp32 for small steps; it is no parameter of its module and not in its
``state_dict``: keep and store what was tuned), and whatever produces the activations (adapters, other
layers).  The functions here are differentiable once in all of these; each is
one entry of ``kernels`` forward and one backward:

  rotate(x, rot)                the RHT (orthogonal: its gradient is its inverse)
  add_rms_norm(x, weight, residual, rot=...)  (y, h), y rotated where rot is given
  linear(lin, xr, out_dtype)    a PackedLinear on rotated rows
  gated(gate, up, xr)           f(gate xr) * (up xr)
  head_loss(lin, xr, targets)   the loss of every token

``xr`` are rotated rows in fp16 or bf16 (``rotate`` or ``add_rms_norm`` give
them), and their gradients are of that type: fp16 rows want a scaled loss.
``runtime``'s modules (``PackedLinear``, ``PackedProjections``, ``PackedMLP``,
``PackedLMHead`` and its ``loss``) are differentiable by themselves, with the
results that they have without a gradient (``PackedMLP``'s single rows: up to
rounding); they rotate inside, and their gradients are of the activations' type, in
fp32 with its range (terms of 11 bits).  Expert pools (``moe``, ``paged``) have no gradient.  The
reference distils and tunes with dequantized weights in torch (vq2/kd.py); here
no dequantized matrix is kept.

A step that is captured into a graph makes its leaves inside (``detach()``,
``requires_grad_()``) and takes their gradients with ``torch.autograd.grad``: a
``backward()`` that is captured while an eager graph of the same leaves lives would
wait for that graph's stream, which a capture does not allow.  The functions are
plain ``torch.autograd.Function``s: ``torch.func``'s transforms do not take them.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K

__all__ = ["rotate", "add_rms_norm", "linear", "gated", "head_loss"]


def _rows16(xr, what):
    if xr.dtype not in (torch.float16, torch.bfloat16):
        raise K.Vq2Error(f"{what}: rotated rows in float16 or bfloat16, got {xr.dtype}")
    return xr.contiguous()


def _planes(lin):
    if lin.planes_released:
        raise K.Vq2Error("gradients need the index planes, which were released")
    return lin._planes()


def _to(t, like):
    return None if t is None else t.view(like.shape).to(like.dtype)


def _own(y):
    """y as no view of another tensor: a function's result may then be written over (y += residual)"""
    return y.new_empty(0).set_(y) if y._is_view() else y


def _row_type(x):
    """the type that rotated rows of x are held in: its own, fp16 for fp32"""
    return torch.float16 if x.dtype == torch.float32 else x.dtype


def _rows_of(ctx, x, rot):
    """The rotated rows of an operator's input: x itself, or x turned by rot.
    Inside one autograd function, so that the gradient of fp32 activations is
    fp32 all the way back, and never that of the fp16 rows: most gradients of
    a mean over many tokens lie below fp16's numbers."""
    ctx.rot, ctx.dtype = rot, x.dtype
    ctx.wide = rot is not None and x.dtype == torch.float32
    return x if rot is None else rot.fwd(x, out_dtype=_row_type(x))


def _input_grad(ctx, dxr):
    if ctx.rot is None or not ctx.needs_input_grad[0]:
        return dxr
    return ctx.rot.inv(dxr, out_dtype=ctx.dtype)


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rot, out_dtype):
        ctx.rot, ctx.dtype = rot, x.dtype
        return rot.fwd(x, out_dtype=out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ctx.rot.inv(dy.contiguous(), out_dtype=ctx.dtype), None, None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, kw, out_dtype):
        ctx.set_materialize_grads(False)
        y, h, _ = K.vq_add_rms_norm(x, weight, residual, out_dtype=out_dtype, **kw)
        ctx.save_for_backward(h, weight)
        ctx.kw, ctx.residual = kw, residual is not None
        return (y, h) if residual is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:  # the norm itself was not used
            return dh, None, dh, None, None
        dx, dw = K.vq_add_rms_norm_backward(dy.contiguous(), h, weight, None if dh is None else dh.contiguous(),
                                            weight_grad=ctx.needs_input_grad[1], **ctx.kw)
        return dx, _to(dw, weight), dx if ctx.residual else None, None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xr, scale, lin, out_dtype):
        from .runtime import vq_matmul

        ctx.save_for_backward(xr, scale)
        ctx.lin = lin
        i0, i1, cb0, cb1 = _planes(lin)
        x2 = xr.reshape(-1, lin.n)
        if x2.shape[0] >= 3 and lin.n % 64 == 0 and lin.n <= K.ROWS_GEMM_MAX_N:
            y = K.vq_rows_gemm(x2, [(i0, i1, scale, lin.out)], cb0, cb1, lin.n, hb=0, act_dtype=xr.dtype, out_dtype=out_dtype)[0]
        else:
            y = vq_matmul(x2, i0, i1, cb0, cb1, scale, lin.out, lin.n, out_dtype)
        return _own(y.view(*xr.shape[:-1], lin.out))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, scale = ctx.saved_tensors
        lin = ctx.lin
        i0, i1, cb0, cb1 = _planes(lin)
        dx, ds = K.vq_gemm_backward(dy.contiguous(), xr, i0, i1, cb0, cb1, scale, lin.out, lin.n,
                                    scale_grad=ctx.needs_input_grad[1])
        return dx, _to(ds, scale), None, None


class _Modules(torch.autograd.Function):
    """Products of PackedLinears that share their input x and its rotation: the
    results are run(x), whatever kernels that takes; rotated rows in 16 bits are
    made again for the scales' gradients alone."""

    @staticmethod
    def forward(ctx, x, run, lins, *scales):
        ctx.set_materialize_grads(False)
        # (without scales to tune x is not needed, and may be written over, as residual streams are)
        ctx.save_for_backward(x if any(ctx.needs_input_grad[3:]) else None, *scales)
        ctx.lins, ctx.shape, ctx.dtype = lins, x.shape, x.dtype
        return tuple(_own(y) for y in run(x))

    @staticmethod
    @once_differentiable
    def backward(ctx, *dys):
        x, *scales = ctx.saved_tensors
        need_x, _, _, *need = ctx.needs_input_grad
        a, wide = ctx.lins[0], ctx.dtype == torch.float32
        rows = torch.float16 if wide else ctx.dtype
        xr = a.rot.fwd(x.reshape(-1, a.n), out_dtype=rows) if any(need) else None
        dx, ds = None, []
        for lin, s, dy, n in zip(ctx.lins, scales, dys, need):
            d = None
            if dy is not None:
                i0, i1, cb0, cb1 = _planes(lin)
                part, d = K.vq_gemm_backward(dy.reshape(-1, lin.out).contiguous(), xr if n else None, i0, i1, cb0, cb1, s, lin.out,
                                             lin.n, scale_grad=n, dx_dtype=rows, wide=wide)
                dx = part if dx is None else dx + part
            ds.append(_to(d, s))
        if dx is not None:
            dx = a.rot.inv(dx, out_dtype=ctx.dtype).view(ctx.shape) if need_x else None
        return dx, None, None, *ds


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_scale, up_scale, gate, up, activation, rot):
        xr = _rows_of(ctx, x, rot)
        ctx.save_for_backward(xr, gate_scale, up_scale)
        ctx.mats, ctx.activation = (gate, up), activation
        (g0, g1, cb0, cb1), (u0, u1, _, _) = _planes(gate), _planes(up)
        act = K.vq_gated_rows(xr, (g0, g1, gate_scale), (u0, u1, up_scale), cb0, cb1, gate.n, activation=activation)
        return act.float() if ctx.wide else act  # (its gradient takes its type)

    @staticmethod
    @once_differentiable
    def backward(ctx, dact):
        xr, gate_scale, up_scale = ctx.saved_tensors
        gate, up = ctx.mats
        (g0, g1, cb0, cb1), (u0, u1, _, _) = _planes(gate), _planes(up)
        dx, dg, du = K.vq_gated_rows_backward(dact.contiguous(), xr, (g0, g1, gate_scale), (u0, u1, up_scale), cb0, cb1,
                                              gate.n, activation=ctx.activation,
                                              scale_grad=ctx.needs_input_grad[1] or ctx.needs_input_grad[2], wide=ctx.wide)
        return _input_grad(ctx, dx), _to(dg, gate_scale), _to(du, up_scale), None, None, None, None


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, lin, targets, ignore_index, rot):
        xr = _rows_of(ctx, x, rot)
        i0, i1, cb0, cb1 = _planes(lin)
        loss, lse = K.vq_head_loss(xr, targets, i0, i1, cb0, cb1, scale, lin.out, lin.n, ignore_index=ignore_index)
        ctx.save_for_backward(xr, scale, targets, lse)
        ctx.lin, ctx.ignore_index = lin, ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        xr, scale, targets, lse = ctx.saved_tensors
        lin = ctx.lin
        i0, i1, cb0, cb1 = _planes(lin)
        dx, ds = K.vq_head_loss_backward(xr, targets, lse, dloss.contiguous(), i0, i1, cb0, cb1, scale, lin.out, lin.n,
                                         ignore_index=ctx.ignore_index, scale_grad=ctx.needs_input_grad[1], wide=ctx.wide)
        return _input_grad(ctx, dx), _to(ds, scale), None, None, None, None


def rotate(x, rot, out_dtype=None):
    """rot.fwd(x): rows in the basis that packed matrices of this rotation take."""
    return _Rotate.apply(x.contiguous(), rot, out_dtype)


def add_rms_norm(x, weight, residual=None, *, eps=1e-6, zero_centred=False, rot=None, out_dtype=None):
    """(y, h) of kernels.vq_add_rms_norm; y is rotated where a ``rot.Rot`` is given.
    out_dtype: 16 or 32 bits (8-bit rows, which are numbers only with their
    scales and have no gradient, are the kernel entry's alone)."""
    if out_dtype in K._DT8:
        raise K.Vq2Error("add_rms_norm: y in 8 bits has no gradient (kernels.vq_add_rms_norm gives it with its scales)")
    kw = dict(eps=eps, zero_centred=zero_centred)
    if rot is not None:
        kw.update(perm=rot._perm32, sign=rot._sign8, hb=rot.hb, rht_scale=rot.scale)
    out = _Norm.apply(x.contiguous(), weight, None if residual is None else residual.contiguous(), kw, out_dtype)
    return out if residual is not None else (out, x)


def linear(lin, xr, out_dtype=None):
    """A PackedLinear's product with rotated rows, in their type or out_dtype."""
    if (lin.n % 64 or lin.n > K.PANEL_MAX_N) and torch.is_grad_enabled() and (xr.requires_grad or lin.scale.requires_grad):
        raise K.Vq2Error(f"linear: a gradient needs a width that is a multiple of 64 up to {K.PANEL_MAX_N}, got {lin.n}")
    return _Linear.apply(_rows16(xr, "linear"), lin.scale, lin, out_dtype or xr.dtype)


def module_products(x, run, lins):
    """run(x), results of PackedLinears of one rotation, differentiable in x and the scales."""
    return _Modules.apply(x, run, lins, *[m.scale for m in lins])


def gated(gate, up, xr, activation="silu"):
    """f(gate xr) * (up xr) of two PackedLinears of one width, cfg, codebooks and rotation."""
    return _Gated.apply(_rows16(xr, "gated"), gate.scale, up.scale, gate, up, activation, None)


def gated_of(gate, up, x, activation):
    """The same of rows that are not rotated, in x's type, for the modules."""
    return _Gated.apply(x.contiguous(), gate.scale, up.scale, gate, up, activation, gate.rot)


def head_loss(lin, xr, targets, ignore_index=-100):
    """kernels.vq_head_loss of a head's PackedLinear: the loss of every row, fp32."""
    return _HeadLoss.apply(_rows16(xr, "head_loss").reshape(-1, lin.n), lin.scale, lin, targets.reshape(-1).contiguous(), ignore_index, None)


def head_loss_of(lin, x, targets, ignore_index):
    """The same of rows that are not rotated, for the modules."""
    return _HeadLoss.apply(x.reshape(-1, lin.n).contiguous(), lin.scale, lin, targets.reshape(-1).contiguous(), ignore_index, lin.rot)
