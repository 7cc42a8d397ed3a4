"""The public ops registered with torch.library (namespace ``mhc``), for code that is
compiled with ``torch.compile(fullgraph=True)`` or exported.

The plain functions in ``mhc.ops`` reach the kernels through ctypes from inside
``torch.autograd.Function``s, which a tracing compiler cannot look into (they are marked opaque and
cause a graph break).  Here every kernel call is a ``torch.library.custom_op`` with a fake
(shape-only) implementation and an autograd formula made of other custom ops, so the tracer sees
ordinary operators:

    from mhc.library import sinkhorn_knopp, fused_stream_mix, fused_add_residual, fused_dynamic_weights

Same signatures and results as the functions of the same names in ``mhc.ops`` (the four above follow the
reference's src/mhc/ops.py:231-323); dropout takes its generator state as a tensor or draws it, and the 8-bit
outputs have no gradient.
"""

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _backward as B
from . import _kernels as K


# ------------------------------------------------------------------------------ Sinkhorn
@torch.library.custom_op("mhc::sinkhorn_fwd", mutates_args=())
def _sinkhorn_fwd(M: Tensor, iters: int, eps: float) -> Tensor:
    return K.sinkhorn_forward(M, iters, eps)


@_sinkhorn_fwd.register_fake
def _(M, iters, eps):
    return torch.empty_like(M, memory_format=torch.contiguous_format)


@torch.library.custom_op("mhc::sinkhorn_bwd", mutates_args=())
def _sinkhorn_bwd(M: Tensor, dP: Tensor, iters: int, eps: float) -> Tensor:
    return B.sinkhorn_backward(M, dP, iters, eps)


@_sinkhorn_bwd.register_fake
def _(M, dP, iters, eps):
    return torch.empty_like(M, memory_format=torch.contiguous_format)


def _sinkhorn_setup(ctx, inputs, output):
    M, ctx.iters, ctx.eps = inputs
    ctx.save_for_backward(M)


def _sinkhorn_grad(ctx, g):
    (M,) = ctx.saved_tensors
    return _sinkhorn_bwd(M, g.contiguous(), ctx.iters, ctx.eps), None, None


_sinkhorn_fwd.register_autograd(_sinkhorn_grad, setup_context=_sinkhorn_setup)


# ---------------------------------------------------------------------------- stream mix
@torch.library.custom_op("mhc::stream_mix_fwd", mutates_args=())
def _stream_mix_fwd(H: Tensor, H_pre: Tensor, H_res: Tensor) -> Tuple[Tensor, Tensor]:
    return K.stream_mix_forward(H, H_pre, H_res)


@_stream_mix_fwd.register_fake
def _(H, H_pre, H_res):
    Bn, S, _, D = H.shape
    return H.new_empty(Bn, S, D), torch.empty_like(H, memory_format=torch.contiguous_format)


@torch.library.custom_op("mhc::stream_mix_bwd", mutates_args=())
def _stream_mix_bwd(d_bi: Tensor, dHr: Tensor, H: Tensor, H_pre: Tensor, H_res: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    return B.stream_mix_backward(d_bi, dHr, H, H_pre, H_res)


@_stream_mix_bwd.register_fake
def _(d_bi, dHr, H, H_pre, H_res):
    Bn = H.shape[0]
    return (torch.empty_like(H, memory_format=torch.contiguous_format),
            H.new_empty(Bn, 4, dtype=torch.float32), H.new_empty(Bn, 4, 4, dtype=torch.float32))


def _mix_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _mix_grad(ctx, g_bi, g_hr):
    H, H_pre, H_res = ctx.saved_tensors
    dH, dH_pre, dH_res = _stream_mix_bwd(g_bi.contiguous(), g_hr.contiguous(), H, H_pre, H_res)
    return dH, dH_pre.to(H_pre.dtype), dH_res.to(H_res.dtype)


_stream_mix_fwd.register_autograd(_mix_grad, setup_context=_mix_setup)


# -------------------------------------------------------------------------- add residual
@torch.library.custom_op("mhc::add_residual_fwd", mutates_args=())
def _add_residual_fwd(H_residual: Tensor, branch_output: Tensor, H_post: Tensor) -> Tensor:
    return K.add_residual_forward(H_residual, branch_output, H_post)


@_add_residual_fwd.register_fake
def _(H_residual, branch_output, H_post):
    return torch.empty_like(H_residual, memory_format=torch.contiguous_format)


@torch.library.custom_op("mhc::add_residual_bwd", mutates_args=())
def _add_residual_bwd(dH_new: Tensor, branch_output: Tensor, H_post: Tensor) -> Tuple[Tensor, Tensor]:
    _, d_bo, dH_post = B.add_residual_backward(dH_new, branch_output, H_post)
    return d_bo, dH_post


@_add_residual_bwd.register_fake
def _(dH_new, branch_output, H_post):
    return (torch.empty_like(branch_output, dtype=dH_new.dtype, memory_format=torch.contiguous_format),
            dH_new.new_empty(dH_new.shape[0], 4, dtype=torch.float32))


def _add_setup(ctx, inputs, output):
    _, branch_output, H_post = inputs
    ctx.save_for_backward(branch_output, H_post)


def _add_grad(ctx, g):
    branch_output, H_post = ctx.saved_tensors
    g = g.contiguous()
    d_bo, dH_post = _add_residual_bwd(g, branch_output, H_post)
    return g, d_bo.to(branch_output.dtype), dH_post.to(H_post.dtype)   # the residual's gradient is g itself


_add_residual_fwd.register_autograd(_add_grad, setup_context=_add_setup)


# ------------------------------------------------------------------------ dynamic weights
@torch.library.custom_op("mhc::dynamic_weights_fwd", mutates_args=())
def _dynamic_weights_fwd(x: Tensor, phi: Tensor, bias: Tensor, alpha_pre: Tensor, alpha_post: Tensor,
                         alpha_res: Tensor, iters: int, eps: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    return K.fused_dynamic_weights_forward(x, phi, bias, alpha_pre, alpha_post, alpha_res, iters, eps,
                                           return_saved=True)


@_dynamic_weights_fwd.register_fake
def _(x, phi, bias, alpha_pre, alpha_post, alpha_res, iters, eps):
    Bn = x.shape[0]
    f = dict(dtype=torch.float32)
    return x.new_empty(Bn, 4, **f), x.new_empty(Bn, 4, **f), x.new_empty(Bn, 4, 4, **f), x.new_empty(Bn, 32, **f)


@torch.library.custom_op("mhc::dynamic_weights_bwd", mutates_args=())
def _dynamic_weights_bwd(x: Tensor, phi: Tensor, bias: Tensor, alpha_pre: Tensor, alpha_post: Tensor,
                         alpha_res: Tensor, saved: Tensor, g_pre: Tensor, g_post: Tensor, g_res: Tensor,
                         iters: int, eps: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    gx, gphi, gbias, galpha = B.fused_dynamic_weights_backward(x, phi, bias, alpha_pre, alpha_post, alpha_res, saved,
                                                               g_pre, g_post, g_res, iters, eps)
    return gx, gphi.clone(), gbias.clone(), galpha.clone()   # the wrapper returns views of one buffer


@_dynamic_weights_bwd.register_fake
def _(x, phi, bias, alpha_pre, alpha_post, alpha_res, saved, g_pre, g_post, g_res, iters, eps):
    f = dict(dtype=torch.float32)
    return (x.new_empty(x.shape, **f), x.new_empty(phi.shape, **f), x.new_empty(24, **f), x.new_empty(3, **f))


def _dw_setup(ctx, inputs, output):
    x, phi, bias, a_pre, a_post, a_res, ctx.iters, ctx.eps = inputs
    ctx.save_for_backward(x, phi, bias, a_pre, a_post, a_res, output[3])


def _dw_grad(ctx, g_pre, g_post, g_res, _g_saved):
    x, phi, bias, a_pre, a_post, a_res, saved = ctx.saved_tensors
    gx, gphi, gbias, galpha = _dynamic_weights_bwd(x, phi, bias, a_pre, a_post, a_res, saved, g_pre.contiguous(),
                                                   g_post.contiguous(), g_res.contiguous(), ctx.iters, ctx.eps)
    return (gx.to(x.dtype), gphi.to(phi.dtype), gbias.to(bias.dtype), galpha[0:1].reshape(a_pre.shape).to(a_pre.dtype),
            galpha[1:2].reshape(a_post.shape).to(a_post.dtype), galpha[2:3].reshape(a_res.shape).to(a_res.dtype),
            None, None)


_dynamic_weights_fwd.register_autograd(_dw_grad, setup_context=_dw_setup)


# --------------------------------------------------------------------------- public names
def sinkhorn_knopp(M: Tensor, num_iters: int = 20, eps: float = 1e-8) -> Tensor:
    return _sinkhorn_fwd(M, num_iters, eps)


def fused_stream_mix(H: Tensor, H_pre: Tensor, H_res: Tensor) -> Tuple[Tensor, Tensor]:
    return _stream_mix_fwd(H, H_pre, H_res)


def fused_add_residual(H_residual: Tensor, branch_output: Tensor, H_post: Tensor, dropout_p: float = 0.0,
                       rng: Optional[Tensor] = None, row_offset: int = 0) -> Tensor:
    threshold = K.drop_threshold(dropout_p)
    if threshold:
        return _add_residual_dropout_fwd(H_residual, branch_output, H_post, _draw(rng, branch_output), threshold, row_offset)
    return _add_residual_fwd(H_residual, branch_output, H_post)


def fused_dynamic_weights(x: Tensor, phi: Tensor, bias: Tensor, alpha_pre, alpha_post, alpha_res,
                          sinkhorn_iters: int = 20, eps: float = 1e-6) -> Tuple[Tensor, Tensor, Tensor]:
    """alpha_* are one-element tensors (they then receive gradients) or Python floats."""
    alpha_pre, alpha_post, alpha_res = [a if isinstance(a, Tensor) else torch.full((1,), float(a), device=x.device)
                                        for a in (alpha_pre, alpha_post, alpha_res)]
    H_pre, H_post, H_res, _ = _dynamic_weights_fwd(x, phi, bias, alpha_pre, alpha_post, alpha_res, sinkhorn_iters, eps)
    return H_pre, H_post, H_res


# ------------------------------------------------------------------------ counter-based dropout
# `rng` (two int64 on the device) is an explicit input of every operator, so a traced program draws where it says it does.
@torch.library.custom_op("mhc::counter_dropout", mutates_args=())
def _counter_dropout(x: Tensor, rng: Tensor, threshold: int, row_offset: int) -> Tensor:
    return K.counter_dropout_forward(x, rng, threshold, row_offset)


@_counter_dropout.register_fake
def _(x, rng, threshold, row_offset):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _dropout_setup(ctx, inputs, output):
    _, rng, ctx.threshold, ctx.row_offset = inputs
    ctx.save_for_backward(rng)


def _dropout_grad(ctx, g):
    (rng,) = ctx.saved_tensors
    return _counter_dropout(g.contiguous(), rng, ctx.threshold, ctx.row_offset), None, None, None


_counter_dropout.register_autograd(_dropout_grad, setup_context=_dropout_setup)


@torch.library.custom_op("mhc::add_residual_dropout_fwd", mutates_args=())
def _add_residual_dropout_fwd(H_residual: Tensor, branch_output: Tensor, H_post: Tensor, rng: Tensor, threshold: int,
                              row_offset: int) -> Tensor:
    return K.add_residual_dropout_forward(H_residual, None, branch_output, H_post, rng, threshold, row_offset)


@_add_residual_dropout_fwd.register_fake
def _(H_residual, branch_output, H_post, rng, threshold, row_offset):
    return torch.empty_like(H_residual, memory_format=torch.contiguous_format)


@torch.library.custom_op("mhc::add_residual_dropout_bwd", mutates_args=())
def _add_residual_dropout_bwd(dH_new: Tensor, branch_output: Tensor, H_post: Tensor, rng: Tensor, threshold: int,
                              row_offset: int) -> Tuple[Tensor, Tensor]:
    _, d_bo, dH_post = B.add_residual_dropout_backward(dH_new, branch_output, H_post, rng, threshold, row_offset)
    return d_bo, dH_post


@_add_residual_dropout_bwd.register_fake
def _(dH_new, branch_output, H_post, rng, threshold, row_offset):
    return (torch.empty_like(branch_output, dtype=dH_new.dtype, memory_format=torch.contiguous_format),
            dH_new.new_empty(dH_new.shape[0], 4, dtype=torch.float32))


def _add_dropout_setup(ctx, inputs, output):
    _, branch_output, H_post, rng, ctx.threshold, ctx.row_offset = inputs
    ctx.save_for_backward(branch_output, H_post, rng)


def _add_dropout_grad(ctx, g):
    branch_output, H_post, rng = ctx.saved_tensors
    g = g.contiguous()
    d_bo, dH_post = _add_residual_dropout_bwd(g, branch_output, H_post, rng, ctx.threshold, ctx.row_offset)
    return g, d_bo.to(branch_output.dtype), dH_post.to(H_post.dtype), None, None, None


_add_residual_dropout_fwd.register_autograd(_add_dropout_grad, setup_context=_add_dropout_setup)


# ------------------------------------------------------------------------------------- RMS norm
@torch.library.custom_op("mhc::add_rms_norm_fwd", mutates_args=())
def _add_rms_norm_fwd(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, rng: Optional[Tensor],
                      threshold: int, row_offset: int) -> Tuple[Tensor, Tensor, Tensor]:
    y, s, rstd = K.add_rms_norm_forward(x, residual, weight, eps, rng, threshold, row_offset)
    return y, (s if residual is not None or threshold else x.new_empty(0)), rstd   # s is x itself then


@_add_rms_norm_fwd.register_fake
def _(x, residual, weight, eps, rng, threshold, row_offset):
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = 1
    for n in x.shape[:-1]:
        rows = rows * n
    return (y, torch.empty_like(y) if residual is not None or threshold else x.new_empty(0),
            x.new_empty(rows, dtype=torch.float32))


@torch.library.custom_op("mhc::rms_norm_bwd", mutates_args=())
def _rms_norm_bwd(dy: Tensor, dsum: Optional[Tensor], x: Tensor, residual: Optional[Tensor], rstd: Tensor,
                  weight: Optional[Tensor], rng: Optional[Tensor], threshold: int,
                  row_offset: int) -> Tuple[Tensor, Tensor, Tensor]:
    dx, dres, dw = B.rms_norm_backward(dy, dsum, x, residual, rstd, weight, rng, threshold, row_offset,
                                       want_dresidual=residual is not None, want_dweight=weight is not None)
    # absent outputs (no residual's own gradient without dropout, no weight): a tensor each, outputs may not alias
    return (dx, dres if threshold and residual is not None else x.new_empty(0), x.new_empty(0) if dw is None else dw)


@_rms_norm_bwd.register_fake
def _(dy, dsum, x, residual, rstd, weight, rng, threshold, row_offset):
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    return (dx, torch.empty_like(dx) if threshold and residual is not None else x.new_empty(0),
            x.new_empty(0) if weight is None else torch.empty_like(weight, memory_format=torch.contiguous_format))


def _norm_setup(ctx, inputs, output):
    x, residual, weight, _, rng, ctx.threshold, ctx.row_offset = inputs
    ctx.save_for_backward(x, residual, weight, rng, output[2])


def _norm_grad(ctx, gy, gs, _g_rstd):
    x, residual, weight, rng, rstd = ctx.saved_tensors
    has_s = residual is not None or ctx.threshold
    dx, dres, dw = _rms_norm_bwd(gy.contiguous(), gs.contiguous() if has_s else None, x, residual, rstd, weight, rng,
                                 ctx.threshold, ctx.row_offset)
    if residual is not None:
        dres = (dres if ctx.threshold else dx).to(residual.dtype)
    return dx, dres if residual is not None else None, dw if weight is not None else None, None, None, None, None


_add_rms_norm_fwd.register_autograd(_norm_grad, setup_context=_norm_setup)


@torch.library.custom_op("mhc::add_rms_norm_quant_fwd", mutates_args=())
def _add_rms_norm_quant_fwd(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, group: int,
                            scale_dtype: torch.dtype) -> Tuple[Tensor, Tensor, Tensor]:
    q, scales, s = K.add_rms_norm_quant_forward(x, residual, weight, eps, group, scale_dtype)
    return q, scales, (s if residual is not None else x.new_empty(0))


@_add_rms_norm_quant_fwd.register_fake
def _(x, residual, weight, eps, group, scale_dtype):
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    G = -(-x.shape[-1] // group) if group else torch.sym_min(x.shape[-1], 1)
    return (q, x.new_empty(tuple(x.shape[:-1]) + (G,), dtype=scale_dtype),
            torch.empty_like(x, memory_format=torch.contiguous_format) if residual is not None else x.new_empty(0))


@torch.library.custom_op("mhc::stream_norm_fwd", mutates_args=())
def _stream_norm_fwd(H: Tensor, H_pre: Tensor, weight: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor]:
    y, _, rstd = K.stream_norm_forward(H, H_pre, weight, eps)
    return y, rstd


@_stream_norm_fwd.register_fake
def _(H, H_pre, weight, eps):
    Bn, S, _, D = H.shape
    return H.new_empty(Bn, S, D), H.new_empty(Bn * S, dtype=torch.float32)


@torch.library.custom_op("mhc::stream_norm_bwd", mutates_args=())
def _stream_norm_bwd(dy: Tensor, H: Tensor, H_pre: Tensor, rstd: Tensor,
                     weight: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    dH, dH_pre, dw = B.stream_norm_backward(dy, H, H_pre, rstd, weight, want_dweight=weight is not None)
    return dH, dH_pre, (H.new_empty(0) if dw is None else dw)


@_stream_norm_bwd.register_fake
def _(dy, H, H_pre, rstd, weight):
    return (torch.empty_like(H, memory_format=torch.contiguous_format), H.new_empty(H.shape[0], 4, dtype=torch.float32),
            H.new_empty(0) if weight is None else torch.empty_like(weight, memory_format=torch.contiguous_format))


def _stream_norm_setup(ctx, inputs, output):
    H, H_pre, weight, _ = inputs
    ctx.save_for_backward(H, H_pre, weight, output[1])


def _stream_norm_grad(ctx, gy, _g_rstd):
    H, H_pre, weight, rstd = ctx.saved_tensors
    dH, dH_pre, dw = _stream_norm_bwd(gy.contiguous(), H, H_pre, rstd, weight)
    return dH, dH_pre.to(H_pre.dtype), dw if weight is not None else None, None


_stream_norm_fwd.register_autograd(_stream_norm_grad, setup_context=_stream_norm_setup)


@torch.library.custom_op("mhc::stream_norm_quant_fwd", mutates_args=())
def _stream_norm_quant_fwd(H: Tensor, H_pre: Tensor, weight: Optional[Tensor], eps: float, group: int,
                           scale_dtype: torch.dtype) -> Tuple[Tensor, Tensor]:
    return K.stream_norm_quant_forward(H, H_pre, weight, eps, group, scale_dtype)


@_stream_norm_quant_fwd.register_fake
def _(H, H_pre, weight, eps, group, scale_dtype):
    Bn, S, _, D = H.shape
    G = -(-D // group) if group else torch.sym_min(D, 1)
    return H.new_empty(Bn, S, D, dtype=torch.float8_e4m3fn), H.new_empty(Bn, S, G, dtype=scale_dtype)


def _draw(rng, like):
    """The generator state as a tensor: rng itself, or a draw from torch's generator."""
    return torch.randint(-(1 << 63), (1 << 63) - 1, (2,), device=like.device, dtype=torch.int64) if rng is None else rng


def counter_dropout(x: Tensor, p: float, rng: Optional[Tensor] = None, row_offset: int = 0) -> Tensor:
    threshold = K.drop_threshold(p)
    return _counter_dropout(x, _draw(rng, x), threshold, row_offset) if threshold else x


def fused_add_rms_norm(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None, eps: float = 1e-6,
                       dropout_p: float = 0.0, rng: Optional[Tensor] = None, row_offset: int = 0) -> Tuple[Tensor, Tensor]:
    threshold = K.drop_threshold(dropout_p)
    y, s, _ = _add_rms_norm_fwd(x, residual, weight, eps, _draw(rng, x) if threshold else None, threshold, row_offset)
    return y, (s if residual is not None or threshold else x)


def fused_add_rms_norm_quant(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None,
                             eps: float = 1e-6, group: Optional[int] = None,
                             scale_dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor, Tensor]:
    q, scales, s = _add_rms_norm_quant_fwd(x, residual, weight, eps, group or 0, scale_dtype)
    return q, scales, (s if residual is not None else x)


def fused_stream_norm(H: Tensor, H_pre: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6) -> Tensor:
    return _stream_norm_fwd(H, H_pre, weight, eps)[0]


def fused_stream_norm_quant(H: Tensor, H_pre: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6,
                            group: Optional[int] = None,
                            scale_dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
    return _stream_norm_quant_fwd(H, H_pre, weight, eps, group or 0, scale_dtype)
