"""Autograd ops of the hyper-connection path, backed by the sm_100a CUDA library.

Public functions and their semantics follow the reference's src/mhc/ops.py:231-323:
sinkhorn_knopp, fused_stream_mix, fused_add_residual, fused_dynamic_weights.
`hyper_connection_mix` is the fused node the module uses: mean-pool + dynamic weights +
stream mix in one autograd Function, so that the gradient of the pooled state is folded into
the single write of dH instead of a separate read-modify-write pass.
"""

import functools
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from ._backward import (add_residual_backward, add_residual_dropout_backward, fused_dynamic_weights_backward,
                        hc_mix_backward, rms_norm_backward, sinkhorn_backward, stream_mix_backward,
                        stream_norm_backward)
from ._kernels import (add_residual_dropout_forward, add_residual_forward, add_residual_mix_forward,
                       add_rms_norm_forward, add_rms_norm_quant_forward, counter_dropout_forward, drop_threshold,
                       dropout_rng, fused_dynamic_weights_forward, hc_mix_forward, hc_mix_norm_forward,
                       meanpool_forward, row_number, sinkhorn_forward, stream_mix_forward, stream_norm_forward,
                       stream_norm_quant_forward)


# The public functions below are opaque to torch.compile (the kernels are reached through ctypes):
# a compiled model calls them eagerly and compiles what surrounds them.


class _SinkhornKnopp(torch.autograd.Function):
    """Saves only M; the backward recomputes the iterations (reference: src/mhc/ops.py:15-29)."""

    @staticmethod
    def forward(ctx, M, num_iters, eps):
        ctx.save_for_backward(M)
        ctx.num_iters, ctx.eps = num_iters, eps
        return sinkhorn_forward(M, num_iters, eps)

    @staticmethod
    def backward(ctx, grad_output):
        (M,) = ctx.saved_tensors
        return sinkhorn_backward(M, grad_output, ctx.num_iters, ctx.eps), None, None


class _FusedStreamMix(torch.autograd.Function):
    """Reference: src/mhc/ops.py:32-49."""

    @staticmethod
    def forward(ctx, H, H_pre, H_res):
        branch_input, H_residual = stream_mix_forward(H, H_pre, H_res)
        ctx.save_for_backward(H, H_pre, H_res)
        ctx.set_materialize_grads(False)
        return branch_input, H_residual

    @staticmethod
    def backward(ctx, grad_branch_input, grad_H_residual):
        H, H_pre, H_res = ctx.saved_tensors
        if grad_branch_input is None and grad_H_residual is None:
            return None, None, None
        if grad_branch_input is None:
            grad_branch_input = torch.zeros(H.shape[0], H.shape[1], H.shape[3], device=H.device, dtype=H.dtype)
        if grad_H_residual is None:
            grad_H_residual = torch.zeros_like(H)
        dH, dH_pre, dH_res = stream_mix_backward(grad_branch_input, grad_H_residual, H, H_pre, H_res)
        return dH, dH_pre.to(H_pre.dtype), dH_res.to(H_res.dtype)


class _FusedAddResidual(torch.autograd.Function):
    """Reference: src/mhc/ops.py:52-69.  The gradient of H_residual is the upstream gradient
    itself and is returned without a copy."""

    @staticmethod
    def forward(ctx, H_residual, branch_output, H_post, pool):
        ctx.save_for_backward(branch_output, H_post)
        ctx.set_materialize_grads(False)
        if pool:
            H_new, partials = add_residual_forward(H_residual, branch_output, H_post, pool=True)
            ctx.mark_non_differentiable(partials)
            return H_new, partials
        return add_residual_forward(H_residual, branch_output, H_post)

    @staticmethod
    def backward(ctx, grad_H_new, _unused=None):
        if grad_H_new is None:
            return None, None, None, None
        branch_output, H_post = ctx.saved_tensors
        dH_residual, d_bo, dH_post = add_residual_backward(grad_H_new, branch_output, H_post)
        return dH_residual, d_bo.to(branch_output.dtype), dH_post.to(H_post.dtype), None


class _AddResidualFromState(torch.autograd.Function):
    """H_new = H_res @ H + H_post * branch_output with the residual mix recomputed from H.

    `stand_in` is the storage-less second output of the fused node run with lazy_residual=True;
    the gradient with respect to the residual mix (which equals the upstream gradient) is returned
    for it, and the fused node turns it into the gradients of H and H_res, exactly as it does for
    a materialised H_residual.  That is why H and H_res receive no gradient from this node."""

    @staticmethod
    def forward(ctx, stand_in, H, H_res, branch_output, H_post, pool):
        ctx.save_for_backward(branch_output, H_post)
        ctx.set_materialize_grads(False)
        if pool:
            H_new, partials = add_residual_mix_forward(H, H_res, branch_output, H_post, pool=True)
            ctx.mark_non_differentiable(partials)
            return H_new, partials
        return add_residual_mix_forward(H, H_res, branch_output, H_post)

    @staticmethod
    def backward(ctx, grad_H_new, _unused=None):
        if grad_H_new is None:
            return None, None, None, None, None, None
        branch_output, H_post = ctx.saved_tensors
        dH_residual, d_bo, dH_post = add_residual_backward(grad_H_new, branch_output, H_post)
        return dH_residual, None, None, d_bo.to(branch_output.dtype), dH_post.to(H_post.dtype), None


class _FusedDynamicWeights(torch.autograd.Function):
    """Reference: src/mhc/ops.py:72-228.  The scales are read on the device (no .item())."""

    @staticmethod
    def forward(ctx, x, phi, bias, alpha_pre, alpha_post, alpha_res, sinkhorn_iters, eps):
        H_pre, H_post, H_res, saved = fused_dynamic_weights_forward(
            x, phi, bias, alpha_pre, alpha_post, alpha_res, sinkhorn_iters, eps, return_saved=True)
        ctx.save_for_backward(x, phi, bias, alpha_pre, alpha_post, alpha_res, saved)
        ctx.sinkhorn_iters, ctx.eps = sinkhorn_iters, eps
        ctx.set_materialize_grads(False)
        return H_pre, H_post, H_res

    @staticmethod
    def backward(ctx, grad_H_pre, grad_H_post, grad_H_res):
        x, phi, bias, alpha_pre, alpha_post, alpha_res, saved = ctx.saved_tensors
        B = x.shape[0]
        if grad_H_pre is None:
            grad_H_pre = torch.zeros(B, 4, device=x.device)
        if grad_H_post is None:
            grad_H_post = torch.zeros(B, 4, device=x.device)
        if grad_H_res is None:
            grad_H_res = torch.zeros(B, 4, 4, device=x.device)
        gx, gphi, gbias, galpha = fused_dynamic_weights_backward(
            x, phi, bias, alpha_pre, alpha_post, alpha_res, saved, grad_H_pre, grad_H_post, grad_H_res,
            ctx.sinkhorn_iters, ctx.eps)
        return (gx.to(x.dtype), gphi.to(phi.dtype), gbias.to(bias.dtype),
                galpha[0:1].reshape_as(alpha_pre).to(alpha_pre.dtype),
                galpha[1:2].reshape_as(alpha_post).to(alpha_post.dtype),
                galpha[2:3].reshape_as(alpha_res).to(alpha_res.dtype), None, None)


class _SequenceMeanPool(torch.autograd.Function):
    """x = H.mean(dim=1).reshape(B, 4*D) in fp32 (reference: src/mhc/module.py:123)."""

    @staticmethod
    def forward(ctx, H):
        ctx.shape, ctx.dtype = H.shape, H.dtype
        return meanpool_forward(H)

    @staticmethod
    def backward(ctx, gx):
        B, S, n, D = ctx.shape
        return (gx.reshape(B, 1, n, D) / S).to(ctx.dtype).expand(B, S, n, D)


class _NoSecondDerivative(torch.autograd.Function):
    """Hands gradients on; differentiating them is an error.  `anchor` requires a gradient, so the result always does."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(g.view_as(g) for g in grads)    # one tensor may stand for two inputs' gradients

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("mhc: this operator has no second derivative")


def _first_order(depends, applies=lambda ctx: True):
    """Decorates the `backward` of a node whose kernels' results cannot be differentiated.  Under create_graph=True (grad mode
    is on in a backward only then) they come out such that differentiating them is an error, where the upstream gradients
    are differentiated or the gradients depend on the node's own differentiated inputs (`depends(ctx, *grads)`).  Elsewhere
    they are constants; an upstream gradient that is handed through stays what it is.  Nodes for which `applies` is false run
    `backward` as it is."""
    def decorate(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            if not (torch.is_grad_enabled() and applies(ctx)):
                return backward(ctx, *grads)
            with torch.no_grad():
                out = backward(ctx, *grads)
            given = [g for g in grads if g is not None]
            if not depends(ctx, *grads) and not any(g.requires_grad for g in given):
                return out
            which = [i for i, o in enumerate(out) if o is not None and not any(o is g for g in given)]
            if not which:
                return out
            anchor = torch.empty(0, device=out[which[0]].device, requires_grad=True)
            marked = dict(zip(which, _NoSecondDerivative.apply(anchor, *[out[i] for i in which])))
            return tuple(marked.get(i, o) for i, o in enumerate(out))
        return run
    return decorate


class _HyperConnectionMix(torch.autograd.Function):
    """Mean-pool + dynamic weights + stream mix as one autograd node.

    Inputs : H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res
    Outputs: branch_input, H_residual, H_post
    Forward and backward are one library call each.  Backward: one reduction pass (dH_pre,
    dH_res), the small weights backward, then one apply pass that writes dH once, including
    grad_x / S.  When `grad_sink` (a flat fp32
    buffer of 4*D*24 + 27 elements) is given, grad_phi / grad_bias / grad_alpha are written
    straight into it, ready for one all-reduce, and `ready_hook` is told so; `ready_event`, if
    given, is recorded on the stream between the kernels that fill the buffer and the pass that
    writes dH, so a collective that waits for it overlaps that pass.
    """

    @staticmethod
    def forward(ctx, H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res,
                sinkhorn_iters, eps, grad_sink, ready_hook, accumulate, pooled, lazy_residual, ready_event=None,
                norm_weight=None, norm_eps=None):
        ctx.has_norm = norm_eps is not None
        if ctx.has_norm:
            branch_input, mixed, rstd, H_post, H_pre, H_res, x, saved = hc_mix_norm_forward(
                H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res, norm_weight, norm_eps,
                sinkhorn_iters, eps, pooled=pooled)
            norm_saved = (mixed, rstd, norm_weight)
        else:
            branch_input, H_residual, H_post, H_pre, H_res, x, saved = hc_mix_forward(
                H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res, sinkhorn_iters, eps,
                pooled=pooled, want_residual=not lazy_residual)
            norm_saved = ()
        if lazy_residual:
            # A stand-in with H's shape and no storage of its own: it only carries the gradient of the
            # (never materialised) residual mix back to this node.  Its values are meaningless.
            H_residual = branch_input.new_empty(1).expand(H.shape)
        ctx.save_for_backward(H, x, phi, H_pre_base, H_post_base, H_res_base, alpha_pre, alpha_post, alpha_res,
                              saved, H_pre, H_res, *norm_saved)
        ctx.sinkhorn_iters, ctx.eps, ctx.grad_sink, ctx.ready_hook = sinkhorn_iters, eps, grad_sink, ready_hook
        ctx.accumulate = bool(accumulate) and grad_sink is not None
        ctx.ready_event = ready_event
        ctx.mark_non_differentiable(H_pre, H_res)
        ctx.set_materialize_grads(False)   # no zero-filled gradients for outputs nobody used
        return branch_input, H_residual, H_post, H_pre, H_res

    # With the norm no term may be left out (its weight's gradient alone does not depend on the weight); without it the
    # gradients have always come back as constants.
    @staticmethod
    @_first_order(lambda ctx, *_: any(ctx.needs_input_grad[:8]), applies=lambda ctx: ctx.has_norm)
    def backward(ctx, d_branch_input, dH_residual, dH_post, _unused_pre, _unused_res):
        (H, x, phi, pre_b, post_b, res_b, alpha_pre, alpha_post, alpha_res, saved, H_pre, H_res) = ctx.saved_tensors[:12]
        B, S, _, D = H.shape
        if d_branch_input is None:
            d_branch_input = torch.zeros(B, S, D, device=H.device, dtype=H.dtype)
        d_norm_weight = None
        if ctx.has_norm:   # the gradient of the normalised branch input -> that of the mix
            mixed, rstd, norm_weight = ctx.saved_tensors[12:]
            d_branch_input, _, d_norm_weight = rms_norm_backward(d_branch_input, None, mixed, None, rstd, norm_weight,
                                                                 want_dweight=ctx.needs_input_grad[16])
        if dH_residual is None:
            dH_residual = torch.zeros_like(H)
        if dH_post is None:
            dH_post = torch.zeros(B, 4, device=H.device, dtype=torch.float32)
        dH, gphi, gbias, galpha = hc_mix_backward(
            d_branch_input, dH_residual, dH_post, H, x, phi, pre_b, post_b, res_b, alpha_pre, alpha_post, alpha_res,
            saved, H_pre, H_res, ctx.sinkhorn_iters, ctx.eps, param_grads=ctx.grad_sink, accumulate=ctx.accumulate,
            ready_event=ctx.ready_event)
        if ctx.ready_hook is not None:
            ctx.ready_hook(ctx.grad_sink)
        if ctx.grad_sink is not None:  # the parameters' .grad tensors are views of the sink already
            return (dH,) + (None,) * 15 + (d_norm_weight, None)
        return (dH, gbias[0:4].reshape(pre_b.shape).to(pre_b.dtype), gbias[4:8].reshape(post_b.shape).to(post_b.dtype),
                gbias[8:24].reshape(res_b.shape).to(res_b.dtype), gphi.to(phi.dtype),
                galpha[0:1].reshape_as(alpha_pre).to(alpha_pre.dtype),
                galpha[1:2].reshape_as(alpha_post).to(alpha_post.dtype),
                galpha[2:3].reshape_as(alpha_res).to(alpha_res.dtype)) + (None,) * 8 + (d_norm_weight, None)


class _AddResidualDropout(torch.autograd.Function):
    """_FusedAddResidual (H_res None) and _AddResidualFromState (first input: the storage-less stand-in) with the
    branch output passed through the counter-based dropout.  The mask is recomputed in the backward from `rng`."""

    @staticmethod
    def forward(ctx, carrier, H, H_res, branch_output, H_post, pool, rng, threshold, row_offset):
        out = add_residual_dropout_forward(carrier if H is None else H, H_res, branch_output, H_post, rng, threshold,
                                           row_offset, pool=pool)
        ctx.save_for_backward(branch_output, H_post, rng)
        ctx.threshold, ctx.row_offset = threshold, row_offset
        ctx.set_materialize_grads(False)
        if pool:
            ctx.mark_non_differentiable(out[1])
        return out

    @staticmethod
    @_first_order(lambda ctx, *_: ctx.needs_input_grad[3] and ctx.needs_input_grad[4])    # each depends on the other input
    def backward(ctx, grad_H_new, _unused=None):
        if grad_H_new is None:
            return (None,) * 9
        branch_output, H_post, rng = ctx.saved_tensors
        dH_residual, d_bo, dH_post = add_residual_dropout_backward(grad_H_new, branch_output, H_post, rng,
                                                                   ctx.threshold, ctx.row_offset)
        return (dH_residual, None, None, d_bo.to(branch_output.dtype), dH_post.to(H_post.dtype)) + (None,) * 4


class _CounterDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rng, threshold, row_offset):
        ctx.save_for_backward(rng)
        ctx.threshold, ctx.row_offset = threshold, row_offset
        return counter_dropout_forward(x, rng, threshold, row_offset)

    @staticmethod
    @_first_order(lambda ctx, *_: False)    # linear
    def backward(ctx, grad):
        (rng,) = ctx.saved_tensors
        return counter_dropout_forward(grad, rng, ctx.threshold, ctx.row_offset), None, None, None


class _AddRmsNorm(torch.autograd.Function):
    """Outputs (y, s); with neither residual nor dropout s is x and only y is an output of the node."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, rng, threshold, row_offset):
        y, s, rstd = add_rms_norm_forward(x, residual, weight, eps, rng, threshold, row_offset)
        ctx.save_for_backward(x, residual, rstd, weight, rng)   # s is formed again: rounded, it would cost dweight its accuracy
        ctx.threshold, ctx.row_offset = threshold, row_offset
        ctx.set_materialize_grads(False)
        return (y, s) if residual is not None or threshold else y

    @staticmethod
    # s is linear in x and the residual, and the weight's gradient does not depend on the weight
    @_first_order(lambda ctx, dy, ds=None: dy is not None and any(ctx.needs_input_grad[:2]))
    def backward(ctx, dy, ds=None):
        if dy is None and ds is None:
            return (None,) * 7
        x, residual, rstd, weight, rng = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        dx, dres, dw = rms_norm_backward(dy, ds, x, residual, rstd, weight, rng, ctx.threshold, ctx.row_offset,
                                         want_dresidual=need_res, want_dweight=need_w)
        if need_res and dres.dtype != residual.dtype:
            dres = dres.to(residual.dtype)
        return dx if need_x else None, dres if need_res else None, dw, None, None, None, None


class _FusedStreamNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, H, H_pre, weight, eps):
        y, _, rstd = stream_norm_forward(H, H_pre, weight, eps)
        ctx.save_for_backward(H, H_pre, weight, rstd)
        return y

    @staticmethod
    @_first_order(lambda ctx, *_: any(ctx.needs_input_grad[:2]))
    def backward(ctx, dy):
        H, H_pre, weight, rstd = ctx.saved_tensors
        dH, dH_pre, dw = stream_norm_backward(dy, H, H_pre, rstd, weight, want_dweight=ctx.needs_input_grad[2])
        return dH, (dH_pre if dH_pre.dtype == H_pre.dtype else dH_pre.to(H_pre.dtype)), dw, None


@torch.compiler.disable
def sinkhorn_knopp(M: torch.Tensor, num_iters: int = 20, eps: float = 1e-8) -> torch.Tensor:
    """Project (batch, 4, 4) matrices to (approximately) doubly stochastic ones by `num_iters`
    alternating row / column normalisations of |M| + eps."""
    return _SinkhornKnopp.apply(M, num_iters, eps)


@torch.compiler.disable
def fused_stream_mix(H: torch.Tensor, H_pre: torch.Tensor, H_res: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """H (batch, seq, 4, dim), H_pre (batch, 4), H_res (batch, 4, 4) ->
    branch_input (batch, seq, dim), H_residual (batch, seq, 4, dim)."""
    return _FusedStreamMix.apply(H, H_pre, H_res)


@torch.compiler.disable
def fused_add_residual(H_residual: torch.Tensor, branch_output: torch.Tensor, H_post: torch.Tensor,
                       pool_for_next: bool = False, dropout_p: float = 0.0, rng=None,
                       row_offset: int = 0) -> torch.Tensor:
    """H_new[n] = H_residual[n] + H_post[n] * branch_output, per batch element.

    With pool_for_next=True the same kernel also accumulates the per-chunk token sums of H_new and
    the returned tensor carries them (attribute `_mhc_pooled`); a HyperConnection that receives
    this very tensor as its input uses them instead of reading H once more for its mean-pool.

    With dropout_p > 0 the branch output goes through counter_dropout(branch_output, dropout_p, rng,
    row_offset) inside the same kernel (rows are batch * seq tokens)."""
    threshold = drop_threshold(dropout_p)
    if threshold:
        return _add_residual_dropout(H_residual, None, None, branch_output, H_post, pool_for_next, rng, threshold, row_offset)
    if not pool_for_next:
        return _FusedAddResidual.apply(H_residual, branch_output, H_post, False)
    H_new, partials = _FusedAddResidual.apply(H_residual, branch_output, H_post, True)
    H_new._mhc_pooled = (partials, version_of(H_new))
    return H_new


@torch.compiler.disable
def add_residual_from_state(stand_in, H, H_res, branch_output, H_post, pool_for_next: bool = False,
                            dropout_p: float = 0.0, rng=None, row_offset: int = 0) -> torch.Tensor:
    """Second half of a layer whose fused node ran with lazy_residual=True (see hyper_connection_mix):
    H_new = H_res @ H + H_post * branch_output, the residual mix recomputed from H.  Dropout of the branch
    output as in fused_add_residual."""
    threshold = drop_threshold(dropout_p)
    if threshold:
        return _add_residual_dropout(stand_in, H, H_res, branch_output, H_post, pool_for_next, rng, threshold, row_offset)
    if not pool_for_next:
        return _AddResidualFromState.apply(stand_in, H, H_res, branch_output, H_post, False)
    H_new, partials = _AddResidualFromState.apply(stand_in, H, H_res, branch_output, H_post, True)
    H_new._mhc_pooled = (partials, version_of(H_new))
    return H_new


def _add_residual_dropout(carrier, H, H_res, branch_output, H_post, pool_for_next, rng, threshold, row_offset):
    rng = dropout_rng(rng, branch_output)
    out = _AddResidualDropout.apply(carrier, H, H_res, branch_output, H_post, bool(pool_for_next), rng, threshold,
                                    row_number(row_offset))
    if not pool_for_next:
        return out
    H_new, partials = out
    H_new._mhc_pooled = (partials, version_of(H_new))
    return H_new


def version_of(t: torch.Tensor):
    """In-place modification counter of t, or None for inference tensors (which keep none)."""
    return None if t.is_inference() else t._version


def pooled_sums_of(H: torch.Tensor):
    """Token sums attached to H by fused_add_residual(pool_for_next=True), or None if absent, of the
    wrong shape, or if H was modified in place since."""
    tag = getattr(H, "_mhc_pooled", None)
    if tag is None:
        return None
    partials, version = tag
    if version_of(H) != version or H.dim() != 4 or partials.shape[0] != H.shape[0] or \
            partials.shape[2] != 4 * H.shape[3] or partials.device != H.device:
        return None
    return partials


@torch.compiler.disable
def fused_dynamic_weights(x, phi, bias, alpha_pre, alpha_post, alpha_res, sinkhorn_iters: int = 20,
                          eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [batch, in_dim], phi [in_dim, 24], bias [24], three one-element scale tensors ->
    H_pre [batch, 4] (rows sum to 1), H_post [batch, 4] in (0, 2), H_res [batch, 4, 4]
    (Sinkhorn-projected).  Outputs are fp32."""
    return _FusedDynamicWeights.apply(x, phi, bias, alpha_pre, alpha_post, alpha_res, sinkhorn_iters, eps)


@torch.compiler.disable
def sequence_mean_pool(H: torch.Tensor) -> torch.Tensor:
    """H (batch, seq, 4, dim) -> fp32 (batch, 4*dim) mean over the sequence axis."""
    return _SequenceMeanPool.apply(H)


@torch.compiler.disable
def hyper_connection_mix(H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res,
                         sinkhorn_iters: int = 20, eps: float = 1e-6, grad_sink=None, ready_hook=None,
                         accumulate: bool = False, pooled=None, lazy_residual: bool = False, ready_event=None,
                         norm_weight: Optional[torch.Tensor] = None, norm_eps: Optional[float] = None):
    """Fused pooled-weights + stream-mix node; returns
    (branch_input, H_residual, H_post, H_pre, H_res); the last two carry no gradient.
    With `grad_sink` the parameter gradients are written into that flat buffer and no
    gradient is returned for the parameters; `ready_hook(grad_sink)` is called as soon as
    the kernels that fill it have been launched; `accumulate` adds to the buffer instead of
    overwriting it; `pooled` are token sums of H from the previous layer (see fused_add_residual).
    With lazy_residual=True the second output is a storage-less stand-in to be passed to
    add_residual_from_state, which recomputes the residual mix from H.  `ready_event`: a
    torch.cuda.Event the backward records once the parameter gradients are complete in stream
    order (before dH is).  With `norm_eps` given (needs lazy_residual=True) branch_input is returned normalised:
    branch_input * rsqrt(mean(branch_input^2) + norm_eps) * norm_weight (None: ones)."""
    if norm_eps is None and norm_weight is not None:
        raise ValueError("norm_weight without norm_eps")
    if norm_eps is not None and not lazy_residual:
        raise ValueError("the norm of branch_input needs lazy_residual=True")
    return _HyperConnectionMix.apply(H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res,
                                     sinkhorn_iters, eps, grad_sink, ready_hook, accumulate, pooled, lazy_residual,
                                     ready_event, norm_weight, norm_eps)


def _records(*tensors) -> bool:
    """Whether autograd would record an operation on these, in reverse or (to refuse it) in forward mode."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:
        return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    return False


@torch.compiler.disable
def counter_dropout(x: torch.Tensor, p: float, rng=None, row_offset: int = 0) -> torch.Tensor:
    """Dropout whose mask is a function of (seed, offset, row, column) and is never stored: x[..., d] is 0 with
    probability p (taken in steps of 1/65536), else scaled by 1 / (1 - p); the backward recomputes the mask.

    rng: two int64 (seed, offset) on x's device, read by the kernels; a pair of integers; or None, which draws
    a pair from torch's CUDA generator (so torch.manual_seed, activation checkpointing and graph capture work as
    with torch's dropout).  The tensor must hold the same values in the backward: to draw anew, pass another one, or
    write to it between the backward and the next forward.  The last axis of x are the columns, all others the
    rows, numbered from row_offset: a shard of rows that is given the index of its first row gets the mask of the
    whole tensor.  Use it while training; with p = 0 it returns x."""
    threshold = drop_threshold(p)
    if threshold == 0:
        return x
    rng = dropout_rng(rng, x)
    if not _records(x):
        return counter_dropout_forward(x, rng, threshold, row_number(row_offset))
    return _CounterDropout.apply(x, rng, threshold, row_number(row_offset))


@torch.compiler.disable
def fused_add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                       weight: Optional[torch.Tensor] = None, eps: float = 1e-6, dropout_p: float = 0.0, rng=None,
                       row_offset: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """s = dropout(x) + residual; y = s * rsqrt(mean(s^2, -1) + eps) * weight.  Returns (y, s), both in x's dtype;
    with neither residual nor dropout s is x itself.

    x and residual (..., dim), weight (dim) in fp32 or x's dtype (None: ones).  Statistics are fp32 and s is
    normalised before it is rounded to x's dtype.  dropout_p, rng, row_offset as in counter_dropout."""
    threshold = drop_threshold(dropout_p)
    rng = dropout_rng(rng, x) if threshold else None
    if not _records(x, residual, weight):
        y, s, _ = add_rms_norm_forward(x, residual, weight, eps, rng, threshold, row_number(row_offset), want_rstd=False)
        return y, (s if residual is not None or threshold else x)
    out = _AddRmsNorm.apply(x, residual, weight, eps, rng, threshold, row_number(row_offset))
    return out if isinstance(out, tuple) else (out, x)


def _no_gradient(what, *tensors):
    if _records(*tensors):
        raise RuntimeError(f"{what} has no gradient (its output is 8 bits wide): call it under torch.no_grad(), or "
                           "use the unquantised form for training")


@torch.compiler.disable
def fused_add_rms_norm_quant(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                             weight: Optional[torch.Tensor] = None, eps: float = 1e-6, group: Optional[int] = None,
                             scale_dtype: torch.dtype = torch.float32):
    """fused_add_rms_norm with y in 8 bits: returns (q, scales, s) with y ~ q * scales.

    q (..., dim) is torch.float8_e4m3fn; scales (..., 1) hold one scale per row, or (..., ceil(dim / group)) one per
    `group` = 32, 64 or 128 columns: max|y| / 448 in fp32, or with scale_dtype=torch.float8_e8m0fnu the next power of
    two not below it (the form block-scaled matrix instructions take for groups of 32).  The smallest scale is
    2^-126.  For inference: no gradient."""
    _no_gradient("fused_add_rms_norm_quant", x, residual, weight)
    q, scales, s = add_rms_norm_quant_forward(x, residual, weight, eps, group, scale_dtype)
    return q, scales, (s if residual is not None else x)


@torch.compiler.disable
def fused_stream_norm(H: torch.Tensor, H_pre: torch.Tensor, weight: Optional[torch.Tensor] = None,
                      eps: float = 1e-6) -> torch.Tensor:
    """The branch input of fused_stream_mix, normalised in the kernel that mixes it:
    b = sum_n H_pre[n] H[n]; y = b * rsqrt(mean(b^2, -1) + eps) * weight.  H (batch, seq, 4, dim), H_pre (batch, 4),
    weight (dim) in fp32 or H's dtype (None: ones) -> y (batch, seq, dim)."""
    if not _records(H, H_pre, weight):
        return stream_norm_forward(H, H_pre, weight, eps, want_rstd=False)[0]
    return _FusedStreamNorm.apply(H, H_pre, weight, eps)


@torch.compiler.disable
def fused_stream_norm_quant(H: torch.Tensor, H_pre: torch.Tensor, weight: Optional[torch.Tensor] = None,
                            eps: float = 1e-6, group: Optional[int] = None,
                            scale_dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """fused_stream_norm with y in 8 bits: (q, scales) as fused_add_rms_norm_quant returns them.  No gradient."""
    _no_gradient("fused_stream_norm_quant", H, H_pre, weight)
    return stream_norm_quant_forward(H, H_pre, weight, eps, group, scale_dtype)
