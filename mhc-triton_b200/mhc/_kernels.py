"""Forward launch wrappers: validate, allocate outputs with torch, call the C ABI.

Names and signatures follow the launch wrappers of the reference
(src/mhc/_kernels.py:597-752 there); `block_dim` is accepted and ignored because the
tiling is fixed inside the CUDA kernels.
"""

from typing import Optional, Tuple

import torch

from . import _lib as L


def _check(cond, msg):
    if not cond:
        raise AssertionError(msg)


def sinkhorn_forward(M: torch.Tensor, num_iters: int = 20, eps: float = 1e-8) -> torch.Tensor:
    """P = Sinkhorn(|M| + eps) for M of shape (..., 4, 4); same dtype as M."""
    _check(M.shape[-2:] == (4, 4), "Expected (..., 4, 4)")
    L.require_cuda(M)
    M = M.contiguous()
    P = torch.empty_like(M)
    with torch.cuda.device(M.device):
        L.call("mhc_sinkhorn_fwd", L.stream_of(M), L.ptr(M), L.ptr(P), M.numel() // 16, L.dtype_code(M), int(num_iters),
                                          float(eps))
    return P


def stream_mix_forward(H: torch.Tensor, H_pre: torch.Tensor, H_res: torch.Tensor,
                       block_dim: int = 128, want_residual: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(branch_input [B,S,D], H_residual [B,S,4,D]) in H's dtype; with want_residual=False the
    residual mix is not written and None is returned in its place."""
    _check(H.dim() == 4, "H must be [batch, seq, 4, dim]")
    B, S, n, D = H.shape
    _check(n == 4, "num_streams must be 4")
    _check(tuple(H_pre.shape) == (B, 4), f"H_pre shape mismatch: {tuple(H_pre.shape)} vs ({B}, 4)")
    _check(tuple(H_res.shape) == (B, 4, 4), f"H_res shape mismatch: {tuple(H_res.shape)} vs ({B}, 4, 4)")
    L.require_cuda(H, H_pre, H_res)
    H = H.contiguous()
    H_pre, H_res = L.f32c(H_pre), L.f32c(H_res)
    bi = torch.empty(B, S, D, device=H.device, dtype=H.dtype)
    Hr = torch.empty_like(H) if want_residual else None
    with torch.cuda.device(H.device):
        L.call("mhc_stream_mix_fwd", L.stream_of(H), L.ptr(H), L.ptr(H_pre), L.ptr(H_res), L.ptr(bi), L.ptr(Hr), B, S, D,
                                            L.dtype_code(H))
    return bi, Hr


def add_residual_forward(H_residual: torch.Tensor, branch_output: torch.Tensor, H_post: torch.Tensor,
                         block_dim: int = 128, pool: bool = False):
    """H_new = H_residual + H_post[:, None, :, None] * branch_output[:, :, None, :].
    With pool=True returns (H_new, partials): partials [B, chunks, 4*D] fp32 are the token sums of
    H_new per chunk, which the next layer's fused forward accepts in place of its own pooling pass."""
    _check(H_residual.dim() == 4, "H_residual must be [batch, seq, 4, dim]")
    B, S, n, D = H_residual.shape
    _check(n == 4, "num_streams must be 4")
    _check(tuple(branch_output.shape) == (B, S, D), "branch_output shape mismatch")
    _check(tuple(H_post.shape) == (B, 4), "H_post shape mismatch")
    L.require_cuda(H_residual, branch_output, H_post)
    H_residual = H_residual.contiguous()
    branch_output = branch_output.to(H_residual.dtype).contiguous()
    H_post = L.f32c(H_post)
    H_new = torch.empty_like(H_residual)
    if pool:
        chunks = L.load().mhc_add_residual_pool_chunks(S, D)
        partials = torch.empty(B, chunks, 4 * D, device=H_residual.device, dtype=torch.float32)
        with torch.cuda.device(H_residual.device):
            L.call("mhc_add_residual_pool_fwd", L.stream_of(H_residual), L.ptr(H_residual), L.ptr(branch_output),
                   L.ptr(H_post), L.ptr(H_new), L.ptr(partials), B, S, D, L.dtype_code(H_residual))
        return H_new, partials
    with torch.cuda.device(H_residual.device):
        L.call("mhc_add_residual_fwd", L.stream_of(H_residual), L.ptr(H_residual), L.ptr(branch_output), L.ptr(H_post), L.ptr(H_new),
                                              B, S, D, L.dtype_code(H_residual))
    return H_new


def meanpool_forward(H: torch.Tensor) -> torch.Tensor:
    """x[b, n*D+d] = mean_s H[b,s,n,d] as fp32 [B, 4*D] (fp32 accumulation, fixed order)."""
    _check(H.dim() == 4 and H.shape[2] == 4, "H must be [batch, seq, 4, dim]")
    B, S, _, D = H.shape
    _check(S > 0, "empty sequence")
    L.require_cuda(H)
    H = H.contiguous()
    x = torch.empty(B, 4 * D, device=H.device, dtype=torch.float32)
    buf, nbytes = L.scratch(L.OP_MEANPOOL_FWD, B, S, D, H)
    with torch.cuda.device(H.device):
        L.call("mhc_meanpool_fwd", L.stream_of(H), L.ptr(H), L.ptr(x), L.ptr(buf), nbytes, B, S, D, L.dtype_code(H))
    return x


last_dynamic_weights_scratch = None


def _alpha_dev(a, like: torch.Tensor) -> torch.Tensor:
    """A scale as a one-element fp32 device tensor (Python floats are uploaded without a sync)."""
    if torch.is_tensor(a):
        _check(a.numel() == 1, "alpha must have one element")
        L.require_cuda(a)
        return L.f32c(a.reshape(1))
    return torch.full((1,), float(a), device=like.device, dtype=torch.float32)


def fused_dynamic_weights_forward(x: torch.Tensor, phi: torch.Tensor, bias: torch.Tensor, alpha_pre, alpha_post,
                                  alpha_res, sinkhorn_iters: int = 20, eps: float = 1e-6, return_saved: bool = False):
    """(H_pre [B,4], H_post [B,4], H_res [B,4,4]), always fp32.

    alpha_* may be Python floats (as in the reference signature) or one-element device
    tensors; tensors are read on the device, so no host synchronisation happens.
    With return_saved=True a fourth tensor [B,32] with the raw projections, sum(x^2) and
    inv_rms is returned for the backward.
    """
    _check(x.dim() == 2, "x must be [batch, in_dim]")
    B, K = x.shape
    _check(tuple(phi.shape) == (K, 24), f"phi shape mismatch: {tuple(phi.shape)} vs ({K}, 24)")
    _check(tuple(bias.shape) == (24,), f"bias shape mismatch: {tuple(bias.shape)} vs (24,)")
    L.require_cuda(x, phi, bias)
    x, phi, bias = L.f32c(x), L.f32c(phi), L.f32c(bias)
    a = [_alpha_dev(v, x) for v in (alpha_pre, alpha_post, alpha_res)]
    H_pre = torch.empty(B, 4, device=x.device, dtype=torch.float32)
    H_post = torch.empty(B, 4, device=x.device, dtype=torch.float32)
    H_res = torch.empty(B, 4, 4, device=x.device, dtype=torch.float32)
    saved = torch.empty(B, 32, device=x.device, dtype=torch.float32)
    buf, nbytes = L.scratch(L.OP_DYNAMIC_WEIGHTS_FWD, B, 0, (K + 3) // 4, x)
    global last_dynamic_weights_scratch
    last_dynamic_weights_scratch = buf     # its first int is the status word of the many-rows kernels (0 = fine)
    with torch.cuda.device(x.device):
        L.call("mhc_dynamic_weights_fwd", L.stream_of(x), L.ptr(x), L.ptr(phi), L.ptr(bias), L.ptr(a[0]), L.ptr(a[1]),
                                                 L.ptr(a[2]), L.ptr(H_pre), L.ptr(H_post), L.ptr(H_res), L.ptr(saved),
                                                 L.ptr(buf), nbytes, B, K, int(sinkhorn_iters), float(eps))
    if return_saved:
        return H_pre, H_post, H_res, saved
    return H_pre, H_post, H_res


def hc_mix_forward(H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res,
                   sinkhorn_iters: int = 20, eps: float = 1e-6, pooled=None, want_residual: bool = True):
    """Fused forward of the module's dynamic path in ONE library call: sequence mean-pool,
    dynamic weights, stream mix.  Returns
    (branch_input, H_residual, H_post, H_pre, H_res, x, saved); x [B,4D] and saved [B,32]
    are what the fused backward needs.  `pooled` ([B, chunks, 4D] fp32 token sums of H from the
    previous layer's add_residual_forward(pool=True)) replaces the pooling pass over H.  With
    want_residual=False H_residual is not written (returned as None): the caller adds the residual
    with add_residual_mix_forward, which recomputes the mix from H."""
    _check(H.dim() == 4 and H.shape[2] == 4, "H must be [batch, seq, 4, dim]")
    B, S, _, D = H.shape
    _check(S > 0 and D > 0, "empty sequence or width")
    _check(tuple(phi.shape) == (4 * D, 24), f"phi shape mismatch: {tuple(phi.shape)} vs ({4 * D}, 24)")
    _check(H_pre_base.numel() == 4 and H_post_base.numel() == 4 and H_res_base.numel() == 16, "base parameter shapes")
    L.require_cuda(H, phi, H_pre_base, H_post_base, H_res_base)
    H = H.contiguous()
    phi, pre_b, post_b, res_b = L.f32c(phi), L.f32c(H_pre_base), L.f32c(H_post_base), L.f32c(H_res_base)
    a = [_alpha_dev(v, H) for v in (alpha_pre, alpha_post, alpha_res)]
    dev = H.device
    small = torch.empty(B * 56, device=dev, dtype=torch.float32)   # one allocation for the small outputs
    H_pre, H_post = small[:4 * B].view(B, 4), small[4 * B:8 * B].view(B, 4)
    H_res, saved = small[8 * B:24 * B].view(B, 4, 4), small[24 * B:].view(B, 32)
    x = torch.empty(B, 4 * D, device=dev, dtype=torch.float32)
    bi = torch.empty(B, S, D, device=dev, dtype=H.dtype)
    Hr = torch.empty_like(H) if want_residual else None
    buf, nbytes = L.scratch(L.OP_HC_MIX_FWD, B, S, D, H)
    chunks = 0
    if pooled is not None:
        _check(pooled.dim() == 3 and pooled.shape[0] == B and pooled.shape[2] == 4 * D and pooled.dtype == torch.float32
               and pooled.is_contiguous() and pooled.device == dev, "pooled must be contiguous fp32 [B, chunks, 4*D]")
        chunks = pooled.shape[1]
    with torch.cuda.device(dev):
        L.call("mhc_hc_mix_fwd", L.stream_of(H), L.ptr(H), L.ptr(phi), L.ptr(pre_b), L.ptr(post_b), L.ptr(res_b),
               L.ptr(a[0]), L.ptr(a[1]), L.ptr(a[2]), L.ptr(x), L.ptr(H_pre), L.ptr(H_post), L.ptr(H_res), L.ptr(saved),
               L.ptr(bi), L.ptr(Hr), L.ptr(pooled), chunks, L.ptr(buf), nbytes, L.tickets(H, B), B, S, D,
               L.dtype_code(H), int(sinkhorn_iters), float(eps))
    return bi, Hr, H_post, H_pre, H_res, x, saved


def add_residual_mix_forward(H: torch.Tensor, H_res: torch.Tensor, branch_output: torch.Tensor, H_post: torch.Tensor,
                             pool: bool = False):
    """H_new = H_res @ H (over the stream axis) + H_post * branch_output in one kernel: the residual
    mix is recomputed from H instead of being read from a materialised H_residual.  With pool=True
    returns (H_new, partials) as add_residual_forward does."""
    _check(H.dim() == 4 and H.shape[2] == 4, "H must be [batch, seq, 4, dim]")
    B, S, _, D = H.shape
    _check(tuple(branch_output.shape) == (B, S, D), "branch_output shape mismatch")
    _check(tuple(H_post.shape) == (B, 4) and tuple(H_res.shape) == (B, 4, 4), "weight shape mismatch")
    L.require_cuda(H, H_res, branch_output, H_post)
    H = H.contiguous()
    branch_output = branch_output.to(H.dtype).contiguous()
    H_post, H_res = L.f32c(H_post), L.f32c(H_res)
    H_new = torch.empty_like(H)
    partials = None
    if pool:
        chunks = L.load().mhc_add_residual_pool_chunks(S, D)
        partials = torch.empty(B, chunks, 4 * D, device=H.device, dtype=torch.float32)
    with torch.cuda.device(H.device):
        L.call("mhc_add_residual_mix_fwd", L.stream_of(H), L.ptr(H), L.ptr(H_res), L.ptr(branch_output), L.ptr(H_post),
               L.ptr(H_new), L.ptr(partials), B, S, D, L.dtype_code(H))
    return (H_new, partials) if pool else H_new


# ------------------------------------------------------------------------------------ counter-based dropout
def drop_threshold(p: float) -> int:
    """The dropout probability in 1/65536ths, the unit the kernels draw in (0: nothing is dropped)."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability must be in [0, 1), got {p}")
    t = int(round(p * 65536.0))
    if t > 65535:
        raise ValueError(f"dropout probability {p} rounds to 1 (it is taken in steps of 1/65536)")
    return t


def dropout_rng(rng, like: torch.Tensor) -> torch.Tensor:
    """The generator state of a dropout call as two int64 (seed, offset) on `like`'s device: `rng` itself if it
    is such a tensor, a pair of integers put there, or, for None, a draw from torch's generator of the device."""
    if rng is None:
        return torch.empty(2, device=like.device, dtype=torch.int64).random_()
    if torch.is_tensor(rng):
        _check(rng.dtype == torch.int64 and rng.numel() == 2, "rng must hold two int64 values (seed, offset)")
        return rng if rng.is_contiguous() else rng.contiguous()
    seed, offset = (int(v) & 0xFFFFFFFFFFFFFFFF for v in rng)
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in (seed, offset)], device=like.device, dtype=torch.int64)


def row_number(row_offset) -> int:
    """row_offset as an int that the library can be given (it refuses what is not in [0, 2^32 - rows])."""
    row_offset = int(row_offset)
    if not -(1 << 63) <= row_offset < 1 << 63:
        raise ValueError(f"row_offset must be in [0, 2^32), got {row_offset}")
    return row_offset


def _rows_of(t: torch.Tensor) -> Tuple[int, int]:
    """(rows, columns) of a tensor whose last axis are the columns."""
    D = t.shape[-1]
    if D:
        return t.numel() // D, D
    n = 1
    for s in t.shape[:-1]:
        n *= s
    return n, D


def counter_dropout_forward(x: torch.Tensor, rng: torch.Tensor, threshold: int, row_offset: int = 0) -> torch.Tensor:
    """x with each element dropped (0) with probability threshold / 65536, or scaled up; rows are all axes but the last."""
    if x.dim() < 1:
        raise AssertionError("x must have at least one axis")
    dev = L.same_device(x, rng)
    x = x.contiguous()
    y = torch.empty_like(x)
    rows, D = _rows_of(x)
    L.call_on(dev, "mhc_counter_dropout", x.data_ptr(), rng.data_ptr(), threshold, row_offset, y.data_ptr(), rows, D,
              L.dtype_code(x))
    return y


def add_residual_dropout_forward(H, H_res, branch_output, H_post, rng, threshold: int, row_offset: int = 0,
                                 pool: bool = False):
    """add_residual_forward (H_res None: H is the materialised residual mix) or add_residual_mix_forward with
    branch_output passed through the counter-based dropout."""
    _check(H.dim() == 4 and H.shape[2] == 4, "H must be [batch, seq, 4, dim]")
    B, S, _, D = H.shape
    _check(branch_output.shape == (B, S, D), "branch_output shape mismatch")
    _check(H_post.shape == (B, 4) and (H_res is None or H_res.shape == (B, 4, 4)), "weight shape mismatch")
    dev = L.same_device(H, H_res, branch_output, H_post, rng)
    H = H.contiguous()
    branch_output = branch_output.to(H.dtype).contiguous()
    H_post = L.f32c(H_post)
    H_res = None if H_res is None else L.f32c(H_res)
    H_new = torch.empty_like(H)
    partials = None
    if pool:
        chunks = L.load().mhc_add_residual_pool_chunks(S, D)
        partials = torch.empty(B, chunks, 4 * D, device=H.device, dtype=torch.float32)
    L.call_on(dev, "mhc_add_residual_dropout_fwd", H.data_ptr(), L.ptr(H_res), branch_output.data_ptr(), H_post.data_ptr(),
              rng.data_ptr(), threshold, row_offset, H_new.data_ptr(), L.ptr(partials), B, S, D, L.dtype_code(H))
    return (H_new, partials) if pool else H_new


# --------------------------------------------------------------------------------------------- RMS norm
_E4M3 = torch.float8_e4m3fn
_SCALES = {torch.float32: L.SCALE_F32, torch.float8_e8m0fnu: L.SCALE_E8M0}


def _norm_weight(weight, dtype, D) -> Tuple[Optional[torch.Tensor], int, Optional[int]]:
    """The weight as the kernels take it (fp32 or the activations' type, contiguous), its type code and its address."""
    if weight is None:
        return None, L.MHC_F32, None
    if weight.shape != (D,):
        raise AssertionError(f"weight shape mismatch: {tuple(weight.shape)} vs ({D},)")
    if weight.dtype != dtype and weight.dtype != torch.float32:
        weight = weight.float()
    weight = weight.contiguous()
    return weight, L.dtype_code(weight), weight.data_ptr()


def _norm_inputs(x, residual):
    if x.dim() < 1:
        raise AssertionError("x must have at least one axis")
    if residual is not None:
        if residual.shape != x.shape:
            raise AssertionError(f"residual shape mismatch: {tuple(residual.shape)} vs {tuple(x.shape)}")
        residual = (residual if residual.dtype == x.dtype else residual.to(x.dtype)).contiguous()
    return x.contiguous(), residual


def add_rms_norm_forward(x, residual=None, weight=None, eps: float = 1e-6, rng=None, threshold: int = 0,
                         row_offset: int = 0, want_rstd: bool = True):
    """(y, s, rstd): s = dropout(x) + residual (x itself when there is neither), y = s * rstd * weight."""
    dev = L.same_device(x, residual, weight, rng)
    x, residual = _norm_inputs(x, residual)
    rows, D = _rows_of(x)
    w, wcode, wptr = _norm_weight(weight, x.dtype, D)
    y = torch.empty_like(x)
    s = torch.empty_like(x) if residual is not None or threshold else None
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if want_rstd else None
    L.call_on(dev, "mhc_add_rms_norm_fwd", x.data_ptr(), None if residual is None else residual.data_ptr(), wptr, wcode,
              L.ptr(rng), threshold, row_offset, None if s is None else s.data_ptr(), y.data_ptr(), L.ptr(rstd), rows, D,
              L.dtype_code(x), eps)
    return y, (x if s is None else s), rstd


def _scales_for(lead, D, group, scale_dtype, device):
    group = 0 if group is None else int(group)
    if group not in (0, 32, 64, 128):
        raise ValueError(f"group must be None (one scale per row), 32, 64 or 128, got {group}")
    if scale_dtype not in _SCALES:
        raise TypeError(f"mhc: unsupported scale dtype {scale_dtype} (float32, float8_e8m0fnu only)")
    G = -(-D // group) if group else min(D, 1)
    return group, _SCALES[scale_dtype], torch.empty((*lead, G), device=device, dtype=scale_dtype)


def add_rms_norm_quant_forward(x, residual=None, weight=None, eps: float = 1e-6, group=None,
                               scale_dtype=torch.float32):
    """(q, scales, s): the norm's output as e4m3 q with one scale per row or per `group` columns."""
    dev = L.same_device(x, residual, weight)
    x, residual = _norm_inputs(x, residual)
    rows, D = _rows_of(x)
    w, wcode, wptr = _norm_weight(weight, x.dtype, D)
    group, scode, scales = _scales_for(x.shape[:-1], D, group, scale_dtype, x.device)
    q = torch.empty_like(x, dtype=_E4M3)
    s = torch.empty_like(x) if residual is not None else None
    L.call_on(dev, "mhc_add_rms_norm_quant_fwd", x.data_ptr(), L.ptr(residual), wptr, wcode, L.ptr(s), q.data_ptr(),
              scales.data_ptr(), group, scode, rows, D, L.dtype_code(x), eps)
    return q, scales, (x if s is None else s)


def _stream_inputs(H, H_pre, weight):
    if H.dim() != 4 or H.shape[2] != 4:
        raise AssertionError("H must be [batch, seq, 4, dim]")
    if H_pre.shape != (H.shape[0], 4):
        raise AssertionError(f"H_pre shape mismatch: {tuple(H_pre.shape)} vs ({H.shape[0]}, 4)")
    dev = L.same_device(H, H_pre, weight)
    return dev, H.contiguous(), L.f32c(H_pre), _norm_weight(weight, H.dtype, H.shape[3])


def stream_norm_forward(H, H_pre, weight=None, eps: float = 1e-6, want_branch_input: bool = False,
                        want_rstd: bool = True):
    """(y, branch_input or None, rstd [B*S]): branch_input = sum_n H_pre[n] H[n], y its norm times weight.  With
    want_branch_input y is the norm of the stored (rounded) branch_input: its backward is rms_norm_backward on that and then
    the mix's; stream_norm_backward belongs to the form without."""
    dev, H, H_pre, (w, wcode, wptr) = _stream_inputs(H, H_pre, weight)
    B, S, _, D = H.shape
    y = torch.empty((B, S, D), device=H.device, dtype=H.dtype)
    bi = torch.empty_like(y) if want_branch_input else None
    rstd = torch.empty(B * S, device=H.device, dtype=torch.float32) if want_rstd else None
    L.call_on(dev, "mhc_stream_norm_fwd", H.data_ptr(), H_pre.data_ptr(), wptr, wcode, L.ptr(bi), y.data_ptr(), L.ptr(rstd),
              B, S, D, L.dtype_code(H), eps)
    return y, bi, rstd


def stream_norm_quant_forward(H, H_pre, weight=None, eps: float = 1e-6, group=None, scale_dtype=torch.float32):
    """(q, scales): stream_norm_forward's y as e4m3 with one scale per token or per `group` columns."""
    dev, H, H_pre, (w, wcode, wptr) = _stream_inputs(H, H_pre, weight)
    B, S, _, D = H.shape
    group, scode, scales = _scales_for((B, S), D, group, scale_dtype, H.device)
    q = torch.empty((B, S, D), device=H.device, dtype=_E4M3)
    L.call_on(dev, "mhc_stream_norm_quant_fwd", H.data_ptr(), H_pre.data_ptr(), wptr, wcode, q.data_ptr(), scales.data_ptr(),
              group, scode, B, S, D, L.dtype_code(H), eps)
    return q, scales


def hc_mix_norm_forward(H, H_pre_base, H_post_base, H_res_base, phi, alpha_pre, alpha_post, alpha_res, norm_weight,
                        norm_eps: float = 1e-6, sinkhorn_iters: int = 20, eps: float = 1e-6, pooled=None):
    """hc_mix_forward(want_residual=False) with the norm of branch_input fused into its last kernel.  Returns
    (y, branch_input, rstd, H_post, H_pre, H_res, x, saved)."""
    _check(H.dim() == 4 and H.shape[2] == 4, "H must be [batch, seq, 4, dim]")
    B, S, _, D = H.shape
    _check(S > 0 and D > 0, "empty sequence or width")
    _check(tuple(phi.shape) == (4 * D, 24), f"phi shape mismatch: {tuple(phi.shape)} vs ({4 * D}, 24)")
    _check(H_pre_base.numel() == 4 and H_post_base.numel() == 4 and H_res_base.numel() == 16, "base parameter shapes")
    index = L.same_device(H, phi, H_pre_base, H_post_base, H_res_base, norm_weight)
    H = H.contiguous()
    w, wcode, wptr = _norm_weight(norm_weight, H.dtype, D)
    phi, pre_b, post_b, res_b = L.f32c(phi), L.f32c(H_pre_base), L.f32c(H_post_base), L.f32c(H_res_base)
    a = [_alpha_dev(v, H) for v in (alpha_pre, alpha_post, alpha_res)]
    dev = H.device
    small = torch.empty(B * 56 + B * S, device=dev, dtype=torch.float32)   # one allocation for the small outputs
    H_pre, H_post = small[:4 * B].view(B, 4), small[4 * B:8 * B].view(B, 4)
    H_res, saved = small[8 * B:24 * B].view(B, 4, 4), small[24 * B:56 * B].view(B, 32)
    rstd = small[56 * B:]
    x = torch.empty(B, 4 * D, device=dev, dtype=torch.float32)
    bi = torch.empty(B, S, D, device=dev, dtype=H.dtype)
    y = torch.empty_like(bi)
    buf, nbytes = L.scratch(L.OP_HC_MIX_FWD, B, S, D, H)
    chunks = 0
    if pooled is not None:
        _check(pooled.dim() == 3 and pooled.shape[0] == B and pooled.shape[2] == 4 * D and pooled.dtype == torch.float32
               and pooled.is_contiguous() and pooled.device == dev, "pooled must be contiguous fp32 [B, chunks, 4*D]")
        chunks = pooled.shape[1]
    L.call_on(index, "mhc_hc_mix_norm_fwd", L.ptr(H), L.ptr(phi), L.ptr(pre_b), L.ptr(post_b), L.ptr(res_b), L.ptr(a[0]),
              L.ptr(a[1]), L.ptr(a[2]), wptr, wcode, float(norm_eps), L.ptr(x), L.ptr(H_pre), L.ptr(H_post),
              L.ptr(H_res), L.ptr(saved), L.ptr(bi), L.ptr(y), L.ptr(rstd), L.ptr(pooled), chunks, L.ptr(buf), nbytes,
              L.eager_tickets(H, B), B, S, D, L.dtype_code(H), int(sinkhorn_iters), float(eps))
    return y, bi, rstd, H_post, H_pre, H_res, x, saved
