"""The operators around a sub-layer where their other tests do not go: extreme batch sizes, the layer's own kernels in the
16-bit types, many rows in fp32, unaligned 8-bit outputs, all against 64 bits.

Tolerances are those of tests/test_gpu_sublayer.py: u = 2^-24 for each fp32 rounding on the way, half a step of the stored
type for the last one."""

import pytest
import torch

from oracle import sublayer_oracle as SO

from . import test_gpu_sublayer as base
from .test_gpu_sublayer import EPS, TYPES, U, check_quant, cuda, draw, half_step, mixed64, steps, stream_case, subnormal, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ more than 2^30 batch elements
# Their 2^32 mixing weights are past 32-bit positions.  Only the first and the last batch elements hold anything but zeros.
MANY = 2 ** 30 + 8


def many_elements(D, dtype):
    need = MANY * (4 * D * dtype.itemsize + 4 * 4 + 2 * D * 4 + 8)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need + (4 << 30):
        pytest.skip(f"needs {need >> 30} GiB of free device memory")
    g = torch.Generator().manual_seed(D)
    ends = torch.cat([torch.arange(8), torch.arange(MANY - 8, MANY)]).cuda()
    H = torch.zeros(MANY, 1, 4, D, device="cuda", dtype=dtype)
    pre = torch.zeros(MANY, 4, device="cuda")
    H[ends] = torch.randn(16, 1, 4, D, generator=g).to(dtype).cuda()
    pre[ends] = (torch.rand(16, 4, generator=g) + 0.05).cuda()
    return H, pre, ends


def mixed64_of(H, pre, at):
    terms = H[at].double().cpu() * pre[at].double().cpu()[:, None, :, None]
    return terms.sum(2), terms.abs().sum(2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_stream_norm_of_a_billion_batch_elements(dtype):
    import mhc
    H, pre, ends = many_elements(1, dtype)
    y = mhc.fused_stream_norm(H, pre, None, 1.0)
    b64, b_mag = mixed64_of(H, pre, ends)
    y64, rstd = SO.rms_norm(b64, torch.ones(1, dtype=torch.float64), 1.0)
    # eps = 1: rstd is at most 1, so the mix's error reaches y with a factor of at most 2
    within(y[ends], y64, half_step(dtype) * y64.abs() + 2 * steps(1) * U * b_mag + 1e-30, "y")
    assert not y[8:16].any() and not y[-16:-8].any()


def test_stream_norm_quant_of_a_billion_batch_elements():
    import mhc
    H, pre, ends = many_elements(4, torch.float32)      # packs of four: the persistent forward
    q, scales = mhc.fused_stream_norm_quant(H, pre, None, 1.0)
    b64, b_mag = mixed64_of(H, pre, ends)
    y64, rstd = SO.rms_norm(b64, torch.ones(4, dtype=torch.float64), 1.0)
    row = (b_mag.square().sum(-1, keepdim=True) / (b64.square().sum(-1, keepdim=True) + 4)).sqrt()
    q = q.view(torch.uint8)[ends].view(torch.float8_e4m3fn)
    check_quant(q, scales[ends], y64, steps(4) * U * (1 + row) * rstd * b_mag + 1e-300, 0, False, 4)


# --------------------------------------------------------------------------- the mix as it is stored, and the norm of that
def check_norm_of_stored(y, bi, rstd, H, pre, w, eps):
    """branch_input is the mix, rounded once; y and rstd belong to the stored value, and so does the norm's own backward."""
    from mhc._backward import rms_norm_backward
    dtype, D = H.dtype, H.shape[3]
    h, k = half_step(dtype), steps(D) * U
    b64, b_mag = mixed64(H, pre)
    within(bi, b64, h * b64.abs() + 8 * U * b_mag + subnormal(dtype), "branch_input")
    s64 = bi.double().cpu()                      # exactly what is normalised: no error of the mix in what follows
    y64, rstd64 = SO.rms_norm(s64, w.double(), eps)
    within(rstd.view(rstd64.shape), rstd64, k * rstd64, "rstd")
    within(y, y64, (h + k) * y64.abs() + subnormal(dtype), "y")
    dy = draw(tuple(y.shape), dtype, 17)
    dx, _, dw = rms_norm_backward(dy.cuda(), None, bi, None, rstd, w.cuda())
    g64, dw64, g_mag, dw_mag = SO.rms_norm_grad(dy.double(), s64, rstd64, w.double())
    within(dx, g64, h * g64.abs() + 2 * k * g_mag + subnormal(dtype), "d_branch_input")
    within(dw, dw64, (y.shape[0] * y.shape[1] + 40 + steps(D)) * U * dw_mag, "dweight")


# packs, single columns (below and above 4096), widths with idle lanes, four packs per thread, too wide for registers
MIXED = [(2, 70, 512), (1, 33, 1021), (2, 9, 1000), (2, 5, 7168), (1, 3, 8191), (1, 4, 16384), (1, 2, 20001)]


@pytest.mark.parametrize("B,S,D", MIXED)
@pytest.mark.parametrize("dt", list(TYPES))
def test_norm_of_the_stored_mix(B, S, D, dt):
    from mhc._kernels import stream_norm_forward
    H, pre, w = stream_case(B, S, D, TYPES[dt], B + S + D)
    y, bi, rstd = stream_norm_forward(*cuda(H, pre, w), EPS, want_branch_input=True)
    check_norm_of_stored(y, bi, rstd, H, pre, w, EPS)


@pytest.mark.parametrize("B,S,D", MIXED[:6])
@pytest.mark.parametrize("dt", list(TYPES))
def test_norm_inside_the_layers_forward(B, S, D, dt):
    import mhc
    from mhc._kernels import hc_mix_norm_forward
    H, _, w = stream_case(B, S, D, TYPES[dt], B + S + D)
    hc = base.layer(D)
    y, bi, rstd, H_post, H_pre, H_res, _, _ = hc_mix_norm_forward(
        H.cuda(), hc.H_pre_base, hc.H_post_base, hc.H_res_base, hc.phi, hc.alpha_pre, hc.alpha_post, hc.alpha_res, w.cuda(), 1e-5)
    check_norm_of_stored(y, bi, rstd, H, H_pre.cpu(), w, 1e-5)
    with torch.no_grad():
        assert torch.equal(hc(H.cuda(), w.cuda(), 1e-5)[0], y)


# ------------------------------------------------------------ the residual update with dropout that recomputes H_res @ H
@pytest.mark.parametrize("B,S,D", [(2, 70, 512), (1, 1, 8), (2, 19, 33), (1, 40, 1021), (3, 50, 1000), (2, 5, 7168), (1, 130, 64)])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("pool", [False, True])
def test_layers_residual_update_with_dropout(B, S, D, dt, pool):
    from mhc._kernels import add_residual_dropout_forward
    dtype, p = TYPES[dt], 0.2
    H, bo = draw((B, S, 4, D), dtype, 1), draw((B, S, D), dtype, 2)
    g = torch.Generator().manual_seed(4)
    post, R = 2 * torch.rand(B, 4, generator=g), torch.rand(B, 4, 4, generator=g)
    out = add_residual_dropout_forward(*cuda(H, R, bo, post), torch.tensor([3, 2 ** 33 + 1], device="cuda"),
                                       SO.threshold_of(p), 11, pool=pool)
    H_new = out[0] if pool else out
    keep = SO.keep_mask(3, 2 ** 33 + 1, B * S, D, p, 11).view(B, S, D)
    add = post.double()[:, None, :, None] * SO.dropout(bo.double(), keep, p).unsqueeze(2)
    want = torch.einsum("bnm,bsmd->bsnd", R.double(), H.double()) + add
    mag = torch.einsum("bnm,bsmd->bsnd", R.double(), H.double().abs()) + add.abs()
    # at most ten roundings: four products and their sums, the dropout's factor, the product with H_post, its sum
    within(H_new, want, half_step(dtype) * want.abs() + 10 * U * mag + subnormal(dtype), "H_new")
    if pool:
        stored = H_new.double().cpu()
        within(out[1].sum(1), stored.sum(1).view(B, 4 * D), (S + 10) * U * stored.abs().sum(1).view(B, 4 * D) + 1e-30, "pool")


@pytest.mark.parametrize("dt,B,S,D", [("bf16", 2, 40, 512), ("f16", 2, 21, 129), ("bf16", 1, 9, 7168), ("f16", 1, 30, 1000)])
def test_layer_in_16_bits_equals_its_parts(dt, B, S, D):
    """hc(H, norm_weight) and add_residual(dropout_p) against the plain layer with the norm and the dropout called beside it.
    Both normalise the stored mix; the parts round the dropout's output and gradient once more on the way."""
    import mhc
    dtype, p = TYPES[dt], 0.25
    hc = base.layer(D)
    H0, g = draw((B, S, 4, D), dtype, 1).cuda(), draw((B, S, 4, D), dtype, 2).cuda()
    w0 = (draw((D,), torch.float32, 3, 0.3) + 1).cuda()
    rng = torch.tensor([5, 6], device="cuda")
    got = []
    for fused in (True, False):
        H, w = H0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
        if fused:
            y, add = hc(H, w, 1e-5)
        else:
            bi, add = hc(H)
            y, _ = mhc.fused_add_rms_norm(bi, None, w, 1e-5)
        y.retain_grad()
        out = add(y, dropout_p=p, rng=rng) if fused else add(mhc.counter_dropout(y, p, rng=rng))
        out.backward(g)
        got.append([y.detach().double(), out.detach().double(), H.grad.double(), w.grad.double(), y.grad.double()])
    (y, out, dH, dw, dy), (y2, out2, dH2, dw2, dy2) = got
    step = torch.finfo(dtype).eps
    tiny = torch.finfo(dtype).smallest_normal
    # the stored mix may be a step apart, y a step more by its own rounding
    assert ((y - y2).abs() <= 2.5 * step * y.abs() + tiny).all()
    # H_post < 2, the factor of kept elements 4 / 3; half a step for the rounded dropout, one for the result
    assert ((out - out2).abs() <= 1.5 * step * out.abs() + 3.5 * step * 2 / (1 - p) * y.abs().unsqueeze(2) + 1e-5).all()
    assert ((dy - dy2).abs() <= 3 * step * dy.abs() + 1e-5).all()
    # d(norm) = rstd (h - n mean(h n)): three steps in h, a step or two in n, its own rounding
    n, h = (y / w0.double()).abs(), (dy * w0.double()).abs()
    with torch.no_grad():
        rstd = (hc(H0)[0].double().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    db = rstd * (h + n * (h * n).mean(-1, keepdim=True))
    assert ((dH - dH2).abs() <= 2 * step * dH.abs() + 12 * step * db.unsqueeze(2) + 2e-5 * float(dH.abs().max())).all()
    assert ((dw - dw2).abs() <= 6 * step * (dy.abs() * n).sum((0, 1)) + 1e-4).all()


# ----------------------------------------------------------------------------------------------- many rows, other instances
@pytest.mark.parametrize("rows,D", [(19013, 40), (9601, 584), (2407, 2048), (1201, 4096)])
def test_many_rows_in_fp32(rows, D):
    """The persistent forward with packs of four."""
    base.test_add_rms_norm(rows, D, "f32", "f32", True, 0.1)
    base.test_add_rms_norm(rows, D, "f32", None, False, 0.5)
    base.test_add_rms_norm_quant(rows, D, "f32", "f32", True, 32, True)
    base.test_add_rms_norm_quant(rows, D, "f32", "f32", False, 128, False)
    base.test_add_rms_norm_quant(rows, D, "f32", None, True, 64, False)
    base.test_add_rms_norm_quant(rows, D, "f32", "f32", True, 0, False)


@pytest.mark.parametrize("B,S,D", [(3, 3201, 584), (5, 482, 4096), (19013, 1, 40)])
def test_many_tokens_in_fp32(B, S, D):
    base.test_stream_norm_quant(B, S, D, "f32", 0, False)
    base.test_stream_norm_quant(B, S, D, "f32", 32, True)
    base.test_stream_norm_quant(B, S, D, "f32", 128, False)


@pytest.mark.parametrize("D", [6001, 12288, 16384, 16385])
def test_more_wide_rows_than_resident_blocks(D):
    """Odd rows of 4097 to 8192 columns, four packs per thread, and rows too wide for registers, walked several per block."""
    for dt in ("bf16", "f32"):
        base.test_add_rms_norm(331, D, dt, "f32", True, 0.0)
        base.test_add_rms_norm(331, D, dt, "f32", True, 0.1)
    base.test_stream_norm(2, 170, D, "bf16", "f32")


@pytest.mark.parametrize("D", [512, 1000, 4096])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("group,e8m0", [(0, False), (32, True), (64, False), (128, True)])
def test_unaligned_8_bit_outputs(D, dt, group, e8m0):
    """Inputs one element past a 16-byte border against 64 bits, each value within half a step of its own size."""
    import mhc
    dtype = TYPES[dt]
    scale_dtype = torch.float8_e8m0fnu if e8m0 else torch.float32

    def odd(t):
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        return flat[1:].view(t.shape).copy_(t)

    x, r, w = base.norm_case(37, D, dtype, torch.float32, True, seed=D)
    q, scales, _ = mhc.fused_add_rms_norm_quant(odd(x), r.cuda(), w.cuda(), EPS, group=group or None, scale_dtype=scale_dtype)
    y64, _ = SO.rms_norm(x.double() + r.double(), w.double(), EPS)
    check_quant(q, scales, y64, 2 * steps(D) * U * y64.abs() + 1e-300, group, e8m0, D)
    H, pre, w = stream_case(3, 13, D, dtype, D + 1)
    q, scales = mhc.fused_stream_norm_quant(odd(H), pre.cuda(), w.cuda(), EPS, group=group or None, scale_dtype=scale_dtype)
    b64, b_mag = mixed64(H, pre)
    y64, rstd = SO.rms_norm(b64, w.double(), EPS)
    row = (b_mag.square().sum(-1, keepdim=True) / (b64.square().sum(-1, keepdim=True) + D * EPS)).sqrt()
    check_quant(q, scales, y64, steps(D) * U * (1 + row) * rstd * w.double().abs() * b_mag + 1e-300, group, e8m0, D)
