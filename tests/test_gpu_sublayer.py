"""The operators around a sub-layer on the GPU, against the 64-bit oracle.

Tolerances.  u = 2^-24 is half an fp32 step, h = eps / 2 half a step of the stored type (both relative).  Every
value is computed in fp32 from exact inputs and rounded once to the stored type, so it is off by at most h times itself
plus K u times the sum of the magnitudes it is made of (computed in 64 bits beside the value), where K counts the fp32
roundings on the way: a row sum is a chain of at most ceil(D / 32) additions in a thread and 15 across threads, and the
other steps are fewer than 20, hence K = D / 32 + 35."""


import pytest
import torch

from oracle import sublayer_oracle as SO

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def steps(D):
    return D / 32 + 35


def within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {want.numel()} outside the bound, worst "
                           f"{float(((got - want).abs() / bound).nan_to_num(1e30).max()):.3g} times it")


def draw(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def subnormal(dtype):
    """Half the spacing below the smallest normal value (fp16 results may land there)."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


# rows, columns: one token, one column, below and over a pack, a warp, a CTA; odd widths; widths of the layer stacks; many rows
SHAPES = [(1, 1), (3, 7), (1, 4096), (2, 8), (5, 64), (37, 129), (1000, 96), (17, 1000), (9, 1021), (6, 2048), (700, 512),
          (4, 7168), (3, 8200), (2, 16384), (2, 12289), (2, 40000), (1500, 584), (3000, 40), (5, 8191), (3, 8193), (650, 279), (700, 3000)]


def norm_case(rows, D, dtype, wdtype, residual, seed=0, p=0.0, zero_row=True):
    x = draw((rows, D), dtype, seed)
    r = draw((rows, D), dtype, seed + 1, 3.0) if residual else None
    if zero_row and rows > 2:      # an empty row: rstd is 1 / sqrt(eps)
        x[1] = 0
        if r is not None:
            r[1] = 0
    w = None if wdtype is None else (draw((D,), torch.float32, seed + 2, 0.3) + 1).to(wdtype)
    return x, r, w


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("rows,D", SHAPES)
@pytest.mark.parametrize("dt,wdt,residual,p", [("f32", "f32", True, 0.0), ("bf16", "f32", True, 0.0),
                                               ("bf16", "bf16", False, 0.0), ("f16", "f16", True, 0.25),
                                               ("f32", None, False, 0.5), ("bf16", "f32", True, 0.1)])
def test_add_rms_norm(rows, D, dt, wdt, residual, p):
    import mhc
    dtype = TYPES[dt]
    x, r, w = norm_case(rows, D, dtype, wdt and TYPES[wdt], residual, seed=rows + D)
    seed, offset, row0 = -(2 ** 63) + 12345, 2 ** 40 + 7, 5
    rng = torch.tensor([seed, offset], device="cuda")
    xd, rd, wd = cuda(x, r, w)
    for t in (xd, rd, wd):
        if t is not None:
            t.requires_grad_(True)
    y, s = mhc.fused_add_rms_norm(xd, rd, wd, EPS, dropout_p=p, rng=rng, row_offset=row0)
    dy, ds = draw((rows, D), dtype, 91), draw((rows, D), dtype, 92)
    leaves = [t for t in (xd, rd, wd) if t is not None]
    both = residual or p > 0
    grads = torch.autograd.grad([y, s] if both else [y], leaves, [dy.cuda(), ds.cuda()] if both else [dy.cuda()])
    grads = dict(zip([n for n, t in (("x", xd), ("r", rd), ("w", wd)) if t is not None], grads))

    s64, factor = x.double(), 1.0
    if p > 0:
        keep, factor = SO.keep_mask(seed, offset, rows, D, p, row0), SO.keep_factor(p)
        s64 = SO.dropout(s64, keep, p)
    if residual:
        s64 = s64 + r.double()
    w64 = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    y64, rstd = SO.rms_norm(s64, w64, EPS)
    h, k = half_step(dtype), steps(D) * U
    # s: a product and a sum, both relative to the terms
    s_mag = s64.abs() + (2 * x.double().abs() * factor if p > 0 else 0)
    if both:
        assert s.dtype == dtype
        within(s, s64, h * s64.abs() + 3 * U * s_mag + subnormal(dtype), "s")
    else:
        assert s is xd
    assert y.dtype == dtype
    within(y, y64, (h + k) * y64.abs() + k * rstd * w64.abs() * s_mag + subnormal(dtype), "y")

    g64, dw64, g_mag, dw_mag = SO.rms_norm_grad(dy.double(), s64, rstd, w64)
    # the product of a kept x by its factor is rounded: next to s, relative to the row, that is at most this much more
    s_rel = 1 + (s_mag.square().sum(-1, keepdim=True) / (s64.square().sum(-1, keepdim=True) + D * EPS)).sqrt() if p > 0 else torch.ones(1)
    if p > 0:
        _, _, g_mag, dw_mag = SO.rms_norm_grad(dy.double(), s_mag, rstd, w64)
    if both:
        g64, g_mag = g64 + ds.double(), g_mag + ds.double().abs()
    tol = h * g64.abs() + 2 * k * g_mag * s_rel + subnormal(dtype)
    if p > 0:
        within(grads["x"], SO.dropout(g64, keep, p), torch.where(keep, (tol + U * g64.abs()) * factor, 0.0), "dx")
    else:
        within(grads["x"], g64, tol, "dx")
    if residual:
        within(grads["r"], g64, tol, "dresidual")
    if w is not None:
        hw = half_step(w.dtype)
        rows_chain = rows + 40        # additions of a column's sum, at most
        within(grads["w"], dw64, hw * dw64.abs() + (rows_chain + steps(D)) * U * dw_mag * s_rel.max() + subnormal(w.dtype), "dw")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("lo", range(0, 4608, 512))
def test_add_rms_norm_every_kind_of_width(dt, lo):
    """Widths that change the threads per row, the rows per block and the last pack, against 64 bits."""
    import mhc
    dtype = TYPES[dt]
    h = half_step(dtype)
    for D in [lo + d for d in (4, 8, 31, 72, 120, 256, 264, 391, 392, 504)]:
        rows = 700 if D < 1024 else 300
        x, r, w = norm_case(rows, D, dtype, torch.float32, True, seed=D, zero_row=False)
        dy, ds = draw((rows, D), dtype, D + 1), draw((rows, D), dtype, D + 2)
        leaves = [t.cuda().requires_grad_(True) for t in (x, r, w)]
        y, s = mhc.fused_add_rms_norm(*leaves, EPS)
        grads = torch.autograd.grad([y, s], leaves, [dy.cuda(), ds.cuda()])
        s64 = x.double() + r.double()
        y64, rstd = SO.rms_norm(s64, w.double(), EPS)
        k = steps(D) * U
        within(y, y64, (h + 2 * k) * y64.abs() + 1e-30, f"y {D}")
        g64, dw64, g_mag, dw_mag = SO.rms_norm_grad(dy.double(), s64, rstd, w.double())
        g64, g_mag = g64 + ds.double(), g_mag + ds.double().abs()
        for got in grads[:2]:
            within(got, g64, h * g64.abs() + 2 * k * g_mag + 1e-30, f"dx {D}")
        within(grads[2], dw64, (rows + 40 + steps(D)) * U * dw_mag, f"dw {D}")


def check_quant(q, scales, y64, y_err, group, e8m0, D):
    """q, scales against fp64 y whose fp32 counterpart is off by at most y_err (elementwise)."""
    G = -(-D // group) if group else 1
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (*y64.shape[:-1], G)
    want = SO.scales_of(y64, group, False)
    worst = torch.stack([e.amax(-1) for e in y_err.split(group or D, -1)], -1) / SO.E4M3_MAX
    rel = worst / want + 4 * U      # of the group's largest value, and its division
    if e8m0:
        assert scales.dtype == torch.float8_e8m0fnu
        got = scales.double().cpu()
        lo, hi = [torch.exp2(torch.ceil(torch.log2(want * f))) for f in (1 - rel, 1 + rel)]
        lo = lo.clamp(min=SO.MIN_SCALE)
        assert ((got == lo) | (got == hi)).all(), "power-of-two scales"
    else:
        assert scales.dtype == torch.float32
        got = scales.double().cpu()
        assert ((got - want).abs() <= rel * want).all(), "scales"
    per = SO.spread_scales(got, D, group)
    v = y64 / per
    err = y_err / per + 2 * U * v.abs()
    step = torch.exp2((torch.frexp(v.abs().clamp(max=448.0)).exponent - 1).clamp(min=-6).double() - 3)
    # within half a step of the quotient; at a binade's edge the step above may be the one that counts
    near = torch.exp2((torch.frexp((v.abs() + err).clamp(max=448.0)).exponent - 1).clamp(min=-6).double() - 3)
    within(q.float(), v, torch.maximum(step, near) / 2 + err, "q")


@pytest.mark.parametrize("rows,D", SHAPES)
@pytest.mark.parametrize("dt,wdt,residual,group,e8m0", [("bf16", "bf16", True, 0, False), ("f32", "f32", False, 0, True),
                                                        ("f16", "f32", True, 32, True), ("bf16", None, False, 64, False),
                                                        ("bf16", "f32", True, 128, False), ("f32", "f32", True, 128, True)])
def test_add_rms_norm_quant(rows, D, dt, wdt, residual, group, e8m0):
    import mhc
    dtype = TYPES[dt]
    x, r, w = norm_case(rows, D, dtype, wdt and TYPES[wdt], residual, seed=rows * 3 + D)
    if rows > 3:
        x[2] *= 1e-3
    q, scales, s = mhc.fused_add_rms_norm_quant(*cuda(x, r, w), EPS, group=group or None,
                                                scale_dtype=torch.float8_e8m0fnu if e8m0 else torch.float32)
    s64 = x.double() + (r.double() if residual else 0)
    w64 = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    y64, rstd = SO.rms_norm(s64, w64, EPS)
    if residual:
        within(s, s64, half_step(dtype) * s64.abs() + 2 * U * s64.abs() + subnormal(dtype), "s")
    check_quant(q, scales, y64, 2 * steps(D) * U * y64.abs() + 1e-300, group, e8m0, D)


def stream_case(B, S, D, dtype, seed):
    H = draw((B, S, 4, D), dtype, seed)
    g = torch.Generator().manual_seed(seed + 5)
    pre = torch.rand(B, 4, generator=g) + 0.05
    w = draw((D,), torch.float32, seed + 6, 0.3) + 1
    return H, pre / pre.sum(1, keepdim=True), w


STREAM_SHAPES = [(1, 1, 8), (2, 3, 64), (3, 5, 33), (1, 130, 256), (5, 1, 4096), (2, 19, 1000), (1, 3, 1021), (2, 2, 7168),
                 (300, 2, 40), (1, 2, 16384), (1, 2, 33000), (2, 700, 512), (2, 333, 584), (1, 301, 999), (3, 40, 2049)]


def mixed64(H, pre):
    terms = H.double() * pre.double()[:, None, :, None]
    return terms.sum(2), terms.abs().sum(2)


@pytest.mark.parametrize("B,S,D", STREAM_SHAPES)
@pytest.mark.parametrize("dt,wdt", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", None)])
def test_stream_norm(B, S, D, dt, wdt):
    import mhc
    dtype = TYPES[dt]
    H, pre, w = stream_case(B, S, D, dtype, B + S + D)
    w = None if wdt is None else w.to(TYPES[wdt])
    Hd, pd, wd = cuda(H, pre, w)
    for t in (Hd, pd, wd):
        if t is not None:
            t.requires_grad_(True)
    y = mhc.fused_stream_norm(Hd, pd, wd, EPS)
    dy = draw((B, S, D), dtype, 77)
    grads = torch.autograd.grad(y, [t for t in (Hd, pd, wd) if t is not None], dy.cuda())
    b64, b_mag = mixed64(H, pre)
    w64 = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    y64, rstd = SO.rms_norm(b64, w64, EPS)
    h, k = half_step(dtype), steps(D) * U
    # an error of the mix reaches the row's sum of squares: relative to the row it is at most its own relative size
    row = (b_mag.square().sum(-1, keepdim=True) / (b64.square().sum(-1, keepdim=True) + D * EPS)).sqrt()
    within(y, y64, h * y64.abs() + k * (1 + row) * rstd * w64.abs() * b_mag + subnormal(dtype), "y")
    g64, dw64, g_mag, dw_mag = SO.rms_norm_grad(dy.double(), b64, rstd, w64)
    _, _, _, dw_mix = SO.rms_norm_grad(dy.double(), b_mag, rstd, w64)
    hs = (dy.double() * w64).abs()
    # the mix enters twice in the term that is subtracted, so its magnitude does too
    g_mag = rstd * hs + rstd ** 3 / D * b_mag * (hs * b_mag).sum(-1, keepdim=True)
    p64 = pre.double()[:, None, :, None]
    tol = 4 * k * (1 + row) * g_mag
    within(grads[0], p64 * g64.unsqueeze(2), p64 * (h * g64.abs() + tol).unsqueeze(2) + subnormal(dtype), "dH")
    dp64 = (H.double() * g64.unsqueeze(2)).sum((1, 3))
    dp_mag = (H.double().abs() * g64.abs().unsqueeze(2)).sum((1, 3))
    dp_tol = (H.double().abs() * tol.unsqueeze(2)).sum((1, 3)) + (S * D / 32 + 60) * U * dp_mag
    within(grads[1], dp64, dp_tol, "dH_pre")
    if w is not None:
        within(grads[2], dw64, half_step(w.dtype) * dw64.abs() + (B * S + 40 + 2 * steps(D)) * U *
               ((1 + row).max() * dw_mix) + subnormal(w.dtype), "dw")


@pytest.mark.parametrize("B,S,D", STREAM_SHAPES)
@pytest.mark.parametrize("dt,group,e8m0", [("bf16", 0, False), ("bf16", 32, True), ("f32", 128, False), ("f16", 64, False)])
def test_stream_norm_quant(B, S, D, dt, group, e8m0):
    import mhc
    H, pre, w = stream_case(B, S, D, TYPES[dt], B + S + D + 1)
    q, scales = mhc.fused_stream_norm_quant(*cuda(H, pre, w), EPS, group=group or None,
                                            scale_dtype=torch.float8_e8m0fnu if e8m0 else torch.float32)
    b64, b_mag = mixed64(H, pre)
    y64, rstd = SO.rms_norm(b64, w.double(), EPS)
    row = (b_mag.square().sum(-1, keepdim=True) / (b64.square().sum(-1, keepdim=True) + D * EPS)).sqrt()
    check_quant(q, scales, y64, steps(D) * U * (1 + row) * rstd * w.double().abs() * b_mag + 1e-300, group, e8m0, D)


# Enough rows for the persistent forward (4 per resident block): narrow rows that share a block, rows of a few warps, wide ones;
# counts that do not divide.
@pytest.mark.parametrize("rows,D", [(19013, 40), (9601, 584), (2407, 4096), (1201, 7168)])
def test_many_rows(rows, D):
    test_add_rms_norm(rows, D, "bf16", "f32", True, 0.1)
    test_add_rms_norm(rows, D, "f16", "f16", False, 0.5)
    test_add_rms_norm_quant(rows, D, "bf16", "bf16", True, 32, True)
    test_add_rms_norm_quant(rows, D, "f16", "f32", False, 128, False)
    test_add_rms_norm_quant(rows, D, "bf16", None, True, 0, False)


@pytest.mark.parametrize("B,S,D", [(3, 3201, 584), (5, 482, 4096)])
def test_many_tokens(B, S, D):
    test_stream_norm_quant(B, S, D, "bf16", 32, True)
    test_stream_norm_quant(B, S, D, "f16", 0, False)
    test_stream_norm(B, S, D, "bf16", "f32")


def test_norm_of_infinities_and_nan_stays_in_its_row():
    import mhc
    x = draw((6, 512), torch.bfloat16, 1)
    x[1, 3], x[3, 500], x[4, 0] = float("nan"), float("inf"), -float("inf")
    w = torch.ones(512)
    y, _ = mhc.fused_add_rms_norm(*cuda(x, None, w), EPS)
    q, scales, _ = mhc.fused_add_rms_norm_quant(*cuda(x, None, w), EPS)
    qg, sg, _ = mhc.fused_add_rms_norm_quant(*cuda(x, None, w), EPS, group=32, scale_dtype=torch.float8_e8m0fnu)
    clean = [0, 2, 5]
    y64, _ = SO.rms_norm(x.double(), w.double(), EPS)
    assert torch.isfinite(y.cpu()[clean].float()).all() and torch.isfinite(q.float().cpu()[clean]).all()
    assert torch.isfinite(scales.cpu()[clean]).all() and torch.isfinite(sg.float().cpu()[clean]).all()
    assert torch.isnan(y.cpu()[1].float()).all() and torch.isnan(scales.cpu()[1]).all() and torch.isnan(q.float().cpu()[1]).all()
    # an infinite entry: rstd 0, so the entry itself is NaN and the others 0
    for r, c in ((3, 500), (4, 0)):
        bad = torch.isnan(y.cpu()[r].float())
        assert bad.sum() == 1 and bad[c] and (y.cpu()[r].float()[~bad] == 0).all()
        assert torch.isnan(scales.cpu()[r]).all()
        assert torch.isnan(sg.float().cpu()[r]).sum() == 1 and torch.isnan(sg.float().cpu()[r, c // 32])
    assert y64.shape == y.shape


def test_zero_rows_and_tiny_values_in_8_bits():
    import mhc
    x = torch.zeros(3, 256)
    x[1] = 1e-30
    w = torch.ones(256)
    for e8m0 in (False, True):
        for group in (None, 32):
            q, s, _ = mhc.fused_add_rms_norm_quant(*cuda(x, None, w), EPS, group=group,
                                                   scale_dtype=torch.float8_e8m0fnu if e8m0 else torch.float32)
            s = s.double().cpu()
            assert (s[0] == SO.MIN_SCALE).all() and (q.float().cpu()[0] == 0).all()
            back = q.double().cpu()[1] * s[1].repeat_interleave(group or 256)
            assert ((back - 1e-27).abs() <= 1e-27 / 16 * 1.01).all()


@pytest.mark.parametrize("size", [1e-20, 1e-34, 3e-36, 2e-37, 3e-38])
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("e8m0", [False, True])
def test_rows_near_the_smallest_numbers_in_8_bits(size, group, e8m0):
    """rstd is 1000 there (eps): the values are normal numbers, their inputs' reciprocals are not."""
    import mhc
    x = draw((5, 256), torch.float32, 7) * size
    x = torch.where(x.abs() < 1.2e-38, torch.zeros(()), x)       # no subnormal inputs
    q, scales, _ = mhc.fused_add_rms_norm_quant(*cuda(x, None, torch.ones(256)), EPS, group=group or None,
                                                scale_dtype=torch.float8_e8m0fnu if e8m0 else torch.float32)
    y64, _ = SO.rms_norm(x.double(), torch.ones(256, dtype=torch.float64), EPS)
    check_quant(q, scales, y64, 2 * steps(256) * U * y64.abs() + 1e-300, group, e8m0, 256)


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (3, 8), (129, 515), (2, 3, 1024), (700, 96), (1, 100003), (33, 4096), (7,)])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("p", [0.1, 0.5, 0.999, 1 / 65536])
def test_counter_dropout(shape, dt, p):
    """Exact: one fp32 product and one rounding, on the oracle's mask; the gradient is the same map."""
    import mhc
    dtype = TYPES[dt]
    x = draw(shape, dtype, 4).requires_grad_(False)
    seed, offset, row0 = 987654321987654321, -3, 2 ** 32 - 1000
    xd = x.cuda().requires_grad_(True)
    y = mhc.counter_dropout(xd, p, rng=torch.tensor([seed, offset], device="cuda"), row_offset=row0)
    dy = draw(shape, dtype, 6)
    (dx,) = torch.autograd.grad(y, xd, dy.cuda())
    D = shape[-1]
    keep = SO.keep_mask(seed, offset, x.numel() // D, D, p, row0).view(shape)
    factor = torch.tensor(SO.keep_factor(p), dtype=torch.float32)
    for got, src in ((y, x), (dx, dy)):
        want = torch.where(keep, src.float() * factor, torch.zeros(())).to(dtype)
        assert torch.equal(got.cpu(), want)


def test_dropout_forms_of_the_generator_state():
    import mhc
    x = torch.ones(64, 256, device="cuda")
    a = mhc.counter_dropout(x, 0.3, rng=(7, 9))
    assert torch.equal(a, mhc.counter_dropout(x, 0.3, rng=torch.tensor([7, 9], device="cuda")))
    assert not torch.equal(a, mhc.counter_dropout(x, 0.3, rng=(7, 10)))
    # a shard of rows that knows its first row gets the whole tensor's mask
    assert torch.equal(a[20:], mhc.counter_dropout(x[20:], 0.3, rng=(7, 9), row_offset=20))
    torch.manual_seed(1)
    b, c = mhc.counter_dropout(x, 0.3), mhc.counter_dropout(x, 0.3)
    torch.manual_seed(1)
    assert torch.equal(b, mhc.counter_dropout(x, 0.3)) and not torch.equal(b, c)
    big = torch.ones(4096, 1024, device="cuda")
    n, p = big.numel(), SO.threshold_of(0.3) / 65536
    dropped = float((mhc.counter_dropout(big, 0.3) == 0).sum())
    assert abs(dropped - n * p) < 6 * (n * p * (1 - p)) ** 0.5      # six standard deviations


def test_dropped_infinities_are_zero():
    import mhc
    x = torch.full((64, 64), float("inf"))
    x[::2] = float("nan")
    y = mhc.counter_dropout(x.cuda(), 0.5, rng=(1, 1)).cpu()
    keep = SO.keep_mask(1, 1, 64, 64, 0.5)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_refuses_what_changes_before_the_backward():
    import mhc
    x = torch.randn(8, 64, device="cuda", requires_grad=True)
    rng = torch.tensor([1, 2], device="cuda")
    y = mhc.counter_dropout(x, 0.5, rng=rng)
    rng.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("B,S,D", [(1, 1, 8), (2, 3, 33), (2, 128, 512), (3, 50, 1000), (1, 9, 7168), (2, 70, 64)])
@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("pool", [False, True])
def test_add_residual_with_dropout(B, S, D, dt, pool):
    import mhc
    dtype, p = TYPES[dt], 0.2
    Hr, bo, dH = draw((B, S, 4, D), dtype, 1), draw((B, S, D), dtype, 2), draw((B, S, 4, D), dtype, 3)
    post = 2 * torch.rand(B, 4, generator=torch.Generator().manual_seed(4))
    rng = torch.tensor([3, 2 ** 33 + 1], device="cuda")
    Hd, bd, pd = [t.cuda().requires_grad_(True) for t in (Hr, bo, post)]
    H_new = mhc.fused_add_residual(Hd, bd, pd, pool_for_next=pool, dropout_p=p, rng=rng, row_offset=11)
    gH, gbo, gpost = torch.autograd.grad(H_new, [Hd, bd, pd], dH.cuda())
    keep = SO.keep_mask(3, 2 ** 33 + 1, B * S, D, p, 11).view(B, S, D)
    bo64 = SO.dropout(bo.double(), keep, p)
    p64, h = post.double()[:, :, None], half_step(dtype)
    add = p64[:, None] * bo64.unsqueeze(2)
    want = Hr.double() + add
    within(H_new, want, h * want.abs() + 4 * U * (Hr.double().abs() + add.abs()) + subnormal(dtype), "H_new")
    assert torch.equal(gH.cpu(), dH)
    terms = dH.double() * p64[:, None]
    d64 = SO.dropout(terms.sum(2), keep, p)
    f = SO.keep_factor(p)
    within(gbo, d64, h * d64.abs() + 8 * U * f * terms.abs().sum(2) + subnormal(dtype), "dbranch_output")
    assert (gbo.cpu()[~keep] == 0).all()
    t = dH.double() * bo64.unsqueeze(2)
    within(gpost, t.sum((1, 3)), (S * D / 64 + 80) * U * t.abs().sum((1, 3)), "dH_post")
    if pool:
        partials, _ = H_new._mhc_pooled
        stored = H_new.detach().double().cpu()
        within(partials.sum(1), stored.sum(1).view(B, 4 * D), (S + 10) * U * stored.abs().sum(1).view(B, 4 * D) + 1e-30, "pool")


# ------------------------------------------------------------------------------- used together, as a layer uses them
def layer(dim, seed=0):
    import mhc
    torch.manual_seed(seed)
    hc = mhc.HyperConnection(dim=dim)
    with torch.no_grad():
        hc.phi.normal_(std=0.02)
        hc.H_res_base.add_(torch.randn(4, 4) * 0.1)
    return hc.cuda()


@pytest.mark.parametrize("mode", ["fused", "materialized", "unfused", "static"])
def test_layer_with_norm_and_dropout_equals_its_parts(mode):
    """hc(H, norm_weight) and add_residual(dropout_p) against the plain layer, fused_add_rms_norm on its branch input and
    counter_dropout on its branch output, in fp32: same numbers up to the order of a few fp32 roundings."""
    import mhc
    B, S, D, p = 2, 40, 256, 0.3
    torch.manual_seed(0)
    hc = layer(D) if mode in ("fused", "materialized") else \
        mhc.HyperConnection(dim=D, dynamic=mode == "unfused", use_fused_weights=False).cuda()
    hc.materialize_residual = mode == "materialized"
    w = torch.rand(D, device="cuda") + 0.5
    H0, g = torch.randn(B, S, 4, D, device="cuda"), torch.randn(B, S, 4, D, device="cuda")
    rng = torch.tensor([5, 6], device="cuda")
    results = []
    for fused in (True, False):
        H, wl = H0.clone().requires_grad_(True), w.clone().requires_grad_(True)
        hc.zero_grad()
        if fused:
            y, add = hc(H, wl, 1e-5)
            out = add(torch.tanh(y), dropout_p=p, rng=rng)
        else:
            bi, add = hc(H)
            y, _ = mhc.fused_add_rms_norm(bi, None, wl, 1e-5)
            out = add(mhc.counter_dropout(torch.tanh(y), p, rng=rng))
        out.backward(g)
        results.append([y, out, H.grad, wl.grad] + [q.grad for q in hc.parameters()])
    for a, b in zip(*results):
        a, b = a.detach(), b.detach()
        assert float((a - b).abs().max()) <= 2e-5 * float(b.abs().max()) + 1e-7


def test_two_layer_stack_against_64_bits():
    """Norm, branch, dropout and pooling across two layers in fp32 against the same stack in plain 64-bit torch."""
    import mhc
    B, S, D, p = 2, 24, 128, 0.25
    hcs = [layer(D, 1), layer(D, 2)]
    ws = [torch.rand(D, device="cuda") + 0.5 for _ in hcs]
    rngs = [torch.tensor([8, i], device="cuda") for i in range(2)]
    torch.manual_seed(3)
    H0, g = torch.randn(B, S, 4, D), torch.randn(B, S, 4, D)

    H = H0.cuda().requires_grad_(True)
    x, wl = H, [w.clone().requires_grad_(True) for w in ws]
    for i, hc in enumerate(hcs):
        y, add = hc(x, wl[i], 1e-6)
        x = add(torch.sin(y), pool_for_next=i == 0, dropout_p=p, rng=rngs[i])
    x.backward(g.cuda())

    H64 = H0.double().requires_grad_(True)
    z, w64 = H64, [w.double().cpu().requires_grad_(True) for w in ws]
    P = [{n: q.detach().double().cpu() for n, q in hc.named_parameters()} for hc in hcs]
    for i in range(2):
        pooled = z.mean(1).reshape(B, 4 * D)
        q = P[i]
        s = torch.cat([q["alpha_pre"].expand(4), q["alpha_post"].expand(4), q["alpha_res"].expand(16)]) * \
            (pooled @ q["phi"]) / torch.sqrt((pooled * pooled).mean(-1, keepdim=True) + 1e-6) + \
            torch.cat([q["H_pre_base"], q["H_post_base"], q["H_res_base"].flatten()])
        pre = torch.sigmoid(s[:, :4])
        pre = pre / (pre.sum(-1, keepdim=True) + 1e-6)
        post, R = 2 * torch.sigmoid(s[:, 4:8]), s[:, 8:].reshape(B, 4, 4).abs() + 1e-6
        for _ in range(20):
            R = R / (R.sum(-1, keepdim=True) + 1e-6)
            R = R / (R.sum(-2, keepdim=True) + 1e-6)
        bi = torch.einsum("bn,bsnd->bsd", pre, z)
        y = SO.rms_norm(bi, w64[i], 1e-6)[0]
        keep = SO.keep_mask(8, i, B * S, D, p).view(B, S, D)
        z = torch.einsum("bnm,bsmd->bsnd", R, z) + post[:, None, :, None] * SO.dropout(torch.sin(y), keep, p).unsqueeze(2)
    z.backward(g.double())
    for a, b in ((x.detach(), z.detach()), (H.grad, H64.grad), (wl[0].grad, w64[0].grad), (wl[1].grad, w64[1].grad)):
        # fp32 chains of a few hundred roundings, largest entries a few times the typical one: 1e-5 of the largest
        assert float((a.double().cpu() - b).abs().max()) <= 1e-5 * float(b.abs().max())


def test_gradient_of_the_kernels_against_differences():
    """Directional central differences of the fp32 kernels themselves (dropout fixed by its counter)."""
    import mhc
    torch.manual_seed(0)
    x, r = torch.randn(6, 200, device="cuda"), torch.randn(6, 200, device="cuda")
    w, dy, ds = torch.rand(200, device="cuda") + 0.5, torch.randn(6, 200, device="cuda"), torch.randn(6, 200, device="cuda")
    vx, vr, vw = (torch.randn_like(t) for t in (x, r, w))

    def loss(a, b, c):
        y, s = mhc.fused_add_rms_norm(a, b, c, 1e-3, dropout_p=0.3, rng=(1, 2))
        return (y.double() * dy + s.double() * ds).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    slope = sum(float((a.double() * v).sum()) for a, v in zip(grads, (vx, vr, vw)))
    h = 2.0 ** -7
    with torch.no_grad():
        diff = float(loss(x + h * vx, r + h * vr, w + h * vw) - loss(x - h * vx, r - h * vr, w - h * vw)) / (2 * h)
    # fp32 noise: 1200 outputs of size <= 8, each off by 2^-22 or so, over 2 h = 2^-6; truncation: h^2 / 6 times a third
    # derivative of some tens per row
    assert abs(diff - slope) <= 0.05 + 1e-3 * abs(slope)


# ------------------------------------------------------------- other streams, alignments, strides, capture, checkpointing
def test_unaligned_and_strided_inputs():
    import mhc
    base = draw((16, 520), torch.bfloat16, 3).cuda()
    w = torch.ones(512, device="cuda")
    want = mhc.fused_add_rms_norm(base[:, 3:515].contiguous(), None, w)[0]
    assert torch.equal(mhc.fused_add_rms_norm(base[:, 3:515], None, w)[0], want)
    flat = torch.empty(16 * 512 + 1, device="cuda", dtype=torch.bfloat16)
    odd = flat[1:].view(16, 512).copy_(base[:, 3:515])      # contiguous, not on 16 bytes
    y = mhc.fused_add_rms_norm(odd, None, w)[0]
    y64 = SO.rms_norm(odd.double().cpu(), torch.ones(512, dtype=torch.float64), EPS)[0]
    within(y, y64, (2.0 ** -8 + steps(512) * U) * y64.abs() + 1e-30, "unaligned")
    a = mhc.counter_dropout(odd, 0.5, rng=(1, 1))
    assert torch.equal(a, mhc.counter_dropout(odd.clone(), 0.5, rng=(1, 1)))
    wt = torch.rand(1024, device="cuda")[::2]
    assert torch.equal(mhc.fused_add_rms_norm(odd, None, wt)[0], mhc.fused_add_rms_norm(odd, None, wt.contiguous())[0])
    q = mhc.fused_add_rms_norm_quant(odd, None, w)
    q2 = mhc.fused_add_rms_norm_quant(odd.clone(), None, w)
    assert (q[0].float() - q2[0].float()).abs().max() <= 32 and (q[1] / q2[1] - 1).abs().max() < 1e-6


def test_empty_inputs():
    import mhc
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y, s = mhc.fused_add_rms_norm(x, torch.empty(0, 64, device="cuda"), w)
    gx, gw = torch.autograd.grad([y, s], [x, w], [torch.empty_like(y), torch.empty_like(s)])
    assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))
    q, sc, _ = mhc.fused_add_rms_norm_quant(x.detach(), None, w.detach(), group=32)
    assert q.shape == (0, 64) and sc.shape == (0, 2)
    assert mhc.counter_dropout(x, 0.5, rng=(1, 1)).shape == x.shape
    H, pre = torch.empty(2, 0, 4, 64, device="cuda", requires_grad=True), torch.rand(2, 4, device="cuda", requires_grad=True)
    out = mhc.fused_stream_norm(H, pre, w)
    gH, gp, gw = torch.autograd.grad(out, [H, pre, w], torch.empty_like(out))
    assert gH.shape == H.shape and torch.equal(gp, torch.zeros_like(pre)) and torch.equal(gw, torch.zeros_like(w))


def test_no_columns():
    import mhc
    x = torch.empty(3, 0, device="cuda", requires_grad=True)
    y, _ = mhc.fused_add_rms_norm(x, torch.empty(3, 0, device="cuda"), torch.empty(0, device="cuda"))
    assert torch.autograd.grad(y.sum(), x)[0].shape == (3, 0)
    q, s, _ = mhc.fused_add_rms_norm_quant(x.detach())
    assert q.shape == (3, 0) and s.shape == (3, 0)
    assert mhc.counter_dropout(x, 0.5, rng=(1, 1)).shape == (3, 0)


def test_one_tensor_as_input_and_residual():
    import mhc
    torch.manual_seed(0)
    x, w, dy, ds = torch.randn(40, 256), torch.rand(256) + 0.5, torch.randn(40, 256), torch.randn(40, 256)
    leaf = x.cuda().requires_grad_(True)
    y, s = mhc.fused_add_rms_norm(leaf, leaf, w.cuda(), EPS)
    (g,) = torch.autograd.grad([y, s], [leaf], [dy.cuda(), ds.cuda()])
    s64 = 2 * x.double()
    _, rstd = SO.rms_norm(s64, w.double(), EPS)
    g64, _, g_mag, _ = SO.rms_norm_grad(dy.double(), s64, rstd, w.double())
    within(g, 2 * (g64 + ds.double()), 4 * steps(256) * U * (g_mag + ds.double().abs()), "dx")


def test_norm_weight_beside_a_gradient_record():
    """A layer whose parameter gradients go to a GradSync record still returns the norm weight's gradient."""
    import mhc
    B, S, D = 2, 16, 128
    H0, g = torch.randn(B, S, 4, D, device="cuda"), torch.randn(B, S, 4, D, device="cuda")
    w0 = torch.rand(D, device="cuda") + 0.5
    got = []
    for sync in (False, True):
        hc = layer(D)
        gs = mhc.GradSync([hc]) if sync else None
        H, w = H0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
        y, add = hc(H, w)
        add(torch.sin(y), dropout_p=0.2, rng=(1, 2)).backward(g)
        if sync:
            gs.finish()
        got.append([H.grad, w.grad, *[p.grad.clone() for p in hc.parameters()]])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_only_some_gradients_are_wanted():
    import mhc
    torch.manual_seed(0)
    x, r, w = torch.randn(9, 128, device="cuda"), torch.randn(9, 128, device="cuda"), torch.rand(128, device="cuda")
    dy = torch.randn_like(x)
    full = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = mhc.fused_add_rms_norm(*full, dropout_p=0.2, rng=(1, 1))
    want = torch.autograd.grad(y, full, dy)
    for i in range(3):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, r, w))]
        y, s = mhc.fused_add_rms_norm(*part, dropout_p=0.2, rng=(1, 1))
        assert torch.equal(torch.autograd.grad(y, part[i], dy)[0], want[i])
    # only the sum is used downstream
    part = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = mhc.fused_add_rms_norm(*part, dropout_p=0.2, rng=(1, 1))
    gx, gr, gw = torch.autograd.grad(s, part, dy)
    assert torch.equal(gr, dy) and torch.equal(gw, torch.zeros_like(w))
    assert torch.equal(gx, mhc.counter_dropout(dy, 0.2, rng=(1, 1)))


def test_results_repeat_and_do_not_depend_on_the_stream():
    import mhc
    torch.manual_seed(0)
    x, r = torch.randn(3000, 1024, device="cuda").bfloat16(), torch.randn(3000, 1024, device="cuda").bfloat16()
    w, dy = torch.rand(1024, device="cuda"), torch.randn(3000, 1024, device="cuda").bfloat16()

    def step():
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
        y, s = mhc.fused_add_rms_norm(*leaves, dropout_p=0.1, rng=(4, 4))
        return [y, s, *torch.autograd.grad([y, s], leaves, [dy, dy])]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, step()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_step_follows_the_generator_state():
    """Forward and backward of a layer with norm and dropout in one CUDA graph: a replay uses what rng holds then."""
    B, S, D = 1, 32, 256
    hc, hc_eager = layer(D), layer(D)      # equal layers; the graph keeps the first one's autograd nodes to itself
    w0, H0 = torch.rand(D, device="cuda"), torch.randn(B, S, 4, D, device="cuda")
    g = torch.randn(B, S, 4, D, device="cuda")
    rng = torch.tensor([1, 0], device="cuda")
    H, w = H0.clone().requires_grad_(True), w0.clone().requires_grad_(True)

    def step(hc=hc, H=H, w=w):
        y, add = hc(H, w)
        out = add(torch.sin(y), dropout_p=0.3, rng=rng)
        return [t.detach() for t in (out, *torch.autograd.grad(out, [H, w, *hc.parameters()], g))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    seen = []
    for offset in (0, 5):
        rng[1] = offset
        graph.replay()
        got = [t.clone() for t in outs]
        for a, b in zip(got, step(hc_eager, H0.clone().requires_grad_(True), w0.clone().requires_grad_(True))):
            assert torch.equal(a, b)
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_captured_draw_from_torchs_generator():
    """rng=None in a graph: every replay draws anew, and the backward of a replay uses that replay's mask."""
    import mhc
    x = torch.rand(64, 256, device="cuda") + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        leaf = x.detach().requires_grad_(True)
        y = mhc.counter_dropout(leaf, 0.4)
        return y.detach(), torch.autograd.grad(y, leaf, torch.ones_like(x))[0]

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, g = step()
    masks = []
    for _ in range(2):
        graph.replay()
        assert torch.equal(y != 0, g != 0)
        masks.append((y != 0).clone())
    assert not torch.equal(*masks)


def test_two_graphs_of_one_stream_replayed_together():
    """Backwards with dropout captured one after the other share nothing that replaying them at once would upset."""
    import mhc
    B, S, D = 2, 256, 1024
    data = [[torch.randn(B, S, 4, D, device="cuda"), torch.randn(B, S, D, device="cuda"), torch.rand(B, 4, device="cuda")]
            for _ in range(2)]
    rng = torch.tensor([1, 2], device="cuda")
    stream = torch.cuda.Stream()

    def step(d):
        leaves = [t.detach().requires_grad_(True) for t in d]
        out = mhc.fused_add_residual(*leaves, dropout_p=0.3, rng=rng)
        return torch.autograd.grad(out, leaves[1:], d[0])

    with torch.cuda.stream(stream):
        want = [[t.clone() for t in step(d)] for d in data]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(step(d))
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for out, ref in zip(outs, want):
        for a, b in zip(out, ref):
            assert torch.equal(a, b)


def test_checkpointing_recomputes_the_same_mask():
    import mhc
    from torch.utils.checkpoint import checkpoint
    x = torch.randn(64, 128, device="cuda")
    grads = []
    for use in (False, True):
        torch.manual_seed(9)
        leaf = x.clone().requires_grad_(True)
        f = lambda t: mhc.counter_dropout(torch.sin(t), 0.4)   # noqa: E731
        out = checkpoint(f, leaf, use_reentrant=False) if use else f(leaf)
        out.sum().backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads)


def test_refusals_on_the_gpu():
    import mhc
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(AssertionError):
        mhc.fused_add_rms_norm(x, torch.randn(4, 32, device="cuda"), w)
    with pytest.raises(AssertionError):
        mhc.fused_add_rms_norm(x, None, torch.ones(32, device="cuda"))
    with pytest.raises(RuntimeError, match="one CUDA device"):
        mhc.fused_add_rms_norm(x, None, torch.ones(64))
    with pytest.raises(RuntimeError, match="one CUDA device"):
        mhc.counter_dropout(x, 0.5, rng=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="dtype"):
        mhc.fused_add_rms_norm(x.double(), None, w)
    with pytest.raises(TypeError, match="scale dtype"):
        mhc.fused_add_rms_norm_quant(x, None, w, scale_dtype=torch.float16)
    with pytest.raises(ValueError, match="group"):
        mhc.fused_add_rms_norm_quant(x, None, w, group=48)
    with pytest.raises(mhc._lib.MhcError, match="eps"):
        mhc.fused_add_rms_norm(x, None, w, -1.0)
    with pytest.raises(mhc._lib.MhcError, match="2\\^32"):
        mhc.counter_dropout(x, 0.5, rng=(1, 1), row_offset=2 ** 32 - 2)
    y, _ = mhc.fused_add_rms_norm(x.requires_grad_(True), None, w)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()           # no second derivative


def test_derivatives_that_do_not_exist_are_refused():
    """Second derivatives and forward-mode tangents raise instead of leaving terms out."""
    import mhc
    from torch.autograd import forward_ad
    B, S, D = 2, 3, 64
    H, bo = torch.randn(B, S, 4, D, device="cuda"), torch.randn(B, S, D, device="cuda")
    Hp, w = torch.rand(B, 4, device="cuda"), torch.ones(D, device="cuda")
    leaf = bo.clone().requires_grad_(True)
    out = mhc.fused_add_residual(H, leaf, Hp, dropout_p=0.25, rng=(1, 2))
    (g,) = torch.autograd.grad((out * out).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    calls = [lambda b, h: mhc.counter_dropout(b, 0.25, rng=(1, 2)), lambda b, h: mhc.fused_add_rms_norm(b, None, w),
             lambda b, h: mhc.fused_stream_norm(h, Hp, w), lambda b, h: mhc.fused_add_rms_norm_quant(b, None, w),
             lambda b, h: mhc.fused_stream_norm_quant(h, Hp, w),
             lambda b, h: mhc.fused_add_residual(h, b, Hp, dropout_p=0.25, rng=(1, 2))]
    for call in calls:
        with torch.no_grad():
            call(bo, H)
        with forward_ad.dual_level():
            call(bo, H)              # nothing carries a tangent
            dual_b = forward_ad.make_dual(bo, torch.ones_like(bo))
            dual_h = forward_ad.make_dual(H, torch.ones_like(H))
            with pytest.raises(RuntimeError):
                call(dual_b, dual_h)


def test_many_rows_past_32_bit_offsets():
    """A tensor of more than 2^31 elements: the last rows must be the last rows."""
    import mhc
    rows, D = 270000, 8192          # 2.2e9 elements, 4.4 GB in bf16
    x = torch.empty(rows, D, device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = torch.ones(D, device="cuda")
    y, _ = mhc.fused_add_rms_norm(x, None, w)
    tail = x[-3:].double().cpu()
    y64 = SO.rms_norm(tail, torch.ones(D, dtype=torch.float64), EPS)[0]
    within(y[-3:], y64, (2.0 ** -8 + steps(D) * U) * y64.abs() + 1e-30, "tail")
    d = mhc.counter_dropout(x, 0.5, rng=(1, 2))
    keep = SO.keep_mask(1, 2, 3, D, 0.5, rows - 3)
    assert torch.equal(d[-3:].cpu(), torch.where(keep, x[-3:].float().cpu() * 2, torch.zeros(())).bfloat16())
    q, scales, _ = mhc.fused_add_rms_norm_quant(x, None, w, group=32, scale_dtype=torch.float8_e8m0fnu)
    check_quant(q[-3:], scales[-3:], y64, 2 * steps(D) * U * y64.abs() + 1e-300, 32, True, D)
    del q, scales, y
    leaf = x.requires_grad_(True)
    out, _ = mhc.fused_add_rms_norm(leaf, None, w)
    (dx,) = torch.autograd.grad(out, leaf, d)
    dy = d[-3:].double().cpu()
    _, rstd = SO.rms_norm(tail, torch.ones(D, dtype=torch.float64), EPS)
    g64, _, g_mag, _ = SO.rms_norm_grad(dy, tail, rstd, torch.ones(D, dtype=torch.float64))
    within(dx[-3:], g64, 2.0 ** -8 * g64.abs() + 2 * steps(D) * U * g_mag + 1e-30, "dx tail")
    del dx, out, d
    H, pre = x.detach()[:269996].view(1, 67499, 4, D).requires_grad_(True), torch.tensor([[0.1, 0.2, 0.3, 0.4]], device="cuda")
    b64, b_mag = mixed64(H[:, -2:].detach().cpu(), pre.cpu())
    y64, rstd = SO.rms_norm(b64, torch.ones(D, dtype=torch.float64), EPS)
    y = mhc.fused_stream_norm(H, pre, w)
    within(y[:, -2:], y64, 2.0 ** -8 * y64.abs() + 4 * steps(D) * U * rstd * b_mag + 1e-30, "stream tail")
    (dH,) = torch.autograd.grad(y, H, y.detach())
    dy = y[:, -2:].detach().double().cpu()
    g64, _, g_mag, _ = SO.rms_norm_grad(dy, b64, rstd, torch.ones(D, dtype=torch.float64))
    p64 = pre.double().cpu()[:, None, :, None]
    within(dH[:, -2:], p64 * g64.unsqueeze(2), p64 * (2.0 ** -8 * g64.abs() + 8 * steps(D) * U * (g_mag + rstd ** 2 * b_mag)
                                                      ).unsqueeze(2) + 1e-30, "dH tail")


def test_kernels_are_the_librarys_own():
    from mhc import _lib as L
    import mhc
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    n = L.load().mhc_launch_count()
    mhc.fused_add_rms_norm(x, None, w)
    mhc.counter_dropout(x, 0.5, rng=torch.tensor([1, 1], device="cuda"))
    assert L.load().mhc_launch_count() == n + 2
