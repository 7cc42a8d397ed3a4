"""64-bit restatement of the operators around a sub-layer (RMS norm, 8-bit output with scales, counter-based
dropout, add residual with dropout), with the magnitudes their rounding errors are bounded by.  Test
infrastructure only; plain tensor algebra on the CPU, nothing of the package under test."""

import numpy as np
import torch

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126


# ------------------------------------------------------------------------------------------ generator
def philox4x32_10(counter, key):
    """Philox4x32 with ten rounds (Salmon et al., SC 2011) on uint64 arrays of 32-bit words: counter [4, n], key (k0, k1)."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c0, c1, c2, c3 = (np.asarray(c, dtype=np.uint64) for c in counter)
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(10):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = ((b >> half) ^ c1 ^ np.uint64(k0), b & low, (a >> half) ^ c3 ^ np.uint64(k1), a & low)
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([c0, c1, c2, c3])


def threshold_of(p):
    return int(round(p * 65536))


def keep_mask(seed, offset, rows, dim, p, row_offset=0):
    """Bool [rows, dim]: which elements the dropout keeps."""
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    groups = (dim + 7) // 8
    col8 = np.tile(np.arange(groups, dtype=np.uint64), rows)
    row = np.repeat(np.arange(row_offset, row_offset + rows, dtype=np.uint64), groups)
    one = np.ones_like(col8)
    w = philox4x32_10([col8, row, one * np.uint64(offset & 0xFFFFFFFF), one * np.uint64(offset >> 32)],
                      (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.empty((rows * groups, 8), dtype=np.uint64)
    for i in range(4):
        halves[:, 2 * i], halves[:, 2 * i + 1] = w[i] & np.uint64(0xFFFF), w[i] >> np.uint64(16)
    return torch.from_numpy(halves.reshape(rows, groups * 8)[:, :dim] >= threshold_of(p))


def keep_factor(p):
    return 65536.0 / (65536 - threshold_of(p))


def dropout(x, keep, p):
    return torch.where(keep, x * keep_factor(p), torch.zeros_like(x))


# ----------------------------------------------------------------------------------------------- norm
def rms_norm(s, weight, eps):
    """(y, rstd) of fp64 rows."""
    rstd = 1.0 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * rstd * weight, rstd


def rms_norm_grad(dy, s, rstd, weight):
    """(ds, dweight) and the magnitude sums (of the terms of ds, of those of dweight) that rounding scales with."""
    D = s.shape[-1]
    h = dy * weight
    k = rstd ** 3 / D * (h * s).sum(-1, keepdim=True)
    k_abs = rstd ** 3 / D * (h * s).abs().sum(-1, keepdim=True)
    terms = (dy * s * rstd).reshape(-1, D)
    return rstd * h - s * k, terms.sum(0), (rstd * h).abs() + s.abs() * k_abs, terms.abs().sum(0)


def round_e4m3(v):
    """Nearest e4m3 value, ties to even (|v| <= 448; NaN stays)."""
    a = v.abs().clamp(max=E4M3_MAX)
    step = torch.exp2((torch.frexp(a).exponent - 1).clamp(min=-6).double() - 3)
    return torch.copysign(torch.round(a / step) * step, v)


def scales_of(y, group, e8m0):
    """fp64 scales [..., G] of y [..., D], one per row (group 0) or per `group` columns."""
    D = y.shape[-1]
    out = []
    for lo in range(0, D, group or D):
        out.append((y[..., lo:lo + (group or D)].abs().amax(-1) / E4M3_MAX).clamp(min=MIN_SCALE))
    s = torch.stack(out, -1)
    return torch.exp2(torch.ceil(torch.log2(s))) if e8m0 else s


def spread_scales(scales, D, group):
    """Scales [..., G] -> [..., D]."""
    return scales.repeat_interleave(group or D, dim=-1)[..., :D]
