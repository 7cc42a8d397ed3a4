"""The operators around a sub-layer without a GPU: the oracle against published vectors, autograd and
differences; argument checks of the C entry points and of the public functions; shape-only registrations."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import sublayer_oracle as SO


# ------------------------------------------------------------------------------------------- the oracle
@pytest.mark.parametrize("counter,key,want", [
    # known answers published with the generator's paper
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_known_answers(counter, key, want):
    got = SO.philox4x32_10([np.array([c]) for c in counter], key)
    assert tuple(int(v) for v in got[:, 0]) == want


def test_oracle_norm_gradient_against_autograd_and_differences():
    g = torch.Generator().manual_seed(3)
    s = torch.randn(5, 7, generator=g, dtype=torch.float64).requires_grad_(True)
    w = torch.randn(7, generator=g, dtype=torch.float64).requires_grad_(True)
    dy = torch.randn(5, 7, generator=g, dtype=torch.float64)
    y, rstd = SO.rms_norm(s, w, 1e-6)
    gs, gw = torch.autograd.grad(y, [s, w], dy)
    with torch.no_grad():
        ds, dw, _, _ = SO.rms_norm_grad(dy, s, rstd, w)
        assert torch.allclose(gs, ds, rtol=1e-12, atol=1e-14) and torch.allclose(gw, dw, rtol=1e-12, atol=1e-14)
        h, v = 1e-5, torch.randn(5, 7, generator=g, dtype=torch.float64)
        diff = ((SO.rms_norm(s + h * v, w, 1e-6)[0] - SO.rms_norm(s - h * v, w, 1e-6)[0]) * dy).sum() / (2 * h)
        # second-order differences: error about h^2 times a third derivative of order one
        assert abs(float(diff - (ds * v).sum())) < 1e-7


def test_oracle_e4m3_matches_the_type():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(SO.round_e4m3(every), every)
    v = torch.randn(4096, dtype=torch.float64, generator=torch.Generator().manual_seed(0)).float() * 60
    v = v.clamp(-448, 448)
    assert torch.equal(SO.round_e4m3(v.double()).float(), v.to(torch.float8_e4m3fn).float())


# ----------------------------------------------------------------------------- C entry points, no launch
# Scalar arguments are checked before pointers and the pointers passed are null (or host addresses of entry points
# that refuse an earlier argument), so nothing is launched even where a check under test were missing.
def _lib():
    from mhc import _lib
    return _lib.load()


def test_c_refusals_of_the_norm():
    lib = _lib()
    f = lib.mhc_add_rms_norm_fwd
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 4, 16, 7, 1e-6, None) == 3      # unknown dtype
    assert f(None, None, None, 0, None, 0, 0, None, None, None, -1, 16, 0, 1e-6, None) == 2     # negative rows
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 1 << 31, 16, 0, 1e-6, None) == 2
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 4, 16, 0, -1.0, None) == 4      # negative eps
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 4, 16, 0, float("nan"), None) == 4
    assert f(None, None, None, 0, None, 65536, 0, None, None, None, 4, 16, 0, 1e-6, None) == 4  # threshold
    assert f(None, None, None, 0, None, 9, 0, None, None, None, 4, 16, 0, 1e-6, None) == 1      # no rng
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 4, 16, 0, 1e-6, None) == 1
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 0, 16, 0, 1e-6, None) == 0      # empty
    assert f(None, None, None, 0, None, 0, 0, None, None, None, 4, 0, 0, 1e-6, None) == 0
    assert f(None, None, 16, 2, None, 0, 0, None, None, None, 4, 16, 1, 1e-6, None) == 3        # fp16 weight, bf16 x
    q = lib.mhc_add_rms_norm_quant_fwd
    assert q(None, None, None, 0, None, None, None, 33, 0, 4, 16, 0, 1e-6, None) == 4           # group
    assert q(None, None, None, 0, None, None, None, 32, 2, 4, 16, 0, 1e-6, None) == 4           # scale type
    assert q(None, None, None, 0, None, None, None, 32, 1, 4, 16, 0, 1e-6, None) == 1
    b = lib.mhc_rms_norm_bwd
    assert b(None, None, None, None, None, None, 0, None, 0, 0, None, None, 64, None, 3, 4, 16, 0, None) == 5   # scratch
    assert b(None, None, None, None, None, None, 0, None, 0, 0, None, None, None, None, 0, 4, 16, 0, None) == 1
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    assert b(p, None, p, None, p, None, 0, None, 0, 0, p, p, None, None, 0, 4, 16, 0, None) == 4      # dresidual without dropout
    s = lib.mhc_stream_norm_fwd
    assert s(None, None, None, 0, None, None, None, 2, 3, 16, 0, 1e-6, None) == 1
    assert s(None, None, None, 0, None, None, None, 1 << 20, 1 << 20, 16, 0, 1e-6, None) == 2   # more tokens than a grid has CTAs
    assert s(None, None, None, 0, None, None, None, 2, 3, 16, 0, -1e-6, None) == 4
    assert lib.mhc_stream_norm_quant_fwd(None, None, None, 0, None, None, 7, 0, 2, 3, 16, 0, 1e-6, None) == 4
    assert lib.mhc_stream_norm_bwd(None, None, None, None, None, 0, None, None, None, None, 8, 2, 3, 16, 0, None) == 5
    assert lib.mhc_stream_norm_bwd(None, None, None, None, None, 0, None, None, None, None, 1 << 30, 2, 3, 16, 0, None) == 1
    h = lib.mhc_hc_mix_norm_fwd
    args = [None] * 9 + [0, -1.0] + [None] * 9 + [0, None, 0, None, 2, 8, 16, 0, 20, 1e-6, None]
    assert h(*args) == 4
    args[10] = 1e-6
    assert h(*args) == 1


def test_c_refusals_of_dropout():
    lib = _lib()
    f = lib.mhc_counter_dropout
    assert f(None, None, 0, 0, None, 4, 16, 0, None) == 4
    assert f(None, None, 65536, 0, None, 4, 16, 0, None) == 4
    assert f(None, None, 9, -1, None, 4, 16, 0, None) == 4
    assert f(None, None, 9, (1 << 32) - 3, None, 4, 16, 0, None) == 4       # rows pass 2^32
    assert f(None, None, 9, 0, None, 4, 16, 5, None) == 3
    assert f(None, None, 9, 0, None, -4, 16, 0, None) == 2
    assert f(None, None, 9, 0, None, 4, 16, 0, None) == 1
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) & ~15
    assert f(None, p + 4, 9, 0, None, 4, 16, 0, None) == 6                  # rng not 8-byte aligned
    assert f(None, p, 9, 0, None, 0, 16, 0, None) == 0                      # empty
    a = lib.mhc_add_residual_dropout_fwd
    assert a(None, None, None, None, None, 9, 0, None, None, 2, 3, 16, 0, None) == 1
    assert a(None, None, None, None, p, 9, 0, None, None, 2, 3, 16, 0, None) == 1
    assert a(None, None, None, None, p, 0, 0, None, None, 2, 3, 16, 0, None) == 4
    assert a(None, None, None, None, p, 9, 0, None, None, 1 << 33, 1 << 30, 16, 0, None) == 4
    b = lib.mhc_add_residual_dropout_bwd
    assert b(None, None, None, p, 9, 0, None, None, None, 8, None, 2, 64, 64, 0, None) == 5
    assert b(None, None, None, p, 9, 0, None, None, None, 1 << 30, None, 2, 64, 64, 0, None) == 1


def test_scratch_sizes_of_the_norm():
    from mhc import _lib as L
    lib = L.load()
    n = lib.mhc_scratch_bytes(L.OP_RMS_NORM_BWD, 0, 32768, 4096, L.MHC_BF16)
    assert 0 < n <= 32 << 20                                 # a row of partial sums per resident CTA
    assert lib.mhc_scratch_bytes(L.OP_RMS_NORM_BWD, 0, 1, 4096, L.MHC_BF16) >= 4 * 4096
    assert 0 < lib.mhc_scratch_bytes(L.OP_STREAM_NORM_BWD, 8, 4096, 4096, L.MHC_BF16) <= 32 << 20


# -------------------------------------------------------------------------------- public functions, no GPU
def test_public_refusals():
    import mhc
    x, w = torch.randn(3, 16), torch.ones(16)
    H, H_pre = torch.randn(1, 2, 4, 16), torch.rand(1, 4)
    for call in (lambda: mhc.fused_add_rms_norm(x, None, w), lambda: mhc.fused_add_rms_norm_quant(x, None, w),
                 lambda: mhc.fused_stream_norm(H, H_pre, w), lambda: mhc.fused_stream_norm_quant(H, H_pre, w),
                 lambda: mhc.counter_dropout(x, 0.5), lambda: mhc.counter_dropout(x, 0.5, (1, 2)),
                 lambda: mhc.fused_add_residual(H, torch.randn(1, 2, 16), torch.rand(1, 4), dropout_p=0.5),
                 lambda: mhc.HyperConnection(dim=16)(H, w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for p in (-0.1, 1.0, 1.5, float("nan"), 0.999999):
        with pytest.raises(ValueError):
            mhc.counter_dropout(x, p)
        with pytest.raises(ValueError):
            mhc.fused_add_residual(H, torch.randn(1, 2, 16), torch.rand(1, 4), dropout_p=p)
    assert mhc.counter_dropout(x, 0.0) is x
    with pytest.raises(AssertionError):
        mhc.counter_dropout(x, 0.5, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(AssertionError):
        mhc.counter_dropout(x, 0.5, torch.zeros(2))
    with pytest.raises(AssertionError):
        mhc.fused_stream_norm(torch.randn(1, 2, 3, 16), H_pre)
    with pytest.raises(AssertionError):
        mhc.fused_stream_norm(H, torch.rand(2, 4))
    for t in (x, H):   # an output of 8 bits has no gradient
        t.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        mhc.fused_add_rms_norm_quant(x, None, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        mhc.fused_stream_norm_quant(H, H_pre, w)
    with pytest.raises(ValueError, match="norm_eps"):
        mhc.hyper_connection_mix(H, *[None] * 7, norm_weight=w)
    with pytest.raises(ValueError, match="lazy_residual"):
        mhc.hyper_connection_mix(H, *[None] * 7, norm_eps=1e-6)
