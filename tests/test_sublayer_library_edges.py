"""mhc.library's norm without a weight: absent gradients of the registered backward are separate tensors, as torch.library
demands of an operator's outputs."""

import itertools

import pytest
import torch

COMBINATIONS = list(itertools.product([False, True], [0.0, 0.25], [False, True]))     # residual, dropout, weight


def _plain_forward(x, residual=None, weight=None, eps=1e-6, rng=None, threshold=0, row_offset=0, want_rstd=True):
    s = x.clone() if residual is None else x + residual
    rstd = (s.square().mean(-1) + eps).rsqrt()
    y = s * rstd.unsqueeze(-1)
    return (y if weight is None else y * weight), s, rstd.reshape(-1)


def _plain_backward(dy, dsum, x, residual, rstd, weight=None, rng=None, threshold=0, row_offset=0, want_dresidual=False,
                    want_dweight=True):
    dx = dy.clone()
    dres = dy * 2 if threshold and want_dresidual else None
    return dx, (dres if threshold else dx), (torch.full_like(weight, 3.0) if want_dweight and weight is not None else None)


def _leaves(residual, weight, device="cpu", dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=g).to(device, dtype).requires_grad_(True)      # noqa: E731
    return make(6, 64), (make(6, 64) if residual else None), (make(64) if weight else None)


@pytest.mark.parametrize("residual,p,weight", COMBINATIONS)
def test_registered_backward_around_stub_kernels(residual, p, weight, monkeypatch):
    """Every combination of inputs reaches the leaves with the gradient that the launch wrapper returned for them."""
    from mhc import library
    monkeypatch.setattr(library.K, "add_rms_norm_forward", _plain_forward)
    monkeypatch.setattr(library.B, "rms_norm_backward", _plain_backward)
    x, r, w = _leaves(residual, weight)
    y, _ = library.fused_add_rms_norm(x, r, w, dropout_p=p, rng=torch.zeros(2, dtype=torch.int64))
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(x.grad, dy)
    if residual:
        assert torch.equal(r.grad, dy * 2 if p else dy)
    if weight:
        assert torch.equal(w.grad, torch.full_like(w, 3.0))


@pytest.mark.parametrize("residual,p,weight", COMBINATIONS)
def test_meta_shapes_of_the_backward(residual, p, weight):
    from mhc import library
    leaves = [None if t is None else torch.empty_like(t, device="meta").requires_grad_(True)
              for t in _leaves(residual, weight, dtype=torch.bfloat16)]
    y, _ = library.fused_add_rms_norm(*leaves, dropout_p=p, rng=torch.empty(2, dtype=torch.int64, device="meta"))
    there = [t for t in leaves if t is not None]
    for t, g in zip(there, torch.autograd.grad(y, there, torch.empty_like(y))):
        assert g.shape == t.shape and g.dtype == t.dtype


@pytest.mark.gpu
@pytest.mark.parametrize("residual,p,weight", COMBINATIONS)
def test_equal_to_the_plain_function(residual, p, weight):
    import mhc
    from mhc import library
    rng = torch.tensor([3, 4], device="cuda")
    results = []
    for ops in (mhc, library):
        leaves = _leaves(residual, weight, "cuda", torch.bfloat16)
        there = [t for t in leaves if t is not None]
        y, s = ops.fused_add_rms_norm(*leaves, dropout_p=p, rng=rng, row_offset=2)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(5)).to(y)
        results.append([y, s, *torch.autograd.grad([y, s] if s is not leaves[0] else [y], there,
                                                   [dy, dy] if s is not leaves[0] else [dy])])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("threshold", [0, 9000])
def test_opcheck_without_a_weight(residual, threshold):
    from mhc import library
    x, r, _ = _leaves(residual, False, "cuda", torch.bfloat16)
    rng = torch.tensor([3, 4], device="cuda") if threshold else None
    torch.library.opcheck(library._add_rms_norm_fwd, (x, r, None, 1e-5, rng, threshold, 0),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                      "test_aot_dispatch_dynamic"))


@pytest.mark.gpu
def test_stream_norm_without_a_weight():
    import mhc
    from mhc import library
    g = torch.Generator().manual_seed(2)
    H0, pre0, dy = torch.randn(2, 5, 4, 64, generator=g), torch.rand(2, 4, generator=g), torch.randn(2, 5, 64, generator=g).cuda()
    results = []
    for ops in (mhc, library):
        H, pre = H0.cuda().requires_grad_(True), pre0.cuda().requires_grad_(True)
        y = ops.fused_stream_norm(H, pre)
        results.append([y, *torch.autograd.grad(y, [H, pre], dy)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
