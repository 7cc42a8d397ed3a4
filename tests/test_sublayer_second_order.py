"""Second derivatives of the operators around a sub-layer are refused wherever a term would be left out, with an upstream
gradient that is itself differentiated or not, and handed through where nothing is left out."""

import pytest
import torch

from mhc import ops


def _first(outputs, inputs, upstream=None):
    outs = outputs if isinstance(outputs, (list, tuple)) else [outputs]
    return torch.autograd.grad(outs, inputs, upstream or [torch.ones_like(o) for o in outs], create_graph=True, allow_unused=True)


def _refused(grads, beside):
    """A loss of these gradients that depends on the leaves another way too must not come back without their part."""
    loss = sum(g.square().sum() for g in grads if g is not None) + sum(t.square().sum() for t in beside)
    with pytest.raises(RuntimeError, match="second derivative"):
        loss.backward()


def _cases(device):
    """name -> (function of the leaves, leaves); every gradient depends on a leaf."""
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=g).to(device).requires_grad_(True)      # noqa: E731
    rng = torch.tensor([1, 2], device=device)
    return {
        "norm": (lambda x, w: ops.fused_add_rms_norm(x, None, w)[0], [make(4, 64), make(64)]),
        "add_norm": (lambda x, r, w: list(ops.fused_add_rms_norm(x, r, w)), [make(4, 64), make(4, 64), make(64)]),
        "dropout_norm": (lambda x, w: list(ops.fused_add_rms_norm(x, None, w, dropout_p=0.25, rng=rng)), [make(4, 64), make(64)]),
        "stream_norm": (lambda H, p, w: ops.fused_stream_norm(H, p, w), [make(2, 3, 4, 64), make(2, 4), make(64)]),
        "add_residual": (lambda H, b, p: ops.fused_add_residual(H, b, p, dropout_p=0.25, rng=rng),
                         [make(2, 3, 4, 64), make(2, 3, 64), make(2, 4)]),
    }


NAMES = list(_cases("cpu"))


def _stub(monkeypatch):
    """Launch wrappers that return tensors of the right shapes."""
    like = torch.ones_like
    monkeypatch.setattr(ops, "add_rms_norm_forward", lambda x, r=None, w=None, *a, **k: (
        x * 2, x + 1, x.new_ones(x.shape[0])))

    def norm_backward(dy, ds, x, r, rstd, w=None, rng=None, threshold=0, row_offset=0, want_dresidual=False, want_dweight=True):
        dx = like(x)
        return dx, (like(x) if threshold else dx), (like(w) if w is not None and want_dweight else None)

    monkeypatch.setattr(ops, "rms_norm_backward", norm_backward)
    monkeypatch.setattr(ops, "stream_norm_forward", lambda H, p, w=None, *a, **k: (H.sum(2), None, H.new_ones(6)))
    monkeypatch.setattr(ops, "stream_norm_backward", lambda dy, H, p, rstd, w=None, **k: (
        like(H), like(p), None if w is None or not k.get("want_dweight", True) else like(w)))
    monkeypatch.setattr(ops, "add_residual_dropout_forward", lambda H, *a, **k: H * 1)
    monkeypatch.setattr(ops, "add_residual_dropout_backward", lambda g, b, p, *a: (g, like(b), like(p)))
    monkeypatch.setattr(ops, "counter_dropout_forward", lambda x, *a: x * 2)


def _run(name, device):
    f, leaves = _cases(device)[name]
    _refused(_first(f(*leaves), leaves), leaves)                             # upstream gradients are constants
    out = f(*leaves)
    outs = out if isinstance(out, list) else [out]
    _refused(_first(sum(o.square().sum() for o in outs), leaves), leaves)    # they depend on the leaves
    for with_graph in (False, True):                                         # first derivatives are what they were
        a = torch.autograd.grad(sum(o.sum() for o in _as_list(f(*leaves))), leaves, create_graph=with_graph)
        b = torch.autograd.grad(sum(o.sum() for o in _as_list(f(*leaves))), leaves)
        for x, y in zip(a, b):
            assert torch.equal(x.detach(), y)


def _as_list(out):
    return out if isinstance(out, list) else [out]


@pytest.mark.parametrize("name", NAMES)
def test_refused_around_stub_kernels(name, monkeypatch):
    _stub(monkeypatch)
    _run(name, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_refused(name):
    _run(name, "cuda")


def _nothing_left_out(device):
    """Gradients that do not depend on any leaf are constants: no refusal, and the rest of the loss is differentiated."""
    g = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=g).to(device)      # noqa: E731
    rng = torch.tensor([1, 2], device=device)
    H, bo, post, x, w = make(2, 3, 4, 64), make(2, 3, 64), make(2, 4), make(4, 64), make(64)
    pre = make(2, 4)
    for f, t in ((lambda t: ops.counter_dropout(t, 0.25, rng), x), (lambda t: ops.fused_add_rms_norm(x, None, t)[0], w),
                 (lambda t: ops.fused_stream_norm(H, pre, t), w), (lambda t: ops.fused_add_residual(H, t, post, dropout_p=0.25, rng=rng), bo),
                 (lambda t: ops.fused_add_residual(H, bo, t, dropout_p=0.25, rng=rng), post)):
        leaf = t.clone().requires_grad_(True)
        (g1,) = _first(f(leaf), [leaf])
        (g1.square().sum() + leaf.square().sum()).backward()
        assert torch.equal(leaf.grad, 2 * leaf.detach())
    a, r, v = (t.clone().requires_grad_(True) for t in (x, 3 * x, w))       # the sum alone is linear in both
    grads = _first(ops.fused_add_rms_norm(a, r, v)[1], [a, r])
    (grads[0].square().sum() + grads[1].square().sum() + a.square().sum() + r.square().sum()).backward()
    assert torch.equal(a.grad, 2 * a.detach()) and torch.equal(r.grad, 2 * r.detach())
    leaf = H.clone().requires_grad_(True)               # the residual's gradient is the upstream one itself
    b, p = bo.clone().requires_grad_(True), post.clone().requires_grad_(True)
    out = ops.fused_add_residual(leaf, b, p, dropout_p=0.25, rng=rng)
    up = torch.ones_like(out).requires_grad_(True)
    (g1,) = _first(out, [leaf], [up])
    (g1.square().sum() + leaf.square().sum()).backward()
    assert torch.equal(leaf.grad, 2 * leaf.detach()) and torch.equal(up.grad, 2 * torch.ones_like(out))


def test_gradients_without_a_second_derivative_around_stub_kernels(monkeypatch):
    _stub(monkeypatch)
    _nothing_left_out("cpu")


@pytest.mark.gpu
def test_gradients_without_a_second_derivative():
    _nothing_left_out("cuda")


# -------------------------------------------------------------------------------------------------- the layer's own node
def _layer(device, norm):
    import mhc
    torch.manual_seed(0)
    hc = mhc.HyperConnection(dim=64).to(device)
    H = torch.randn(2, 5, 4, 64).to(device).requires_grad_(True)
    w = torch.rand(64).to(device).add_(0.5).requires_grad_(True)
    y, add = hc(H, w) if norm else hc(H)
    return y, add, H, w


def _layer_with_norm(device):
    y, add, H, w = _layer(device, True)
    _refused(_first(y, [H, w]), [H, w])
    y, add, H, w = _layer(device, True)
    _refused(_first(y.square().sum(), [H, w]), [H, w])
    y, add, H, w = _layer(device, True)
    _refused(_first(add(torch.tanh(y), dropout_p=0.25, rng=torch.tensor([1, 2], device=device)), [H, w]), [H, w])
    for with_graph in (False, True):
        y, add, H, w = _layer(device, True)
        a = torch.autograd.grad(y.sum(), [H, w], create_graph=with_graph)
        y, add, H, w = _layer(device, True)
        for p, q in zip(a, torch.autograd.grad(y.sum(), [H, w])):
            assert torch.equal(p.detach(), q)


def test_layer_with_norm_around_stub_kernels(monkeypatch):
    _stub(monkeypatch)
    like = torch.ones_like

    def mix_norm(H, *a, **k):
        B, S, _, D = H.shape
        return (H.sum(2), H.sum(2), H.new_ones(B * S), H.new_ones(B, 4), H.new_ones(B, 4), H.new_ones(B, 4, 4),
                H.new_ones(B, 4 * D), H.new_ones(B, 32))

    monkeypatch.setattr(ops, "hc_mix_norm_forward", mix_norm)
    monkeypatch.setattr(ops, "hc_mix_backward", lambda dbi, dHr, dp, H, x, phi, *a, **k: (
        like(H), like(phi), phi.new_ones(24), phi.new_ones(3)))
    _layer_with_norm("cpu")


@pytest.mark.gpu
def test_layer_with_norm():
    _layer_with_norm("cuda")


@pytest.mark.gpu
def test_layer_without_norm_is_as_it_was():
    y, add, H, w = _layer("cuda", False)
    (g,) = _first(y, [H])
    (g.square().sum() + H.square().sum()).backward()
    assert torch.equal(H.grad, 2 * H.detach())
