"""The torch.library registration of the norm and dropout operators (mhc.library): schemas and shapes on meta tensors,
and on the GPU the same results as the plain functions, opcheck, and a full-graph trace."""

import pytest
import torch

B, S, D = 2, 24, 64


def _inputs(device, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)

    def r(*shape, dt=torch.float32):
        t = torch.randn(*shape, generator=g).to(dt)
        return (torch.empty(t.shape, dtype=dt, device="meta") if device == "meta" else t.to(device)).requires_grad_(True)

    return dict(H=r(B, S, 4, D, dt=dtype), pre=r(B, 4), post=r(B, 4), w=r(D), w2=r(D, dt=dtype), bo=r(B, S, D, dt=dtype))


def _rng(device):
    return torch.empty(2, dtype=torch.int64, device="meta") if device == "meta" else torch.tensor([3, 4], device=device)


def _block(ops, t, rng):
    """A sub-layer with its norms and dropouts."""
    y = ops.fused_stream_norm(t["H"], t["pre"], t["w"], 1e-6)
    z, s = ops.fused_add_rms_norm(t["bo"], y, t["w2"], 1e-5, dropout_p=0.2, rng=rng, row_offset=3)
    z2, _ = ops.fused_add_rms_norm(s, None, t["w"], 1e-5)
    out = ops.counter_dropout(z + z2, 0.3, rng)
    return ops.fused_add_residual(t["H"], out, t["post"], dropout_p=0.1, rng=rng)


def test_schemas_registered():
    import mhc.library  # noqa: F401
    for name, nret in [("counter_dropout", 1), ("add_residual_dropout_fwd", 1), ("add_residual_dropout_bwd", 2),
                       ("add_rms_norm_fwd", 3), ("rms_norm_bwd", 3), ("add_rms_norm_quant_fwd", 3), ("stream_norm_fwd", 2),
                       ("stream_norm_bwd", 3), ("stream_norm_quant_fwd", 2)]:
        op = getattr(torch.ops.mhc, name).default
        assert len(op._schema.returns) == nret, name
        assert not op._schema.is_mutable, name


def test_meta_shapes():
    from mhc import library
    t = _inputs("meta", torch.bfloat16)
    out = _block(library, t, _rng("meta"))
    assert out.shape == (B, S, 4, D) and out.dtype == torch.bfloat16
    grads = torch.autograd.grad(out, list(t.values()), torch.empty_like(out))
    for (k, v), g in zip(t.items(), grads):
        assert g.shape == v.shape and g.dtype == v.dtype, k
    with torch.no_grad():
        q, sc, s = library.fused_add_rms_norm_quant(t["bo"], t["bo"], t["w"], group=32, scale_dtype=torch.float8_e8m0fnu)
        assert q.shape == (B, S, D) and q.dtype == torch.float8_e4m3fn and sc.shape == (B, S, 2) and s.shape == q.shape
        q, sc = library.fused_stream_norm_quant(t["H"], t["pre"])
        assert q.shape == (B, S, D) and sc.shape == (B, S, 1) and sc.dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_to_the_plain_functions(dtype):
    import mhc
    from mhc import library
    results = []
    for ops in (mhc, library):
        t = _inputs("cuda", dtype)
        out = _block(ops, t, _rng("cuda"))
        grads = torch.autograd.grad(out, list(t.values()), torch.ones_like(out))
        with torch.no_grad():
            quant = [*ops.fused_add_rms_norm_quant(t["bo"], t["bo"], t["w"], group=32),
                     *ops.fused_stream_norm_quant(t["H"], t["pre"], t["w"])]
        results.append([out, *grads, *[q.float() for q in quant]])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_opcheck_and_full_graph():
    from mhc import library
    t = _inputs("cuda", torch.bfloat16)
    rng = _rng("cuda")
    checks = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    torch.library.opcheck(library._counter_dropout, (t["bo"], rng, 9000, 1), test_utils=checks)
    torch.library.opcheck(library._add_rms_norm_fwd, (t["bo"], t["bo"].detach().clone().requires_grad_(True), t["w"], 1e-5, rng,
                                                      9000, 0), test_utils=checks)
    torch.library.opcheck(library._stream_norm_fwd, (t["H"], t["pre"], t["w"], 1e-5), test_utils=checks)
    torch.library.opcheck(library._add_residual_dropout_fwd, (t["H"], t["bo"], t["post"], rng, 9000, 0), test_utils=checks)
    torch.library.opcheck(library._add_rms_norm_quant_fwd, (t["bo"].detach(), None, t["w"].detach(), 1e-5, 32, torch.float32),
                          test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(lambda t, rng: _block(library, t, rng), fullgraph=True, backend="aot_eager")
    eager, traced = _block(library, t, rng), compiled(t, rng)
    assert torch.equal(eager, traced)
    g = torch.ones_like(eager)
    for a, b in zip(torch.autograd.grad(eager, list(t.values()), g), torch.autograd.grad(traced, list(t.values()), g)):
        assert torch.equal(a, b)
