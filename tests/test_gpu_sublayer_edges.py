"""The operators around a sub-layer where their other tests do not go: extreme batch sizes, the layer's own kernels in the
16-bit types, many rows in fp32, unaligned 8-bit outputs, all against 64 bits.

Tolerances are those of tests/test_gpu_sublayer.py: u = 2^-24 for each fp32 rounding on the way, half a step of the stored
type for the last one."""

import pytest
import torch

from oracle import sublayer_oracle as SO

from .test_gpu_sublayer import EPS, U, check_quant, half_step, steps, within

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
