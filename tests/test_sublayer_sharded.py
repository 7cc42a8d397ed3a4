"""Norm and dropout of the sequence-sharded wrapper: every rank's rows of the dropout's counter are its own, and with one rank
the wrapper is the layer."""

import os
from unittest import mock

import pytest
import torch
import torch.distributed as dist

from oracle import sublayer_oracle as SO
from tests.util import run_ranks

D, P = 32, 0.5
# batch elements, tokens of each rank, total_len given to the wrapper
SHARDS = [(1, (6, 6), None), (3, (5, 5), None), (2, (5, 5), 10), (2, (1, 7), 8), (3, (7, 2), 9)]


def _fake_mix(H, *a):
    B, S, _, D = H.shape
    return H.sum(2), H.new_empty(1).expand(H.shape), H.new_ones(B, 4), H.new_ones(B, 4), H.new_ones(B, 4, 4)


def _fake_update(stand_in, H, H_res, branch_output, H_post, pool, p, rng, row_offset):
    """The mask that the kernel draws for these arguments (row = b * S + s)."""
    B, S, D = branch_output.shape
    return SO.keep_mask(rng[0], rng[1], B * S, D, p, row_offset).view(B, S, D)


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import mhc
        from mhc import ops, parallel
        layer = mhc.HyperConnection(dim=D)
        with mock.patch.object(parallel._SequenceShardedMix, "apply", _fake_mix), \
                mock.patch.object(ops, "add_residual_from_state", _fake_update):
            for B, tokens, total in SHARDS:
                sp = parallel.SequenceShardedHyperConnection(layer, total_len=total)
                bi, add = sp(torch.zeros(B, tokens[rank], 4, D))
                every = [None] * world
                dist.all_gather_object(every, [add(bi, P, rng=(7, 9)), add(bi, P, rng=(7, 9), row_offset=0)])
                masks = [m[0] for m in every]
                rows = torch.cat([m.reshape(-1, D) for m in masks])
                assert len(torch.unique(rows, dim=0)) == B * sum(tokens), "a row of the counter serves two tokens"
                if B == 1 and total is None:
                    whole = SO.keep_mask(7, 9, sum(tokens), D, P)
                    assert torch.equal(rows, whole), "one sequence in equal shards has the whole tensor's mask"
                for r in range(world):      # a row_offset that is given is taken as it is
                    assert torch.equal(every[r][1].reshape(-1, D), SO.keep_mask(7, 9, B * tokens[r], D, P, 0))
        q.put((rank, "ok"))
    except Exception as e:  # report instead of hanging the peer
        q.put((rank, f"{type(e).__name__}: {e}"))
    finally:
        dist.destroy_process_group()


def test_ranks_draw_masks_of_their_own():
    assert run_ranks(_worker, 2) == [(0, "ok"), (1, "ok")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,S,D", [(torch.float32, 2, 30, 64), (torch.bfloat16, 3, 17, 129), (torch.float16, 1, 40, 512)])
def test_one_rank_equals_the_layer(dtype, B, S, D):
    """Same mask, same norm of the mix as it is stored, whose last bit may differ."""
    import mhc
    from mhc.parallel import SequenceShardedHyperConnection
    torch.manual_seed(5)
    hc = mhc.HyperConnection(dim=D).cuda()
    with torch.no_grad():
        hc.phi.normal_(std=0.02)
    H0 = torch.randn(B, S, 4, D).to(dtype).cuda()
    g = torch.randn(B, S, 4, D).to(dtype).cuda()
    w0 = (torch.rand(D) + 0.5).cuda()
    rng = torch.tensor([3, 4], device="cuda")
    got = []
    for m in (hc, SequenceShardedHyperConnection(hc)):
        hc.zero_grad()
        H, w = H0.clone().requires_grad_(True), w0.clone().requires_grad_(True)
        y, add = m(H, w, 1e-5)
        y.retain_grad()
        out = add(y, dropout_p=0.3, rng=rng)
        out.backward(g)
        got.append([y.detach().double(), out.detach().double(), H.grad.double(), w.grad.double(), y.grad.double()])
    (y, out, dH, dw, dy), (y2, out2, dH2, dw2, dy2) = got
    # both normalise the mix as it is stored, from the same products in the same order up to their fusing: a stored value
    # may be a step of the type apart, and what is made of it that and two half steps of its own
    step = torch.finfo(dtype).eps
    assert ((y - y2).abs() <= 2.5 * step * y.abs() + 1e-6).all()
    bo = (out - out2).abs()
    assert (bo <= 3 * step * out.abs() + 2.5 * step * 2 / 0.7 * y.abs().unsqueeze(2) + 1e-5).all()
    assert ((dy - dy2).abs() <= 2 * step * dy.abs() + 1e-5).all()
    # d(norm) = rstd (h - n mean(h n)), with a step or two in h and in n each; n = y / w
    n, h = (y / w0.double()).abs(), (dy * w0.double()).abs()
    with torch.no_grad():
        rstd = (hc(H0)[0].double().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    db = rstd * (h + n * (h * n).mean(-1, keepdim=True))
    assert ((dH - dH2).abs() <= 2 * step * dH.abs() + 8 * step * db.unsqueeze(2) + 2e-5 * float(dH.abs().max())).all()
    assert ((dw - dw2).abs() <= 5 * step * (dy.abs() * n).sum((0, 1)) + 1e-4).all()
