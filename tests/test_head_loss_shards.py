"""The cross entropy of a head over the shards of a volume: uneven ones, and one without voxels."""
import pytest
import torch

from helpers.launch import ROOT, results, torchrun_gloo
from scaffold_b200.ops import _lib
from scaffold_b200.ops.head_loss import head_cross_entropy
from test_head_loss import IGNORED, _definition, _inputs

ON = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Shard:
    """What the loss uses of a spatial context: this shard's sums are noted, the other shards' are added."""

    size, lead_swap = 2, None

    def __init__(self, others=()):
        self.sent, self.others = [], list(others)

    def all_reduce_sum(self, t):
        self.sent.append(t.detach().clone())
        for o in self.others:
            assert o.dtype == t.dtype and o.shape == t.shape  # a collective's ranks bring the same
            t += o
        return t


def _sharded(parts, w, b, cw):
    """(loss, dx, dw, db) of each part of the voxels, with the sums of all."""
    sums = []
    for x, y in parts:
        shard = Shard()
        head_cross_entropy(x, w, b, y, cw, ignore_label=IGNORED, spatial=shard)
        (one,) = shard.sent
        sums.append(one)
    assert len({(s.dtype, s.shape) for s in sums}) == 1
    out = []
    for i, (x, y) in enumerate(parts):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        loss = head_cross_entropy(*leaves, y, cw, ignore_label=IGNORED, spatial=Shard(sums[:i] + sums[i + 1:]))
        assert loss.dtype == torch.float32 and loss.shape == ()
        out.append((loss.detach(), *torch.autograd.grad(loss, leaves)))
    return out


@pytest.mark.parametrize("dev", ON)
@pytest.mark.parametrize("c,k", [(64, 147), (320, 70), (16, 34)])
@pytest.mark.parametrize("cuts", [(0, 300), (100, 300), (300, 300), (5, 297)], ids=str)
def test_shards_add_up_to_the_whole_volume(c, k, cuts, dev):
    x, w, b, y, cw = _inputs(300, c, k, ignored=0.2, weighted=True, w_type=torch.float32, dev=dev)
    edges = [0, *cuts, 300]
    parts = [(x[i:j], y[i:j]) for i, j in zip(edges, edges[1:])]
    got = _sharded(parts, w, b, cw)
    if dev == "cuda":
        _lib.check_status()
    w16 = w.to(torch.bfloat16)
    loss, dx, dw, db, *_ = _definition(x, w16 if dev == "cuda" else w, b, y, cw)
    for one, *_ in got:
        assert abs(float(one) - float(loss)) <= 1e-5 * float(loss)
    # P in bf16 and dX in bf16: 2^-8 of a value at most each, at random; dW and db come in fp32 (as for the whole volume)
    for i, want in ((1, dx), (2, dw), (3, db)):
        have = torch.cat([g[1] for g in got]) if i == 1 else sum(g[i].double() for g in got)
        assert have.shape == want.shape and float((have.double() - want).norm()) <= 4e-3 * float(want.norm())
    for (part, _), (_, gx, gw, gb) in zip(parts, got):
        assert gx.shape == part.shape and gw.shape == w.shape
        if len(part) == 0:
            assert not gw.any() and not gb.any()


@pytest.mark.parametrize("dev", ON)
def test_no_voxel_in_any_shard(dev):
    x, w, b, y, _ = _inputs(4, 16, 34, dev=dev)
    y.fill_(IGNORED)
    for loss, *grads in _sharded([(x, y), (x[:0], y[:0])], w, b, None):
        assert float(loss) == 0 and not any(g.any() for g in grads)


def test_uneven_and_empty_shards_over_two_ranks():
    proc = torchrun_gloo(ROOT / "tests" / "helpers" / "rank_scripts" / "head_loss_2rank.py", 2)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
    assert results(proc.stdout)["checked"] == ["2 2"]
