"""The head's cross entropy on two gloo ranks whose shards of a volume are uneven, and empty."""
import faulthandler
import os
import sys
from pathlib import Path

import torch
import torch.distributed as dist

ROOT = Path(__file__).resolve().parents[3]
sys.path.insert(0, str(ROOT))

from scaffold_b200.ops.head_loss import head_cross_entropy  # noqa: E402


class Shards:
    size, lead_swap = 2, None

    @staticmethod
    def all_reduce_sum(t):
        dist.all_reduce(t)
        return t


def main():
    faulthandler.dump_traceback_later(int(os.environ.get("SCAFFOLD_TEST_FAULT_TIMEOUT", "200")), exit=True)
    dist.init_process_group("gloo")
    rank = dist.get_rank()
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(50, 16, generator=g), torch.randn(34, 16, generator=g), torch.randn(34, generator=g)
    y, cw = torch.randint(0, 34, (50,), generator=g), torch.rand(34, generator=g) + 0.5
    whole = [t.clone().requires_grad_() for t in (x, w, b)]
    want = head_cross_entropy(*whole, y, cw)
    want_grads = torch.autograd.grad(want, whole)
    checked = 0
    for cut in (17, 0):  # voxels of rank 0
        mine = slice(0, cut) if rank == 0 else slice(cut, None)
        leaves = [x[mine].clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
        loss = head_cross_entropy(*leaves, y[mine], cw, spatial=Shards)
        grads = torch.autograd.grad(loss, leaves)
        for t in grads[1:]:
            dist.all_reduce(t)
        torch.testing.assert_close(loss, want, rtol=1e-6, atol=0)
        torch.testing.assert_close(grads[0], want_grads[0][mine], rtol=1e-5, atol=1e-8)
        torch.testing.assert_close(grads[1:], want_grads[1:], rtol=1e-5, atol=1e-7)
        checked += 1
    n = torch.tensor([checked])
    dist.all_reduce(n, op=dist.ReduceOp.MIN)
    if rank == 0:
        print(f"RESULT checked {int(n)} {checked}", flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
