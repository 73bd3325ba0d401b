"""CPU, two gloo ranks: when a gradient bucket is summed over the ranks, for parameters whose gradient the nodes in front add to the buffer themselves
(autograd gets None and calls the parameter's hook all the same), for ordinary ones and for a mix, with the additions in the backward pass or queued
behind it."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


class AddsItself(torch.autograd.Function):
    """y = x w, its weight gradient added to the static buffer: at once, or by whoever empties ``queue``"""

    @staticmethod
    def forward(ctx, x, w, queue):
        from bmt_amd import ops
        ops.note_use(w)
        ctx.save_for_backward(x)
        ctx.w, ctx.queue = w, queue
        return x * w

    @staticmethod
    def backward(ctx, d):
        (x,), w = ctx.saved_tensors, ctx.w

        @torch.no_grad()
        def add():
            w.grad.add_(d * x)
            w._bmt_uses -= 1
            if w._bmt_uses <= 0:
                w._bmt_on_grad(w)
        if ctx.queue is None:
            add()
        else:
            ctx.queue.append(add)
        return d * w, None, None


def _worker(rank, world, port, queued, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from bmt_amd.parallel import GradientReducer
    params = [torch.nn.Parameter(torch.full((50,), 1.0 + i)) for i in range(4)]
    reducer = GradientReducer(params, bucket_bytes=2 * 50 * 4)
    assert len(reducer.buckets) == 2
    got = []
    for it in range(2):
        reducer.zero_grad()
        x = torch.arange(50.0) + 100 * rank + it
        queue = [] if queued else None
        y = x
        for p in params[:3]:
            y = AddsItself.apply(y, p, queue)
        y = y * params[3] + AddsItself.apply(x, params[0], queue) + params[1].square()      # (an ordinary use, a second one, and both of one parameter)
        y.sum().backward()
        for add in queue or ():
            add()
        reducer.finish()
        got.append([p.grad.clone() for p in params])
        x = x.requires_grad_(True)
        y = x
        for p in params[:3]:
            y = y * p
        y = y * params[3] + x * params[0] + params[1].square()
        want = torch.autograd.grad(y.sum(), params)
        for g, w in zip(got[-1], want):
            total = w.clone()
            dist.all_reduce(total)
            assert torch.allclose(g, total, rtol=1e-5), (rank, it)
    if rank == 0:
        torch.save(True, out)
    dist.destroy_process_group()


@pytest.mark.parametrize("queued", [False, True])
def test_two_ranks_sum_every_bucket_once_and_complete(tmp_path, queued):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "ok.pt")
    mp.spawn(_worker, args=(2, port, queued, out), nprocs=2, join=True)
    assert torch.load(out, weights_only=True)
