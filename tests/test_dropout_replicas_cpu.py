"""Dropout masks that have to be independent of each other: of two modules and of the replicas of a model."""
import datetime
import os
import socket
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import residual_oracle as ro
from spiky_b200 import residual

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_modules_have_seeds_of_their_own():
    torch.manual_seed(5)
    one, two = residual.CounterDropout(0.5), residual.CounterDropout(0.5)
    torch.manual_seed(5)
    again = residual.CounterDropout(0.5)
    assert one.state[0] != two.state[0] and torch.equal(one.state, again.state)
    assert residual.CounterDropout(0.5, 9).state.tolist() == [9, 0] and residual.CounterDropout(0.5, seed=0).state.tolist() == [0, 0]
    with torch.device("meta"):
        assert residual.CounterDropout(0.5).state.is_meta


def test_replica_sites():
    assert [residual.replica_site(r) for r in (None, 0, 1, 2 ** 15 - 1)] == [0, 0, 2 ** 48, 2 ** 63 - 2 ** 48]
    for bad in (-1, 2 ** 15):
        with pytest.raises(ValueError):
            residual.replica_site(bad)
        with pytest.raises(ValueError):
            residual.CounterDropout(0.5, replica=bad)


def _on_the_host(x, p, state, site=0):
    """counter_dropout's definition, for tensors of the host."""
    kept = ro.keeps(p, int(state[0]), int(state[1]) + site, x.numel()).view(x.shape)
    return torch.where(kept, x * ro.drop_scale(p), torch.zeros((), dtype=x.dtype))


def _worker(rank, world, port, out):
    for d in (ROOT, os.path.join(ROOT, "tests")):
        sys.path.insert(0, d)
    from spiky_b200.data_parallel import broadcast_structure

    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    try:
        residual.counter_dropout = _on_the_host

        def take(state, count):
            used = state.clone()
            state[1] += count
            return used

        residual.take_dropout_state = take
        x, got = torch.ones(4, 64), []
        for given in (None, 5):   # the rank, and one number for all
            drop = residual.CounterDropout(0.5, seed=100 + rank, replica=given)
            broadcast_structure(drop)
            ddp = torch.nn.parallel.DistributedDataParallel(torch.nn.Sequential(torch.nn.Linear(64, 64), drop), broadcast_buffers=True)
            with torch.no_grad():
                ddp.module[0].weight.copy_(torch.eye(64))
                ddp.module[0].bias.zero_()
            got += [ddp(x).detach() for _ in range(2)]
            assert drop.state.tolist() == [100, 2]
        torch.save(got, os.path.join(out, f"{rank}.pt"))
        dist.barrier()
    finally:
        dist.destroy_process_group()


def test_replicas_keep_their_masks_after_a_broadcast(tmp_path):
    """Two ranks whose buffers were made alike, by broadcast_structure and by DistributedDataParallel at every pass."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    one, two = (torch.load(tmp_path / f"{r}.pt") for r in range(2))
    for rank, got in ((0, one), (1, two)):
        for k in range(2):
            assert torch.equal(got[k], _on_the_host(torch.ones(4, 64), 0.5, residual.dropout_state(100, "cpu", k), rank << 48))
            assert torch.equal(got[2 + k], _on_the_host(torch.ones(4, 64), 0.5, residual.dropout_state(100, "cpu", k), 5 << 48))
    assert not any(torch.equal(one[k], two[j]) for k in range(2) for j in range(2))
