"""Batched generation on several ranks, without a GPU: what the ranks have to agree on."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from qmoe_b200.decoder import common_uniform, worst_of_ranks


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _uniform_worker(rank, world, port, result_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.manual_seed(100 + rank)                       # a seed per rank, as usual
        drawn = common_uniform(None, 3, 5, "cpu", world)
        mine = torch.full((3, 5), 0.25 * (rank + 1))
        given = common_uniform(mine, 3, 5, "cpu", world)
        # a group in which the first rank is not the process group's first
        sub = dist.new_group([1, 2])
        in_sub = common_uniform(None, 2, 2, "cpu", 2, sub) if rank in (1, 2) else torch.zeros(2, 2)
        torch.save((drawn, given, mine, in_sub), os.path.join(result_dir, f"r{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_ranks_sample_from_the_same_numbers(tmp_path):
    world = 3
    mp.spawn(_uniform_worker, args=(world, _free_port(), str(tmp_path)), nprocs=world, join=True)
    results = [torch.load(tmp_path / f"r{r}.pt") for r in range(world)]
    for r, (drawn, given, mine, in_sub) in enumerate(results):
        assert torch.equal(drawn, results[0][0]) and bool(((drawn >= 0) & (drawn < 1)).all())
        assert torch.equal(given, results[0][2])            # the first rank's
        assert bool((mine == 0.25 * (r + 1)).all())         # what the caller gave is left alone
        if r in (1, 2):
            assert torch.equal(in_sub, results[1][3])


def test_one_rank_needs_no_process_group():
    torch.manual_seed(7)
    want = torch.rand(2, 3)
    torch.manual_seed(7)
    assert torch.equal(common_uniform(None, 2, 3, "cpu"), want)
    for bad in (torch.rand(3, 2), torch.rand(2, 3, dtype=torch.float64)):
        with pytest.raises(ValueError):
            common_uniform(bad, 2, 3, "cpu")


def test_generate_batch_takes_the_common_numbers(monkeypatch):
    """The model hands its ranks and group on before anything is sampled."""
    from qmoe_b200 import decoder

    class Seen(Exception):
        pass

    def stop(uniform, n_new, n, device, world, group):
        raise Seen(uniform, n_new, n, world, group)

    monkeypatch.setattr(decoder, "common_uniform", stop)
    model = object.__new__(decoder.SwitchDecoderLM)
    model.dev, model.world, model.group = torch.device("cpu"), 4, "a group"
    with pytest.raises(Seen) as seen:
        model.generate_batch([torch.zeros(2, dtype=torch.int64)] * 3, 6, temperature=1.0)
    assert seen.value.args == (None, 6, 3, 4, "a group")


def _count_worker(rank, world, port, result_dir):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.save(worst_of_ranks([rank, 0, 5 - rank], "cpu", world), os.path.join(result_dir, f"r{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_every_rank_learns_of_a_failure_on_one(tmp_path):
    mp.spawn(_count_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)
    for r in range(2):
        assert torch.load(tmp_path / f"r{r}.pt") == [1, 0, 5]
    assert worst_of_ranks([3, 0], "cpu") == [3, 0]
