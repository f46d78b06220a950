"""CPU tests of joining vocabulary shards, over gloo."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from megatron_dion_amd import lm_ops


def _ranks(rank, world, port, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    g = torch.Generator().manual_seed(0)
    z = torch.randn(9, 40, generator=g) * 5
    t = torch.randint(0, 40, (9,), generator=g)
    ignored = torch.zeros(9, dtype=torch.bool)
    ignored[2] = True
    if rank == 0:
        lse = torch.where(ignored, torch.zeros(9), torch.logsumexp(z, 1))
        tl = torch.where(ignored, torch.zeros(9), z.gather(1, t[:, None])[:, 0])
    else:  # all padding
        lse, tl = torch.full((9,), float("-inf")), torch.zeros(9)
    loss, whole = lm_ops.combine_vocab_shards(lse, tl, ignored, dist.group.WORLD)
    ref = torch.nn.functional.cross_entropy(z.double(), torch.where(ignored, -100, t), reduction="none")
    # logits of up to 20, whose fp32 logarithm and sums are off by a few 20 * 2^-24
    ret[rank] = torch.allclose(loss.double(), ref, atol=2e-5, rtol=0) and bool((loss[2] == 0) & (whole[2] == 0))
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_without_a_word_join_over_gloo(world):
    with mp.Manager() as m:
        ret = m.dict()
        mp.spawn(_ranks, args=(world, 29641 + world, ret), nprocs=world, join=True)
        assert all(ret[r] for r in range(world))
