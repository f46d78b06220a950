"""Vocabulary shards through the public calls: `group` in the loss and in its gradients."""
import socket
import threading

import pytest
import torch
import torch.distributed as dist

import megatron_dion_amd as mda
from megatron_dion_amd import lm_ops
from tests import _lm_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


class _Ranks:
    """Threads of one process as the ranks of a group: each reduction meets at a barrier."""

    def __init__(self, world):
        self.world, self.slots, self.rank = world, [None] * world, threading.local()
        self.barrier = threading.Barrier(world, timeout=60)

    def all_reduce(self, t, op=None, group=None):
        assert group is self
        self.slots[self.rank.value] = t
        self.barrier.wait()
        all_ = torch.stack(list(self.slots))
        out = all_.amax(0) if op == dist.ReduceOp.MAX else all_.sum(0)
        self.barrier.wait()
        t.copy_(out)
        self.barrier.wait()

    def run(self, fn):
        results, errors = [None] * self.world, []

        def work(rank):
            self.rank.value = rank
            try:
                results[rank] = fn(rank)
            except Exception as e:  # noqa: BLE001
                errors.append(e)
                self.barrier.abort()

        threads = [threading.Thread(target=work, args=(r,)) for r in range(self.world)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        if errors:
            raise next((e for e in errors if not isinstance(e, threading.BrokenBarrierError)), errors[0])
        return results


def _case(tokens, hidden, vocab, dtype):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    w = (torch.randn(vocab, hidden, generator=g) * 2 * hidden ** -0.5).to(dtype)
    t = torch.randint(0, vocab, (tokens,), generator=g)
    t[::9] = -100
    return x, w, t, torch.rand(tokens, generator=g) / tokens


# 500 words in shards of 128: the last has 116 and padding; of 200, 100 and 150 words the last ranks have none
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("words,world,rows", [(500, 4, 128), (200, 4, 128), (100, 2, 128), (150, 3, 75)])
def test_shards_as_ranks(monkeypatch, dtype, out_dtype, words, world, rows):
    x, w, t, gl = _case(70, 64, words, dtype)
    padded = torch.full((world * rows, 64), float("nan"), dtype=dtype)
    padded[:words] = w
    ref = R.xent(x, w, t, -100, gl, out_dtype=out_dtype)
    ranks = _Ranks(world)
    monkeypatch.setattr(lm_ops.dist, "all_reduce", ranks.all_reduce)

    def rank(r):
        kw = dict(vocab_start=r * rows, vocab_size=words, group=ranks)
        mine = padded[r * rows:(r + 1) * rows].cuda()
        loss, lse = mda.linear_cross_entropy_forward(x.cuda(), mine, t.cuda(), **kw)
        gw = torch.full((rows, 64), float("nan"), dtype=out_dtype, device="cuda")
        gh, gw = mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), mine, t.cuda(), lse, grad_weight=gw, **kw)
        main = torch.ones(rows, 64, dtype=out_dtype, device="cuda")
        mda.linear_cross_entropy_backward(gl.cuda(), x.cuda(), mine, t.cuda(), lse, grad_weight=main, accumulate=True,
                                          need_hidden=False, **kw)
        torch.cuda.synchronize()
        return loss.cpu(), lse.cpu(), gh.cpu(), gw.cpu(), main.cpu()

    out = ranks.run(rank)
    for r, (loss, lse, gh, gw, main) in enumerate(out):
        # the shards' joining: an exponential, a sum and a logarithm in fp32
        assert bool(((loss.double() - ref["loss"]).abs() <= ref["e_loss"] + 16 * R.U32 * (1 + ref["lse"].abs())).all())
        assert torch.equal(loss, out[0][0]) and torch.equal(lse, out[0][1]) and torch.equal(gh, out[0][2])
        # each share is rounded once, and so is each sum over the ranks
        tol = 1.01 * ref["e_grad_hidden"] + 2 * world * R.half_step(dtype) * ref["grad_hidden"].abs().amax()
        assert bool(((gh.double() - ref["grad_hidden"]).abs() <= tol).all())
        n = max(0, min(rows, words - r * rows))
        part = slice(r * rows, r * rows + n)
        assert bool(((gw[:n].double() - ref["grad_weight"][part]).abs() <= 1.01 * ref["e_grad_weight"][part]).all())
        assert (gw[n:] == 0).all() and (main[n:] == 1).all()


def test_a_group_of_one_rank():
    """The collectives themselves."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    try:
        x, w, t, gl = _case(70, 64, 500, BF16)
        t[5] = 500  # no word
        a = (x.cuda(), w.cuda(), t.cuda())
        kw = dict(vocab_size=500, group=dist.group.WORLD)
        loss, lse = mda.linear_cross_entropy_forward(*a)
        loss1, lse1 = mda.linear_cross_entropy_forward(*a, **kw)
        assert torch.equal(loss.isnan(), loss1.isnan()) and torch.equal(loss.nan_to_num(), loss1.nan_to_num())
        assert torch.equal(lse, lse1)
        for u, v in zip(mda.linear_cross_entropy_backward(gl.cuda(), *a, lse),
                        mda.linear_cross_entropy_backward(gl.cuda(), *a, lse1, **kw)):
            assert torch.equal(u.nan_to_num(), v.nan_to_num())
        xg, wg = a[0].clone().requires_grad_(), a[1].clone().requires_grad_()
        t[5] = 0
        a = (x.cuda(), w.cuda(), t.cuda())
        (mda.linear_cross_entropy(xg, wg, a[2], **kw) * gl.cuda()).sum().backward()
        _, lse = mda.linear_cross_entropy_forward(*a)
        gh, gw = mda.linear_cross_entropy_backward(gl.cuda(), *a, lse)
        assert torch.equal(xg.grad, gh) and torch.equal(wg.grad, gw)
        # rows that hold no word of the vocabulary
        _, lse0 = mda.linear_cross_entropy_forward(*a, vocab_start=500, vocab_size=500, group=dist.group.WORLD)
        assert (lse0[t.cuda() != -100] == float("-inf")).all() and (lse0[t.cuda() == -100] == 0).all()
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("kw", [dict(vocab_start=100, vocab_size=100), dict(vocab_start=128, vocab_size=100),
                                dict(vocab_start=50), dict(vocab_size=101), dict(vocab_start=20, vocab_size=120)])
def test_a_part_of_the_vocabulary_needs_a_group(kw):
    """Its loss would lack the other words, and the logits of targets among them."""
    x, w, t, _ = _case(20, 64, 100, BF16)
    with pytest.raises(RuntimeError, match="DION_BAD_VOCAB"):
        mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda(), **kw)
    with pytest.raises(RuntimeError, match="DION_BAD_VOCAB"):
        mda.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), **kw)
    mda.linear_cross_entropy_forward(x.cuda(), w.cuda(), t.cuda(), vocab_size=90)  # 10 rows of padding
