"""The token that tensor-parallel ranks choose together, on gloo ranks: each has its slice of the vocabulary, the largest
logit of it and that one's id."""
import os
import socket
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
import torch.distributed as dist  # noqa: E402
import torch.multiprocessing as mp  # noqa: E402

VOCAB = 151936


def cases():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, VOCAB, generator=g)
    x[1] = 0.0                                   # all equal: token 0
    x[2] = -float("inf")                         # everything masked: token 0
    x[3, [5, 80000, 151935]] = 50.0              # the first of equals over the ranks
    x[4, 151935] = 90.0                          # the last token
    x[5] = -float("inf")
    x[5, 75968] = -3.0                           # one allowed
    x[6, [140000, 9]] = torch.tensor([float("nan"), float("inf")])  # NaN above all, as argmax has it
    x[7, 100000] = float("inf")
    x[8, 33333] = 1e30
    return x


def _rank(rank, world, port, q):
    from saccade_core import qwen2 as q2
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        cfg = q2.Qwen2Config(64, 128, 1, 1, 1, 64, VOCAB)
        v0, v1 = q2.vocab_split(cfg, rank, world)
        x = cases()
        n = x.shape[0]
        val, idx = x[:, v0:v1].max(-1)
        m = SimpleNamespace(group=None, world=world)
        cand, gath = torch.zeros(n, 2), torch.zeros(world, n, 2)
        out = torch.full((n,), -1, dtype=torch.int64)
        assert q2.best_of_ranks(m, val, idx + v0, out, cand, gath) is out
        best = idx + v0                          # as the paged decoder calls it: the ids are the output
        q2.best_of_ranks(m, val, best, best, cand, gath)
        some = (idx + v0)[:4].clone()            # fewer rows than the buffers
        q2.best_of_ranks(m, val[:4], some, some, cand[:4], gath[:, :4].contiguous())
        q.put((rank, out.tolist(), best.tolist(), some.tolist()))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_choose_as_one_argmax(world):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.SimpleQueue()
    procs = [ctx.Process(target=_rank, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(120)
        assert p.exitcode == 0
    want = cases().argmax(-1).tolist()
    assert want[1:3] == [0, 0] and want[6] == 140000
    for _ in range(world):
        rank, out, best, some = q.get()
        assert out == want and best == want and some == want[:4], rank


@pytest.mark.parametrize("world,heads", [(1, (28, 4)), (2, (28, 4)), (4, (28, 4)), (8, (28, 4)), (2, (14, 2)), (8, (64, 8))])
def test_a_ranks_paged_cache_holds_its_kv_heads(world, heads):
    from saccade_core import qwen2 as q2
    cfg = q2.Qwen2Config(64, 1024, 2, *heads, 64, 512)
    ck = SimpleNamespace(cfg=cfg, blocks=[{}, {}], embed=torch.zeros(1))
    for rank in range(world):
        q0, q1, k0, k1 = q2.head_split(cfg, rank, world)
        c = q2.Qwen2Model.paged_cache(ck, 3, max_seqs=2, max_positions=48, page_size=16, tp=(rank, world, None))
        assert len(c.k) == 2 and c.k[0].shape == (3, k1 - k0, 16, 64)
        # the rank's query heads are a multiple of its KV heads, which the attention asks for
        assert (q1 - q0) % (k1 - k0) == 0 and (q1 - q0) // (k1 - k0) <= 64
