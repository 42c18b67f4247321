"""Fused routers on the paged path: the tokens of the unfused one, captured and eager, beside passes on another stream."""
import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import no_repeats, prompts, q2  # noqa: F401 - fixture

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [12, 40])
def test_paged_decoding_with_fused_routers(q2, batch):  # noqa: F811
    cfg = q2.Qwen2Config(hidden=256, intermediate=704, layers=3, heads=4, kv_heads=2, head_dim=64, vocab=4096)
    ck = q2.random_checkpoint(cfg, seed=3, fill=0.01)
    g = torch.Generator().manual_seed(3)
    q2.calibrate(ck, torch.randint(0, cfg.vocab, (batch, 12), generator=g).cuda(), max_pos=32)
    ps = prompts([3 + i * 7 % 11 for i in range(batch)], cfg.vocab, 8)
    want = None
    for fused in ("none", "norm", "all"):
        for graph in (True, False):
            cache = q2.Qwen2Model.paged_cache(ck, 3 * batch + 6, max_seqs=batch + 1, max_positions=48, page_size=16)
            m = q2.Qwen2Model(ck, max_pos=48, fused_route=fused, cache=cache)
            dec = q2.PagedDecoder(m, batch, no_repeats(batch))
            toks = dec.generate(ps, 8, graph=graph).tolist()
            m.check_device()
            used = {k[1] for k in m._bufs if k[0] == "route"}
            assert used == {"none": set(), "norm": {"qkv", "gateup"}, "all": {"qkv", "gateup", "down"}}[fused]
            want = want or toks
            assert toks == want
            # as many tokens of another sequence on a stream of their own, while the decoder steps
            cache.reserve(batch, batch)
            ids = torch.arange(batch, device="cuda")
            i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
            args = (ids, cache.block_table[batch:batch + 1], i32(0, batch), i32(batch), ids[-1:].clone(), batch, batch)
            alone = m.forward_paged(*args).clone()
            got, side = [dec.start(ps).tolist()], torch.cuda.Stream()
            torch.cuda.synchronize()
            for _ in range(7):
                dec.step()
                with torch.cuda.stream(side):
                    beside = m.forward_paged(*args)
                got.append(dec.ids.tolist())
                torch.cuda.synchronize()
                assert torch.equal(beside, alone)
            assert [list(t) for t in zip(*got)] == want
            dec.finish()
