"""The passes that PagedDecoder.start() cuts its prompts into."""
import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import ck, decoder, prompts, q2  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk,max_tokens", [(2048, 50), (2048, 1), (16, 40), (7, 7), (30, 1 << 40)])
def test_passes_hold_at_most_max_tokens(q2, ck, chunk, max_tokens):  # noqa: F811
    """Prompts in passes of every size: all of their tokens once and in order, none above the bounds, and the cache
    that one pass leaves (an f32 cache: to f32 rounding, of keys of size 1)."""
    lens, vocab = [5, 40, 17, 1], ck.cfg.vocab
    ps = prompts(lens, vocab, 2)

    def run(**kw):
        cache = q2.Qwen2Model.paged_cache(ck, 40, max_seqs=4, max_positions=160, page_size=16, dtype=torch.float32)
        m = q2.Qwen2Model(ck, max_pos=160, mode="exact", cache=cache)
        sizes, seen = [], [[] for _ in lens]
        inner = m.forward_paged

        def counted(ids, table, cu, kv, last, max_q, max_kv):
            sizes.append((ids.numel(), max_q))
            rows = [cache.block_table[:, 0].tolist().index(p) for p in table[:, 0].tolist()]
            for b, i, j, end in zip(rows, cu.tolist(), cu.tolist()[1:], kv.tolist()):
                seen[b] += ids[i:j].tolist()
                assert len(seen[b]) == end
            return inner(ids, table, cu, kv, last, max_q, max_kv)
        m.forward_paged = counted
        dec = q2.PagedDecoder(m, 4)
        first = dec.start(ps, **kw)
        assert seen == [p.tolist() for p in ps]
        assert dec.kv_len.tolist() == lens and dec.hist_len.tolist() == [n + 1 for n in lens]
        assert [int(dec.history[b, n]) for b, n in enumerate(lens)] == first.tolist()
        keys = [torch.cat([cache.k[-1][p] for p in cache.pages(b)], 1)[:, :n].clone() for b, n in enumerate(lens)]
        dec.finish()
        return sizes, keys

    _, whole = run()
    sizes, keys = run(chunk=chunk, max_tokens=max_tokens)
    assert all(t <= max_tokens and q <= chunk for t, q in sizes)
    # the last layer's keys of nothing-routed exact linears: f16 inputs that f32 rounding may move by a step (2^-10)
    for a, b in zip(whole, keys):
        assert (a - b).abs().max() <= 2.0 ** -10 * 8 * a.abs().max()


def test_bounds_below_one_are_refused(q2, ck):  # noqa: F811
    dec = decoder(q2, ck)
    for kw in (dict(chunk=0), dict(max_tokens=0), dict(max_tokens=-3)):
        with pytest.raises(ValueError):
            dec.start(prompts([3, 4], 100, 1), **kw)
