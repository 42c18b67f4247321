"""What the paged passes record on the device reaches the decoder's user."""
import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import ck, decoder, prompts, q2  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_a_page_outside_the_cache_is_raised(q2, ck, graph):  # noqa: F811
    import saccade_core as sc
    ps = prompts([9, 20], ck.cfg.vocab, 1)
    dec = decoder(q2, ck)
    c, m = dec.cache, dec.model
    want = dec.generate(ps, 5, graph=graph).tolist()
    keep = int(c.block_table[1, 0])
    c.block_table[1, 0] = c.num_pages
    with pytest.raises(sc.CTarqError, match="outside the paged cache"):
        dec.start(ps)
    with pytest.raises(RuntimeError, match="start"):
        dec.step()  # the prompts have not passed
    c.block_table[1, 0] = keep
    assert dec.start(ps).tolist() == [t[0] for t in want]
    c.block_table[1, 0] = -1
    dec.step()
    with pytest.raises(sc.CTarqError, match="outside the paged cache"):
        m.check_device()
    m.check_device()  # told once
    c.block_table[1, 0] = keep
    # in the middle of generate()
    inner, n = dec._reserve_next, []

    def later():
        n.append(1)
        if len(n) == 3:
            c.block_table[1, 0] = -1
        inner()
    dec._reserve_next = later
    with pytest.raises(sc.CTarqError, match="outside the paged cache"):
        dec.generate(ps, 6, graph=graph)
    dec._reserve_next = inner
    c.block_table[1, 0] = keep
    assert dec.generate(ps, 5, graph=graph).tolist() == want
    dec.finish()


def test_a_token_outside_the_vocabulary_is_raised_once(q2, ck):  # noqa: F811
    import saccade_core as sc
    dec = decoder(q2, ck)
    good = prompts([3, 4], ck.cfg.vocab, 1)
    want = dec.start(good).tolist()
    for bad in (ck.cfg.vocab, -1, 2 ** 40):
        with pytest.raises(sc.CTarqError, match="outside the vocabulary"):
            dec.start([good[0], torch.tensor([1, bad, 2])])
        assert dec.start(good).tolist() == want
    dec.finish()
