import gc

import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import ck, decoder, prompts, q2  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu


def test_a_dropped_decoder_leaves_nothing_behind(q2, ck):  # noqa: F811
    """A wide decoder dropped in the middle of its run, a narrow one after it: all pages come back."""
    ps = prompts([20, 7, 60, 33], ck.cfg.vocab, 6)
    dec = decoder(q2, ck, batch=4)
    m, c = dec.model, dec.cache
    alone = dec.generate(ps, 4).tolist()
    dec.step()
    assert c.free_pages < 40
    del dec
    gc.collect()
    narrow = q2.PagedDecoder(m, 1)
    assert narrow.generate(ps[:1], 4).tolist() == [alone[0]]  # exact linears: a row does not depend on the others
    assert c.free_pages == 40 - len(c.pages(0)) and c.pages(1) == []
    narrow.finish()
    assert c.free_pages == 40
