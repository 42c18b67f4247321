"""What PagedDecoder refuses at its construction."""
import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import ck, decoder, q2  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu


def test_rules_that_do_not_fit_the_decoder(q2, ck):  # noqa: F811
    import saccade_core as sc
    m = decoder(q2, ck).model
    words = ck.cfg.vocab // 32
    ok = sc.LogitRules(2, "cuda", repetition=1.1, mask=torch.full((2, words), -1, dtype=torch.int32))
    q2.PagedDecoder(m, 2, ok)
    short = sc.LogitRules(2, "cuda", mask=torch.full((2, words - 1), -1, dtype=torch.int32))
    for batch, rules in ((3, ok), (1, ok), (2, short), (2, sc.LogitRules(2, "cpu", presence=0.5))):
        with pytest.raises(ValueError):
            q2.PagedDecoder(m, batch, rules)
