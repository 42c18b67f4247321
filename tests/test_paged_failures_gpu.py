"""Steps and captures that fail on the host."""
import pytest

torch = pytest.importorskip("torch")

from test_paged_streams_gpu import ck, decoder, prompts, q2  # noqa: F401 - fixtures

pytestmark = pytest.mark.gpu


class Failed(Exception):
    pass


def failing_rules(dec, at):
    """The rules raise at their `at`-th use from now on."""
    inner, left = dec.rules.apply, [at]

    def apply(*a, **kw):
        left[0] -= 1
        if left[0] == 0:
            raise Failed
        return inner(*a, **kw)
    dec.rules.apply = apply


def test_a_failed_step_ends_the_run(q2, ck):  # noqa: F811
    """Its sequences have moved on by a position that holds no token: they are not stepped again."""
    ps = prompts([9, 20], ck.cfg.vocab, 1)
    dec = decoder(q2, ck)
    want = dec.generate(ps, 6, graph=False).tolist()
    dec.start(ps)
    dec.step()
    failing_rules(dec, 2)
    dec.step()
    with pytest.raises(Failed):
        dec.step()
    with pytest.raises(RuntimeError, match="start"):
        dec.step()
    assert dec.generate(ps, 6, graph=False).tolist() == want
    dec.finish()
    assert dec.cache.free_pages == 40


def test_a_failed_capture_leaves_eager_steps(q2, ck):  # noqa: F811
    ps = prompts([9, 20], ck.cfg.vocab, 1)
    dec = decoder(q2, ck)
    want = dec.generate(ps, 6, graph=False).tolist()
    got = [dec.start(ps)]
    failing_rules(dec, 2)  # the eager step passes, the recorded one fails
    with pytest.raises(Failed):
        dec.capture()
    assert dec.graph is None
    got.append(dec.ids.clone())
    for _ in range(2):
        got.append(dec.step().clone())
    dec.capture()
    got += [dec.ids.clone(), dec.step().clone()]
    assert torch.stack(got, 1).tolist() == want
    dec.finish()
