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


def test_arguments_that_are_no_truth_values_or_numbers():
    import saccade_core as sc
    from paged_cases import Paged
    c = Paged([(1, 20)], 4, 2, 64, 16, torch.float16, "cuda")
    call = lambda **kw: sc.paged_attention(  # noqa: E731
        *({"q": c.q, "k": c.k_pages, "v": c.v_pages, "t": c.table, "cu": c.cu_q, "kv": c.kv_len, "mq": 1, "mk": 20} | {
            k: v for k, v in kw.items() if k in ("mq", "mk")}).values(), **{k: v for k, v in kw.items() if k not in ("mq", "mk")})
    pair = torch.tensor([True, False])
    with pytest.raises(ValueError, match="return_lse"):
        call(return_lse=pair)
    with pytest.raises(ValueError, match="return_best"):
        sc.process_logits(torch.zeros(1, 8, device="cuda"), return_best=pair)
    for kw in (dict(mq=1.5), dict(mk=None), dict(mq="1"), dict(mk=1 << 64), dict(scale="1"), dict(scale=pair)):
        with pytest.raises(ValueError):
            call(**kw)
    out, lse = call(return_lse=1)
    assert torch.equal(call(), out) and lse.shape == (1, 4)
    torch.cuda.synchronize()
