"""PagedDecoder's stream and the caller's: each step sees what the caller's stream has written before it, and the caller's
stream sees what the step has written."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BUSY = 40_000_000  # cycles: about 20 ms


@pytest.fixture(scope="module")
def q2():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import saccade_core
    from saccade_core import qwen2
    saccade_core.set_bypass_c_tarq(False)
    return qwen2


@pytest.fixture(scope="module")
def ck(q2):
    cfg = q2.Qwen2Config(hidden=256, intermediate=704, layers=3, heads=4, kv_heads=2, head_dim=64, vocab=4096)
    return q2.random_checkpoint(cfg, seed=5, fill=0.01)


def prompts(lens, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lens]


def decoder(q2, ck, rules=None, batch=2):
    cache = q2.Qwen2Model.paged_cache(ck, 40, max_seqs=4, max_positions=160, page_size=16)
    return q2.PagedDecoder(q2.Qwen2Model(ck, max_pos=160, mode="exact", cache=cache), batch, rules)


def no_repeats(n):
    """Every token once: a stale one shows."""
    import saccade_core as sc
    return sc.LogitRules(n, "cuda", presence=1000.0)


def only(token, vocab):
    """A mask row that allows one token."""
    m = torch.zeros(vocab // 32, dtype=torch.int64)
    m[token // 32] = 1 << (token % 32)
    return torch.where(m >= 2 ** 31, m - 2 ** 32, m).to(torch.int32)


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_a_step_sees_the_rules_written_before_it(q2, ck, graph):
    """The mask's next content arrives late on the caller's stream; the step waits for it."""
    import saccade_core as sc
    vocab = ck.cfg.vocab
    mask = torch.full((2, vocab // 32), -1, dtype=torch.int32, device="cuda")
    rules = sc.LogitRules(2, "cuda", mask=mask)
    dec = decoder(q2, ck, rules)
    dec.start(prompts([9, 20], vocab, 1))
    if graph:
        dec.capture()
    for token in (77, 4095, 31, 1200):
        new = only(token, vocab).cuda()
        torch.cuda.synchronize()
        torch.cuda._sleep(BUSY)
        rules.mask.copy_(new.expand(2, -1))
        dec.step()
        torch.cuda.synchronize()
        assert dec.ids.tolist() == [token, token]
    dec.finish()


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_what_is_written_behind_a_step_does_not_reach_it(q2, ck, graph):
    """The rules of the next step, written while this one is in its layers."""
    import saccade_core as sc
    vocab = ck.cfg.vocab
    rules = sc.LogitRules(2, "cuda", mask=torch.full((2, vocab // 32), -1, dtype=torch.int32, device="cuda"))
    dec = decoder(q2, ck, rules)
    dec.start(prompts([9, 20], vocab, 1))
    if graph:
        dec.capture()
    a, b = only(50, vocab).cuda().expand(2, -1), only(60, vocab).cuda().expand(2, -1)
    rules.mask.copy_(a)
    torch.cuda.synchronize()
    with torch.cuda.stream(dec.stream):
        torch.cuda._sleep(BUSY)  # the step begins late
    dec.step()
    rules.mask.copy_(b)
    torch.cuda.synchronize()
    assert dec.ids.tolist() == [50, 50]
    dec.step()
    torch.cuda.synchronize()
    assert dec.ids.tolist() == [60, 60]
    dec.finish()


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_the_callers_stream_reads_the_step_it_has_made(q2, ck, graph):
    """Tokens copied and read with no synchronisation but the read's own, on the default stream and on another."""
    ps = prompts([9, 20], ck.cfg.vocab, 1)
    dec = decoder(q2, ck, no_repeats(2))
    want = dec.generate(ps, 9, graph=False)
    torch.cuda.synchronize()
    dec.finish()
    dec = decoder(q2, ck, no_repeats(2))
    got = [dec.start(ps)]
    if graph:
        dec.capture()
        got.append(dec.ids.clone())
    side = torch.cuda.Stream()
    while len(got) < 9:
        with torch.cuda.stream(dec.stream):
            torch.cuda._sleep(BUSY)
        if len(got) % 2:
            got.append(dec.step().clone())
        else:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(dec.step().clone())
            torch.cuda.current_stream().wait_stream(side)
    got = torch.stack(got, 1).tolist()
    assert got == want.tolist()
    dec.finish()


def test_generate_keeps_each_steps_tokens(q2, ck):
    """generate() with a busy caller's stream gives what an idle one gives."""
    ps = prompts([30, 3], ck.cfg.vocab, 2)
    dec = decoder(q2, ck, no_repeats(2))
    want = dec.generate(ps, 12)
    torch.cuda.synchronize()
    want = want.tolist()
    assert all(len(set(row)) == 12 for row in want)
    dec.finish()
    for graph in (True, False):
        dec = decoder(q2, ck, no_repeats(2))
        torch.cuda._sleep(BUSY)
        assert dec.generate(ps, 12, graph=graph).tolist() == want
        dec.finish()


def test_ragged_passes_keep_no_memory(q2, ck):
    """Passes of many different token counts, and decoders that come and go: what is allocated stays the same."""
    dec = decoder(q2, ck, batch=4)
    m, c = dec.model, dec.cache
    for b in range(4):
        c.reserve(b, 160)
    kv = lambda t: torch.tensor([t], dtype=torch.int32, device="cuda")  # noqa: E731

    def one(t):
        ids = torch.zeros(t, dtype=torch.int64, device="cuda")
        m.forward_paged(ids, c.block_table[:1], torch.tensor([0, t], dtype=torch.int32, device="cuda"), kv(t),
                        torch.tensor([t - 1], device="cuda"), t, t)

    for t in (160, 1, 8, 9, 64, 65):
        one(t)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for t in range(1, 161):
        one(t)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    for b in range(4):
        c.release(b)
    dec.generate(prompts([150, 150, 150, 150], ck.cfg.vocab, 1), 2)
    dec.finish()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for i in range(12):
        dec.generate(prompts([3 + 11 * i, 140 - 7 * i, 1 + i, 77], ck.cfg.vocab, i), 3)
        dec.finish()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() <= before + 4 * 4 * ck.cfg.vocab * 4  # a step's logits, before and after the rules


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_a_pass_on_another_stream_beside_the_decoder(q2, ck, graph):
    """The model runs another sequence, of as many new tokens as the decoder's batch, on a stream that nothing orders
    with the decoder's steps: both give what they give alone."""
    ps = prompts([9, 20], ck.cfg.vocab, 1)
    dec = decoder(q2, ck, no_repeats(2))
    m, c = dec.model, dec.cache
    want = dec.generate(ps, 25, graph=graph).tolist()
    c.reserve(3, 2)
    ids = torch.tensor([5, 6], device="cuda")
    args = (ids, c.block_table[3:4], torch.tensor([0, 2], dtype=torch.int32, device="cuda"),
            torch.tensor([2], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], device="cuda"), 2, 2)
    alone = m.forward_paged(*args).clone()
    side, beside = torch.cuda.Stream(), []
    got = [dec.start(ps).tolist()]
    torch.cuda.synchronize()
    for _ in range(24):
        dec.step()
        with torch.cuda.stream(side):
            beside += [m.forward_paged(*args) for _ in range(2)]
        got.append(dec.ids.tolist())
    torch.cuda.synchronize()
    assert [list(t) for t in zip(*got)] == want
    assert all(torch.equal(x, alone) for x in beside)
    dec.finish()
