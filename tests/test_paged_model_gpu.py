"""The serving operators together: a small Qwen2 model on a paged cache, decoding ragged prompts with
penalties, biases and grammar masks."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


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
    # nothing routed (thresholds at infinity): the logits are a smooth function of the attention's outputs
    cfg = q2.Qwen2Config(hidden=256, intermediate=704, layers=3, heads=4, kv_heads=2, head_dim=64, vocab=4096)
    return q2.random_checkpoint(cfg, seed=5, fill=0.01)


def prompts(lens, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g) for n in lens]


def paged(q2, ck, dtype, slots=4, pages=40, positions=160, page=16):
    cache = q2.Qwen2Model.paged_cache(ck, pages, max_seqs=slots, max_positions=positions, page_size=page, dtype=dtype)
    return q2.Qwen2Model(ck, max_pos=positions, mode="exact", cache=cache)


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 0.02), (torch.float16, 0.03), (torch.bfloat16, 0.15)],
                         ids=["f32", "f16", "bf16"])
def test_prefill_logits_are_the_contiguous_models(q2, ck, dtype, bound):
    """The attention output of every head goes to the linears as 16 bits in both models.  An f32 cache differs
    in f32 rounding only, which now and then moves an output by one step of f16 (2^-10 of it); an f16 cache
    rounds q, k, v and the output by 2^-11 each, a bf16 cache by 2^-8.  Three layers of residual adds carry
    each to the logits with a factor of a few: 3 x 4 x 2^-10 = 0.012, 3 x 3 x 4 x 2^-11 = 0.018 and 0.14 of
    the logits' root mean square."""
    lens = [1, 37, 90]
    ps = prompts(lens, ck.cfg.vocab, 1)
    ref = q2.Qwen2Model(ck, max_batch=1, max_pos=160, mode="exact")
    model = paged(q2, ck, dtype)
    for b, n in enumerate(lens):
        model.cache.reserve(b, n)
    ids = torch.cat(ps).cuda()
    cu = torch.tensor([0, 1, 38, 128], dtype=torch.int32, device="cuda")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = model.forward_paged(ids, model.cache.block_table[:3], cu, kv, torch.tensor([0, 37, 127], device="cuda"), 90, 90)
    model.check_device(), model.cache.check_device()
    for b, p in enumerate(ps):
        i, s, pos = q2.prefill_indices(p[None].cuda())
        want = ref.forward_tokens(i, s, pos, torch.tensor([p.numel() - 1], device="cuda"), p.numel() - 1)[0]
        rms = want.square().mean().sqrt()
        assert float((got[b] - want).abs().max() / rms) <= bound * 4  # the largest of 4096: 4 sigma


@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
@pytest.mark.parametrize("chunk", [2048, 16])
def test_decoding_follows_the_rules(q2, ck, graph, chunk):
    """Every step's token is the best of its own raw logits under the rules, computed plainly from the tokens so
    far; the cache grows page by page and gives everything back."""
    import saccade_core as sc
    lens, steps, vocab = [5, 40, 17], 30, ck.cfg.vocab
    ps = prompts(lens, vocab, 2)
    model = paged(q2, ck, torch.float16)
    words = vocab // 32
    mask = torch.zeros(1, words, dtype=torch.int32)
    allowed = torch.arange(0, vocab, 7)
    for t in allowed.tolist():
        mask[0, t // 32] |= (1 << (t % 32)) - (1 << 32 if t % 32 == 31 else 0)
    bias = [{}, {3: 0.5, 70: -1.0}, {7: 0.25}]
    rep, pres, freq = [1.3, 1.0, 1.1], [0.4, 0.0, 0.2], [0.1, 0.0, 0.3]
    rules = sc.LogitRules(3, "cuda", repetition=rep, presence=pres, frequency=freq, bias=bias, mask=mask, mask_row=[-1, -1, 0])
    dec = q2.PagedDecoder(model, 3, rules)
    toks = [[], [], []]

    def check(raw, chosen, b):
        x = raw.double().cpu().clone()
        seen = ps[b].tolist() + toks[b]
        for v in set(seen):
            x[v] = x[v] / rep[b] if x[v] > 0 else x[v] * rep[b]
            n = toks[b].count(v)
            x[v] -= freq[b] * n + (pres[b] if n else 0.0)
        for v, w in bias[b].items():
            x[v] += w
        if b == 2:
            keep = torch.full_like(x, -math.inf)
            keep[allowed] = x[allowed]
            x = keep
        assert x[chosen] >= x.max() - 1e-5 * raw.abs().max()  # f32 steps against 64 bits
        toks[b].append(chosen)

    first = dec.start(ps, chunk=chunk).tolist()
    for b in range(3):
        if chunk == 2048:  # one pass: its logits are the last ones
            check(dec.raw[b], first[b], b)
        else:
            toks[b].append(first[b])
    for i in range(steps):
        if graph and i == 0:
            dec.capture()
        else:
            dec.step()
        dec.stream.synchronize()
        chosen = dec.ids.tolist()
        for b in range(3):
            check(dec.raw[b], chosen[b], b)
    assert dec.lengths == [n + steps for n in lens]
    assert [len(model.cache.pages(b)) for b in range(3)] == [-(-n // 16) for n in dec.lengths]
    model.check_device(), model.cache.check_device()
    assert all(t % 7 == 0 for t in toks[2])
    dec.finish()
    assert model.cache.free_pages == 40 and dec.lengths == [0, 0, 0]


def test_graph_and_eager_and_chunks_give_the_same_tokens(q2, ck):
    """The same prompts through captured and eager steps: the same bits, so the same tokens; and again after
    other sequences have used the pages."""
    ps = prompts([33, 2, 64], ck.cfg.vocab, 3)
    model = paged(q2, ck, torch.float16)
    out = []
    for graph in (True, False, True):
        dec = q2.PagedDecoder(model, 3)
        out.append(dec.generate(ps, 20, graph=graph))
        dec.finish()
        other = q2.PagedDecoder(model, 2)
        other.generate(prompts([50, 9], ck.cfg.vocab, 4), 5)
        other.finish()
    model.cache.check_device()
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def test_decoder_refusals(q2, ck):
    model = paged(q2, ck, torch.float16, slots=2, pages=3, positions=64)
    dec = q2.PagedDecoder(model, 2)
    with pytest.raises(ValueError):
        q2.PagedDecoder(model, 3)
    with pytest.raises(ValueError):
        dec.start(prompts([3], 100, 1))
    with pytest.raises(ValueError):
        dec.start([torch.zeros(0, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)])
    with pytest.raises(ValueError):
        dec.start(prompts([65, 1], 100, 1))
    with pytest.raises(RuntimeError):
        dec.start(prompts([33, 16], 100, 1))  # 3 + 1 pages of 3
    dec.finish()
    with pytest.raises(ValueError):
        model.forward_tokens(None, None, None, None, 0)
    ref = q2.Qwen2Model(ck, max_pos=8)
    with pytest.raises(ValueError):
        q2.PagedDecoder(ref, 1)
    with pytest.raises(ValueError):
        ref.forward_paged(None, None, None, None, None, 1, 1)
    cache = q2.Qwen2Model.paged_cache(ck, 4, max_seqs=1, max_positions=64, page_size=16)
    with pytest.raises(ValueError):
        q2.Qwen2Model(ck, max_pos=32, cache=cache)
    dec = q2.PagedDecoder(model, 1)
    with pytest.raises(RuntimeError):
        dec.step()  # before any prompt
    with pytest.raises(RuntimeError):
        dec.capture()
    dec.start(prompts([47], 100, 1))
    dec.step()
    with pytest.raises(RuntimeError):
        for _ in range(20):
            dec.step()  # position 48 needs a fourth page
    dec.finish()


def test_one_decoder_at_a_time(q2, ck):
    """A second decoder on the same cache is refused until the first has finished, and finishing one that does
    not run takes nothing from the one that does; a start() without enough pages leaves the run as it was."""
    ps = prompts([20, 7], ck.cfg.vocab, 6)
    model = paged(q2, ck, torch.float16, slots=2, pages=5)
    want = q2.PagedDecoder(model, 2)
    tokens = want.generate(ps, 6, graph=False)
    want.finish()
    first, second = q2.PagedDecoder(model, 2), q2.PagedDecoder(model, 1)
    got = [first.start(ps)]
    with pytest.raises(RuntimeError, match="another decoder"):
        second.start(ps[:1])
    second.finish()
    with pytest.raises(RuntimeError, match="pages wanted"):
        first.start(prompts([150, 7], ck.cfg.vocab, 7))
    for _ in range(5):
        got.append(first.step().clone())
        first.stream.synchronize()
    assert torch.equal(torch.stack(got, 1), tokens)
    first.finish()
    assert model.cache.free_pages == 5
    second.start(ps[:1])
    del second  # a decoder that is gone holds nothing up
    assert torch.equal(first.generate(ps, 3), tokens[:, :3])
    first.finish()
