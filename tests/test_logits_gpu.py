"""process_logits on the GPU against its formulas in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from paged_cases import U

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def sc():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import saccade_core
    return saccade_core


def make(rows, vocab, begin, width, bias, masks, dtype, seed):
    g = torch.Generator("cpu").manual_seed(seed)
    whole = begin + vocab + 40
    r = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g)  # noqa: E731
    hist = r(0, width + 1, rows)
    hist[0] = width
    kw = dict(history=r(begin, begin + max(1, min(vocab, 50)), rows, width) if width else torch.zeros(rows, 0, dtype=torch.int64))
    stray = torch.rand(rows, width, generator=g) < 0.2
    kw["history"][stray] = r(-3, whole, rows, width)[stray]  # other slices' tokens, and negative ids
    kw["hist_len"], kw["prompt_len"] = hist, (hist * torch.rand(rows, generator=g)).long()
    for t in ("history", "hist_len", "prompt_len"):
        kw[t] = kw[t].to(torch.int32).cuda()
    kw["repetition"] = (0.7 + 0.8 * torch.rand(rows, generator=g)).cuda()
    kw["presence"], kw["frequency"] = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    if bias:
        n = r(0, bias + 1, rows)
        kw["bias_ptr"] = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32).cuda()
        total = int(n.sum()) + 5
        kw["bias_ids"] = r(begin - 2, begin + min(vocab, 60), total).to(torch.int32).cuda()  # many listed twice
        kw["bias_vals"] = torch.randn(total, generator=g).cuda()
    if masks:
        words = (begin + vocab + 31) // 32
        m = r(-2**31, 2**31, masks, words)
        m[0] = 0  # allows nothing
        kw["mask"] = m.to(torch.int32).cuda()
        kw["mask_row"] = r(-1, masks, rows).to(torch.int32).cuda()
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    return x, kw


def plain(x, begin, kw):
    """Processed logits in 64 bits and the magnitudes their roundings are relative to."""
    y, mag = x.double().cpu(), x.double().abs().cpu()
    for i in range(x.shape[0]):
        n, m = int(kw["hist_len"][i]), int(kw["prompt_len"][i])
        h = (kw["history"][i, :n].cpu().long() - begin).tolist()
        r, p, f = (float(kw[t][i]) for t in ("repetition", "presence", "frequency"))
        for v in set(h):
            if 0 <= v < x.shape[1]:
                c = h[m:].count(v)
                y[i, v] = y[i, v] / r if y[i, v] > 0 else y[i, v] * r
                y[i, v] -= f * c + (p if c else 0.0)
                mag[i, v] = abs(float(mag[i, v])) * max(r, 1 / r) + abs(f * c) + abs(p)
        if "bias_ptr" in kw:
            lo, hi = kw["bias_ptr"][i:i + 2].tolist()
            for v, b in dict(zip(kw["bias_ids"][lo:hi].tolist(), kw["bias_vals"][lo:hi].tolist())).items():
                if 0 <= v - begin < x.shape[1]:
                    y[i, v - begin] += b
                    mag[i, v - begin] += abs(b)
        if "mask" in kw and int(kw["mask_row"][i]) >= 0:
            words = kw["mask"][int(kw["mask_row"][i])].cpu().long() & 0xFFFFFFFF
            tok = torch.arange(x.shape[1]) + begin
            y[i][(words[tok // 32] >> (tok % 32)) & 1 == 0] = -math.inf
    return y, mag


def check(sc, x, begin, kw, **more):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, best, value = sc.process_logits(x, vocab_begin=begin, return_best=True, status=status, **kw, **more)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    y, mag = plain(x, begin, kw)
    got = out.double().cpu()
    assert torch.equal(got == -math.inf, y == -math.inf)
    live = y > -math.inf
    # at most five f32 roundings of values up to mag, then the output's
    tol = 5 * 2.0 ** -24 * mag + U[x.dtype] * 1.001 * y.abs() + (2.0 ** -25 if x.dtype == F16 else 0.0)
    assert ((got - y).abs()[live] <= tol[live]).all()
    top = out.amax(-1)
    assert torch.equal(value, top)
    tok = torch.arange(x.shape[1], device="cuda")
    assert torch.equal(best, torch.where(out == top[:, None], tok, x.shape[1]).amin(-1) + begin)
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,begin,width,bias,masks", [
    (1, 1, 0, 3, 2, 0), (1, 7, 0, 0, 0, 1), (3, 33, 64, 50, 10, 2), (2, 1000, 0, 300, 0, 0), (5, 4099, 37, 700, 40, 3),
    (9, 20481, 0, 64, 5, 0), (2, 38017, 38016, 2000, 300, 2), (1, 151936, 0, 128, 0, 0), (3, 200003, 32, 5000, 0, 1),
    (40, 5000, 0, 9, 0, 40)])
def test_matches_64_bits(sc, dtype, rows, vocab, begin, width, bias, masks):
    x, kw = make(rows, vocab, begin, width, bias, masks, dtype, seed=rows * vocab)
    out = check(sc, x, begin, kw)
    again = sc.process_logits(x, vocab_begin=begin, **kw)
    assert torch.equal(out, again)
    y = x.clone()
    assert sc.process_logits(y, vocab_begin=begin, out=y, **kw) is y and torch.equal(y, out)  # in place


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strided_rows_and_shifted_outputs(sc, dtype):
    """Rows and outputs that start off 16-byte boundaries, each by its own offset."""
    x, kw = make(4, 3001, 0, 100, 20, 2, dtype, seed=3)
    want = check(sc, x, 0, kw)
    for a, b in ((0, 1), (1, 0), (3, 3), (5, 2)):
        wide = torch.full((4, 3010), 9.0, dtype=dtype, device="cuda")
        wide[:, a:a + 3001] = x
        dst = torch.full((4, 3017), 5.0, dtype=dtype, device="cuda")
        sc.process_logits(wide[:, a:a + 3001], out=dst[:, b:b + 3001], **kw)
        assert torch.equal(dst[:, b:b + 3001], want)
        assert (dst[:, :b] == 5.0).all() and (dst[:, b + 3001:] == 5.0).all()


def test_nothing_asked_is_a_copy_and_special_values_pass(sc):
    x = torch.randn(3, 9001, device="cuda")
    x[0, 5], x[1, 7], x[1, 9], x[2, 100] = math.inf, math.nan, math.inf, -math.inf
    out, best, value = sc.process_logits(x, return_best=True)
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))
    assert best[:2].tolist() == [5, 7] and math.isnan(float(value[1])) and int(best[2]) == int(x[2].argmax())
    # a masked NaN or infinity is -inf like any other masked token; a row with nothing left gives its first token
    mask = torch.full((2, 282), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = ~((1 << 5) | (1 << 7) | (1 << 9))
    mask[1] = 0
    out, best, value = sc.process_logits(x, mask=mask, mask_row=torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda"),
                                         vocab_begin=0, return_best=True)
    assert out[0, 5] == -math.inf and out[1, 7] == -math.inf and out[1, 9] == -math.inf
    assert torch.isfinite(value[:2]).all() and int(best[2]) == 0 and value[2] == -math.inf
    assert (out[2] == -math.inf).all()


def test_equal_values_give_the_first(sc):
    x = torch.zeros(3, 40000, device="cuda", dtype=BF16)
    x[1, 777:] = 1.0
    x[2, ::2] = -0.0
    assert sc.process_logits(x, return_best=True)[1].tolist() == [0, 777, 0]


def test_history_counts_every_occurrence(sc):
    """One token over and over, in the prompt and generated, and a history of the longest kind."""
    n = 70000
    h = torch.full((2, n), 3, dtype=torch.int32, device="cuda")
    h[:, ::7] = 4
    x = torch.ones(2, 500, device="cuda")
    one = torch.ones(2, device="cuda")
    out = sc.process_logits(x, history=h, hist_len=torch.tensor([n, 10], dtype=torch.int32, device="cuda"),
                            prompt_len=torch.tensor([100, 10], dtype=torch.int32, device="cuda"), frequency=one,
                            presence=one * 2, repetition=one * 4)
    c4 = len(range(0, n, 7)) - len(range(0, 100, 7))
    assert out[0, 4] == 0.25 - c4 - 2 and out[0, 3] == 0.25 - (n - 100 - c4) - 2
    assert out[1, 3] == 0.25 and out[1, 4] == 0.25 and (out[:, 5:] == 1).all()


def test_lengths_out_of_range_are_recorded_and_cut(sc):
    x, kw = make(4, 3001, 0, 100, 20, 2, F32, seed=6)
    want = sc.process_logits(x, **kw)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    def with_(name, i, v):
        t = dict(kw, **{name: kw[name].clone()})
        t[name][i] = v
        status.zero_()
        out = sc.process_logits(x, status=status, **t)
        torch.cuda.synchronize()
        return out, int(status.item())
    for name, v in (("hist_len", 101), ("hist_len", 2**31 - 1), ("hist_len", -1), ("prompt_len", 101), ("prompt_len", -7),
                    ("mask_row", 2), ("mask_row", 2**31 - 1), ("bias_ptr", -1), ("bias_ptr", 2**31 - 1)):
        out, st = with_(name, 2, v)
        assert st != 0, (name, v)
        assert torch.equal(out[0], want[0]) and torch.equal(out[3], want[3]) or name == "bias_ptr"
    ids = torch.arange(5000, dtype=torch.int32, device="cuda") % 3001
    status.zero_()
    sc.process_logits(x[:1], bias_ptr=torch.tensor([0, 5000], dtype=torch.int32, device="cuda"), bias_ids=ids,
                      bias_vals=torch.ones(5000, device="cuda"), status=status)
    assert int(status.item()) != 0


def test_in_a_graph(sc):
    x, kw = make(3, 9000, 0, 200, 8, 2, F32, seed=2)
    y, kw2 = make(3, 9000, 0, 200, 8, 2, F32, seed=3)
    kw2["bias_ptr"], kw2["bias_ids"], kw2["bias_vals"] = kw["bias_ptr"], kw["bias_ids"], kw["bias_vals"]
    want = [sc.process_logits(a, return_best=True, **k) for a, k in ((x, kw), (y, kw2))]
    hold, kh = x.clone(), {k: v.clone() for k, v in kw.items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sc.process_logits(hold, return_best=True, **kh)
    for (a, k), w in (((y, kw2), want[1]), ((x, kw), want[0])):
        hold.copy_(a)
        for name in kh:
            kh[name].copy_(k[name])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, w))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("share", [0.05, 0.5, 1.0])
def test_many_tokens_touched(sc, dtype, share):
    """Any share of a row's tokens in its history or bias list, results of either zero, infinities and NaN of any
    bits among them: exactly the formula's f32 roundings."""
    g = torch.Generator().manual_seed(17)
    vocab = 20011
    x = torch.randn(2, vocab, generator=g).to(dtype)
    x[:, 0::11], x[:, 1::11], x[:, 2::11], x[:, 3::11] = 0.5, 0.0, math.inf, -math.inf
    x[:, 4::11] = -0.0
    if dtype == F32:
        x.view(torch.int32)[:, 5::11] = 0x7FC0DEAD
    h = torch.stack([torch.randperm(vocab, generator=g) for _ in range(2)])[:, :int(share * vocab)].to(torch.int32)
    n = torch.zeros(2, vocab).scatter_(1, h.long(), 1.0)
    ids = torch.arange(5, 4000, dtype=torch.int32)
    b = torch.randn(len(ids), generator=g)
    half = torch.full((2,), 0.5, device="cuda")
    out, best, value = sc.process_logits(
        x.cuda(), history=h.cuda(), hist_len=torch.full((2,), h.shape[1], dtype=torch.int32, device="cuda"), frequency=half,
        bias_ptr=torch.tensor([0, 0, len(ids)], dtype=torch.int32, device="cuda"), bias_ids=ids.cuda(), bias_vals=b.cuda(),
        return_best=True)
    want = x.float() - 0.5 * n
    want[1, 5:4000] += b
    want = want.to(dtype).cuda()
    nan = want.isnan()
    assert torch.equal(out.isnan(), nan)
    bits = torch.int32 if dtype == F32 else torch.int16
    assert torch.equal(out.view(bits)[~nan], want.view(bits)[~nan])
    assert torch.equal(best, want.argmax(-1)) if dtype == F32 else torch.equal(best, want.float().argmax(-1))
