"""The paged cache on the GPU: appending and attention against a plain implementation in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

from paged_cases import U, Paged

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def sc():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import saccade_core
    return saccade_core


def attend(sc, c, **kw):
    """The call, with length bounds of its own if the case has them."""
    out = torch.full((c.tokens, c.nh, c.hd), 7.0, dtype=kw.pop("out_dtype", c.dtype), device=c.q.device)
    status = torch.zeros(1, dtype=torch.int32, device=c.q.device)
    got, lse = sc.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, c.max_kv, out=out,
                                  return_lse=True, status=status, **kw)
    torch.cuda.synchronize()
    assert got is out and int(status.item()) == 0
    return got, lse


def compare(c, got, lse, scale):
    ref, rl, tol, ltol = c.attention(scale)
    end = c.cu[-1]
    err = (got[:end].cpu().double() - ref[:end]).abs()
    assert torch.isfinite(got[:end]).all()
    assert (err <= tol[:end]).all(), float((err / tol[:end].clamp(min=1e-300)).max())
    assert (got[end:] == 7.0).all(), "rows behind the last sequence are left as they were"
    empty = rl[:end] == -math.inf
    assert torch.equal(lse[:end].cpu() == -math.inf, empty)
    lerr = torch.where(empty, 0.0, (lse[:end].cpu().double() - rl[:end]).abs().nan_to_num(0.0))
    assert (lerr <= ltol[:end]).all()


LENS = {
    "decode": [(1, n) for n in (1, 2, 7, 8, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 257, 300)],
    "decode-long": [(1, 4096), (1, 3001), (1, 1), (1, 2047)],
    "ragged": [(1, 100), (0, 50), (33, 33), (2, 2), (130, 200), (1, 1), (0, 0), (64, 300), (17, 1000)],
    "chunk": [(300, 1111), (257, 257)],
    "short": [(2, 70), (5, 5), (3, 400), (4, 129)],
    "one": [(1, 1)],
    "none": [(0, 0), (0, 12)],
}


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 1, 128), (8, 8, 64), (16, 2, 128), (20, 1, 64)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", list(LENS), ids=list(LENS))
def test_attention_matches_64_bits(sc, dtype, heads, lens, bound=None):
    page = {"decode": 16, "decode-long": 64, "ragged": 8, "chunk": 32, "short": 128, "one": 256, "none": 8}[lens]
    c = Paged(LENS[lens], *heads, page, dtype, "cuda", seed=len(lens) + heads[0], behind=3)
    c.max_kv = bound or c.max_kv
    scale = heads[2] ** -0.5
    compare(c, *attend(sc, c), scale)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (20, 1, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", ["decode", "short", "one", "none", "decode-long", "ragged", "chunk"])
@pytest.mark.parametrize("bound", [1, 200, 2048, 1 << 24])
def test_any_bound_on_the_positions_gives_the_attention(sc, dtype, heads, lens, bound):
    """The bound chooses between clusters (of 1 to 8 CTAs) and the cut line; sequences may even exceed it."""
    test_attention_matches_64_bits(sc, dtype, heads, lens, bound)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
def test_attention_page_sizes_strides_and_bounds(sc, dtype, page):
    """Pages that end inside a tile, pages apart from one another, q as a slice of a wider buffer, a
    scale of its own, and length bounds far above the lengths."""
    c = Paged([(1, 37), (40, 513), (1, 1000), (9, 9)], 14, 2, 64, page, dtype, "cuda", seed=page, behind=1, gap=64)
    wide = torch.full((c.tokens, 18, 64), math.nan, dtype=dtype, device="cuda")
    wide[:, :14] = c.q
    c.q = wide[:, :14]
    c.max_q, c.max_kv = c.tokens, 1 << 20
    compare(c, *attend(sc, c, scale=0.3), 0.3)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("bound", [64, 1 << 20])
@pytest.mark.parametrize("q_len", [1, 3])
def test_more_sequences_than_threads(sc, dtype, bound, q_len):
    """A thousand short sequences, some without new tokens: the work is divided over several blocks of them.
    (One token is few for every kernel, three tokens of 7 heads are many.)"""
    lens = [((i % 5 != 3) * q_len, q_len + i * 7 % 41) for i in range(1000)]
    c = Paged(lens, 14, 2, 64, 8, dtype, "cuda", seed=7, behind=2)
    c.max_kv = bound
    compare(c, *attend(sc, c), 0.125)


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("lens", [[(1, 70), (5, 5)], [(33, 200), (1, 1)]], ids=["few", "many"])
def test_64_query_heads_of_a_kv_head(sc, dtype, lens):
    c = Paged(lens, 64, 1, 64, 16, dtype, "cuda", seed=21)
    compare(c, *attend(sc, c), 0.125)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("lens", ["decode", "chunk", "ragged"])
@pytest.mark.parametrize("bound", [None, 1 << 20])
def test_output_over_the_queries(sc, dtype, lens, bound):
    c = Paged(LENS[lens], 14, 2, 64, 16, dtype, "cuda", seed=31)
    c.max_kv = bound or c.max_kv
    want, _ = attend(sc, c)
    q = c.q.clone()
    assert sc.paged_attention(q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, c.max_kv, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
def test_attention_extreme_scores(sc, dtype):
    """Scores of hundreds: weights from 1 down to zero, maxima that move by more than any exponent."""
    c = Paged([(1, 700), (150, 400)], 8, 2, 128, 32, dtype, "cuda", seed=5, scale=6.0)
    compare(c, *attend(sc, c), 128 ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
def test_negative_positions_attend_nothing(sc, dtype):
    """More new tokens than positions: the first rows' positions are negative and attend no key."""
    c = Paged([(5, 2), (1, 9), (200, 150), (1, 0), (3, 0)], 14, 2, 64, 16, dtype, "cuda", seed=9, behind=2)
    got, lse = attend(sc, c)
    compare(c, got, lse, 0.125)
    assert (got[:3] == 0).all() and (lse[:3] == -math.inf).all() and (got[c.cu[3]:c.cu[5]] == 0).all()


def test_f32_cache_to_f16_output(sc):
    c = Paged([(1, 300), (20, 77)], 14, 2, 64, 16, F32, "cuda", seed=3)
    full, _ = attend(sc, c)
    half, _ = attend(sc, c, out_dtype=F16)
    assert torch.equal(half, full.to(F16))


@pytest.mark.parametrize("lens", ["decode", "chunk"])
def test_two_calls_are_the_same_bits_and_streams_do_not_mix(sc, lens):
    c = Paged(LENS[lens], 28, 4, 128, 16, BF16, "cuda", seed=1)
    d = Paged(LENS[lens], 28, 4, 128, 16, BF16, "cuda", seed=2)
    a0, b0 = attend(sc, c)[0], attend(sc, d)[0]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(s1):
            a = sc.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, c.max_kv)
        with torch.cuda.stream(s2):
            b = sc.paged_attention(d.q, d.k_pages, d.v_pages, d.table, d.cu_q, d.kv_len, d.max_q, d.max_kv)
    torch.cuda.synchronize()
    assert torch.equal(a, a0) and torch.equal(b, b0)


@pytest.mark.parametrize("q_len,bound", [(1, 512), (1, 1 << 20), (60, 512)])
@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
def test_attention_in_a_graph_follows_lengths_and_tables(sc, dtype, q_len, bound):
    """A captured call replays with other lengths and pages in the same tensors, and a second graph
    beside it on another stream does not touch its scratch."""
    c = Paged([(q_len, 140), (q_len, 500), (q_len, 63)], 14, 2, 64, 16, dtype, "cuda", seed=11)
    d = Paged([(q_len, 333), (q_len, 60), (q_len, 511)], 14, 2, 64, 16, dtype, "cuda", seed=12)
    width = max(c.table.shape[1], d.table.shape[1])
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    pages = max(c.pages, d.pages)
    kp = torch.full((pages, 2, 16, 64), math.nan, dtype=dtype, device="cuda")
    vp, q, kv, cu = kp.clone(), torch.empty_like(c.q), c.kv_len.clone(), c.cu_q.clone()

    def fill(x):
        table.fill_(-1)[:, :x.table.shape[1]] = x.table
        kp[:x.pages], vp[:x.pages] = x.k_pages, x.v_pages
        q.copy_(x.q), kv.copy_(x.kv_len)

    fill(c)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        sc.paged_attention(q, kp, vp, table, cu, kv, q_len, bound)
    stream.synchronize()
    graph, other, side = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        got = sc.paged_attention(q, kp, vp, table, cu, kv, q_len, bound)
    with torch.cuda.graph(other, stream=side):
        beside = sc.paged_attention(d.q, d.k_pages, d.v_pages, d.table, d.cu_q, d.kv_len, q_len, bound)
    want = {x: sc.paged_attention(x.q, x.k_pages, x.v_pages, x.table, x.cu_q, x.kv_len, q_len, bound) for x in (c, d)}
    for x in (c, d, c):
        fill(x)
        torch.cuda.synchronize()
        for _ in range(3):
            with torch.cuda.stream(side):
                other.replay()
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[x]) and torch.equal(beside, want[d])


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("q_len", [1, 40])
def test_bad_pages_and_lengths_are_recorded_and_not_followed(sc, dtype, q_len):
    c = Paged([(q_len, 100), (q_len, 60), (q_len, 90)], 14, 2, 64, 16, dtype, "cuda", seed=4)
    good, _ = attend(sc, c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def again():
        status.zero_()
        out = torch.full_like(good, 7.0)
        sc.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, c.max_kv, out=out, status=status)
        torch.cuda.synchronize()
        return out, int(status.item())

    assert again()[1] == 0
    for bad in (-1, c.pages, 2**31 - 1, -2**31):
        keep = int(c.table[1, 2])
        c.table[1, 2] = bad
        out, st = again()
        assert st != 0 and torch.equal(out[:q_len], good[:q_len]) and torch.equal(out[2 * q_len:], good[2 * q_len:])
        c.table[1, 2] = keep
    for bad in (c.table.shape[1] * 16 + 1, 2**31 - 1, -5):
        c.kv_len[1] = bad
        out, st = again()
        assert st != 0 and (out[q_len:2 * q_len] == 7.0).all()
        assert torch.equal(out[:q_len], good[:q_len]) and torch.equal(out[2 * q_len:], good[2 * q_len:])
        c.kv_len[1] = 60
    # a sequence of more new tokens than the bound, one that reaches behind the rows
    c.max_q = q_len - 1 if q_len > 1 else 1
    if q_len > 1:
        out, st = again()
        assert st != 0 and (out == 7.0).all()
    c.max_q = q_len
    keep = c.cu_q.clone()
    c.cu_q[3] = c.tokens + 1
    out, st = again()
    assert st != 0 and torch.equal(out[:2 * q_len], good[:2 * q_len]) and (out[2 * q_len:] == 7.0).all()
    c.cu_q.copy_(keep)
    assert torch.equal(again()[0], good)


# ---------------------------------------------------------------- append


def tables(n, hd, device):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * (1.0e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    ang = torch.cat([ang, ang], 1)
    return ang.cos().float().to(device), ang.sin().float().to(device)


@pytest.mark.parametrize("src,dtype", [(F32, F16), (F32, BF16), (F32, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 1, 128), (64, 8, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("layout", ["apart", "fused", "odd"])
def test_append_matches_64_bits(sc, src, dtype, heads, layout):
    nh, nkv, hd = heads
    lens = [(1, 1), (5, 40), (0, 30), (1, 17), (70, 70), (3, 129)]
    c = Paged(lens, nh, nkv, hd, 16, dtype, "cuda", seed=nh, behind=2, gap=8 if layout == "odd" else 0)
    g = torch.Generator("cuda").manual_seed(1)
    extra = 1 if layout == "odd" else 0  # rows that start off any 16-byte boundary
    buf = torch.randn(c.tokens, (nh + 2 * nkv) * hd + extra, device="cuda", generator=g).to(src)
    q, k, v = (buf[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    if layout == "apart":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos, sin = tables(130, hd, "cuda")
    kp, vp = c.k_pages.clone(), c.v_pages.clone()
    if layout == "odd":
        kp, vp = c.k_pages, c.v_pages
    before_k, before_v = kp.clone(), vp.clone()
    out = torch.full((c.tokens, nh, hd), 7.0, dtype=dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = sc.paged_append(q, k, v, cos, sin, kp, vp, c.table, c.cu_q, c.kv_len, out=out, status=status)
    torch.cuda.synchronize()
    assert got is out and int(status.item()) == 0
    want_k, want_v, u = before_k.double(), before_v.double(), U[dtype]
    tol_k = torch.zeros_like(want_k)
    for b, (n, kv) in enumerate(lens):
        rows, pos = slice(c.cu[b], c.cu[b + 1]), torch.arange(kv - n, kv, device="cuda")
        if n == 0:
            continue
        cs, sn = cos[pos][:, None].double(), sin[pos][:, None].double()
        sign = torch.cat([-torch.ones(hd // 2), torch.ones(hd // 2)]).double().cuda()
        rot = lambda t: t.double() * cs + t.double().roll(hd // 2, -1) * sign * sn  # noqa: E731
        # two products and their sum, each rounded in f32, then one rounding to the cache's type
        mag = lambda t: (t.double() * cs).abs() + (t.double().roll(hd // 2, -1) * sn).abs()  # noqa: E731
        tol = lambda t: mag(t) * 2.0 ** -23 + u * rot(t).abs() * 1.001 + (2.0 ** -25 if dtype == F16 else 0)  # noqa: E731
        assert ((out[rows].double() - rot(q[rows])).abs() <= tol(q[rows])).all()
        page = c.table[b].long()[pos // 16]
        want_k[page, :, pos % 16], want_v[page, :, pos % 16] = rot(k[rows]), v[rows].to(dtype).double()
        tol_k[page, :, pos % 16] = tol(k[rows])
    assert (out[c.cu[-1]:] == 7.0).all()
    same = torch.isnan(want_k) & torch.isnan(kp.double())
    assert (same | ((kp.double() - want_k).abs() <= tol_k)).all()
    assert torch.equal(vp.double().nan_to_num(99.0), want_v.nan_to_num(99.0))
    if src == dtype and layout == "apart":  # in place: the same bits
        sc.paged_append(q, k, v, cos, sin, kp, vp, c.table, c.cu_q, c.kv_len, out=q)
        assert torch.equal(q[:c.cu[-1]], out[:c.cu[-1]])


def test_append_for_more_sequences_than_a_warp(sc):
    lens = [(i % 3, 1 + i % 3 + i % 29) for i in range(300)]
    c = Paged(lens, 4, 2, 64, 8, F16, "cuda", seed=1)
    q, k, v = (torch.randn(c.tokens, n, 64, device="cuda") for n in (4, 2, 2))
    cos, sin = tables(40, 64, "cuda")
    kp, vp = torch.zeros_like(c.k_pages), torch.zeros_like(c.v_pages)
    sc.paged_append(q, k, v, cos, sin, kp, vp, c.table, c.cu_q, c.kv_len)
    for b, (n, kv) in enumerate(lens):
        for i in range(n):
            p, row = kv - n + i, c.cu[b] + i
            assert torch.equal(vp[int(c.table[b, p // 8]), :, p % 8], v[row].half())


def test_append_skips_what_has_no_place(sc):
    c = Paged([(2, 20), (1, 33), (2, 1), (1, 5)], 14, 2, 64, 16, F16, "cuda", seed=8)
    q, k, v = (torch.randn(c.tokens, n, 64, device="cuda") for n in (14, 2, 2))
    cos, sin = tables(40, 64, "cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run():
        kp, vp = torch.full_like(c.k_pages, 3.0), torch.full_like(c.v_pages, 3.0)
        out = torch.full((c.tokens, 14, 64), 7.0, dtype=F16, device="cuda")
        status.zero_()
        sc.paged_append(q, k, v, cos, sin, kp, vp, c.table, c.cu_q, c.kv_len, out=out, status=status)
        torch.cuda.synchronize()
        return out, kp, vp, int(status.item())

    out, kp, vp, st = run()  # sequence 2 has one position for two tokens: the first has none
    assert st != 0 and (out[3] == 7.0).all() and not (out[4] == 7.0).any()
    c.kv_len[2] = 2
    out, kp, vp, st = run()
    assert st == 0
    for bad in (-1, c.pages, 2**31 - 1):
        keep = int(c.table[1, 2])
        c.table[1, 2] = bad  # position 32's page
        out2, kp2, vp2, st = run()
        assert st != 0 and torch.equal(out2, out)
        assert (kp2[keep] == 3.0).all() and (vp2[keep] == 3.0).all()
        kp2[keep], vp2[keep] = kp[keep], vp[keep]
        assert torch.equal(kp2, kp) and torch.equal(vp2, vp)
        c.table[1, 2] = keep
    for bad in (41, 10**6, 2**31 - 1, -3):  # beyond the rotation tables, and the block table, and before 0
        c.kv_len[3] = bad
        out2, _, _, st = run()
        assert st != 0 and (out2[5] == 7.0).all() and torch.equal(out2[:5], out[:5])
        c.kv_len[3] = 5
    assert run()[3] == 0


def test_append_then_attend_is_one_prefill(sc):
    """A prompt appended and attended in chunks of any size gives what one pass gives, within the
    rounding of a few keys' order (f32), and decoding continues it."""
    nh, nkv, hd, page, n = 14, 2, 64, 16, 203
    g = torch.Generator("cuda").manual_seed(2)
    q, k, v = (torch.randn(n, h, hd, device="cuda", generator=g) for h in (nh, nkv, nkv))
    cos, sin = tables(n, hd, "cuda")
    table = torch.randperm(16, device="cuda", generator=g)[None].to(torch.int32)

    def run(cuts):
        kp, vp = torch.zeros(16, nkv, page, hd, device="cuda"), torch.zeros(16, nkv, page, hd, device="cuda")
        outs = []
        for a, b in zip([0] + cuts, cuts + [n]):
            cu = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
            kv = torch.tensor([b], dtype=torch.int32, device="cuda")
            qr = sc.paged_append(q[a:b], k[a:b], v[a:b], cos, sin, kp, vp, table, cu, kv)
            outs.append(sc.paged_attention(qr, kp, vp, table, cu, kv, b - a, n))
        return torch.cat(outs), kp, vp

    whole, kp, vp = run([])
    for cuts in ([1], [64, 128], [100, 101, 102, 150], list(range(180, n))):
        part, kp2, vp2 = run(cuts)
        assert torch.equal(kp, kp2) and torch.equal(vp, vp2)
        assert (part - whole).abs().max() <= 2e-5  # f32 sums of up to 203 terms of size ~1, regrouped


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (20, 1, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", ["ragged", "chunk", "short", "decode"])
@pytest.mark.parametrize("bound", [None, 1 << 20])
def test_values_that_are_not_finite_stay_with_the_rows_that_attend_them(sc, dtype, heads, lens, bound):
    """NaN and infinities among the values, in old and new positions: the same bits as with zeros there in
    every row before the position and in every other column, and nothing finite in their own."""
    c = Paged(LENS[lens], *heads, 16, dtype, "cuda", seed=21)
    c.max_kv = max(c.max_kv, bound or 0)
    g = torch.Generator().manual_seed(5)
    bad, G = torch.zeros(c.tokens, c.nh, c.hd, dtype=torch.bool), heads[0] // heads[1]
    put = []
    for b, (n, kv) in enumerate(c.lens):
        for i in range(min(n, 5)):
            new = int(torch.randint(kv - n, kv, (1,), generator=g)) if i < 4 else kv - 1
            p = int(torch.randint(0, kv, (1,), generator=g)) if i == 0 and n > 3 else new
            h, col = int(torch.randint(c.nkv, (1,), generator=g)), int(torch.randint(c.hd, (1,), generator=g))
            put.append((int(c.table[b, p // 16]), h, p % 16, col))
            bad[c.cu[b] + max(0, p - (kv - n)):c.cu[b] + n, h * G:(h + 1) * G, col] = True
    for at in put:
        c.v_pages[at] = 0.0
    clean, clean_lse = (t.clone() for t in attend(sc, c))
    assert torch.isfinite(clean).all()
    for value in (math.nan, math.inf, -math.inf):
        for at in put:
            c.v_pages[at] = value
        got, lse = attend(sc, c)
        assert torch.equal(torch.isfinite(got).cpu(), ~bad)
        assert torch.equal(torch.where(bad.cuda(), clean, got), clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("lens", ["ragged", "chunk", "short"])
@pytest.mark.parametrize("bound", [None, 1 << 20])
def test_keys_that_are_not_finite_stay_with_the_rows_that_attend_them(sc, dtype, lens, bound):
    c = Paged(LENS[lens], 14, 2, 64, 16, dtype, "cuda", seed=22)
    c.max_kv = max(c.max_kv, bound or 0)
    clean, clean_lse = (t.clone() for t in attend(sc, c))
    bad = torch.zeros(c.tokens, c.nh, dtype=torch.bool)
    for b, (n, kv) in enumerate(c.lens):
        if n > 0:
            p = kv - (n + 1) // 2
            c.k_pages[int(c.table[b, p // 16]), 1, p % 16, 40] = math.nan
            bad[c.cu[b] + p - (kv - n):c.cu[b] + n, 7:] = True
    got, lse = attend(sc, c)
    assert torch.equal(torch.isnan(got).all(-1).cpu(), bad) and torch.equal(torch.isnan(lse).cpu(), bad)
    assert torch.equal(got[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])


@pytest.mark.parametrize("dtype", [F16, F32], ids=["f16", "f32"])
@pytest.mark.parametrize("q_len,bound", [(1, 512), (1, 1 << 20), (70, 512)])
def test_pages_more_than_2_31_elements_apart(sc, dtype, q_len, bound):
    """Attention and appending in a cache whose last pages lie behind 2^31 elements: the bits of a small cache."""
    c = Paged([(q_len, 2100), (q_len, 190)], 14, 2, 64, 256, dtype, "cuda", seed=31)
    size, apart = 2 * 256 * 64, 2 ** 31 // (c.pages - 2) // 8 * 8 + 8 * 1024
    far = [torch.empty(apart * (c.pages - 1) + size, dtype=dtype, device="cuda").as_strided(
        (c.pages, 2, 256, 64), (apart, 256 * 64, 64, 1)) for _ in range(2)]
    assert apart * (c.pages - 2) > 2 ** 31
    far[0].copy_(c.k_pages), far[1].copy_(c.v_pages)
    cos, sin = tables(2200, 64, "cuda")
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(c.tokens, 2, 64, device="cuda", generator=g).to(dtype) for _ in range(2))
    out = []
    for kp, vp in ((c.k_pages, c.v_pages), far):
        q = sc.paged_append(c.q, k, v, cos, sin, kp, vp, c.table, c.cu_q, c.kv_len)
        out.append((q, *sc.paged_attention(q, kp, vp, c.table, c.cu_q, c.kv_len, q_len, bound, return_lse=True)))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and torch.isfinite(out[0][1]).all()
    assert torch.equal(far[0].nan_to_num(7.0), c.k_pages.nan_to_num(7.0))
    assert torch.equal(far[1].nan_to_num(7.0), c.v_pages.nan_to_num(7.0))
