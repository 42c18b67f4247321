"""Attention where one position has nearly all of the weight: what the many small weights add up to stays in the output."""
import math

import pytest

torch = pytest.importorskip("torch")

from paged_cases import Paged, _tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sc():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import saccade_core
    return saccade_core


def sink_case(lens, heads, score, dtype, seed):
    """Every query is 5 along the first axis; one old key per sequence is score / 5 along it with a value of zero, the
    others are zero: their scores are 0 and their values 0.5..1.5."""
    nh, nkv, hd = heads
    c = Paged(lens, nh, nkv, hd, 64, dtype, "cuda", seed=seed, behind=1)
    g = torch.Generator().manual_seed(seed)
    c.q.zero_()
    c.q[..., 0] = 5.0
    for b, (n, kv) in enumerate(lens):
        at = int(torch.randint(0, kv - n, (1,), generator=g))
        c.seq_k[b].zero_()
        c.seq_k[b][at, :, 0] = score / 5.0
        c.seq_v[b].copy_(0.5 + torch.rand(c.seq_v[b].shape, generator=g))
        c.seq_v[b][at] = 0.0
        for p0 in range(0, kv, 64):
            m, pg = min(64, kv - p0), int(c.table[b, p0 // 64])
            c.k_pages[pg, :, :m] = c.seq_k[b][p0:p0 + m].transpose(0, 1).cuda()
            c.v_pages[pg, :, :m] = c.seq_v[b][p0:p0 + m].transpose(0, 1).cuda()
    return c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens,bound", [([(1, 16000)], 16384), ([(1, 20011), (1, 900)], 1 << 20), ([(2, 9000)], 9000)],
                         ids=["clusters", "cut", "two"])
@pytest.mark.parametrize("score", [12.0, 20.0])
def test_small_weights_of_few_new_tokens_add_up(sc, dtype, heads, lens, bound, score):
    """exp(-12) and exp(-20) of the largest weight, 2^-17 and 2^-29, up to 20,010 times.  The bound is the plain
    case's without its allowance for weights that f16 cannot hold: f16 weights are kept in two parts, scaled by 2^15,
    so the low part's half step of 2^-25 is 2^-40 of the largest weight; the output's own is 2^-25."""
    c = sink_case(lens, heads, score, dtype, seed=int(score) + len(lens))
    out = torch.full((c.tokens, c.nh, c.hd), 7.0, dtype=dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _, lse = sc.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, bound, scale=1.0, out=out,
                                return_lse=True, status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and (out[c.cu[-1]:] == 7.0).all()
    ref, rl, tol, ltol = c.attention(1.0)
    if dtype == torch.float16:
        tol = tol - _tiny(dtype) + 2.0 ** -25 + 2.0 ** -40 * 1.5 * max(kv for _, kv in lens)
    end = c.cu[-1]
    err = (out[:end].cpu().double() - ref[:end]).abs()
    assert (ref[:end] > 0).all() and (err <= tol[:end]).all(), float((err / tol[:end]).max())
    assert ((lse[:end].cpu().double() - rl[:end]).abs() <= ltol[:end]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", [[(40, 20011), (3, 900)], [(150, 5000)]], ids=["long", "chunk"])
@pytest.mark.parametrize("score", [12.0, 20.0])
def test_small_weights_of_many_new_tokens_add_up(sc, dtype, heads, lens, score):
    """The plain case's bound without its allowance for weights that f16 cannot hold: the kernel of many new tokens
    holds a weight in one part, of which the largest is 2^6 at least, so f16's half step of 2^-25 is 2^-31 of it."""
    c = sink_case(lens, heads, score, dtype, seed=int(score) + len(lens))
    out = torch.full((c.tokens, c.nh, c.hd), 7.0, dtype=dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    sc.paged_attention(c.q, c.k_pages, c.v_pages, c.table, c.cu_q, c.kv_len, c.max_q, c.max_kv, scale=1.0, out=out,
                       status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0 and (out[c.cu[-1]:] == 7.0).all()
    ref, _, tol, _ = c.attention(1.0)
    if dtype == torch.float16:
        tol = tol - _tiny(dtype) + 2.0 ** -25 + 2.0 ** -31 * 1.5 * max(kv for _, kv in lens)
    end = c.cu[-1]
    err = (out[:end].cpu().double() - ref[:end]).abs()
    assert (ref[:end] > 0).all() and (err <= tol[:end]).all(), float((err / tol[:end]).max())
