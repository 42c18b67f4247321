"""The serving operators of the Qwen2 decoder, as they are called and as their formulas say.

Three operators: appending rotated keys and values to a paged cache (saccade_core.paged_append), causal
attention of every sequence's newest tokens over that cache (saccade_core.paged_attention), and the
penalties, biases and grammar masks on the logits with the best token (saccade_core.process_logits).
run() computes them from elementary torch operations in 32 bits, or with the framework's kernels
where `own` is true; exact() is the same from the definition in 64 bits, sequence by sequence.

A cache page is [kv heads][page size][head dim]; a sequence's pages are in its row of the block
table.  Sequence b owns the token rows cu_q[b]..cu_q[b+1], its cache holds kv_len[b] positions after
them, and its i-th new token sits at position kv_len[b] - q_len[b] + i.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
# (query heads, KV heads, head dim): Qwen2-0.5B, 7B and 72B, a rank's share of 7B at 8 ranks (3 heads
# on a shared KV head), the small models of the tests, and no sharing at all
HEADS = [(14, 2, 64), (28, 4, 128), (64, 8, 128), (3, 1, 128), (4, 2, 64), (2, 1, 64), (8, 8, 64)]


def listed():
    return [
        # one decode step's append for 64 sequences of the 7B model: the linears give f32, the cache is f16
        dict(name="append-decode-64", op="append", seqs=64, q_min=1, q_max=1, kv_min=513, kv_max=768, heads=28,
             kv_heads=4, dim=128, page=64, src="f32", cache="f16", fused=False),
        # a prefill pass of two 2048-token prompts of the 72B model: q, k, v are slices of one bf16 buffer
        dict(name="append-prefill-2x2048", op="append", seqs=2, q_min=2048, q_max=2048, kv_min=2048, kv_max=2048,
             heads=64, kv_heads=8, dim=128, page=16, src="bf16", cache="bf16", fused=True),
        # a ragged step of the 0.5B model, decodes beside chunks of prompts, the cache in f32
        dict(name="append-ragged-f32", op="append", seqs=7, q_min=1, q_max=301, kv_min=1, kv_max=1211, heads=14,
             kv_heads=2, dim=64, page=32, src="f32", cache="f32", fused=False),
        # one sequence's decode step of the 7B model: the smallest call, where latency counts
        dict(name="attend-decode-1", op="attend", seqs=1, q_min=1, q_max=1, kv_min=640, kv_max=640, heads=28, kv_heads=4,
             dim=128, page=64, cache="f16", lse=False),
        # the batched decode step of the 7B model: 64 sequences of 512-token prompts, up to 256 steps in
        dict(name="attend-decode-64", op="attend", seqs=64, q_min=1, q_max=1, kv_min=513, kv_max=768, heads=28,
             kv_heads=4, dim=128, page=64, cache="f16", lse=False),
        # few long sequences of the 72B model: the cache read once is all that counts
        dict(name="attend-decode-8-long", op="attend", seqs=8, q_min=1, q_max=1, kv_min=20001, kv_max=32768, heads=64,
             kv_heads=8, dim=128, page=16, cache="bf16", lse=False),
        # chunks of 512 new tokens over long cached prefixes: the largest, tensor-core bound
        dict(name="attend-chunk-4x512", op="attend", seqs=4, q_min=512, q_max=512, kv_min=7001, kv_max=8192, heads=64,
             kv_heads=8, dim=128, page=16, cache="bf16", lse=True),
        # a prefill pass of 16 ragged prompts of the 7B model
        dict(name="attend-prefill-16", op="attend", seqs=16, q_min=129, q_max=512, kv_min=129, kv_max=512, heads=28,
             kv_heads=4, dim=128, page=64, cache="f16", lse=False),
        # a mixed step of the 0.5B model with the f32 cache of the reference: decodes beside short chunks
        dict(name="attend-mixed-f32", op="attend", seqs=12, q_min=1, q_max=24, kv_min=1, kv_max=1500, heads=14, kv_heads=2,
             dim=64, page=8, cache="f32", lse=True),
        # one row of the 0.5B model's logits with a short history: latency
        dict(name="logits-1", op="logits", rows=1, vocab=151936, begin=0, prompt=128, generated=128, bias=0, masks=0,
             dtype="f32"),
        # the batched decode step of the 7B model: every row penalised, some biased, half under a grammar
        dict(name="logits-64", op="logits", rows=64, vocab=152064, begin=0, prompt=512, generated=256, bias=64, masks=8,
             dtype="f32"),
        # many rows over one rank's odd slice of the vocabulary in bf16, long histories
        dict(name="logits-200-bf16", op="logits", rows=200, vocab=38017, begin=38016, prompt=6000, generated=2000, bias=300,
             masks=200, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logits"])
    if op == "logits":
        case = dict(op=op, rows=_spread(rng, 1, 200), vocab=_spread(rng, 1000, 152064), begin=32 * rng.randrange(0, 1200),
                    prompt=_spread(rng, 1, 6000), generated=_spread(rng, 1, 2000), bias=rng.choice([0, rng.randrange(1, 400)]),
                    masks=rng.choice([0, 1, rng.randrange(2, 40)]), dtype=rng.choice(["f32", "f32", "f16", "bf16"]))
        return case
    heads, kv_heads, dim = rng.choice(HEADS)
    cache = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    q_max = rng.choice([1, _spread(rng, 2, 24), _spread(rng, 25, 700)])
    q_min = rng.choice([1, max(1, q_max // 2), q_max])
    kv_max = _spread(rng, max(q_max, 2), 32768)
    kv_min = rng.choice([1, max(1, kv_max // 2)])
    seqs = _spread(rng, 1, 96)
    case = dict(op=op, q_min=q_min, q_max=q_max, kv_min=kv_min, kv_max=kv_max, heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([8, 16, 32, 64, 128]), cache=cache)
    if op == "append":
        case.update(seqs=seqs, src=rng.choice([cache, "f32"]), fused=rng.random() < 0.5)
        case["kv_max"] = min(kv_max, 4096 if q_max < 4096 else q_max)
        case["kv_min"] = min(kv_min, case["kv_max"])
        case["seqs"] = max(1, min(seqs, 8192 // q_max, 120000 // case["kv_max"]))
        return case
    # no more scores, cached values or products than the largest listed cases
    f32_part = 4 if cache == "f32" else 1
    seqs = min(seqs, int(1.0e9 / f32_part / (heads * q_max * kv_max)), int(2.6e8 / f32_part / (kv_heads * dim * kv_max)))
    if seqs < 1:
        seqs = 1
        case["kv_max"] = min(kv_max, int(1.0e9 / f32_part / (heads * q_max)))
        case["kv_max"] = max(q_max, min(case["kv_max"], int(2.6e8 / f32_part / (kv_heads * dim))))
        case["kv_min"] = min(kv_min, case["kv_max"])
    case.update(seqs=seqs, lse=rng.random() < 0.5)
    return case


def _lens(case):
    """The sequences' new tokens and cached positions: a property of the case, not of the seed."""
    rng = random.Random("%(seqs)d %(q_min)d %(q_max)d %(kv_min)d %(kv_max)d" % case)
    out = []
    for _ in range(case["seqs"]):
        q = rng.randint(case["q_min"], case["q_max"])
        out.append((q, max(q, rng.randint(case["kv_min"], case["kv_max"]))))
    return out


def work(case):
    if case["op"] == "logits":
        n, s = case["rows"] * case["vocab"], BYTES[case["dtype"]]
        hist = case["rows"] * (case["prompt"] + case["generated"]) * 4
        masks = case["masks"] * ((case["vocab"] + 31) // 32) * 4
        return {"bytes": 2 * n * s + hist + masks + case["rows"] * (case["bias"] * 8 + 12), "flops": 2 * n}
    lens, cb = _lens(case), BYTES[case["cache"]]
    tokens, hq, hkv, d = sum(q for q, _ in lens), case["heads"], case["kv_heads"], case["dim"]
    meta = sum(4 * (-(-kv // case["page"])) + 8 for _, kv in lens)
    if case["op"] == "append":
        elems = tokens * (hq + 2 * hkv) * d
        return {"bytes": elems * (BYTES[case["src"]] + cb) + tokens * 2 * d * 4 + meta, "flops": 3 * tokens * (hq + hkv) * d}
    pairs = sum(q * (kv - q) + q * (q + 1) // 2 for q, kv in lens)
    out = tokens * hq * d * cb * 2 + (tokens * hq * 4 if case["lse"] else 0)
    return {"bytes": sum(kv for _, kv in lens) * hkv * d * cb * 2 + out + meta, "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)

    if case["op"] == "logits":
        rows, vocab, begin = case["rows"], case["vocab"], case["begin"]
        whole = begin + vocab + 64
        width = case["prompt"] + case["generated"]

        def often(*shape):  # token ids of text: few of them make up most of it
            u = torch.rand(*shape, device=dev, generator=g)
            ids = (whole * u ** 4).long().clamp_(0, whole - 1)
            return ((ids * 7919) % whole).to(torch.int32)

        def some(lo, hi):
            return lo + (hi - lo) * torch.rand(rows, device=dev, generator=g)

        prompt_len = torch.randint(0, case["prompt"] + 1, (rows,), device=dev, generator=g)
        made = torch.randint(0, case["generated"] + 1, (rows,), device=dev, generator=g)
        st = dict(case=case, logits=normal(rows, vocab, scale=3.0, dtype=DTYPES[case["dtype"]]), history=often(rows, width),
                  prompt_len=prompt_len.to(torch.int32), hist_len=(prompt_len + made).to(torch.int32),
                  repetition=some(1.0, 1.3), presence=some(-0.2, 0.8), frequency=some(0.0, 0.5),
                  bias_ptr=None, bias_ids=None, bias_vals=None, mask=None, mask_row=None,
                  out=torch.empty(rows, vocab, device=dev, dtype=DTYPES[case["dtype"]]))
        if case["bias"]:
            n = torch.randint(0, case["bias"] + 1, (rows,), device=dev, generator=g)
            st["bias_ptr"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), n.cumsum(0)]).to(torch.int32)
            total = rows * case["bias"]
            st["bias_ids"] = (begin + torch.randint(0, vocab, (total,), device=dev, generator=g)).to(torch.int32)
            st["bias_vals"] = normal(total, scale=2.0)
        if case["masks"]:
            words = (begin + vocab + 31) // 32
            def bits():
                return torch.randint(-2**31, 2**31, (case["masks"], words), device=dev, generator=g)
            st["mask"] = (bits() & bits() & bits()).to(torch.int32)  # an eighth of the tokens may come next
            st["mask_row"] = torch.randint(-case["masks"], case["masks"], (rows,), device=dev, generator=g).clamp_(
                min=-1).to(torch.int32)
        return st

    lens, dt = _lens(case), DTYPES[case["cache"]]
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    tokens = sum(q for q, _ in lens)
    need = [-(-kv // page) for _, kv in lens]
    pages, width = sum(need) + 3, max(need)
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for q, _ in lens:
        cu.append(cu[-1] + q)
    st = dict(case=case, table=table, cu_q=torch.tensor(cu, dtype=torch.int32, device=dev),
              kv_len=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev),
              k_pages=normal(pages, hkv, page, d, dtype=dt), v_pages=normal(pages, hkv, page, d, dtype=dt))
    if case["op"] == "attend":
        st["q"] = normal(tokens, hq, d, dtype=dt, scale=1.5)
        st["q_max"], st["kv_max"] = max(q for q, _ in lens), max(kv for _, kv in lens)
        st["scale"] = 1.0 / math.sqrt(d)
        return st
    src = DTYPES[case["src"]]
    if case["fused"]:
        buf = normal(tokens, hq + 2 * hkv, d, dtype=src)
        st["q"], st["k"], st["v"] = buf[:, :hq], buf[:, hq:hq + hkv], buf[:, hq + hkv:]
    else:
        st["q"], st["k"], st["v"] = (normal(tokens, n, d, dtype=src) for n in (hq, hkv, hkv))
    pos = torch.arange(max(kv for _, kv in lens), dtype=torch.float64, device=dev)
    angle = pos[:, None] * (1.0e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d))[None, :]
    angle = torch.cat([angle, angle], dim=1)
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    return st


# ------------------------------------------------------------------------------------------- one pass


def run(st):
    op = st["case"]["op"]
    if own:
        return _framework(st, op)
    return {"append": _append, "attend": _attend, "logits": _logits}[op](st)


def _framework(st, op):
    if "saccade_core" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "saccade-x2_b200"))
    import saccade_core as sc
    if op == "append":
        q = sc.paged_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["k_pages"], st["v_pages"], st["table"],
                            st["cu_q"], st["kv_len"])
        return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "attend":
        r = sc.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["cu_q"], st["kv_len"], st["q_max"],
                               st["kv_max"], scale=st["scale"], return_lse=st["case"]["lse"])
        return {"out": r[0], "lse": r[1]} if st["case"]["lse"] else {"out": r}
    out, best, value = sc.process_logits(
        st["logits"], history=st["history"], prompt_len=st["prompt_len"], hist_len=st["hist_len"],
        repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"], bias_ptr=st["bias_ptr"],
        bias_ids=st["bias_ids"], bias_vals=st["bias_vals"], mask=st["mask"], mask_row=st["mask_row"],
        vocab_begin=st["case"]["begin"], out=st["out"], return_best=True)
    return {"logits": out, "best": best, "value": value}


def _places(st):
    """Each new token's sequence, position, page and row in the page."""
    n = st["q"].shape[0]
    row = torch.arange(n, device=st["q"].device, dtype=torch.int32)
    seq = torch.searchsorted(st["cu_q"], row, right=True) - 1
    pos = (st["kv_len"] - st["cu_q"][1:])[seq] + row
    page = st["table"][seq, pos // st["case"]["page"]]
    return seq, pos.long(), page.long(), (pos % st["case"]["page"]).long()


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    x = x.float()
    return x * cos[:, None] + torch.cat([-x[..., h:], x[..., :h]], dim=-1) * sin[:, None]


def _append(st):
    _, pos, page, row = _places(st)
    cos, sin, dt = st["cos"][pos], st["sin"][pos], st["k_pages"].dtype
    st["k_pages"][page, :, row] = _rotate(st["k"], cos, sin).to(dt)
    st["v_pages"][page, :, row] = st["v"].to(dt)
    return {"q": _rotate(st["q"], cos, sin).to(dt), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _attend(st):
    c, q = st["case"], st["q"]
    hkv, d, group = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    n, seqs, qm, km = q.shape[0], c["seqs"], st["q_max"], st["kv_max"]
    seq, pos, _, _ = _places(st)
    place = torch.arange(n, device=q.device) - st["cu_q"].long()[seq]
    qp = torch.zeros(seqs, qm, hkv, group, d, device=q.device)
    qp[seq, place] = q.float().view(n, hkv, group, d)
    last = torch.full((seqs, qm), -1, dtype=torch.long, device=q.device)  # each query's own position
    last[seq, place] = pos
    key = torch.arange(km, device=q.device)
    page, row = st["table"][:, key // c["page"]].long(), (key % c["page"]).expand(seqs, km)
    held = (key < st["kv_len"][:, None])[..., None, None]  # [seqs, keys, 1, 1]
    k = st["k_pages"][page, :, row].float()
    v = torch.where(held, st["v_pages"][page, :, row].float(), 0.0)
    s = torch.matmul(qp.permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * qm, d), k.permute(0, 2, 3, 1))
    s = (s * st["scale"]).view(seqs, hkv, group, qm, km)
    s = s.masked_fill_((key > last[..., None])[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, hkv, group * qm, km), v.permute(0, 2, 1, 3)).view(seqs, hkv, group, qm, d)
    o = (o / total).permute(0, 3, 1, 2, 4)[seq, place].reshape(n, c["heads"], d).to(q.dtype)
    if not c["lse"]:
        return {"out": o}
    return {"out": o, "lse": (m + total.log())[..., 0].permute(0, 3, 1, 2)[seq, place].reshape(n, c["heads"])}


def _logits(st):
    c, x = st["case"], st["logits"].float()
    rows, vocab, begin = c["rows"], c["vocab"], c["begin"]
    ids = st["history"].long() - begin
    at = torch.arange(ids.shape[1], device=ids.device)
    here = (at < st["hist_len"][:, None]) & (ids >= 0) & (ids < vocab)
    ids = ids.clamp(0, vocab - 1)
    count = torch.zeros(rows, vocab, device=x.device).scatter_add_(1, ids, (here & (at >= st["prompt_len"][:, None])).float())
    seen = torch.zeros(rows, vocab, device=x.device).scatter_add_(1, ids, here.float()) > 0
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count
    x = x - torch.where(count > 0, st["presence"][:, None], 0.0)
    if c["bias"]:
        n = st["bias_ids"].shape[0]
        entry = torch.arange(n, device=x.device, dtype=torch.int32)
        row = torch.searchsorted(st["bias_ptr"], entry, right=True) - 1
        used = row < rows
        place = torch.where(used, row.clamp(max=rows - 1) * vocab + st["bias_ids"].long() - begin, 0)
        which = torch.full((rows * vocab,), -1, dtype=torch.int32, device=x.device)
        which.scatter_reduce_(0, place, torch.where(used, entry, -1), "amax")  # of a token listed twice the last entry
        which = which.view(rows, vocab).long()
        x = torch.where(which >= 0, x + st["bias_vals"][which.clamp(min=0)], x)
    if c["masks"]:
        tok = begin + torch.arange(vocab, device=x.device)
        word = st["mask"][:, tok // 32]
        allowed = ((word >> (tok % 32).int()) & 1).bool()
        free = st["mask_row"] < 0
        x = torch.where(allowed[st["mask_row"].clamp(min=0).long()] | free[:, None], x, -math.inf)
    out = x.to(st["logits"].dtype)
    value = out.amax(-1)
    tok = torch.arange(vocab, device=x.device)
    best = torch.where(out == value[:, None], tok, vocab).amin(-1) + begin  # the first of equals
    return {"logits": out, "best": best, "value": value}


# ------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(st)
    cu, kvs = st["cu_q"].tolist(), st["kv_len"].tolist()
    table, page = st["table"].long(), case["page"]
    if case["op"] == "append":
        d = case["dim"]
        kp, vp, qs = st["k_pages"].double(), st["v_pages"].double(), []
        sign = torch.ones(d, dtype=torch.float64, device=kp.device)
        sign[:d // 2] = -1
        for b, kv in enumerate(kvs):
            rows, pos = slice(cu[b], cu[b + 1]), torch.arange(kv - (cu[b + 1] - cu[b]), kv, device=kp.device)
            cs, sn = st["cos"].double()[pos][:, None], st["sin"].double()[pos][:, None]
            q, k = (t[rows].double() * cs + t[rows].double().roll(d // 2, -1) * sign * sn for t in (st["q"], st["k"]))
            kp[table[b][pos // page], :, pos % page] = k
            vp[table[b][pos // page], :, pos % page] = st["v"][rows].double()
            qs.append(q)
        return {"q": torch.cat(qs), "k_pages": kp, "v_pages": vp}
    group, d = case["heads"] // case["kv_heads"], case["dim"]
    outs, lses = [], []
    for b, kv in enumerate(kvs):
        n = cu[b + 1] - cu[b]
        pages = table[b][:-(-kv // page)]
        k, v = (st[t][pages].transpose(0, 1).reshape(case["kv_heads"], -1, d)[:, :kv].double() for t in ("k_pages", "v_pages"))
        masked = torch.arange(kv, device=k.device)[None, :] > torch.arange(kv - n, kv, device=k.device)[:, None]
        o, z = [], []
        for h in range(case["heads"]):  # a head at a time: the scores of all would not be small in 64 bits
            s = st["q"][cu[b]:cu[b + 1], h].double() @ k[h // group].T * st["scale"]
            s = s.masked_fill_(masked, -math.inf)
            z.append(torch.logsumexp(s, -1))
            o.append(torch.softmax(s, -1) @ v[h // group])
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(z, 1))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)} if case["lse"] else {"out": torch.cat(outs)}


def _exact_logits(st):
    c = st["case"]
    out = st["logits"].double()
    tok = torch.arange(c["vocab"], device=out.device) + c["begin"]
    whole = c["begin"] + c["vocab"] + 64
    for i in range(c["rows"]):
        n, m = int(st["hist_len"][i]), int(st["prompt_len"][i])
        past = st["history"][i, :n].long()
        seen = torch.bincount(past, minlength=whole)[tok] > 0
        count = torch.bincount(past[m:], minlength=whole)[tok].double()
        x, r = out[i], st["repetition"][i].double()
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - st["frequency"][i].double() * count - st["presence"][i].double() * (count > 0)
        if c["bias"]:
            lo, hi = int(st["bias_ptr"][i]), int(st["bias_ptr"][i + 1])
            last = dict(zip(st["bias_ids"][lo:hi].tolist(), st["bias_vals"][lo:hi].tolist()))
            if last:
                keys = torch.tensor(list(last.keys()), device=out.device) - c["begin"]
                x[keys] += torch.tensor(list(last.values()), dtype=torch.float64, device=out.device)
        if c["masks"] and int(st["mask_row"][i]) >= 0:
            words = st["mask"][int(st["mask_row"][i])].long()
            x = torch.where((words[tok // 32] >> (tok % 32)) % 2 == 1, x, -math.inf)
        out[i] = x
    return {"logits": out, "best": None, "value": out.amax(-1)}
