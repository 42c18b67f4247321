"""Ragged paged-cache cases and their plain 64-bit implementation."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Paged:
    """Sequences with (new tokens, cached positions) `lens`; pages in a shuffled order, everything the
    lengths do not cover NaN, unused block table entries -1, `behind` token rows behind the last sequence."""

    def __init__(self, lens, nh, nkv, hd, page, dtype, device, seed=0, behind=0, gap=0, scale=1.0):
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.lens, self.nh, self.nkv, self.hd, self.page, self.dtype = lens, nh, nkv, hd, page, dtype
        need = [-(-max(kv, 0) // page) for _, kv in lens]
        self.pages, width = sum(need) + 2, max(need + [1]) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        cu = [0]
        for q, _ in lens:
            cu.append(cu[-1] + q)
        self.tokens, self.cu = cu[-1] + behind, cu
        self.max_q, self.max_kv = max([q for q, _ in lens] + [1]), max([kv for _, kv in lens] + [1])
        self.table, self.cu_q = table.to(device), torch.tensor(cu, dtype=torch.int32, device=device)
        self.kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=device)
        self.seq_k = [torch.randn(max(kv, 0), nkv, hd, generator=g).mul_(scale).to(dtype) for _, kv in lens]
        self.seq_v = [torch.randn(max(kv, 0), nkv, hd, generator=g).to(dtype) for _, kv in lens]
        # each page `gap` elements away from the end of the one before
        size = nkv * page * hd + gap
        def pool():
            return torch.full((self.pages, size), math.nan, dtype=dtype, device=device)[:, :size - gap].unflatten(
                1, (nkv, page, hd))
        self.k_pages, self.v_pages = pool(), pool()
        for b, (_, kv) in enumerate(lens):
            for p0 in range(0, max(kv, 0), page):
                n, pg = min(page, kv - p0), int(table[b, p0 // page])
                self.k_pages[pg, :, :n] = self.seq_k[b][p0:p0 + n].transpose(0, 1).to(device)
                self.v_pages[pg, :, :n] = self.seq_v[b][p0:p0 + n].transpose(0, 1).to(device)
        self.q = torch.randn(self.tokens, nh, hd, generator=g).mul_(scale).to(dtype).to(device)

    def attention(self, scale):
        """Output, lse and their error bounds in 64 bits, for every row of every sequence.

        Bounds: a score's f32 sum of hd products (in any order, scaled once) is off by at most
        e = (hd + 2) 2^-24 sum |q k| scale; a weight exp(s - m), its exponent's argument rounded (|s - m| 2^-23),
        by a factor 1 +- (2 e + |s - m| 2^-22 + 2^-21); the 16-bit kernels round each weight once
        more (U); sums of up to L weights or products, regrouped and rescaled, by (L + 64) 2^-24 of the sum of
        the magnitudes.  Numerator and denominator both carry them; the output is rounded once."""
        G = self.nh // self.nkv
        out = torch.zeros(self.tokens, self.nh, self.hd, dtype=torch.float64)
        lse = torch.full((self.tokens, self.nh), -math.inf, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        u = U[self.dtype]
        up = 0.0 if self.dtype == torch.float32 else u
        for b, (n, kv) in enumerate(self.lens):
            if n == 0 or kv == 0:
                continue
            q = self.q[self.cu[b]:self.cu[b] + n].cpu().double()
            k, v = (t[b].double().repeat_interleave(G, 1) for t in (self.seq_k, self.seq_v))
            s = torch.einsum("ihd,jhd->hij", q, k) * scale
            mag = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * abs(scale)
            pos = torch.arange(kv - n, kv)
            dead = (torch.arange(kv)[None, :] > pos[:, None])[None]
            s = s.masked_fill(dead, -math.inf)
            live = pos >= 0
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m).masked_fill(dead, 0.0)
            total = p.sum(-1, keepdim=True)
            w = p / total
            rows = torch.arange(self.cu[b], self.cu[b] + n)[live]
            o = torch.einsum("hij,jhd->ihd", w, v)
            out[rows], lse[rows] = o[live], (m + total.log())[..., 0].T[live]
            arg = torch.where(dead, 0.0, (s - m).abs().clamp(max=200.0))
            e = torch.where(dead, 0.0, (self.hd + 2) * 2.0 ** -24 * mag)
            e = e + e.gather(-1, s.argmax(-1, keepdim=True))  # the maximum's own error
            rel = e + arg * 2.0 ** -22 + 2.0 ** -21
            sums = (kv + 64) * 2.0 ** -24
            num = torch.einsum("hij,jhd->ihd", w * (rel + up + sums), v.abs())
            den = (w * rel).sum(-1).T + sums
            tol[rows] = (1.01 * (num + den[..., None] * o.abs()) + u * 1.01 * o.abs() + 1e-30 + _tiny(self.dtype))[live]
            ltol[rows] = (1.01 * den + 2.0 ** -22 * lse[self.cu[b]:self.cu[b] + n].abs().clamp(min=1.0))[live]
        return out, lse, tol, ltol


def _tiny(dtype):
    """Half the smallest subnormal step of the output's type, plus f16 weights' own (far keys' weights below
    it vanish: at most 2^-25 each of values up to 8, over up to 4096 keys)."""
    return {torch.float16: 2.0 ** -25 + 4096 * 8 * 2.0 ** -25 * 2.0 ** -8, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
