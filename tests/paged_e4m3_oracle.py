"""The paged cache in e4m3 from its definition, in 64 bits: a sequence is a list of tokens, a page what a table row says."""
import math

import torch

TOP, LEAST, MOST = 448.0, -100, 119


def round8(x):
    """Nearest e4m3 number, ties to even, in 64 bits; beyond 448 the largest, NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    step = torch.where(x.isinf(), 1.0, step)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def exponent(most: float) -> int:
    for e in range(LEAST, MOST + 1):
        if most <= TOP * 2.0 ** e:
            return e
    return MOST


class Cache:
    """Pages as 64-bit numbers of codes [blocks, heads, block_size, D] and integers [blocks, heads]."""

    def __init__(self, pages):
        self.c = {"k": pages.k.cpu().double(), "v": pages.v.cpu().double()}
        self.e = {"k": pages.k_exp.cpu().long(), "v": pages.v_exp.cpu().long()}
        self.w = None if pages.weight is None else pages.weight.cpu().double()
        self.bs = pages.k.shape[2]

    def append(self, k, v, tables, lens, starts):
        for b in range(len(lens)):
            r0, r1 = starts[b], starts[b + 1]
            for name, new in (("k", k), ("v", v)):
                by_page = {}
                for r in range(r0, r1):
                    pos = lens[b] - (r1 - r)
                    if pos >= 0 and pos // self.bs < tables.shape[1]:
                        by_page.setdefault(pos // self.bs, []).append((pos % self.bs, r))
                for i, rows in by_page.items():
                    p, begin = int(tables[b, i]), rows[0][0]
                    for h in range(self.c[name].shape[1]):
                        D = self.c[name].shape[3]
                        x = torch.stack([new[r, h * D:(h + 1) * D].double().cpu() for _, r in rows])
                        e = exponent(float(torch.where(x.isfinite(), x.abs(), 0.0).max()))
                        if begin:
                            had = int(self.e[name][p, h])
                            e = max(e, had)
                            self.c[name][p, h, :begin] = round8(self.c[name][p, h, :begin] * 2.0 ** (had - e))
                        self.c[name][p, h, begin:begin + len(rows)] = round8(x * 2.0 ** -e)
                        self.e[name][p, h] = e
                    if self.w is not None:
                        self.w[p, :, begin:begin + len(rows)] = 0.0

    def tokens(self, name, tables, b, n):
        """[n, heads, D]"""
        if n == 0:
            return torch.zeros(0, self.c[name].shape[1], self.c[name].shape[3], dtype=torch.float64)
        t = [int(tables[b, i]) for i in range((n + self.bs - 1) // self.bs)]
        return torch.cat([self.c[name][p] * torch.exp2(self.e[name][p].double())[:, None, None] for p in t], 1).transpose(0, 1)[:n]

    def attend(self, q, tables, lens, scale=None):
        """(out, most error of an output in exact arithmetic but with 11-bit softmax weights and fp32 scores, weights per sequence, their relative error)"""
        G, D = self.c["k"].shape[1], self.c["k"].shape[3]
        scale = 1 / math.sqrt(D) if scale is None else scale
        outs, errs, ws, wrel = [], [], [], []
        for b, n in enumerate(lens):
            x = q[b].double().cpu().view(G, -1, D)
            if n == 0:
                outs.append(torch.zeros(x.numel(), dtype=torch.float64))
                errs.append(torch.zeros(x.numel(), dtype=torch.float64))
                ws.append(torch.zeros(0, G, dtype=torch.float64))
                wrel.append(0.0)
                continue
            k, v = self.tokens("k", tables, b, n), self.tokens("v", tables, b, n)
            s = torch.einsum("hgd,nhd->hgn", x, k) * scale
            p = torch.softmax(s, -1)
            o = torch.einsum("hgn,nhd->hgd", p, v)
            # a score: D products summed in 32 bits (2^-24 each at most of the sum of magnitudes), the query scaled to 16-bit floats (2^-24 of its
            # largest number at most), four roundings behind them; a weight: twice that (its own score and the largest), the two exponentials
            sizes = torch.einsum("hgd,nhd->hgn", x.abs(), k.abs()).max() + (x.abs().amax(-1, keepdim=True) * k.abs().sum(-1).t()[:, None]).max()
            rel = 2.0 * float(sizes) * abs(scale) * (D + 4) * 2.0 ** -24 + 2.0 ** -20
            many = torch.einsum("hgn,nhd->hgd", p, v.abs())
            # 16-bit weights: half a step, 2^-11, and 2^-25 where they are subnormal, of values up to the largest
            err = (rel + 2.0 ** -11) * many + n * 2.0 ** -25 * 2 * v.abs().max()
            outs.append(o.reshape(-1))
            errs.append(err.reshape(-1))
            ws.append(p.sum(1).t())
            wrel.append(rel)
        return torch.stack(outs), torch.stack(errs), ws, wrel

    def evict(self, tables, lens, keep, recent, first, out_tables=None):
        G = self.w.shape[1]
        kept = torch.full((len(lens), G, keep), -1, dtype=torch.int32)
        for b, n in enumerate(lens):
            m = min(n, keep)
            moved = []
            for h in range(G):
                place = list(range(n))
                at = lambda t: (int(tables[b, t // self.bs]), t % self.bs)  # noqa: E731
                if n > keep:
                    w = [float(self.w[at(t)[0], h, at(t)[1]]) for t in range(n)]
                    w = [math.inf if x != x else x for x in w]
                    nan = [math.isnan(float(self.w[at(t)[0], h, at(t)[1]])) for t in range(n)]
                    middle = sorted(range(first, n - recent), key=lambda t: (not nan[t], -w[t], t))[:m - first - recent]
                    place = list(range(first)) + sorted(middle) + list(range(n - recent, n))
                kept[b, h, :m] = torch.tensor(place, dtype=torch.int32)
                if n <= keep and out_tables is None:
                    continue
                for j, t in enumerate(place):
                    p, o = at(t)
                    moved.append((j, h, {x: (self.c[x][p, h, o].clone(), int(self.e[x][p, h])) for x in ("k", "v")}, float(self.w[p, h, o])))
            to = tables if out_tables is None else out_tables
            tops = {}
            for j, h, kv, _ in moved:
                for x in ("k", "v"):
                    key = (x, int(to[b, j // self.bs]), h)
                    tops[key] = max(tops.get(key, -1000), kv[x][1])
            for j, h, kv, w in moved:
                p = int(to[b, j // self.bs])
                for x in ("k", "v"):
                    self.c[x][p, h, j % self.bs] = round8(kv[x][0] * 2.0 ** (kv[x][1] - tops[(x, p, h)]))
                self.w[p, h, j % self.bs] = w
            for (x, p, h), e in tops.items():
                self.e[x][p, h] = e
        return torch.tensor([min(n, keep) for n in lens], dtype=torch.int32), kept

    def same(self, pages):
        """Codes, exponents and (but for their rounding) weights of `pages` are these."""
        for name, codes, exps in (("k", pages.k, pages.k_exp), ("v", pages.v, pages.v_exp)):
            torch.testing.assert_close(codes.cpu().double(), self.c[name], rtol=0, atol=0, equal_nan=True)
            assert torch.equal(exps.cpu().long(), self.e[name])
        if self.w is not None:
            torch.testing.assert_close(pages.weight.cpu().double(), self.w, rtol=0, atol=0, equal_nan=True)
