"""Performance cases of the paged cache in e4m3: append, attention of single tokens, eviction by attention weight.

A page holds `bs` tokens of a sequence for every KV head, keys and values in e4m3 with a power of two for each page and head (`exponent`: the
least one in -100 .. 119 under which the page's largest number is at most 448).  Four kinds of work on one layer of it:

* "append":  the keys and values of new tokens go into their pages, then all positions are read back in order, as a later portion of a prompt needs
             them for its attention;
* "attend":  attention of one new token per sequence over its pages;
* "track":   the same, and every cached token's attention weight, summed over the heads of its group, is added to a sum kept beside the cache;
* "evict":   of every sequence the first and the last tokens and the heaviest of the others stay and go, in order, to pages of their own (the old ones
             may be shared with another sequence), which are then read back.

`listed` names the standing cases, `draw` gives more of the same ranges, `exact` restates each in 64 bits, one sequence after the other.
"""
from __future__ import annotations

import math
import random

import torch

own = False

LEAST, MOST, TOP = -100, 119, 448.0


def listed() -> list:
    return [
        # one token of a small model's only user, and its 300 positions read back: launches and little else
        dict(name="append_one", kind="append", batch=1, kv=12, dim=64, bs=16, dtype="bf16", low=299, high=299, new_low=1, new_high=1),
        # continuous batching: portions of prompts of odd lengths behind contexts of odd lengths, half-filled pages on either side
        dict(name="append_mixed", kind="append", batch=16, kv=8, dim=64, bs=16, dtype="bf16", low=0, high=2001, new_low=1, new_high=700),
        # the second half of a long prompt
        dict(name="append_prompt", kind="append", batch=1, kv=8, dim=128, bs=16, dtype="bf16", low=8192, high=8192, new_low=8192, new_high=8192),
        # one user of a small model
        dict(name="attend_one_small", kind="attend", batch=1, kv=12, group=1, dim=64, bs=16, dtype="bf16", low=300, high=300),
        # one user with a very long context: work for the whole GPU from 8 KV heads
        dict(name="attend_one_long", kind="attend", batch=1, kv=8, group=4, dim=128, bs=16, dtype="bf16", low=131072, high=131072),
        # a busy server: contexts of all lengths
        dict(name="attend_ragged", kind="attend", batch=64, kv=4, group=4, dim=128, bs=16, dtype="bf16", low=100, high=4000),
        # a full server with long contexts: the cache's bytes and nothing else
        dict(name="attend_full", kind="attend", batch=64, kv=8, group=4, dim=128, bs=16, dtype="bf16", low=4096, high=8192),
        # heads of 64, larger pages, 16-bit floats
        dict(name="attend_heads64", kind="attend", batch=48, kv=8, group=4, dim=64, bs=32, dtype="fp16", low=16, high=1024),
        # the same with attention weights: one user
        dict(name="track_one", kind="track", batch=1, kv=4, group=4, dim=128, bs=16, dtype="bf16", low=2047, high=2047),
        # the serving workload's prompt and output lengths
        dict(name="track_wide", kind="track", batch=24, kv=8, group=4, dim=128, bs=16, dtype="bf16", low=128, high=2560),
        # one sequence down to its budget
        dict(name="evict_one", kind="evict", batch=1, kv=4, dim=128, bs=16, low=2500, high=2500, keep=1024, recent=128, first=4),
        # a server that runs out of pages: sequences of all lengths, some of them within the budget
        dict(name="evict_batch", kind="evict", batch=24, kv=8, dim=128, bs=16, low=1500, high=8192, keep=2048, recent=256, first=4),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(("append", "attend", "track", "evict"))
        c = dict(kind=kind, batch=_log(rng, 1, 64), kv=rng.choice((1, 2, 4, 8, 12)), dim=rng.choice((64, 128)), bs=rng.choice((16, 16, 32, 64)))
        if kind == "append":
            low, new = _log(rng, 1, 8192) - 1, _log(rng, 1, 4096)
            c.update(dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), low=low, high=rng.randint(low, 8192), new_low=new, new_high=rng.randint(new, 4096))
        elif kind == "evict":
            keep, low = _log(rng, 17, 4096), _log(rng, 1, 16384)
            first, recent = rng.randint(0, 8), rng.randint(0, keep // 2)
            c.update(low=low, high=rng.randint(low, 16384), keep=keep, recent=recent, first=first)
        else:
            low = _log(rng, 1, 16384)
            c.update(group=rng.choice((1, 2, 4, 7, 8, 16)), dtype=rng.choice(("bf16", "bf16", "fp16")), low=low, high=rng.randint(low, 16384))
        padded = c["batch"] * (c["high"] + c.get("new_high", 0)) * c["kv"] * c["dim"]       # numbers of a padded batch's keys
        if padded <= 64 * 8192 * 8 * 128 and work(c)["bytes"] <= 4e8:
            return c


# ---- sizes ---------------------------------------------------------------------------------------------------------------------
def _between(count, low, high, salt) -> list:
    """`count` lengths from low to high: a property of the case, not of its seed."""
    if count == 1:
        return [high]
    r = random.Random(salt)
    return [low, high] + [r.randint(low, high) for _ in range(count - 2)]


def _lengths(c) -> list:
    return _between(c["batch"], c["low"], c["high"], 1)


def _new(c) -> list:
    return _between(c["batch"], c["new_low"], c["new_high"], 2)


def work(c) -> dict:
    """Codes, exponents, rows and sums that are read once, and results that are written once."""
    held, G, D, bs = _lengths(c), c["kv"], c["dim"], c["bs"]
    size = 4 if c.get("dtype") == "fp32" else 2
    pages = lambda lens: sum((n + bs - 1) // bs for n in lens)  # noqa: E731
    if c["kind"] == "append":
        new = _new(c)
        all_, rows = [a + b for a, b in zip(held, new)], sum(new)
        # new rows are read and their codes written; the codes of earlier positions are read; every position's row is written
        return dict(bytes=2.0 * (rows * G * D * (size + 1) + sum(held) * G * D + pages(all_) * G + sum(all_) * G * D * size), flops=2.0 * sum(all_) * G * D)
    if c["kind"] == "evict":
        kept = [min(n, c["keep"]) for n in held]
        # sums are read; codes and sums of what stays are read and written; the places are written; the pages are read back as bf16 rows
        return dict(bytes=4.0 * sum(held) * G + sum(kept) * G * (2 * D * 2 + 8 + 4) + 4.0 * pages(kept) * G + 2.0 * sum(kept) * G * D * 2, flops=2.0 * sum(held) * G)
    T, H = sum(held), G * c["group"]
    return dict(bytes=2.0 * T * G * D + 2.0 * pages(held) * G + 4.0 * c["batch"] * H * D + (8.0 * T * G if c["kind"] == "track" else 0.0), flops=4.0 * T * H * D)


# ---- what a program holds before the call ----------------------------------------------------------------------------------------
def _type(c):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[c.get("dtype", "bf16")]


def _two(e):
    """2^e in fp32 for whole numbers e from -126 to 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(a):
    """The least exponent under which a magnitude is at most 448 = 0.875 * 2^9."""
    m, x = torch.frexp(a)
    return torch.where(a > 0, x - 9 + (m > 0.875).to(x.dtype), LEAST).clamp(LEAST, MOST)


def _codes(x):
    return x.clamp(-TOP, TOP).to(torch.float8_e4m3fn)


def _pool(c, blocks, g):
    """Pages as earlier tokens left them: keys with a few strong channels, values without."""
    G, D, bs = c["kv"], c["dim"], c["bs"]
    got = []
    for strong in (4.0, 1.0):
        x = torch.empty((blocks, G, bs, D), device="cuda").normal_(0.0, 1.0, generator=g)
        x[..., :D // 16] *= strong
        x *= _two(torch.randint(-1, 2, (blocks, G, 1, 1), generator=g, device="cuda"))          # pages differ in size
        e = _exponent(x.abs().amax((2, 3)))
        got += [_codes(x.mul_(_two(-e)[:, :, None, None])), e.to(torch.int8)]
    return dict(k=got[0], k_exp=got[1], v=got[2], v_exp=got[3])


def _tables(lens, bs, order, at=0):
    """Block tables of sequences whose pages come out of `order` one after the other, and how many they are."""
    need = [(n + bs - 1) // bs for n in lens]
    t = torch.zeros((len(lens), max(max(need), 1)), dtype=torch.int32)
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t.cuda(), at


def _starts(lens) -> torch.Tensor:
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=g)  # noqa: E731
    held, G, D, bs = _lengths(c), c["kv"], c["dim"], c["bs"]
    new = _new(c) if c["kind"] == "append" else [0] * len(held)
    lens = [a + b for a, b in zip(held, new)]
    kept = [min(n, c["keep"]) for n in held] if c["kind"] == "evict" else []
    blocks = sum((n + bs - 1) // bs for n in lens + kept) + 3
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    s = dict(case=c, **_pool(c, blocks, g))
    s["tables"], at = _tables(lens, bs, order)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if c["kind"] == "append":
        s["k_new"], s["v_new"] = rand(sum(new), G * D).to(_type(c)), rand(sum(new), G * D).to(_type(c))
        s["first"], s["starts"], s["rows"] = _starts(new), _starts(lens), sum(lens)
    elif c["kind"] == "evict":
        s["out_tables"], _ = _tables(kept, bs, order, at)
        s["starts"], s["rows"] = _starts(kept), sum(kept)
        # sums of softmax weights: a few tokens have most of it, the newest have none yet
        w = torch.rand((blocks, G, bs), generator=g, device="cuda")
        s["weight"] = (w ** 8 * 20.0) * (torch.rand((blocks, G, bs), generator=g, device="cuda") < 0.95)
    else:
        s["q"] = rand(c["batch"], G * c["group"] * D).to(_type(c))
        s["weight"] = torch.rand((blocks, G, bs), generator=g, device="cuda") if c["kind"] == "track" else None
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        return _own(s)
    if c["kind"] == "append":
        _append(s)
        return _read(s, s["tables"], s["lens"], _type(c))
    if c["kind"] == "evict":
        return _evict(s)
    return _attend(s)


def _own(s):
    from rustral_b200 import ops

    c = s["case"]
    pages = ops.PagesE4M3(s["k"], s["v"], s["k_exp"], s["v_exp"], s.get("weight"))
    if c["kind"] == "append":
        ops.kv_append_e4m3(pages, s["k_new"], s["v_new"], s["tables"], s["lens"], s["first"])
        return ops.kv_read_e4m3(pages, s["tables"], s["lens"], s["starts"], s["rows"], dtype=_type(c))
    if c["kind"] == "evict":
        lens, kept = ops.kv_evict_e4m3(pages, s["tables"], s["lens"], c["keep"], recent=c["recent"], keep_first=c["first"], out_tables=s["out_tables"])
        k, v = ops.kv_read_e4m3(pages, s["out_tables"], lens, s["starts"], s["rows"])
        return dict(lens=lens, kept=kept, k=k, v=v, weight=pages.weight)
    if c["kind"] == "attend":
        return ops.paged_attention_decode_e4m3(s["q"], pages, s["tables"], s["lens"])
    return ops.paged_attention_decode_e4m3(s["q"], pages, s["tables"], s["lens"], accumulate=True), pages.weight


def _rows_of(starts, rows):
    """(sequence, place in it) of every row of sequences that lie one behind the other."""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(starts[1:].contiguous(), r.to(torch.int32), right=True)
    return b, r - starts[b]


def _append(s):
    c, bs, G, D = s["case"], s["case"]["bs"], s["case"]["kv"], s["case"]["dim"]
    b, i = _rows_of(s["first"], s["k_new"].shape[0])
    pos = s["lens"][b] - (s["first"][b + 1] - s["first"][b]) + i
    page, off = s["tables"][b, pos // bs].long(), (pos % bs).long()
    blocks = s["k"].shape[0]
    begin = torch.full((blocks,), bs, device="cuda").scatter_reduce(0, page, off, "amin")            # first new slot of a page; bs: it gets none
    touched, fresh = (begin < bs)[:, None], (begin == 0)[:, None]
    held = torch.arange(bs, device="cuda") < torch.where(begin < bs, begin, 0)[:, None]
    for codes, exps, new in ((s["k"], s["k_exp"], s["k_new"]), (s["v"], s["v_exp"], s["v_new"])):
        x = new.float().view(-1, G, D)
        most = torch.zeros((blocks, G), device="cuda").scatter_reduce(0, page[:, None].expand(-1, G), x.abs().amax(-1), "amax")
        e = torch.where(touched, torch.where(fresh, _exponent(most), torch.maximum(exps.int(), _exponent(most))), exps.int())
        again = _codes(codes.float() * _two(exps.int() - e)[:, :, None, None])
        codes.view(torch.uint8).copy_(torch.where(held[:, None, :, None], again.view(torch.uint8), codes.view(torch.uint8)))
        codes.view(torch.uint8)[page, :, off] = _codes(x * _two(-e)[page][:, :, None]).view(torch.uint8)
        exps.copy_(e)


def _padded(s, codes, exps, tables):
    """Values [sequences, KV heads, positions, D] of the pages of every table."""
    t = tables.long()
    c = codes.view(torch.uint8)[t].view(torch.float8_e4m3fn).float()                                # [B, pages, G, bs, D]
    c *= _two(exps[t])[..., None, None]
    return c.transpose(1, 2).reshape(t.shape[0], codes.shape[1], -1, codes.shape[3])


def _read(s, tables, lens, dtype):
    b, i = _rows_of(s["starts"], s["rows"])
    out = [_padded(s, s[n], s[n + "_exp"], tables)[b, :, i].reshape(s["rows"], -1).to(dtype) for n in ("k", "v")]
    return tuple(out)


def _attend(s):
    c, tables, lens = s["case"], s["tables"], s["lens"]
    B, G, D, bs = c["batch"], c["kv"], c["dim"], c["bs"]
    k = _padded(s, s["k"], s["k_exp"], tables)
    there = torch.arange(k.shape[2], device="cuda") < lens[:, None]                                 # [B, positions]
    x = (s["q"].float().view(B, G, c["group"], D) @ k.transpose(2, 3)) / math.sqrt(D)
    del k
    x.masked_fill_(~there[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    v = _padded(s, s["v"], s["v_exp"], tables).masked_fill_(~there[:, None, :, None], 0.0)
    out = (p @ v).reshape(B, -1).to(_type(c))
    if c["kind"] == "attend":
        return out
    b, i = there.nonzero(as_tuple=True)
    s["weight"][tables[b, i // bs].long(), :, i % bs] += p.sum(2)[b, :, i]
    return out, s["weight"]


def _evict(s):
    c, tables, lens = s["case"], s["tables"], s["lens"]
    B, G, D, bs, keep = c["batch"], c["kv"], c["dim"], c["bs"], c["keep"]
    t = tables.long()
    w = s["weight"][t].transpose(1, 2).reshape(B, G, -1)
    L = max(w.shape[2], keep)
    w = torch.nn.functional.pad(w, (0, L - w.shape[2]))
    at, n = torch.arange(L, device="cuda"), lens[:, None, None]
    key = torch.where((at < c["first"]) | (at >= n - c["recent"]), math.inf, w)
    key = torch.where(at < n, key, -math.inf)
    kept = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values      # [B, G, keep]
    kept = torch.where(kept < n, kept, -1)
    out_lens = lens.clamp(max=keep)
    # pages, slots and exponents that the kept tokens come from
    safe, h = kept.clamp_min(0), torch.arange(G, device="cuda")[None, :, None]
    page, off = t.gather(1, (safe // bs).view(B, -1)).view_as(safe), safe % bs
    pad = -keep % bs
    out_t = torch.nn.functional.pad(s["out_tables"].long(), (0, (keep + bs - 1) // bs - s["out_tables"].shape[1]))
    b, place = (torch.arange(keep, device="cuda") < out_lens[:, None]).nonzero(as_tuple=True)
    for name in ("k", "v"):
        e = torch.where(kept >= 0, s[name + "_exp"][page, h].int(), -128)
        top = torch.nn.functional.pad(e, (0, pad), value=-128).view(B, G, -1, bs).amax(-1)
        to = top.repeat_interleave(bs, -1)[..., :keep]
        x = s[name].view(torch.uint8)[page, h, off].view(torch.float8_e4m3fn).float() * _two((e - to).clamp(-126, 0))[..., None]
        s[name].view(torch.uint8)[out_t[b, place // bs], :, place % bs] = _codes(x).view(torch.uint8)[b, :, place]
        s[name + "_exp"][out_t[b, place // bs]] = to[b, :, place].to(torch.int8)
    s["weight"][out_t[b, place // bs], :, place % bs] = s["weight"][page, h, off][b, :, place]
    k, v = _read(s, s["out_tables"], out_lens, torch.bfloat16)
    return dict(lens=out_lens, kept=kept.int(), k=k, v=v, weight=s["weight"])


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------------------
def _round8(x):
    """The nearest e4m3 numbers, ties to even: a step is 2^-9 below 2^-6, an eighth of the power of two below it elsewhere."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _least(a) -> torch.Tensor:
    """The exponents of magnitudes, by trying."""
    e = torch.floor(torch.log2(a.clamp_min(1e-300))) - 9
    for _ in range(2):
        e = torch.where(TOP * torch.exp2(e) < a, e + 1, e)
    return e.clamp(LEAST, MOST)


def _sequence(s, name, b, tables, n, bs):
    """(values [positions, KV heads, D], exponents [pages, KV heads]) of one sequence, 64 bits."""
    table = tables[b, :(n + bs - 1) // bs].long()
    e = s[name + "_exp"][table].double()
    x = s[name][table].double() * torch.exp2(e)[:, :, None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n], e


def exact(c, seed):
    if c["batch"] * c["high"] * c["kv"] * c["dim"] > 64 * 8192 * 8 * 128:
        return None
    s = prepare(c, seed)
    held, bs, G, D = _lengths(c), c["bs"], c["kv"], c["dim"]
    if c["kind"] == "append":
        out, at = dict(k=[], v=[]), 0
        for b, (n, m) in enumerate(zip(held, _new(c))):
            for name in ("k", "v"):
                new = s[name + "_new"][at:at + m].double().view(m, G, D)
                old, e = _sequence(s, name, b, s["tables"], n, bs)
                whole = n // bs * bs                                              # positions in pages that get no new token
                parts = [old[:whole]]
                rest, at_page = torch.cat([old[whole:], new]), n // bs
                for i in range(0, rest.shape[0], bs):                             # page by page behind them
                    x, had = rest[i:i + bs], max(0, min(bs, n - whole - i))
                    scale = _least(x[had:].abs().amax((0, 2))) if x.shape[0] > had else None
                    if had and i == 0:
                        scale = e[at_page] if scale is None else torch.maximum(e[at_page], scale)
                    two = torch.exp2(scale)[None, :, None]
                    parts.append(_round8(x / two) * two)
                out[name].append(torch.cat(parts).reshape(n + m, -1))
            at += m
        return torch.cat(out["k"]), torch.cat(out["v"])
    if c["kind"] == "evict":
        lens, kept_all, weight, out = [], [], s["weight"].double(), dict(k=[], v=[])
        for b, n in enumerate(held):
            w, _ = _sequence(dict(w=s["weight"][..., None], w_exp=torch.zeros_like(s["k_exp"])), "w", b, s["tables"], n, bs)
            w = w[..., 0]                                                          # [positions, KV heads]
            m = min(n, c["keep"])
            kept = torch.full((G, c["keep"]), -1, dtype=torch.int32, device="cuda")
            for h in range(G):
                if n <= c["keep"]:
                    places = torch.arange(n, device="cuda")
                else:
                    f, r = c["first"], c["recent"]
                    middle = sorted(range(f, n - r), key=lambda j, x=w[:, h].tolist(): (-x[j], j))[:m - f - r]
                    places = torch.tensor(list(range(f)) + sorted(middle) + list(range(n - r, n)), device="cuda")
                kept[h, :m] = places
            for name in ("k", "v"):
                x, e = _sequence(s, name, b, s["tables"], n, bs)
                rows = torch.stack([x[kept[h, :m].long(), h] for h in range(G)], 1)          # [m, G, D]
                from_ = torch.stack([e[kept[h, :m].long() // bs, h] for h in range(G)], 1)
                for i in range(0, m, bs):
                    two = torch.exp2(from_[i:i + bs].amax(0))[None, :, None]
                    rows[i:i + bs] = _round8(rows[i:i + bs] / two) * two
                out[name].append(rows.reshape(m, -1))
            at = torch.arange(m, device="cuda")
            for h in range(G):
                weight[s["out_tables"][b, at // bs].long(), h, at % bs] = w[kept[h, :m].long(), h]
            lens.append(m)
            kept_all.append(kept)
        return dict(lens=torch.tensor(lens, dtype=torch.int32), kept=torch.stack(kept_all), k=torch.cat(out["k"]), v=torch.cat(out["v"]), weight=weight)
    outs, weight = [], s["weight"].double() if c["kind"] == "track" else None
    for b, n in enumerate(held):
        q = s["q"][b].double().view(G, c["group"], D)
        k, v = (_sequence(s, name, b, s["tables"], n, bs)[0] for name in ("k", "v"))
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(D), -1)
        outs.append(torch.einsum("hgn,nhd->hgd", p, v).reshape(-1))
        if weight is not None:
            at = torch.arange(n, device="cuda")
            weight[s["tables"][b, at // bs].long(), :, at % bs] += p.sum(1).t()
    return torch.stack(outs) if weight is None else (torch.stack(outs), weight)
