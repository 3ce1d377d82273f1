"""Performance cases of decoding several continuations of a prompt: selection of beams, their states, their pages, attention over what they share.

Four kinds of work:

* "select":  of every group of beams the best continuations over beams and vocabulary, by the sums of their tokens' logarithmic probabilities;
* "reorder": states of a batch (dense caches of keys and values, recurrent cells) take the order of the selected beams, in place;
* "copy":    blocks of a paged cache (or slots of recurrent state) are copied to other blocks, in all layers;
* "attend":  attention of one new token per sequence over a paged cache in which the sequences of a group share their first tokens' pages.

`listed` names the standing cases, `draw` gives more of the same ranges, `exact` restates each in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False


def listed() -> list:
    return [
        # the first step of beam search on one prompt: one live beam, a small model's vocabulary
        dict(name="select_first", kind="select", groups=1, beams=4, vocab=50257, count=8, dtype="bf16", alive=1, ended=0),
        # one user, later on: two beams have ended, logits in 32 bits
        dict(name="select_ended", kind="select", groups=1, beams=8, vocab=128256, count=16, dtype="fp32", alive=8, ended=2),
        # a batch of prompts, the wide vocabulary
        dict(name="select_batch", kind="select", groups=64, beams=4, vocab=128256, count=8, dtype="bf16", alive=4, ended=0),
        # hidden states of a two-layer recurrent model under one beam search
        dict(name="reorder_cells", kind="reorder", form="cells", groups=1, beams=8, layers=2, width=512, dtype="fp32"),
        # dense caches of a small decoder: four prompts, the filled part of the cache
        dict(name="reorder_caches", kind="reorder", form="caches", groups=4, beams=4, layers=4, heads=12, room=1024, length=1000, dim=64, dtype="bf16"),
        # a step of beam search on a small model: the last, half-filled page of three beams, in every layer
        dict(name="copy_step", kind="copy", form="pages", layers=12, blocks=200, bs=16, heads=12, dim=64, pairs=3, dtype="bf16"),
        # recurrent states of sequences that were forked
        dict(name="copy_states", kind="copy", form="slots", layers=4, blocks=24, heads=32, state=128, dim=128, taps=3, channels=10240, pairs=7, dtype="bf16"),
        # pages moved together: what is in use goes to the front of a fragmented cache
        dict(name="copy_compact", kind="copy", form="pages", layers=8, blocks=700, bs=16, heads=8, dim=128, pairs=256, dtype="bf16"),
        # four beams of a small model's only user
        dict(name="attend_beams", kind="attend", groups=1, low=4, high=4, shared_low=300, shared_high=300, own_low=1, own_high=24, kv=12, group=1, dim=64, bs=16,
             dtype="bf16"),
        # prompts of all lengths with eight beams each, grouped heads
        dict(name="attend_groups", kind="attend", groups=12, low=8, high=8, shared_low=100, shared_high=8000, own_low=1, own_high=200, kv=8, group=4, dim=128, bs=16,
             dtype="bf16"),
        # one long document, several answers sampled from it
        dict(name="attend_document", kind="attend", groups=1, low=16, high=16, shared_low=32771, shared_high=32771, own_low=40, own_high=600, kv=8, group=4, dim=128, bs=16,
             dtype="bf16"),
        # a full server behind one long system prompt
        dict(name="attend_system", kind="attend", groups=1, low=256, high=256, shared_low=16384, shared_high=16384, own_low=16, own_high=512, kv=8, group=4, dim=128, bs=16,
             dtype="bf16"),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(("select", "reorder", "copy", "attend"))
        c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp16")))
        if kind == "select":
            beams = _log(rng, 1, 32)
            c.update(groups=_log(rng, 1, 256), beams=beams, vocab=_log(rng, 256, 131072), count=rng.randint(beams, 2 * beams),
                     alive=rng.choice((1, beams)), ended=rng.randint(0, beams // 3), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
        elif kind == "reorder":
            c.update(groups=_log(rng, 1, 32), beams=rng.randint(2, 16), layers=rng.randint(1, 8), dtype=rng.choice(("bf16", "fp16", "fp32")))
            if rng.random() < 0.5:
                c.update(form="cells", width=_log(rng, 30, 8192))
            else:
                room = _log(rng, 8, 2048)
                c.update(form="caches", heads=rng.choice((1, 2, 4, 8, 12)), room=room, length=rng.randint(1, room), dim=rng.choice((64, 128)))
        elif kind == "copy":
            blocks = _log(rng, 8, 1000)
            c.update(layers=rng.randint(1, 16), blocks=blocks, heads=rng.choice((1, 2, 4, 8, 12)), pairs=rng.randint(1, blocks // 2))
            if rng.random() < 0.5:
                c.update(form="pages", bs=rng.choice((16, 16, 32, 64)), dim=rng.choice((64, 128)), dtype=rng.choice(("bf16", "fp16", "fp32")))
            else:
                c.update(form="slots", state=rng.choice((16, 64, 128)), dim=rng.choice((64, 128)), taps=3, channels=rng.randint(30, 2000))
        else:
            low, shared, mine = _log(rng, 1, 256), _log(rng, 1, 32768), _log(rng, 1, 1024)
            c.update(groups=_log(rng, 1, 64), low=low, high=rng.randint(low, 256), shared_low=shared, shared_high=rng.randint(shared, 32768), own_low=mine,
                     own_high=rng.randint(mine, 1024), kv=rng.choice((1, 2, 4, 8, 12)), group=rng.choice((1, 2, 4, 7, 8, 16)), dim=rng.choice((64, 128)),
                     bs=rng.choice((16, 16, 32, 64)))
            if sum(_sizes(c)) > 256:
                continue
        w = work(c)
        if w["bytes"] <= 3.4e8 and w["flops"] <= 7e10 and _held(c) <= 1e9:
            return c


# ---- sizes ---------------------------------------------------------------------------------------------------------------------
def _between(count, low, high, salt) -> list:
    """`count` numbers from low to high: a property of the case, not of its seed."""
    r = random.Random(salt)
    return ([high] if count == 1 else [low, high] + [r.randint(low, high) for _ in range(count - 2)]) if count else []


def _sizes(c) -> list:
    return _between(c["groups"], c["low"], c["high"], 1)


def _lengths(c) -> tuple:
    """(shared tokens of every group, own tokens of every sequence)."""
    return _between(c["groups"], c["shared_low"], c["shared_high"], 2), _between(sum(_sizes(c)), c["own_low"], c["own_high"], 3)


def _parents(c) -> list:
    """The rows that a selection left: good beams have several children, each group's in the order of their scores."""
    r = random.Random(4)
    return [g * c["beams"] + min(r.randrange(c["beams"]), r.randrange(c["beams"])) for g in range(c["groups"]) for _ in range(c["beams"])]


def _blocks_of(c) -> tuple:
    """(blocks copied from, blocks copied to): all different."""
    order = random.Random(5).sample(range(c["blocks"]), 2 * c["pairs"])
    return order[:c["pairs"]], order[c["pairs"]:]


def _size(c) -> int:
    return 4 if c["dtype"] == "fp32" else 2


def _row(c) -> int:
    """Bytes of one row (block, slot) in all tensors."""
    if c["kind"] == "reorder":
        return 2 * c["layers"] * _size(c) * (c["width"] if c["form"] == "cells" else c["heads"] * c["length"] * c["dim"])
    if c["form"] == "pages":
        return 2 * c["layers"] * _size(c) * c["bs"] * c["heads"] * c["dim"]
    return c["layers"] * (4 * c["heads"] * c["state"] * c["dim"] + _size(c) * c["taps"] * c["channels"])


def _held(c) -> float:
    """Bytes of the state."""
    if c["kind"] == "select":
        return c["groups"] * c["beams"] * c["vocab"] * _size(c)
    if c["kind"] == "reorder":
        return _row(c) * c["groups"] * c["beams"] * (c["room"] / c["length"] if c["form"] == "caches" else 1.0)
    if c["kind"] == "copy":
        return _row(c) * c["blocks"]
    return work(c)["bytes"]


def work(c) -> dict:
    """Logits, states, keys and values that are read once, and results that are written once."""
    if c["kind"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return dict(bytes=float(n * _size(c) + c["groups"] * (4 * c["beams"] + 20 * c["count"])), flops=3.0 * n)
    if c["kind"] == "reorder":
        moved = [p for i, p in enumerate(_parents(c)) if p != i]
        return dict(bytes=float((len(moved) + len(set(moved))) * _row(c) + 8 * c["groups"] * c["beams"]), flops=0.0)
    if c["kind"] == "copy":
        return dict(bytes=2.0 * c["pairs"] * _row(c), flops=0.0)
    shared, mine = _lengths(c)
    sizes, heads = _sizes(c), c["kv"] * c["group"]
    tokens = sum(shared) + sum(mine)
    pairs = sum(n * p for n, p in zip(sizes, shared)) + sum(mine)
    return dict(bytes=4.0 * tokens * c["kv"] * c["dim"] + 4.0 * sum(sizes) * heads * c["dim"], flops=4.0 * pairs * heads * c["dim"])


# ---- what a program holds before the call ----------------------------------------------------------------------------------------
def _type(c):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[c["dtype"]]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, dtype=None, std=1.0):
        return torch.empty(shape, dtype=dtype or _type(c), device="cuda").normal_(0.0, std, generator=g)

    s = dict(case=c)
    if c["kind"] == "select":
        rows, vocab = c["groups"] * c["beams"], c["vocab"]
        # a head's logits for a vocabulary that was padded for the product; every hundredth token is not allowed here
        x = rand(rows, (vocab + 127) // 128 * 128, std=2.5)
        s["logits"] = x[:, :vocab]
        s["logits"][:, torch.randperm(vocab, generator=g, device="cuda")[:vocab // 100]] = -math.inf
        scores = -20.0 - 4.0 * torch.rand((c["groups"], c["beams"]), generator=g, device="cuda")
        scores[:, c["alive"]:] = -math.inf
        s["scores"], s["end"] = scores, vocab // 2
        s["ended"] = None
        if c["ended"]:
            s["ended"] = torch.zeros((c["groups"], c["beams"]), dtype=torch.bool, device="cuda")
            s["ended"][:, -c["ended"]:] = True
    elif c["kind"] == "reorder":
        rows = c["groups"] * c["beams"]
        if c["form"] == "cells":
            s["tensors"], s["dim"] = [rand(c["layers"], rows, c["width"]) for _ in range(2)], 1
        else:
            whole = [rand(rows, c["heads"], c["room"], c["dim"]) for _ in range(2 * c["layers"])]
            s["tensors"], s["dim"] = [t[:, :, :c["length"]] for t in whole], 0
        s["index"] = torch.tensor(_parents(c), dtype=torch.int64, device="cuda")
    elif c["kind"] == "copy":
        if c["form"] == "pages":
            s["tensors"], s["dim"] = [rand(c["layers"], c["blocks"], c["bs"], c["heads"], c["dim"]) for _ in range(2)], 1
        else:
            s["tensors"], s["dim"] = [], 0
            for _ in range(c["layers"]):
                s["tensors"] += [rand(c["blocks"], c["heads"], c["state"], c["dim"], dtype=torch.float32), rand(c["blocks"], c["taps"], c["channels"])]
        s["src"], s["dst"] = _blocks_of(c)
    else:
        _prepare_pages(c, s, rand, seed)
    return s


def _prepare_pages(c, s, rand, seed):
    """Pages of groups of sequences that were forked from one: full pages of what they share are the same, a page that it ends in was copied."""
    sizes, (shared, mine), bs = _sizes(c), _lengths(c), c["bs"]
    owner = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [shared[i] + n for i, n in zip(owner, mine)]
    common = [p // bs for p in shared]
    tail = [(n + bs - 1) // bs - common[i] for i, n in zip(owner, lens)]
    order = torch.randperm(sum(common) + sum(tail) + 3, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    s["k"], s["v"] = (rand(order.numel(), bs, c["kv"], c["dim"]) for _ in range(2))
    tables, at = torch.zeros((len(lens), max((n + bs - 1) // bs for n in lens)), dtype=torch.int32), 0
    firsts = [sum(sizes[:i]) for i in range(len(sizes))]
    for i, n in enumerate(common):
        tables[firsts[i]:firsts[i] + sizes[i], :n] = order[at:at + n]
        at += n
    for b, n in enumerate(tail):
        tables[b, common[owner[b]]:common[owner[b]] + n] = order[at:at + n]
        at += n
    for i, p in enumerate(shared):
        if p % bs:
            pages = tables[firsts[i]:firsts[i] + sizes[i], p // bs].long().cuda()
            for t in (s["k"], s["v"]):
                t[pages, :p % bs] = t[pages[:1], :p % bs]
    s["sizes"], s["firsts"], s["shared_host"], s["lens_host"] = sizes, firsts, shared, lens
    s["q"] = rand(len(lens), c["kv"] * c["group"] * c["dim"], std=2.0)
    s["tables"] = tables.cuda()
    s["shared"], s["lens"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (shared, lens))
    if own:
        from rustral_b200 import ops
        s["plan"] = ops.PrefixGroups(sizes, "cuda")


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s, kind)
    return {"select": _select, "reorder": _reorder, "copy": _copy, "attend": _attend}[kind](s)


def _own(s, kind):
    from rustral_b200 import ops

    if kind == "select":
        scores, rows, tokens = ops.beam_select(s["logits"], s["scores"], s["case"]["count"], ended=s["ended"], end_token=s["end"])
        return dict(scores=scores, rows=rows, tokens=tokens)
    if kind == "reorder":
        ops.reorder_rows_(s["tensors"], s["index"], dim=s["dim"], group=s["case"]["beams"])
        return s["tensors"]
    if kind == "copy":
        ops.copy_blocks_(s["tensors"], s["src"], s["dst"], dim=s["dim"])
        return s["tensors"]
    return ops.paged_attention_shared(s["q"], s["k"], s["v"], s["plan"], s["shared"], s["tables"], s["lens"])


def _select(s):
    """In 64 bits: of two continuations with nearly the same sum only one may be selected."""
    c = s["case"]
    x = s["logits"].double()
    x -= x.amax(1, keepdim=True)
    x -= torch.exp(x).sum(1, keepdim=True).log_()
    total = x.view(c["groups"], c["beams"], -1).add_(s["scores"].double()[..., None])
    if s["ended"] is not None:
        total.masked_fill_(s["ended"][..., None], -math.inf)
        total[:, :, s["end"]] = torch.where(s["ended"], s["scores"].double(), total[:, :, s["end"]])
    best = torch.sort(total.view(c["groups"], -1), dim=1, descending=True, stable=True)
    at = best.indices[:, :c["count"]]
    first = torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]
    return dict(scores=best.values[:, :c["count"]].float(), rows=first + at // c["vocab"], tokens=at % c["vocab"])


def _reorder(s):
    for t in s["tensors"]:
        t.copy_(t.index_select(s["dim"], s["index"]))
    return s["tensors"]


def _copy(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    for t in s["tensors"]:
        t.index_copy_(s["dim"], dst, t.index_select(s["dim"], src))
    return s["tensors"]


def _attend(s):
    """Group by group: scores over what it shares and over a padded gather of its sequences' own tokens, one softmax over both."""
    c = s["case"]
    G, R, D, bs = c["kv"], c["group"], c["dim"], c["bs"]
    out = torch.empty_like(s["q"])
    for b, n, shared in zip(s["firsts"], s["sizes"], s["shared_host"]):
        lens = s["lens"][b:b + n]
        most = max(s["lens_host"][b:b + n])
        common, pages = shared // bs, (most + bs - 1) // bs
        q = s["q"][b:b + n].float().view(n, G, R, D) / math.sqrt(D)
        first = s["tables"][b, :common].long()
        rest = s["tables"][b:b + n, common:pages].long()
        there = torch.arange(common * bs, pages * bs, device="cuda") < lens[:, None]
        # [KV heads, tokens, D] of the shared pages, [n, KV heads, tokens, D] of the others
        ks, vs = (s[t][first].float().view(-1, G, D).transpose(0, 1) for t in ("k", "v"))
        kr, vr = (s[t][rest].float().view(n, -1, G, D).transpose(1, 2) for t in ("k", "v"))
        flat = q.transpose(0, 1).reshape(G, n * R, D)
        x = torch.cat([(flat @ ks.transpose(1, 2)).view(G, n, R, -1).transpose(0, 1),
                       (q @ kr.transpose(2, 3)).masked_fill_(~there[:, None, None], -math.inf)], -1)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        x /= x.sum(-1, keepdim=True)
        cut = common * bs
        o = (x[..., :cut].transpose(0, 1).reshape(G, n * R, cut) @ vs).view(G, n, R, D).transpose(0, 1)
        o = o + x[..., cut:] @ vr.masked_fill_(~there[:, None, :, None], 0.0)
        out[b:b + n] = o.reshape(n, -1).to(out.dtype)
    return out


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "select":
        picked = dict(scores=[], rows=[], tokens=[])
        for g in range(c["groups"]):
            lo = g * c["beams"]
            x = s["logits"][lo:lo + c["beams"]].double()
            total = torch.log_softmax(x, 1) + s["scores"][g].double()[:, None]
            if s["ended"] is not None:
                for k in s["ended"][g].nonzero()[:, 0].tolist():
                    total[k] = -math.inf
                    total[k, s["end"]] = s["scores"][g, k].double()
            flat = total.flatten()
            taken = torch.zeros_like(flat, dtype=torch.bool)
            for _ in range(c["count"]):
                most = flat.masked_fill(taken, -math.inf).max()
                at = int(((flat == most) & ~taken).int().argmax())         # the first of equal ones
                taken[at] = True
                picked["scores"].append(most)
                picked["rows"].append(lo + at // c["vocab"])
                picked["tokens"].append(at % c["vocab"])
        shape = (c["groups"], c["count"])
        return dict(scores=torch.stack(picked["scores"]).view(shape), rows=torch.tensor(picked["rows"]).view(shape),
                    tokens=torch.tensor(picked["tokens"]).view(shape))
    if c["kind"] in ("reorder", "copy"):
        at = list(range(c["groups"] * c["beams"])) if c["kind"] == "reorder" else list(range(c["blocks"]))
        pairs = zip(at, _parents(c)) if c["kind"] == "reorder" else zip(*reversed(_blocks_of(c)))
        for to, of in pairs:
            at[to] = of
        return [t[:, at].double() if s["dim"] else t[at].double() for t in s["tensors"]]
    G, D, bs = c["kv"], c["dim"], c["bs"]
    outs = []
    for b, n in enumerate(s["lens_host"]):
        pages = s["tables"][b, :(n + bs - 1) // bs].long()
        k, v = (s[t][pages].reshape(-1, G, D)[:n].double() for t in ("k", "v"))
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", s["q"][b].double().view(G, -1, D), k) / math.sqrt(D), -1)
        outs.append(torch.einsum("hgn,nhd->hgd", p, v).reshape(-1))
    return torch.stack(outs)
