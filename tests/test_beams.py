"""Continuations of one prompt (ops.beams) against their definitions in 64 bits: on the host and, marked `gpu`, the kernels.

Selected rows and tokens and moved rows are compared bit for bit.  A score's 64-bit sum is rounded once to fp32 (half a step), and the 32-bit sum of exponentials under
it may be off: each exponential by 2^-21 of itself (the argument of the base-2 exponential is rounded to 24 bits at sizes up to 2^5 where its term counts, and
the instruction's own error is 2^-22), the additions of n numbers in chains of at most 64 and trees of 8 levels by 72 * 2^-24; together below 2^-17, which is the error of
the logarithm.  Attention: see `bound`."""
import math

import pytest
import torch

from rustral_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
I32 = torch.int32
INF = math.inf


# ---- selection -----------------------------------------------------------------------------------------------------------------------------
def choose(logits, scores, count, ended=None, end_token=0):
    """The definition, one place after the other, in Python's 64-bit floats."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    top = torch.finfo(torch.float32).max
    got = ([], [], [])
    for g in range(groups):
        totals = []
        for k in range(beams):
            r = g * beams + k
            s = float(scores[g, k])
            s = -INF if s != s else min(s, top)
            if ended is not None and bool(ended[g, k]):
                line = [-INF] * vocab
                line[end_token] = s
            else:
                x = [-INF if v != v else min(v, top) for v in logits[r].double().tolist()]
                m = max(x)
                if m == -INF or s == -INF:
                    line = [-INF] * vocab
                else:
                    lse = math.log(math.fsum(math.exp(v - m) for v in x))
                    line = [s + ((v - m) - lse) for v in x]
            totals += line
        order = sorted(range(len(totals)), key=lambda i: (-totals[i], i))[:count]
        got[0].append([totals[i] for i in order])
        got[1].append([g * beams + i // vocab for i in order])
        got[2].append([i % vocab for i in order])
    return torch.tensor(got[0], dtype=torch.float64), torch.tensor(got[1]), torch.tensor(got[2])


def same_choice(got, want):
    scores, rows, tokens = (t.cpu() for t in got)
    assert scores.dtype is torch.float32 and rows.dtype is tokens.dtype is torch.int64
    assert torch.equal(rows, want[1]) and torch.equal(tokens, want[2])
    finite = want[0].isfinite()
    assert torch.equal(scores.isfinite(), finite) or (want[0].abs() > 3.4e38).any()
    w, s = want[0][finite], scores[finite].double()
    assert ((s - w).abs() <= 2.0 ** -17 + w.abs() * 2.0 ** -24).all()


SELECTIONS = [
    # groups, beams, vocabulary, count, type, live beams, ended beams, share of tokens that are not allowed
    (1, 1, 1, 1, torch.float32, 1, 0, 0.0),
    (1, 4, 1, 4, torch.bfloat16, 4, 0, 0.0),
    (2, 3, 7, 21, torch.float32, 3, 0, 0.0),                  # every continuation there is
    (3, 3, 5, 12, torch.float16, 3, 1, 0.5),                  # fewer than asked for
    (1, 4, 1000, 8, torch.bfloat16, 1, 0, 0.01),              # the first step
    (5, 6, 2049, 12, torch.float32, 6, 2, 0.01),
    (2, 2, 8192, 4, torch.bfloat16, 2, 0, 0.0),
    (2, 4, 8193, 8, torch.float16, 4, 1, 0.0),
    (1, 32, 5003, 64, torch.bfloat16, 32, 4, 0.02),
    (1, 2, 50257, 128, torch.float32, 2, 0, 0.001),
    (70, 3, 300, 5, torch.float32, 3, 0, 0.0),
    (1, 2, 9000, 3, torch.bfloat16, 2, 0, 0.999),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(SELECTIONS)))
def test_beam_select(device, case):
    groups, beams, vocab, count, dtype, alive, over, banned = SELECTIONS[case]
    g = torch.Generator().manual_seed(case)
    padded = torch.full((groups * beams, vocab + 3 + 5 * (case % 3)), 1e4, dtype=dtype)
    logits = padded[:, :vocab]
    logits.copy_(torch.randn(groups * beams, vocab, generator=g) * 2.5)
    logits[torch.rand(logits.shape, generator=g) < banned] = -INF
    scores = -20.0 - 3.0 * torch.rand(groups, beams, generator=g)
    scores[:, alive:] = -INF
    ended = None
    if over:
        ended = torch.zeros(groups, beams, dtype=torch.bool)
        ended[:, torch.randperm(beams, generator=g)[:over]] = True
    want = choose(logits, scores, count, ended, vocab // 2)
    got = ops.beam_select(padded.to(device)[:, :vocab], scores.to(device), count, None if ended is None else ended.to(device), vocab // 2)
    same_choice(got, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_beam_select_of_infinities_and_nan(device, dtype):
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0, 3], x[0, 9] = math.nan, -INF
    x[1, 5] = x[1, 30] = INF                                     # share what there is
    x[2] = -INF                                                  # nothing allowed
    x[3] = torch.finfo(dtype).min                                # masked by the type's least number: all equal
    x[4] = math.nan
    x[5, 7] = torch.finfo(dtype).max
    scores = torch.tensor([[-1.0, -2.0, -3.0], [-0.5, math.nan, -2.0]])
    for count in (1, 4, 60, 120):
        same_choice(ops.beam_select(x.to(device), scores.to(device), count), choose(x, scores, count))


@pytest.mark.parametrize("device", DEVICES)
def test_beam_select_of_equal_logits(device):
    """Equal sums go to the lowest row and token, however many there are; -0 and 0 are equal."""
    scores = torch.tensor([[-1.0, -1.0, -2.0]])
    x = torch.zeros(3, 30000)
    x[:, ::2] = -0.0
    scores_, rows, tokens = ops.beam_select(x.to(device), scores.to(device), 128)
    assert rows.tolist() == [[0] * 128] and tokens.tolist() == [list(range(128))]
    assert (scores_.cpu().double() + 1.0 + math.log(30000)).abs().max() <= 2.0 ** -17 + 12 * 2.0 ** -24
    x = torch.zeros(3, 100)
    same_choice(ops.beam_select(x.to(device), scores.to(device), 128), choose(x, scores, 128))
    x = torch.full((3, 20000), -5.0)                              # plateaus in the second beam
    x[1, 4000:9000] = 2.0
    same_choice(ops.beam_select(x.bfloat16().to(device), scores.to(device), 100), choose(x, scores, 100))


@pytest.mark.parametrize("device", DEVICES)
def test_beam_select_sorted_logits(device):
    """Neighbouring tokens in order of their size: the best of a row all lie in the hands of a few threads."""
    x = torch.stack([torch.linspace(-3, 9, 20001), torch.linspace(9, -3, 20001), torch.linspace(-8, 8, 20001)])
    scores = torch.tensor([[-1.0, -1.5, -0.25]])
    for count in (1, 7, 128):
        same_choice(ops.beam_select(x.to(device), scores.to(device), count), choose(x, scores, count))


@pytest.mark.parametrize("device", DEVICES)
def test_beam_select_no_groups(device):
    scores, rows, tokens = ops.beam_select(torch.zeros(0, 10, device=device), torch.zeros(0, 2, device=device), 4)
    assert scores.shape == rows.shape == tokens.shape == (0, 4)


@pytest.mark.parametrize("device", DEVICES)
def test_beam_select_refuses(device):
    x, s = torch.zeros(6, 10, device=device), torch.zeros(2, 3, device=device)
    for bad in (0, 31, -1):
        with pytest.raises(ValueError):
            ops.beam_select(x, s, bad)
    with pytest.raises(ValueError):
        ops.beam_select(x[:5], s, 2)
    with pytest.raises(TypeError):
        ops.beam_select(x.double(), s, 2)
    with pytest.raises(TypeError):
        ops.beam_select(x, s.half(), 2)
    ended = torch.zeros(2, 3, dtype=torch.bool, device=device)
    for token in (-1, 10):
        with pytest.raises(ValueError):
            ops.beam_select(x, s, 2, ended, token)
    with pytest.raises(TypeError):
        ops.beam_select(x, s, 2, ended.int(), 1)
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(2, 0, device=device), torch.zeros(1, 2, device=device), 1)


@pytest.mark.gpu
def test_beam_select_refuses_what_the_kernel_does_not_serve():
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(300, 4, device="cuda"), torch.zeros(1, 300, device="cuda"), 2)
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(2, 400, device="cuda"), torch.zeros(1, 2, device="cuda"), 129)
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros(2, 400, device="cuda"), torch.zeros(1, 2), 12)


# ---- moves -----------------------------------------------------------------------------------------------------------------------------------
def pieces(device, rows, dtype=torch.float32, seed=0):
    """Tensors whose rows (dimension 1) lie in memory in different ways, and copies of what they were made from."""
    g = torch.Generator().manual_seed(seed)
    whole = [torch.randn(3, rows, 5, generator=g), torch.randn(2, rows + 2, 4, 33, generator=g), torch.randn(1, rows, 1, generator=g), torch.randn(2, rows, 700, generator=g),
             torch.randn(rows, 2, 64, generator=g)]
    whole = [t.to(dtype).to(device) for t in whole]
    views = [whole[0], whole[1][:, 1:rows + 1, :, 1:17], whole[2], whole[3][:, :, 3:], whole[4].transpose(0, 1)]
    return whole, views


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype is not torch.bool else t


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn, torch.int64])
@pytest.mark.parametrize("rows,pairs", [(2, 1), (12, 5), (100, 50), (1500, 700)])
def test_copy_blocks(device, dtype, rows, pairs):
    whole, views = pieces(device, rows, dtype, rows)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    src[-1] = src[0]                                              # one block may be copied twice
    want = [t.clone() for t in whole]
    want_views = [want[0], want[1][:, 1:rows + 1, :, 1:17], want[2], want[3][:, :, 3:], want[4].transpose(0, 1)]
    for w, v in zip(want_views, views):
        for s, d in zip(src, dst):
            w[:, d] = v[:, s]
    ops.copy_blocks_(views, src, dst, dim=1)
    for w, t in zip(want, whole):
        assert torch.equal(bits(w), bits(t))


@pytest.mark.gpu
def test_copy_blocks_of_more_pairs_than_a_launch_takes():
    t = torch.randn(9000, 6, device="cuda")
    want = t.clone()
    want[4500:] = want[:4500]
    ops.copy_blocks_([t], range(4500), range(4500, 9000))
    assert torch.equal(t, want)


@pytest.mark.gpu
def test_copy_blocks_of_many_tensors():
    ts = [torch.randn(10, 3 + i, device="cuda") for i in range(75)]
    want = [t.clone() for t in ts]
    for w in want:
        w[[7, 2]] = w[[3, 9]]
    ops.copy_blocks_(ts, [3, 9], [7, 2])
    assert all(torch.equal(a, b) for a, b in zip(ts, want))


@pytest.mark.gpu
def test_copy_blocks_past_four_gigabytes():
    """Offsets of blocks and of layers that do not fit 32 bits."""
    t = torch.zeros(3, 50, 1 << 25, dtype=torch.uint8, device="cuda")           # 5 GB
    t[:, 1, ::4099] = torch.tensor([[3], [5], [7]], dtype=torch.uint8, device="cuda")
    ops.copy_blocks_([t], [1], [49], dim=1)
    assert torch.equal(t[:, 49], t[:, 1]) and t[:, 48].max() == 0 and t[:, 2].max() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_copy_blocks_refuses_and_copies_nothing(device):
    t = torch.arange(40.0, device=device).view(20, 2)
    want = t.clone()
    many = list(range(17, 0, -1))
    for src, dst in (([0], [20]), ([-1], [0]), ([20], [1]), ([0, 1], [2, 2]), ([0, 1], [2, 1]), ([0], [0]), ([0, 1], [2]), ([1 << 40], [2]), (["a"], [1]),
                     ([18] * 17, many[:-1] + [many[0]]), (many, [18] * 16 + [17]), (many, [0] + many[:-1])):
        with pytest.raises(ValueError):
            ops.copy_blocks_([t], src, dst)
    with pytest.raises(ValueError):
        ops.copy_blocks_([t, t], [0], [1])
    with pytest.raises(ValueError):
        ops.copy_blocks_([t, t[:10]], [0], [1])
    with pytest.raises(ValueError):
        ops.copy_blocks_([t], [0], [1], dim=2)
    with pytest.raises(ValueError):
        ops.copy_blocks_([t[:1].expand(5, 2)], [0], [1])
    assert torch.equal(t, want)
    ops.copy_blocks_([t], [], [])
    ops.copy_blocks_([], [0], [1])
    assert torch.equal(t, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("groups,group", [(1, 1), (1, 2), (3, 8), (2, 9), (4, 16), (1, 17), (2, 64), (1, 256)])
def test_reorder_rows(device, dtype, groups, group):
    rows = groups * group
    whole, views = pieces(device, rows, dtype, rows)
    g = torch.Generator().manual_seed(group)
    first = torch.arange(rows) // group * group
    maps = [first + torch.randint(0, group, (rows,), generator=g),                                   # any map
            torch.cat([i * group + torch.randperm(group, generator=g) for i in range(groups)]),      # cycles
            first + (torch.arange(rows) + 1) % group,                                                # one long cycle
            first, torch.arange(rows)]
    for index in maps:
        want = [t.clone() for t in whole]
        want_views = [want[0], want[1][:, 1:rows + 1, :, 1:17], want[2], want[3][:, :, 3:], want[4].transpose(0, 1)]
        for w in want_views:
            w.copy_(w.clone()[:, index.to(device)])
        ops.reorder_rows_(views, index.to(device), dim=1, group=group)
        for w, t in zip(want, whole):
            assert torch.equal(bits(w), bits(t))


@pytest.mark.parametrize("device", DEVICES)
def test_reorder_rows_without_groups_and_with_indices_outside(device):
    t = torch.randn(6, 4, device=device)
    was = t.clone()
    ops.reorder_rows_([t], torch.tensor([5, 4, 3, 2, 1, 0], device=device))
    assert torch.equal(t, was.flip(0))
    t.copy_(was)
    ops.reorder_rows_([t], torch.tensor([1, -1, 3, 5, 1 << 40, 4], device=device), group=2)
    # rows 1, 2, 3 and 4 name rows outside their groups (or none) and stay
    assert torch.equal(t, was[[1, 1, 3, 3, 4, 4]])


@pytest.mark.parametrize("device", DEVICES)
def test_reorder_rows_refuses(device):
    t, i = torch.zeros(6, 4, device=device), torch.zeros(6, dtype=torch.int64, device=device)
    with pytest.raises(TypeError):
        ops.reorder_rows_([t], i.int())
    for bad in (dict(index=i[:5]), dict(index=i, group=4), dict(index=i, group=0), dict(index=i, dim=1)):
        with pytest.raises(ValueError):
            ops.reorder_rows_([t], **bad)
    with pytest.raises(ValueError):
        ops.reorder_rows_([torch.zeros(2, 3, 4, 5, device=device).permute(3, 1, 0, 2)], i[:5])
    ops.reorder_rows_([], i)
    ops.reorder_rows_([torch.zeros(0, 4, device=device)], i[:0])
    ops.reorder_rows_([torch.zeros(6, 0, device=device)], i)


@pytest.mark.parametrize("device", DEVICES)
def test_moves_refuse_memory_that_is_there_twice(device):
    """One tensor in place of a list, rows that overlap, an index among the tensors; tensors may come from a generator."""
    base, i = torch.arange(36.0, device=device), torch.tensor([1, 0, 2, 3, 4, 5], device=device)
    rows = base[:30].view(6, 5)
    for t in (base.as_strided((6, 8), (4, 1)), base.as_strided((2, 6, 3), (4, 4, 1)), base.as_strided((6, 2, 3), (4, 2, 1))):
        with pytest.raises(ValueError):
            ops.reorder_rows_([t], i, dim=1 if t.shape[0] == 2 else 0)
        with pytest.raises(ValueError):
            ops.copy_blocks_([t], [0], [1], dim=1 if t.shape[0] == 2 else 0)
    with pytest.raises(ValueError):
        ops.reorder_rows_([rows, i], i)
    with pytest.raises(TypeError):
        ops.reorder_rows_(base[:36].view(6, 6), i)
    with pytest.raises(TypeError):
        ops.copy_blocks_(base[:36].view(6, 6), [0], [1])
    assert torch.equal(base.cpu(), torch.arange(36.0)) and i.tolist() == [1, 0, 2, 3, 4, 5]
    ops.reorder_rows_((t for t in [rows]), i)
    ops.copy_blocks_((t for t in [rows.t()]), [2], [4], dim=1)
    assert rows[:, 0].tolist() == [5, 0, 10, 15, 10, 25]


@pytest.mark.gpu
def test_reorder_rows_refuses_what_the_kernel_does_not_serve():
    with pytest.raises(ValueError):
        ops.reorder_rows_([torch.zeros(257, 4, device="cuda")], torch.zeros(257, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.reorder_rows_([torch.zeros(6, 4, device="cuda")], torch.zeros(6, dtype=torch.int64))


# ---- attention over a shared prefix ------------------------------------------------------------------------------------------------------------
def forked(sizes, shared, lens, bs, kv, dim, dtype, seed, width=0, hole=math.nan):
    """Caches and tables of groups that were forked: full pages of what they share are the same, a page that it ends in was copied.  Slots behind every
    sequence's tokens hold `hole`, table entries behind its pages name none."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + bs - 1) // bs for n in lens]
    blocks = sum(need) + sum((p + bs - 1) // bs for p in shared) + 2
    order = torch.randperm(blocks, generator=g).tolist()
    k, v = (torch.full((blocks, bs, kv, dim), hole, dtype=dtype) for _ in range(2))
    t = torch.full((len(lens), max(need + [width, 1])), 1 << 30, dtype=I32)
    b = 0
    for n, p in zip(sizes, shared):
        full = [order.pop() for _ in range(p // bs)]
        tail = [torch.randn(p % bs, kv, dim, generator=g).to(dtype) for _ in range(2)]
        for x in (k, v):
            for page in full:
                x[page] = torch.randn(bs, kv, dim, generator=g).to(dtype)
        for i in range(b, b + n):
            pages = full[:need[i]] + [order.pop() for _ in range(max(0, need[i] - len(full)))]
            t[i, :need[i]] = torch.tensor(pages, dtype=I32)
            for x, end in zip((k, v), tail):
                for at in range(len(full) * bs, lens[i]):
                    x[pages[at // bs], at % bs] = end[at - len(full) * bs] if at < p else torch.randn(kv, dim, generator=g).to(dtype)
        b += n
    return k, v, t


def attend64(q, k, v, t, lens, scale):
    """softmax(q k scale) v of every sequence through its own table, 64 bits; and the largest magnitude of its values for each head and column."""
    bs, kv, dim = k.shape[1:]
    out, most = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(lens):
        if n:
            at = torch.arange(n)
            pages = t[b, at // bs].long()
            kk, vv = k[pages, at % bs].double(), v[pages, at % bs].double()
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b].double().view(kv, -1, dim), kk) * scale, -1)
            out[b] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(-1)
            most[b] = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(-1)
    return out, most


def bound(want, most, dtype):
    """A row's weights are rounded to `dtype` (half a step each, relative; fp16 ones below 2^-14 of the largest by 2^-25 of it), so its sum of weighted values is off by half a step of the
    sum of their weighted magnitudes at most; the 32-bit scores (sums of up to 128 products, |s| below 2^6) put 2^-14 on each weight's exponent at most; the result is
    rounded once."""
    half = torch.finfo(dtype).eps / 2
    return (half + 2.0 ** -12) * most + half * want.abs() + 2.0 ** -12


ATTENDED = [
    # group sizes, shared tokens, own tokens of every sequence, block size, KV heads, heads of each, head size, type
    ([1], [0], [1], 16, 1, 1, 64, torch.bfloat16),
    ([1], [1], [0], 16, 1, 4, 128, torch.bfloat16),
    ([4], [300], [1, 5, 17, 24], 16, 12, 1, 64, torch.bfloat16),
    ([4], [16], [1, 1, 1, 1], 16, 2, 4, 128, torch.bfloat16),
    ([3], [15], [1, 2, 130], 16, 2, 4, 64, torch.float16),
    ([2, 3, 1], [129, 0, 500], [3, 1, 0, 200, 1, 128], 16, 2, 8, 128, torch.bfloat16),
    ([5, 1, 7], [2000, 640, 33], [1, 40, 300, 2, 9, 77, 1, 2, 3, 4, 5, 6, 7], 16, 4, 4, 128, torch.float16),
    ([9], [257], [1] * 9, 16, 1, 7, 64, torch.bfloat16),
    ([40], [1000], list(range(40)), 16, 2, 4, 128, torch.bfloat16),
    ([33], [4097], [200] * 33, 32, 1, 12, 64, torch.bfloat16),
    ([20, 60], [900, 100], [7] * 80, 64, 2, 4, 128, torch.float16),
    ([70], [384], [1] * 70, 128, 1, 2, 128, torch.bfloat16),
    ([17], [200], [30] * 17, 256, 2, 8, 64, torch.bfloat16),
    ([6], [100], [30] * 6, 24, 2, 8, 64, torch.bfloat16),            # pages that no tile is a multiple of
    ([50], [100], [30] * 50, 5, 1, 8, 64, torch.bfloat16),
    ([3], [700], [1, 100, 10], 16, 1, 16, 128, torch.bfloat16),
    ([3], [700], [1, 100, 10], 16, 1, 40, 64, torch.bfloat16),        # more heads of a group than a tile has rows
    ([10], [260], [1] * 10, 16, 1, 71, 64, torch.bfloat16),
    ([300], [130], [2] * 300, 16, 1, 1, 64, torch.bfloat16),
    ([1] * 4090 + [3, 3], [1] * 4090 + [140, 20], [1 + i % 3 for i in range(4096)], 16, 1, 2, 64, torch.bfloat16),    # as many sequences as there may be
    ([2000, 2096], [40, 3], [1 + i % 3 for i in range(4096)], 16, 1, 1, 128, torch.float16),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(ATTENDED)))
def test_attention_shared(device, case):
    sizes, shared, mine, bs, kv, per, dim, dtype = ATTENDED[case]
    owner = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [shared[g] + n for g, n in zip(owner, mine)]
    k, v, t = forked(sizes, shared, lens, bs, kv, dim, dtype, case, width=(0, 40)[case % 2])
    packed = torch.full((len(lens), kv * per * dim + 24), 1e4, dtype=dtype)
    q = packed[:, 8:8 + kv * per * dim]
    q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(1000 + case)) * 2)
    scale = 1.0 / math.sqrt(dim) if case % 3 else 0.05
    want, most = attend64(q, k, v, t, lens, scale)
    dev = [x.to(device) for x in (packed, k, v, t, torch.tensor(shared, dtype=I32), torch.tensor(lens, dtype=I32))]
    got = ops.paged_attention_shared(dev[0][:, 8:8 + kv * per * dim], dev[1], dev[2], ops.PrefixGroups(sizes, device), dev[4], dev[3], dev[5], scale=scale)
    assert got.dtype is dtype and got.shape == q.shape
    assert ((got.cpu().double() - want).abs() <= bound(want, most, dtype)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sizes", [[5], [48]])
def test_attention_shared_of_short_sequences(device, sizes):
    """Sequences without tokens get zeros and take no part; of a group whose shortest has fewer tokens than it is said to share only those count, and what
    others hold behind them does not reach it."""
    n, bs, kv, per, dim = sizes[0], 16, 2, 4, 64
    lens = [500] * n
    lens[0], lens[2] = 0, 90
    k, v, t = forked([n], [400], lens, bs, kv, dim, torch.bfloat16, 3)
    t[0] = t[1]                                                    # the first row's table is the group's
    k[t[1, 200 // bs].long(), 200 % bs] = math.nan                 # a place that the short one does not see
    q = torch.randn(n, kv * per * dim, generator=torch.Generator().manual_seed(4)).bfloat16()
    out = torch.full_like(q, 7.0).to(device)
    for said in (400, 100000, -5):
        got = ops.paged_attention_shared(q.to(device), k.to(device), v.to(device), ops.PrefixGroups([n], device), torch.tensor([said], dtype=I32, device=device),
                                         t.to(device), torch.tensor(lens, dtype=I32, device=device), out=out)
        assert got is out and torch.equal(got[0].cpu(), torch.zeros(kv * per * dim, dtype=torch.bfloat16))
        want, most = attend64(q, k, v, t, lens, 0.125)
        assert ((got[2].cpu().double() - want[2]).abs() <= bound(want, most, torch.bfloat16)[2]).all()
        assert got[1].isnan().all() and got[3].isnan().all()       # theirs has the NaN


@pytest.mark.parametrize("device", DEVICES)
def test_attention_shared_refuses(device):
    k, v, t = forked([2], [16], [17, 18], 16, 2, 64, torch.bfloat16, 0)
    k, v, t = k.to(device), v.to(device), t.to(device)
    q = torch.zeros(2, 256, dtype=torch.bfloat16, device=device)
    shared, lens, groups = torch.tensor([16], dtype=I32, device=device), torch.tensor([17, 18], dtype=I32, device=device), ops.PrefixGroups([2], device)
    good = dict(q=q, k_cache=k, v_cache=v, groups=groups, shared_lens=shared, block_tables=t, context_lens=lens)
    for name, bad in (("q", q.float()), ("q", q.view(2, 4, 64)), ("k_cache", k.half()), ("k_cache", k[:, ::2]), ("shared_lens", shared.long()), ("shared_lens", lens),
                      ("block_tables", t[:1]), ("block_tables", t.long()), ("context_lens", shared), ("out", q.half())):
        with pytest.raises(TypeError):
            ops.paged_attention_shared(**{**good, name: bad})
    for name, bad in (("q", q[:, :200]), ("groups", ops.PrefixGroups([1, 2], device)), ("q", q[:, :64])):
        with pytest.raises(ValueError):
            ops.paged_attention_shared(**{**good, name: bad})
    with pytest.raises(ValueError):
        ops.PrefixGroups([2, 0])
    empty = ops.paged_attention_shared(q[:0], k, v, ops.PrefixGroups([], device), shared[:0], t[:0], lens[:0])
    assert empty.shape == (0, 256)


@pytest.mark.gpu
def test_attention_shared_refuses_what_the_kernel_does_not_serve():
    k = torch.zeros(4, 16, 1, 64, device="cuda")
    lens, t = torch.tensor([3], dtype=I32, device="cuda"), torch.zeros(1, 2, dtype=I32, device="cuda")
    with pytest.raises(ValueError):
        ops.paged_attention_shared(torch.zeros(1, 64, device="cuda"), k, k, ops.PrefixGroups([1], "cuda"), lens, t, lens)
    k = torch.zeros(4, 16, 1, 96, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.paged_attention_shared(torch.zeros(1, 96, device="cuda", dtype=torch.bfloat16), k, k, ops.PrefixGroups([1], "cuda"), lens, t, lens)


@pytest.mark.gpu
def test_attention_shared_captured_and_twice_the_same():
    """Two captured graphs and eager calls between their replays, new lengths without a new capture, bit for bit."""
    sizes, shared, bs, kv, per, dim = [6, 30], [700, 300], 16, 2, 4, 128
    lens = [s + 20 + i for i, s in enumerate([700] * 6 + [300] * 30)]
    k, v, t = (x.cuda() for x in forked(sizes, shared, lens, bs, kv, dim, torch.bfloat16, 9))
    q = torch.randn(36, kv * per * dim, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    groups, sh, ln = ops.PrefixGroups(sizes, "cuda"), torch.tensor(shared, dtype=I32, device="cuda"), torch.tensor(lens, dtype=I32, device="cuda")
    call = lambda: ops.paged_attention_shared(q, k, v, groups, sh, t, ln)  # noqa: E731
    want = call()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    ln.sub_(torch.arange(36, device="cuda", dtype=I32) % 7)
    less = call()
    for g, out in graphs:
        g.replay()
        assert torch.equal(out, less)
    ln.copy_(torch.tensor(lens, dtype=I32))
    for g, out in reversed(graphs):
        g.replay()
        again = call()
        assert torch.equal(out, want) and torch.equal(again, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_beam_select_of_many_rows(dtype):
    """Rows of several tiles each: random ones, rising, falling, level, with a plateau, and with infinities and NaN; a vocabulary that ends inside a tile, rows that begin on 16
    bytes and rows that do not."""
    beams, vocab, groups = 16, 40011, 40
    g = torch.Generator(device="cuda").manual_seed(5)
    for pad in (5, 6 if dtype is torch.float32 else 4):
        x = torch.empty(groups * beams, vocab + pad, device="cuda").normal_(0.0, 2.5, generator=g).to(dtype)[:, :vocab]
        ramp = torch.linspace(-6, 6, vocab, device="cuda").to(dtype)
        x[1 * beams:2 * beams] = ramp
        x[2 * beams:3 * beams] = ramp.flip(0)
        x[3 * beams:4 * beams] = 0.5
        x[4 * beams:5 * beams, 7000:30000] = 9.0
        x[5 * beams:6 * beams, 39000:] = -math.inf
        x[6 * beams + 1, 5], x[6 * beams + 2, 33333], x[6 * beams + 3, 20000:20007] = math.nan, math.inf, math.inf
        x[7 * beams:8 * beams] = -math.inf
        x[7 * beams + 3, 40000:40005] = 1.0
        scores = -5.0 - torch.rand(groups, beams, generator=g, device="cuda")
        for count in (3, 32, 128):
            got = ops.beam_select(x, scores, count)
            want = ops.beam_select(x.cpu(), scores.cpu(), count)               # the definition in 64 bits, tested above
            assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
            finite = want[0].isfinite()
            assert torch.equal(got[0].cpu().isfinite(), finite)
            w = want[0][finite].double()
            assert ((got[0].cpu()[finite].double() - w).abs() <= 2.0 ** -17 + w.abs() * 2.0 ** -23).all()     # both rounded to fp32
