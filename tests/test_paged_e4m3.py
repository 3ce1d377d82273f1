"""The paged cache in e4m3 (ops.paged_e4m3) against its definition in 64 bits: on the host and, marked `gpu`, the kernels.

Codes, exponents, places and moved weights are compared bit for bit.  Attention outputs: the oracle gives the error that 16-bit softmax weights and
32-bit scores can make, and the output's own rounding is at most half a step (torch.finfo(type).eps / 2)."""
import pytest
import torch

from paged_e4m3_oracle import Cache
from rustral_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
I32 = torch.int32


def tables_of(lens, bs, blocks, seed, width=0):
    """A table row per sequence, pages in random order, entries behind a sequence's pages out of range."""
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
    need = [(n + bs - 1) // bs for n in lens]
    t = torch.full((len(lens), max(max(need), width, 1)), 1 << 30, dtype=I32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    assert at <= blocks
    return t


def filled(blocks, bs, G, D, seed, weights=False, spread=3):
    """Pages of random codes: what earlier owners left."""
    g = torch.Generator().manual_seed(seed)
    p = ops.PagesE4M3.zeros(blocks, bs, G, D, weights=weights)
    for codes, exps in ((p.k, p.k_exp), (p.v, p.v_exp)):
        codes.view(torch.uint8).copy_((torch.randn(codes.shape, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        exps.copy_(torch.randint(-spread - 5, spread - 4, exps.shape, generator=g))
    if weights:
        p.weight.copy_(torch.rand(p.weight.shape, generator=g))
    return p


def to(pages, device):
    return ops.PagesE4M3(*(None if t is None else t.to(device, copy=True) for t in (pages.k, pages.v, pages.k_exp, pages.v_exp, pages.weight)))


def starts_of(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def ints(x, device):
    return torch.tensor(x, dtype=I32, device=device)


APPENDS = [
    # batch of (tokens before, new), block size, KV heads, head size, type
    ([(0, 1)], 16, 1, 64, torch.bfloat16),
    ([(15, 1), (16, 1), (17, 1), (0, 1), (31, 2)], 16, 3, 64, torch.bfloat16),
    ([(0, 16), (0, 17), (5, 40), (16, 16), (3, 0), (100, 33)], 16, 2, 128, torch.bfloat16),
    ([(0, 0), (0, 129), (0, 0), (7, 1), (0, 0)], 32, 2, 64, torch.float16),
    ([(63, 65), (64, 64), (1, 200)], 64, 1, 128, torch.float32),
    ([(9, 300)], 48, 5, 64, torch.bfloat16),
    ([(100, 300), (0, 128)], 128, 2, 64, torch.float32),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(device, case):
    seqs, bs, G, D, dtype = APPENDS[case]
    lens, new = [a + n for a, n in seqs], [n for _, n in seqs]
    p0 = filled(sum((n + bs - 1) // bs for n in lens) + 4, bs, G, D, case, weights=case % 2 == 0)
    t = tables_of(lens, bs, p0.k.shape[0], case)
    g = torch.Generator().manual_seed(100 + case)
    rows = sum(new)
    # sizes from far below to far above what the pages hold: exponents that grow by much, by little and not at all
    size = torch.exp2(torch.randint(-18, 12, (rows, 1), generator=g).float())
    k = (torch.randn(rows, G * D, generator=g) * size).to(dtype)
    v = (torch.randn(rows, G * D, generator=g) * size.flip(0)).to(dtype)
    want = Cache(p0)
    want.append(k, v, t, lens, starts_of(new))
    p = to(p0, device)
    # rows as columns of a packed projection, and rows behind the last sequence that must not be stored
    packed = torch.full((rows + 3, 2 * G * D + 8), 1e4, dtype=dtype)
    packed[:rows, :G * D], packed[:rows, G * D + 8:] = k, v
    packed = packed.to(device)
    ops.kv_append_e4m3(p, packed[:, :G * D], packed[:, G * D + 8:], t.to(device), ints(lens, device), ints(starts_of(new), device))
    want.same(p)


@pytest.mark.parametrize("device", DEVICES)
def test_append_one_row_each(device):
    lens, bs, G, D = [1, 0, 16, 17, 40, 48, 900], 16, 4, 128
    p0 = filled(80, bs, G, D, 7, weights=True)
    t = tables_of(lens, bs, 80, 7)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(len(lens), G * D, generator=g).bfloat16() * s for s in (1.0, 30.0))
    want = Cache(p0)
    want.append(k, v, t, lens, list(range(len(lens) + 1)))
    p = to(p0, device)
    ops.kv_append_e4m3(p, k.to(device), v.to(device), t.to(device), ints(lens, device))
    want.same(p)


@pytest.mark.parametrize("device", DEVICES)
def test_append_token_by_token_is_the_page_at_once_but_for_subnormals(device):
    """Growing exponents keep numbers: with exponents that differ by 5 at most no code gets below the normal ones, and every number but those of
    the smallest sizes is what one rounding gives."""
    G, D, bs, n = 2, 64, 16, 37
    g = torch.Generator().manual_seed(3)
    size = torch.exp2(torch.randint(0, 6, (n, 1), generator=g).float())
    k = (torch.sign(torch.randn(n, G * D, generator=g)) * (1 + torch.rand(n, G * D, generator=g)) * size).to(device)
    t = ints([[2, 0, 1]], device)
    a, b = (ops.PagesE4M3.zeros(3, bs, G, D, device) for _ in range(2))
    ops.kv_append_e4m3(a, k, k, t, ints([n], device), ints([0, n], device))
    for i in range(n):
        ops.kv_append_e4m3(b, k[i:i + 1], k[i:i + 1], t, ints([i + 1], device))
    for x, y in ((a.k, b.k), (a.v, b.v), (a.k_exp, b.k_exp)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_special_numbers(device, dtype):
    """Zeros, infinities, NaN, the smallest and largest numbers, exact ties and the border of an exponent (448 and what follows it)."""
    G, D, bs = 1, 64, 16
    rows = torch.zeros(6, D)
    rows[1, :8] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0, -448.0, 449.0, 0.0, -0.0])
    rows[2, :3] = torch.tensor([1e-38, 2.0 ** -110, 1e-44])
    rows[3, :3] = torch.tensor([3.0e38, -1.0, 2.0 ** 100])
    rows[4, :8] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -7, 3 * 2.0 ** -10, 2.0 ** -10, 2.0 ** -11, 27.0])
    rows[5, :2] = torch.tensor([450.0, 2.0 ** -9])
    rows = rows.to(dtype)
    p0 = filled(8, bs, G, D, 1)
    t = torch.arange(6, dtype=I32).view(6, 1)
    want = Cache(p0)
    want.append(rows, rows, t, [1] * 6, list(range(7)))
    p = to(p0, device)
    ops.kv_append_e4m3(p, rows.to(device), rows.to(device), t.to(device), ints([1] * 6, device))
    want.same(p)
    assert p.k_exp[:6, 0].tolist() == want.e["k"][:6, 0].tolist()
    assert p.k_exp[0, 0] == -100 and p.k_exp[4, 0] == 0 and p.k_exp[5, 0] == 1
    assert torch.isnan(p.k.cpu().float()[1, 0, 0, 2])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("G,D,bs", [(1, 64, 16), (3, 128, 32), (8, 128, 16)])
def test_read(device, dtype, G, D, bs):
    lens = [0, 1, 15, 33, 0, 100, 64]
    p0 = filled(40, bs, G, D, 5)
    t, starts = tables_of(lens, bs, 40, 5, width=9), starts_of(lens)
    rows = starts[-1] + 5
    p = to(p0, device)
    k, v = (torch.full((rows, G * D + 8), 7.0, dtype=dtype, device=device)[:, :G * D] for _ in range(2))
    got = ops.kv_read_e4m3(p, t.to(device), ints(lens, device), ints(starts, device), rows, out=(k, v))
    assert got[0] is k and got[1] is v
    want = Cache(p0)
    for name, x in (("k", k), ("v", v)):
        ref = torch.cat([want.tokens(name, t, b, n).reshape(n, G * D) for b, n in enumerate(lens)])
        assert torch.equal(x[:starts[-1]].cpu().double(), ref)
        assert bool((x[starts[-1]:] == 7.0).all())                    # rows behind the last sequence
    k2, v2 = ops.kv_read_e4m3(p, t.to(device), ints(lens, device), ints(starts, device), starts[-1], dtype=dtype)
    assert torch.equal(k2, k[:starts[-1]]) and torch.equal(v2, v[:starts[-1]])


def check_attention(device, lens, G, group, D, bs, dtype, accumulate, seed=0, scale=None, spread=3, pages=None, width=0):
    blocks = sum((n + bs - 1) // bs for n in lens) + 2
    p0 = pages or filled(blocks, bs, G, D, seed, weights=accumulate, spread=spread)
    t = tables_of(lens, bs, p0.k.shape[0], seed, width)
    for b, n in enumerate(lens):                                      # what lies behind a sequence's last token in its page: NaN
        if n % bs:
            for codes in (p0.k, p0.v):
                codes.view(torch.uint8)[int(t[b, n // bs]), :, n % bs:] = 0x7f
    q = torch.randn(len(lens), G * group * D, generator=torch.Generator().manual_seed(seed + 50)).to(dtype)
    want, err, ws, wrel = Cache(p0).attend(q, t, lens, scale)
    p = to(p0, device)
    out = ops.paged_attention_decode_e4m3(q.to(device), p, t.to(device), ints(lens, device), scale, accumulate=accumulate)
    assert out.dtype is dtype
    off = (out.cpu().double() - want).abs()
    most = err + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal
    assert bool((off <= most).all()), f"worst {float((off / most).max())} of the bound"
    for x, y in ((p.k, p0.k), (p.v, p0.v)):
        assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8))
    if accumulate:
        w = p0.weight.double().clone()
        most = w * 2.0 ** -23
        for b, n in enumerate(lens):
            for i in range(n):
                at = (int(t[b, i // bs]), slice(None), i % bs)
                w[at] += ws[b][i]
                most[at] = w[at] * 2.0 ** -23 + ws[b][i] * (wrel[b] + group * 2.0 ** -23)
        off = (p.weight.cpu().double() - w).abs()
        assert bool((off <= most).all()), f"worst {float((off / most.clamp_min(1e-30)).max())} of the bound"
    return p0, t, q, out


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("G,group,D,bs,dtype", [(2, 4, 128, 16, torch.bfloat16), (1, 1, 64, 16, torch.bfloat16), (3, 7, 64, 32, torch.float16),
                                                (2, 8, 128, 64, torch.float16), (1, 16, 128, 48, torch.bfloat16), (1, 20, 64, 16, torch.bfloat16),
                                                (1, 33, 128, 16, torch.bfloat16)])
def test_attention(device, G, group, D, bs, dtype, accumulate):
    check_attention(device, EDGES, G, group, D, bs, dtype, accumulate, seed=G + group)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1], [0], [300], [2047], [513, 1, 0, 5000, 16, 777]])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_lengths(device, lens, accumulate):
    check_attention(device, lens, 2, 4, 128, 16, torch.bfloat16, accumulate, seed=len(lens), width=400 if len(lens) == 1 else 0)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_with_far_exponents(device):
    """Pages whose exponents are 60 apart, keys and values alike; scores of all sizes."""
    lens = [400, 31, 16]
    p0 = filled(32, 16, 2, 64, 2, weights=True)
    g = torch.Generator().manual_seed(4)
    p0.k_exp.copy_(torch.randint(-30, -6, p0.k_exp.shape, generator=g))
    p0.v_exp.copy_(torch.randint(-60, 1, p0.v_exp.shape, generator=g))
    check_attention(device, lens, 2, 4, 64, 16, torch.bfloat16, True, seed=2, pages=p0)
    p0.v_exp.fill_(-100)
    p0.k_exp.fill_(-100)
    check_attention(device, lens, 2, 4, 64, 16, torch.bfloat16, True, seed=2, pages=p0)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_where_one_key_has_all_the_weight(device):
    lens = [300, 17]
    p0 = filled(24, 16, 1, 128, 9)
    check_attention(device, lens, 1, 4, 128, 16, torch.bfloat16, False, seed=9, scale=3.0, pages=p0)
    check_attention(device, lens, 1, 4, 128, 16, torch.bfloat16, False, seed=9, scale=-3.0, pages=p0)
    check_attention(device, lens, 1, 4, 128, 16, torch.bfloat16, False, seed=9, scale=0.0, pages=p0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[40, 300], [300, 2500] * 40])
def test_attention_over_tables_with_pages_that_are_not_there(device, lens):
    """Whatever number a table has for a page that is not there, it counts as page 0, and no weight is added for it."""
    p0 = filled(sum((n + 15) // 16 for n in lens) + 1, 16, 2, 64, 6, weights=True)
    t = tables_of(lens, 16, p0.k.shape[0], 6)
    q = torch.randn(len(lens), 8 * 64, generator=torch.Generator().manual_seed(7)).bfloat16().to(device)
    got = []
    for gone in (-1, 1 << 30, -2 ** 31, 2 ** 31 - 1):
        t[:, 1], p = gone, to(p0, device)
        out = ops.paged_attention_decode_e4m3(q, p, t.to(device), ints(lens, device), accumulate=True)
        got.append((out, p.weight))
    for out, weight in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(weight, got[0][1])
    t[:, 1] = 0
    assert torch.equal(ops.paged_attention_decode_e4m3(q, to(p0, device), t.to(device), ints(lens, device)), got[0][0])


@pytest.mark.gpu
def test_attention_of_queries_of_all_sizes():
    """Query rows far apart in size, of bf16's smallest and largest numbers too; strided rows, an output in place of columns."""
    G, group, D, bs, lens = 1, 4, 64, 16, [100, 5, 40]
    p0 = filled(16, bs, G, D, 11)
    t = tables_of(lens, bs, 16, 11)
    q = torch.randn(3, group * D, generator=torch.Generator().manual_seed(1))
    q[0] *= 2.0 ** 20
    q[1] *= 2.0 ** -100
    q[2, D:2 * D] = 0.0
    q[2, 2 * D] = 2.0 ** 10
    q = q.bfloat16()
    p0.k_exp[t[0, :7].long()] -= 22
    want, err, _, _ = Cache(p0).attend(q, t, lens)
    wide = torch.full((3, group * D + 24), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 10:10 + group * D] = q.cuda()
    out = torch.full((3, group * D + 8), 5.0, dtype=torch.bfloat16, device="cuda")
    p = to(p0, "cuda")
    ops.paged_attention_decode_e4m3(wide[:, 10:10 + group * D], p, t.cuda(), ints(lens, "cuda"), out=out[:, 1:1 + group * D])
    off = (out[:, 1:1 + group * D].cpu().double() - want).abs()
    assert bool((off <= err + want.abs() * 2.0 ** -8).all())
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 1 + group * D:] == 5).all())


@pytest.mark.gpu
def test_attention_has_the_same_bits_alone_and_beside_others():
    lens, G, group, D, bs = [5000, 1, 300, 256, 0, 2500] + [700] * 60, 2, 4, 128, 16
    p0 = filled(sum((n + bs - 1) // bs for n in lens), bs, G, D, 3, weights=True)
    t, p = tables_of(lens, bs, p0.k.shape[0], 3).cuda(), to(p0, "cuda")
    q = torch.randn(len(lens), G * group * D, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    together = ops.paged_attention_decode_e4m3(q, p, t, ints(lens, "cuda"), accumulate=True)
    again, p2 = [], to(p0, "cuda")
    for b in range(len(lens)):
        width = max(1, (lens[b] + bs - 1) // bs)
        again.append(ops.paged_attention_decode_e4m3(q[b:b + 1], p2, t[b:b + 1, :width].contiguous(), ints(lens[b:b + 1], "cuda"), accumulate=True))
    assert torch.equal(together, torch.cat(again))
    assert torch.equal(p.weight, p2.weight)


@pytest.mark.gpu
@pytest.mark.parametrize("group,D,dtype", [(4, 128, torch.bfloat16), (1, 64, torch.float16), (12, 64, torch.bfloat16)])
def test_attention_over_many_slices(group, D, dtype):
    """Tables with room for more than 64 slices: long sequences, and short ones in such tables."""
    check_attention("cuda", [17000, 40, 0, 16641], 1, group, D, 16, dtype, True, seed=5)
    check_attention("cuda", [300, 1, 2049], 2, group, D, 16, dtype, True, seed=6, width=1200)
    check_attention("cuda", [511] * 40 + [0, 7], 2, group, D, 64, dtype, False, seed=7, width=80)


EVICTS = [
    # lengths, keep, recent, first, block size, KV heads, head size
    ([40], 20, 4, 2, 16, 1, 64),
    ([0, 1, 16, 17, 33, 100, 64], 17, 5, 1, 16, 3, 128),
    ([50, 31, 200], 32, 0, 0, 32, 2, 64),
    ([50, 31, 200], 32, 32, 0, 16, 2, 64),
    ([50, 31, 200], 32, 0, 32, 16, 2, 64),
    ([130, 129, 128, 127], 1, 0, 0, 64, 2, 128),
    ([700, 90], 600, 100, 8, 48, 2, 64),
    ([300, 50, 200, 129], 150, 20, 3, 128, 2, 64),
    ([300, 81, 500], 170, 0, 0, 80, 1, 128),
]


def weights_for(pages, seed, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(pages.weight.shape, generator=g) ** 6
    if kind == "ties":                                                # few different values: the lowest place wins
        w = torch.round(w * 3) / 3
        w = torch.where(torch.rand(w.shape, generator=g) < 0.3, -0.0, w)
    if kind == "odd":
        r = torch.rand(w.shape, generator=g)
        w = torch.where(r < 0.1, float("inf"), torch.where(r < 0.2, float("nan"), torch.where(r < 0.3, -w, torch.where(r < 0.4, 1e-42, w))))
        w = torch.where(r > 0.95, -float("inf"), w)
    pages.weight.copy_(w)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("own_pages", [False, True])
@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_evict(device, case, kind, own_pages):
    lens, keep, recent, first, bs, G, D = EVICTS[case]
    need = sum((n + bs - 1) // bs for n in lens)
    p0 = filled(need + sum((min(n, keep) + bs - 1) // bs for n in lens) + 2, bs, G, D, case, weights=True, spread=12)
    weights_for(p0, case, kind)
    t = tables_of(lens, bs, p0.k.shape[0], case)
    out_t = None
    if own_pages:
        free = sorted(set(range(p0.k.shape[0])) - set(t.flatten().tolist()))
        out_t = torch.zeros(len(lens), max(1, (min(max(lens), keep) + bs - 1) // bs), dtype=I32)
        for b, n in enumerate(lens):
            for i in range((min(n, keep) + bs - 1) // bs):
                out_t[b, i] = free.pop()
    want, p = Cache(p0), to(p0, device)
    want_lens, want_kept = want.evict(t, lens, keep, recent, first, out_t)
    got, kept = ops.kv_evict_e4m3(p, t.to(device), ints(lens, device), keep, recent, first, None if out_t is None else out_t.to(device))
    assert torch.equal(got.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    want.same(p)


@pytest.mark.gpu
@pytest.mark.parametrize("own_pages", [False, True])
def test_evict_long(own_pages):
    """Lengths of many tiles, against the host's path (which the tests above hold to the definition)."""
    lens, keep, bs, G, D = [40000, 9000, 5000, 2048, 100], 4099, 16, 2, 64
    p0 = filled(sum((n + bs - 1) // bs for n in lens) + 5 * 260, bs, G, D, 5, weights=True, spread=6)
    weights_for(p0, 5, "ties")
    t = tables_of(lens, bs, p0.k.shape[0], 5)
    out_t = None
    if own_pages:
        free = sorted(set(range(p0.k.shape[0])) - set(t.flatten().tolist()))
        out_t = torch.tensor([[free.pop() for _ in range(257)] for _ in lens], dtype=I32)
    host, dev = to(p0, "cpu"), to(p0, "cuda")
    a = ops.kv_evict_e4m3(host, t, ints(lens, "cpu"), keep, 500, 4, out_t)
    b = ops.kv_evict_e4m3(dev, t.cuda(), ints(lens, "cuda"), keep, 500, 4, None if out_t is None else out_t.cuda())
    assert all(torch.equal(x, y.cpu()) for x, y in zip(a, b))
    for x, y in zip((host.k.view(torch.uint8), host.v.view(torch.uint8), host.k_exp, host.v_exp, host.weight),
                    (dev.k.view(torch.uint8), dev.v.view(torch.uint8), dev.k_exp, dev.v_exp, dev.weight)):
        assert torch.equal(x, y.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "odd", "equal", "narrow", "wide"])
@pytest.mark.parametrize("lens,keep,recent,first", [([40000, 16385, 300], 9000, 100, 4), ([16300, 4000, 2048], 2000, 0, 0), ([140000, 20000], 15000, 64, 1),
                                                    ([140000], 139998, 139990, 4)])
def test_evict_of_weights_of_all_spreads(kind, lens, keep, recent, first):
    """Weights that are all equal, that differ in their last bits only, or in all; against the host's path."""
    p0 = filled(sum((n + 15) // 16 for n in lens), 16, 1, 64, 3, weights=True)
    g = torch.Generator().manual_seed(8)
    if kind in ("plain", "odd"):
        weights_for(p0, 3, kind)
    elif kind == "equal":
        p0.weight.fill_(0.25)
    elif kind == "narrow":
        p0.weight.copy_(1.0 + torch.randint(0, 1500, p0.weight.shape, generator=g) * 2.0 ** -23)
    else:                                                             # both signs, every exponent
        p0.weight.copy_(torch.randint(-2 ** 31, 2 ** 31, p0.weight.shape, generator=g, dtype=torch.int64).to(I32).view(torch.float32))
    t = tables_of(lens, 16, p0.k.shape[0], 3)
    host, dev = to(p0, "cpu"), to(p0, "cuda")
    a = ops.kv_evict_e4m3(host, t, ints(lens, "cpu"), keep, recent, first)
    b = ops.kv_evict_e4m3(dev, t.cuda(), ints(lens, "cuda"), keep, recent, first)
    assert all(torch.equal(x, y.cpu()) for x, y in zip(a, b))
    assert torch.equal(host.k.view(torch.uint8), dev.k.cpu().view(torch.uint8)) and torch.equal(host.weight.view(I32), dev.weight.cpu().view(I32))


@pytest.mark.parametrize("device", DEVICES)
def test_a_run_of_all(device):
    """A prompt in two portions, decoded tokens, eviction, more decoded tokens: state bit for bit, outputs within the bound."""
    G, group, D, bs, B = 2, 4, 64, 16, 3
    g = torch.Generator().manual_seed(0)
    p = ops.PagesE4M3.zeros(40, bs, G, D, device, weights=True)
    want = Cache(p)
    t = tables_of([120, 80, 50], bs, 40, 1)
    td = t.to(device)
    lens = [0, 0, 0]
    for new in ([50, 17, 1], [33, 40, 0]):
        lens = [a + b for a, b in zip(lens, new)]
        k, v = (torch.randn(sum(new), G * D, generator=g).bfloat16() for _ in range(2))
        ops.kv_append_e4m3(p, k.to(device), v.to(device), td, ints(lens, device), ints(starts_of(new), device))
        want.append(k, v, t, lens, starts_of(new))
    want.same(p)
    rows = starts_of(lens)
    k, _ = ops.kv_read_e4m3(p, td, ints(lens, device), ints(rows, device), rows[-1])
    assert torch.equal(k.cpu().double(), torch.cat([want.tokens("k", t, b, n).reshape(n, -1) for b, n in enumerate(lens)]))

    def decode(steps):
        for _ in range(steps):
            for b in range(B):
                lens[b] += 1
            k, v, q = (torch.randn(B, n * D, generator=g).bfloat16() for n in (G, G, G * group))
            ops.kv_append_e4m3(p, k.to(device), v.to(device), td, ints(lens, device))
            want.append(k, v, t, lens, list(range(B + 1)))
            want.w = p.weight.cpu().double()                          # what the kernel has summed; its own error is bounded elsewhere
            out = ops.paged_attention_decode_e4m3(q.to(device), p, td, ints(lens, device), accumulate=True)
            ref, err, ws, _ = want.attend(q, t, lens)
            assert bool(((out.cpu().double() - ref).abs() <= err + ref.abs() * 2.0 ** -8).all())
            grown = (p.weight.cpu().double() - want.w).sum()
            assert abs(float(grown) - B * G * group) < 1e-3           # every head's weights sum to one
            want.w = p.weight.cpu().double()

    decode(6)
    new_lens, kept = ops.kv_evict_e4m3(p, td, ints(lens, device), 32, 8, 2)
    want_lens, want_kept = want.evict(t, lens, 32, 8, 2)
    assert torch.equal(new_lens.cpu(), want_lens) and torch.equal(kept.cpu(), want_kept)
    want.same(p)
    lens[:] = want_lens.tolist()
    decode(5)


@pytest.mark.gpu
def test_captured_graphs_and_streams():
    """Two captured steps replayed on two streams at once, with new inputs in the same buffers, give what the calls give."""
    G, group, D, bs, lens = 2, 4, 128, 16, [700, 33, 1]
    made = []
    for seed in range(2):
        p0 = filled(60, bs, G, D, seed, weights=True)
        t = tables_of(lens, bs, 60, seed).cuda()
        p, q = to(p0, "cuda"), torch.randn(3, G * group * D, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        k, n = torch.randn(3, G * D, generator=torch.Generator().manual_seed(seed + 9)).bfloat16().cuda(), ints(lens, "cuda")

        def step(p=p, q=q, k=k, t=t, n=n):
            ops.kv_append_e4m3(p, k, k, t, n)
            out = ops.paged_attention_decode_e4m3(q, p, t, n, accumulate=True)
            lens2, kept = ops.kv_evict_e4m3(p, t, n, 64, 16, 2)
            starts = torch.zeros(4, dtype=I32, device="cuda")
            torch.cumsum(lens2, 0, dtype=I32, out=starts[1:])
            return (out, lens2, kept, *ops.kv_read_e4m3(p, t, lens2, starts, 98))
        step()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            got = step()
        made.append((graph, stream, got, step, p, p0, q, k, n))
    for graph, stream, got, step, p, p0, q, k, n in made:
        for a, b in ((p.k.view(torch.uint8), p0.k.view(torch.uint8)), (p.v.view(torch.uint8), p0.v.view(torch.uint8)), (p.k_exp, p0.k_exp),
                     (p.v_exp, p0.v_exp), (p.weight, p0.weight)):
            a.copy_(b)
        q.mul_(0.5)
        n[0] = 650
    torch.cuda.synchronize()
    for graph, stream, *_ in made:
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for graph, stream, got, step, p, p0, q, k, n in made:
        first = [x.clone() for x in got]
        fresh = to(p0, "cuda")
        for a, b in ((p.k.view(torch.uint8), fresh.k.view(torch.uint8)), (p.v.view(torch.uint8), fresh.v.view(torch.uint8)), (p.k_exp, fresh.k_exp),
                     (p.v_exp, fresh.v_exp), (p.weight, fresh.weight)):
            a.copy_(b)
        for a, b in zip(first, step()):
            assert torch.equal(a[:98] if a.dim() == 2 else a, b[:98] if b.dim() == 2 else b)


@pytest.mark.gpu
def test_offsets_behind_32_bits():
    """Pages whose codes lie more than 2^32 bytes into the arrays."""
    G, D, bs = 8, 128, 16
    blocks = (1 << 32) // (G * D * bs) + 64
    p = ops.PagesE4M3(*(torch.empty((blocks, G, bs, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)),
                      *(torch.zeros((blocks, G), dtype=torch.int8, device="cuda") for _ in range(2)),
                      torch.zeros((blocks, G, bs), dtype=torch.float32, device="cuda"))
    lens = [50, 40]
    t = torch.tensor([[blocks - 1, 3, blocks - 2, blocks - 7], [blocks - 9, blocks - 8, 0, 5]], dtype=I32)
    g = torch.Generator().manual_seed(1)
    k, v, q = torch.randn(90, G * D, generator=g).bfloat16(), torch.randn(90, G * D, generator=g).bfloat16(), torch.randn(2, 4 * G * D, generator=g).bfloat16()
    small = ops.PagesE4M3.zeros(8, bs, G, D, weights=True)
    ts = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=I32)
    want = Cache(small)
    want.append(k, v, ts, lens, [0, 50, 90])
    ops.kv_append_e4m3(p, k.cuda(), v.cuda(), t.cuda(), ints(lens, "cuda"), ints([0, 50, 90], "cuda"))
    got = ops.kv_read_e4m3(p, t.cuda(), ints(lens, "cuda"), ints([0, 50, 90], "cuda"), 90, dtype=torch.float32)
    for x, name in zip(got, "kv"):
        assert torch.equal(x.cpu().double(), torch.cat([want.tokens(name, ts, b, n).reshape(n, -1) for b, n in enumerate(lens)]))
    out = ops.paged_attention_decode_e4m3(q.cuda(), p, t.cuda(), ints(lens, "cuda"), accumulate=True)
    ref, err, _, _ = want.attend(q, ts, lens)
    assert bool(((out.cpu().double() - ref).abs() <= err + ref.abs() * 2.0 ** -8).all())
    want.w[:4], want.w[4:] = p.weight.cpu().double()[t[0].long()], p.weight.cpu().double()[t[1].long()]
    a = want.evict(ts, lens, 20, 4, 1)
    b = ops.kv_evict_e4m3(p, t.cuda(), ints(lens, "cuda"), 20, 4, 1)
    assert all(torch.equal(x, y.cpu()) for x, y in zip(a, b))
    got = ops.kv_read_e4m3(p, t.cuda(), b[0], ints([0, 20, 40], "cuda"), 40, dtype=torch.float32)
    for x, name in zip(got, "kv"):
        assert torch.equal(x.cpu().double(), torch.cat([want.tokens(name, ts, b, 20).reshape(20, -1) for b in range(2)]))


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------
def small(device="cpu", **kw):
    p = ops.PagesE4M3.zeros(4, kw.pop("bs", 16), kw.pop("G", 2), kw.pop("D", 64), device, weights=kw.pop("weights", True))
    return p, torch.zeros(2, 2, dtype=I32, device=device), torch.ones(2, dtype=I32, device=device)


def calls(p, t, n):
    x = torch.zeros(2, 128, device=p.k.device).bfloat16()
    s = torch.tensor([0, 1, 2], dtype=I32, device=p.k.device)
    return [lambda: ops.kv_append_e4m3(p, x, x, t, n), lambda: ops.kv_read_e4m3(p, t, n, s, 2), lambda: ops.paged_attention_decode_e4m3(x, p, t, n),
            lambda: ops.kv_evict_e4m3(p, t, n, 1)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("break_", ["tables", "lens", "lens_size", "codes", "exps", "exps_size", "order", "weight", "values"])
def test_refuses_pages_and_tables(device, break_):
    p, t, n = small(device)
    if break_ == "tables":
        t = t.long()
    elif break_ == "lens":
        n = n.long()
    elif break_ == "lens_size":
        n = torch.cat([n, n])
    elif break_ == "codes":
        p.k = p.k.view(torch.uint8)
    elif break_ == "exps":
        p.v_exp = p.v_exp.int()
    elif break_ == "exps_size":
        p.k_exp = p.k_exp[:2]
    elif break_ == "order":
        p.k = p.k.transpose(1, 2).contiguous().transpose(1, 2)
    elif break_ == "weight":
        p.weight = p.weight.double()
    else:
        p.v = p.v[:3]
    for call in calls(p, t, n):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("device", DEVICES)
def test_refuses_operands(device):
    p, t, n = small(device)
    x = torch.zeros(2, 128, device=device).bfloat16()
    s = ints([0, 1, 2], device)
    with pytest.raises(TypeError):
        ops.kv_append_e4m3(p, x[:, :64], x[:, :64], t, n)
    with pytest.raises(TypeError):
        ops.kv_append_e4m3(p, x, x.float(), t, n)
    with pytest.raises(TypeError):
        ops.kv_append_e4m3(p, x.double(), x.double(), t, n)
    with pytest.raises(ValueError):
        ops.kv_append_e4m3(p, x[:1], x[:1], t, n)                     # one row for two sequences
    with pytest.raises(TypeError):
        ops.kv_append_e4m3(p, x, x, t, n, s[:2].contiguous())
    with pytest.raises(TypeError):
        ops.kv_append_e4m3(p, x, x, t, n, s.long())
    with pytest.raises(TypeError):
        ops.kv_read_e4m3(p, t, n, s, 2, dtype=torch.float64)
    with pytest.raises(TypeError):
        ops.kv_read_e4m3(p, t, n, s, 3, out=(x, x))
    with pytest.raises(TypeError):
        ops.kv_read_e4m3(p, t, n, s[1:].contiguous(), 2)
    with pytest.raises(TypeError):
        ops.paged_attention_decode_e4m3(x[:, :96], p, t, n)
    with pytest.raises(TypeError):
        ops.paged_attention_decode_e4m3(x[:1], p, t, n)
    with pytest.raises(TypeError):
        ops.paged_attention_decode_e4m3(x, p, t, n, out=x.float())
    for bad in (dict(keep=0), dict(keep=4, recent=3, keep_first=2), dict(keep=4, recent=-1), dict(keep=4, keep_first=-1)):
        with pytest.raises(ValueError):
            ops.kv_evict_e4m3(p, t, n, **bad)
    with pytest.raises(TypeError):
        ops.kv_evict_e4m3(p, t, n, 1, out_tables=t.long())
    with pytest.raises(TypeError):
        ops.kv_evict_e4m3(p, t, n, 1, out_tables=t[:1])
    with pytest.raises(ValueError):
        ops.kv_evict_e4m3(p, t, n, 20, out_tables=t[:, :1].contiguous())
    q, t2, n2 = small(device, weights=False)
    with pytest.raises(ValueError):
        ops.kv_evict_e4m3(q, t, n, 1)
    with pytest.raises(ValueError):
        ops.paged_attention_decode_e4m3(x, q, t, n, accumulate=True)


@pytest.mark.gpu
def test_refuses_what_no_kernel_takes():
    for kw in (dict(bs=8), dict(bs=24), dict(D=32), dict(D=96)):
        p, t, n = small("cuda", **kw)
        with pytest.raises(ValueError):
            ops.kv_evict_e4m3(p, t, n, 1)
    p, t, n = small("cuda")
    with pytest.raises(TypeError):
        ops.paged_attention_decode_e4m3(torch.zeros(2, 128, device="cuda"), p, t, n)
    with pytest.raises(ValueError):
        ops.paged_attention_decode_e4m3(torch.zeros(2, 128, device="cuda").bfloat16(), p, t.cpu(), n)
    x = torch.zeros(2, 136, device="cuda").bfloat16()[:, 1:129]
    with pytest.raises(ValueError):
        ops.kv_read_e4m3(p, t, n, ints([0, 1, 2], "cuda"), 2, out=(x, x))


@pytest.mark.gpu
def test_refuses_more_tokens_than_the_kernels_count():
    for bs, width in ((1 << 20, 1024), ((1 << 20) + 16, 1)):
        p = ops.PagesE4M3.zeros(1, bs, 1, 64, "cuda", weights=True)
        t, n = torch.zeros(1, width, dtype=I32, device="cuda"), ints([1], "cuda")
        x = torch.zeros(1, 64, device="cuda").bfloat16()
        for call in (lambda: ops.kv_append_e4m3(p, x, x, t, n), lambda: ops.kv_read_e4m3(p, t, n, ints([0, 1], "cuda"), 1),
                     lambda: ops.paged_attention_decode_e4m3(x, p, t, n), lambda: ops.kv_evict_e4m3(p, t, n, 1)):
            with pytest.raises(ValueError):
                call()


@pytest.mark.parametrize("device", DEVICES)
def test_empty_calls(device):
    p, t, n = small(device)
    x, s = torch.zeros(0, 128, device=device).bfloat16(), torch.zeros(1, dtype=I32, device=device)
    t0, n0 = t[:0].contiguous(), n[:0].contiguous()
    before = p.k.clone()
    ops.kv_append_e4m3(p, x, x, t0, n0)
    ops.kv_append_e4m3(p, x, x, t, n, torch.zeros(3, dtype=I32, device=device))
    assert ops.kv_read_e4m3(p, t0, n0, s, 0)[0].shape == (0, 128)
    assert ops.paged_attention_decode_e4m3(x, p, t0, n0).shape == (0, 128)
    lens, kept = ops.kv_evict_e4m3(p, t0, n0, 3)
    assert lens.shape == (0,) and kept.shape == (0, 2, 3)
    no_pages = torch.zeros(2, 0, dtype=I32, device=device)
    assert bool((ops.paged_attention_decode_e4m3(torch.ones(2, 128, device=device).bfloat16(), p, no_pages, n) == 0).all())
    lens, kept = ops.kv_evict_e4m3(p, no_pages, n, 3)
    assert lens.tolist() == [0, 0] and bool((kept == -1).all())
    assert torch.equal(before.view(torch.uint8), p.k.view(torch.uint8))


@pytest.mark.parametrize("device", DEVICES)
def test_rows_and_lengths_that_do_not_match(device):
    """More rows than tokens, tokens behind the table, page numbers out of range: such rows are not stored, and nothing else is touched."""
    G, D, bs = 1, 64, 16
    p0 = filled(6, bs, G, D, 0, weights=True)
    t = torch.tensor([[0, 1], [2, 99], [-1, 3]], dtype=I32)
    lens, starts = [2, 40, 20], [0, 5, 30, 50]
    k = torch.randn(50, G * D, generator=torch.Generator().manual_seed(0)).bfloat16()
    p = to(p0, device)
    ops.kv_append_e4m3(p, k.to(device), k.to(device), t.to(device), ints(lens, device), ints(starts, device))
    want = Cache(p0)
    want.append(k[3:5], k[3:5], torch.tensor([[0]]), [2], [0, 2])                   # the last two rows are positions 0 and 1
    want.append(k[5:6], k[5:6], torch.tensor([[2]]), [16], [0, 1])                  # position 15; 16 to 31 have page 99, 32 to 39 none
    want.append(k[46:50], k[46:50], torch.tensor([[5, 3]]), [20], [0, 4])           # positions 16 to 19; page -1 in front
    want.same(p)
    out = torch.full((50, G * D), 2.0, dtype=torch.float32, device=device)
    ops.kv_read_e4m3(p, t.to(device), ints(lens, device), ints(starts, device), 50, out=(out, out.clone()))
    for row, filled_ in ((0, True), (1, True), (2, False), (5, True), (20, True), (21, False), (29, False), (30, False), (45, False), (46, True), (49, True)):
        assert bool((out[row] == 2.0).all()) != filled_


@pytest.mark.gpu
def test_read_with_starts_that_do_not_ascend():
    """A row in front of the sequence that it is counted to has no position: it stays as it was."""
    p = to(filled(8, 16, 1, 64, 0), "cuda")
    t = torch.arange(1, 6, dtype=I32, device="cuda").view(5, 1)
    out = [torch.full((40, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    ops.kv_read_e4m3(p, t, ints([16] * 5, "cuda"), ints([0, 5, 20, 21, 5, 40], "cuda"), 40, out=out)
    # of rows 16 to 31, whose search begins with sequence 2: 16 to 19 lie in front of it, 20 is its first, 21 on are counted to sequence 4
    for x in out:
        assert bool((x[16:20] == 7.0).all()) and not bool((x[20] == 7.0).all())


@pytest.mark.gpu
def test_evict_right_after_a_prompt():
    """Weights that are all zero, as appending leaves them: of short sequences most of a CTA's warps have no token and are done at once, and two CTAs
    share an SM.  The earliest stay beside the last, call after call."""
    G, D, bs, keep, recent = 8, 64, 16, 16, 5
    lens = [17 + 3 * b % 190 for b in range(160)]
    p = ops.PagesE4M3.zeros(sum((n + bs - 1) // bs for n in lens), bs, G, D, "cuda", weights=True)
    t = tables_of(lens, bs, p.k.shape[0], 0).cuda()
    k = torch.randn(sum(lens), G * D, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    ops.kv_append_e4m3(p, k, k, t, ints(lens, "cuda"), ints(starts_of(lens), "cuda"))
    assert not bool(p.weight.any())
    want = torch.tensor([[*range(keep - recent), *range(n - recent, n)] for n in lens], dtype=I32)[:, None].expand(-1, G, -1)
    starts = ints([keep * b for b in range(len(lens) + 1)], "cuda")
    rows = torch.cat([starts_of(lens)[b] + want[b, 0].long() for b in range(len(lens))])
    host = ops.PagesE4M3.zeros(sum((n + bs - 1) // bs for n in lens), bs, G, D)
    ops.kv_append_e4m3(host, k.cpu(), k.cpu(), t.cpu(), ints(lens, "cpu"), ints(starts_of(lens), "cpu"))
    exact = ops.kv_read_e4m3(host, t.cpu(), ints(lens, "cpu"), ints(starts_of(lens), "cpu"), sum(lens), dtype=torch.float32)[0][rows]
    for _ in range(50):
        q = to(p, "cuda")
        got, kept = ops.kv_evict_e4m3(q, t, ints(lens, "cuda"), keep, recent)
        assert bool((got == keep).all()) and torch.equal(kept.cpu(), want)
    # codes are rounded once to a larger exponent, that of numbers below 2^3, -5 at most: by half a step of a code, 2^-4 of it, or of a subnormal one, 2^-10 * 2^-5
    back = ops.kv_read_e4m3(q, t, got, starts, keep * len(lens), dtype=torch.float32)[0].cpu()
    assert bool(((back - exact).abs() <= exact.abs() * 2.0 ** -4 + 2.0 ** -15).all())


# one sequence in a cluster; several slices and a merge; tables with room for more than 64 slices
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,width", [([1, 16, 40, 300], 0), ([520] * 30 + [1, 17], 0), ([1, 300, 5000], 1200)])
@pytest.mark.parametrize("group,D", [(4, 128), (12, 64)])
@pytest.mark.parametrize("lean", [0.0, 330.0, -330.0, 2600.0, -2600.0])
def test_attention_over_pages_at_both_ends_of_the_exponents(device, lens, width, group, D, lean):
    """Pages of zeros (exponent -100) beside pages of exponent 119.  `lean`: the scores of the former lie lean / 32 above those of the latter (up to 81, 117 powers
    of two), so that they have nearly all of the denominator, half or nearly nothing, and the latter nearly all of the sums."""
    G, bs = 2, 16
    p0 = filled(sum((n + bs - 1) // bs for n in lens) + 2, bs, G, D, 12, weights=True)
    zeros = torch.arange(p0.k.shape[0]) % 3 == 0
    zeros[tables_of(lens, bs, p0.k.shape[0], 13, width)[:, 0].long()] = False           # every sequence has a page of either kind where it has two
    p0.k_exp.fill_(-6)
    p0.v_exp.fill_(119)
    p0.v_exp[zeros] = -100
    p0.v.view(torch.uint8)[zeros] = 0
    # dimension 0: code 64 for pages of zeros and -64 for the others, under an exponent of -6, times lean / 8 in the query
    p0.k.view(torch.uint8)[..., 0] = torch.where(zeros, 0x68, 0xe8).to(torch.uint8)[:, None, None]
    t = tables_of(lens, bs, p0.k.shape[0], 13, width)
    q = torch.randn(len(lens), G * group, D, generator=torch.Generator().manual_seed(3))
    q[..., 0] = lean / 8
    q = q.view(len(lens), -1).bfloat16()
    want, err, ws, wrel = Cache(p0).attend(q, t, lens, 0.125)
    p = to(p0, device)
    out = ops.paged_attention_decode_e4m3(q.to(device), p, t.to(device), ints(lens, device), 0.125, accumulate=True).cpu().double()
    off, most = (out - want).abs(), err + want.abs() * 2.0 ** -8
    assert bool((off <= most).all()), f"worst {float((off / most).max())} of the bound"
    for b, n in enumerate(lens):
        at = torch.arange(n)
        pages = t[b, at // bs].long()
        was, got = p0.weight[pages, :, at % bs].double(), p.weight.cpu()[pages, :, at % bs].double()
        most = (was + ws[b]) * 2.0 ** -23 + ws[b] * (wrel[b] + group * 2.0 ** -23)
        assert bool(((got - was - ws[b]).abs() <= most).all())
        assert abs(float((got - was).sum()) - G * group) <= n * G * 2.0 ** -23 * 2 + G * group * wrel[b]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[300], [17, 2000], [9000, 700]])
@pytest.mark.parametrize("group,D,dtype", [(4, 128, torch.bfloat16), (1, 64, torch.float16), (12, 64, torch.bfloat16)])
def test_attention_beside_one_token_with_nearly_all_the_weight(device, lens, group, D, dtype):
    """The first token has nearly all the weight and a value of zero, so that the output is what the others add, each with 2^-27 of its weight."""
    G, bs = 2, 16
    p0 = filled(sum((n + bs - 1) // bs for n in lens), bs, G, D, 14, spread=0)
    t = tables_of(lens, bs, p0.k.shape[0], 14)
    p0.k_exp.fill_(-6)
    p0.k.view(torch.uint8)[..., 0] = 0xe8                             # -64: -1 with the exponent
    p0.v.view(torch.uint8).bitwise_and_(0x7f)                         # values without signs: no sum is smaller than its terms
    for b in range(len(lens)):
        p0.k.view(torch.uint8)[int(t[b, 0]), :, 0, 0] = 0x68
        p0.v.view(torch.uint8)[int(t[b, 0]), :, 0] = 0
    q = torch.zeros(len(lens), G * group, D)
    q[..., 0] = 75.0                                                  # scores 150 / 8 apart, 27.05 powers of two
    q = q.view(len(lens), -1).to(dtype)
    want, _, _, _ = Cache(p0).attend(q, t, lens, 0.125)
    out = ops.paged_attention_decode_e4m3(q.to(device), to(p0, device), t.to(device), ints(lens, device), 0.125).cpu().double()
    # factors: half a step of an f16, 2^-11, or 2^-39 of the largest; scores of 9.4 in 32 bits (twice, 2^-24 each) and two exponentials, below 2^-17 together;
    # the output's own rounding, half a step
    largest = float(p0.v.float().max()) * 2.0 ** int(p0.v_exp.max())
    f = torch.finfo(dtype)
    most = want * (2.0 ** -11 + 2.0 ** -17 + f.eps / 2) + max(lens) * 2.0 ** -39 * largest + f.smallest_normal * f.eps / 2
    off = (out - want).abs()
    assert bool((off <= most).all()), f"worst {float((off / most).max())} of the bound"


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens,width", [([40, 300], 0), ([520] * 30 + [1, 17], 0)])
@pytest.mark.parametrize("group,D,dtype", [(4, 128, torch.bfloat16), (12, 64, torch.float16)])
@pytest.mark.parametrize("first", [0.0, -64.0])
def test_attention_of_scores_past_the_range(device, lens, width, group, D, dtype, first):
    """Keys of 2^125 in dimension 0 of some tokens, alone in their pages.  A query without that dimension has scores of zero with them, one with -64 there scores of
    -2^131 / 8, below what 32 bits have: no weight."""
    G, bs = 2, 16
    p0 = filled(sum((n + bs - 1) // bs for n in lens), bs, G, D, 15, weights=True, spread=2)
    t = tables_of(lens, bs, p0.k.shape[0], 15, width)
    g = torch.Generator().manual_seed(4)
    for b, n in enumerate(lens):
        for i in range(1, (n + bs - 1) // bs, 2):                     # two of a warp's tiles in a row too
            page = int(t[b, i])
            p0.k.view(torch.uint8)[page] = 0
            p0.k.view(torch.uint8)[page, ..., 0] = 0x68               # 64 under 2^119
            p0.k_exp[page] = 119
    q = torch.randn(len(lens), G * group, D, generator=g)
    q[..., 0] = first
    q[..., 1] = 2.0 ** 13                                             # 2^119 times the query's power of two is past the range; keys are zero there
    p0.k.view(torch.uint8)[..., 1] = 0
    q = q.view(len(lens), -1).to(dtype)
    want, err, ws, wrel = Cache(p0).attend(q, t, lens, 0.125)
    p = to(p0, device)
    out = ops.paged_attention_decode_e4m3(q.to(device), p, t.to(device), ints(lens, device), 0.125, accumulate=True).cpu().double()
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(p.weight).all())
    # The oracle's bound goes by the largest key and says nothing here.  A query's numbers lie 2^-13 below its largest, in f16 off by 2^-25 of that at most; D products are
    # summed in 32 bits; a weight is off by twice what its score is (its own and the largest's); factors by 2^-11 or 2^-39 of the largest, exponentials by 2^-17.
    most = torch.zeros(len(lens))
    for b, n in enumerate(lens):
        k, v = (Cache(p0).tokens(x, t, b, n).abs() for x in "kv")
        k = torch.where(k > 1e30, 0.0, k)
        scores = 0.125 * (k.sum(-1).max() * 2.0 ** -12 + (q[b].double().view(G, group, 1, D).abs() * k.transpose(0, 1)[:, None]).sum(-1).max() * (D + 4) * 2.0 ** -24)
        most[b] = (torch.expm1(2 * scores) + 2.0 ** -11 + 2.0 ** -17 + n * 2.0 ** -39) * v.max()
    assert bool(((out - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + most[:, None] + 2.0 ** -24).all())
    grown = (p.weight.cpu() - p0.weight).double()
    assert abs(float(grown.sum()) - len(lens) * G * group) < 1e-2
    if first:
        gone = torch.cat([t[b, 1:(n + bs - 1) // bs:2] for b, n in enumerate(lens)]).long()
        assert not bool(grown[gone].any())


@pytest.mark.parametrize("device", DEVICES)
def test_tables_without_pages(device):
    """No position has a page: nothing is stored, no row is written."""
    p, _, n = small(device)
    before = to(p, device)
    t, s = torch.zeros(2, 0, dtype=I32, device=device), ints([0, 1, 2], device)
    x = torch.ones(2, 128, device=device).bfloat16()
    ops.kv_append_e4m3(p, x, x, t, n)
    ops.kv_append_e4m3(p, x, x, t, n, s)
    for a, b in ((p.k, before.k), (p.v, before.v), (p.k_exp, before.k_exp), (p.weight, before.weight)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    out = (x.clone(), x.clone())
    assert ops.kv_read_e4m3(p, t, n, s, 2, out=out) is not None and all(bool((y == 1).all()) for y in out)
    assert ops.kv_read_e4m3(p, t, n, s, 2)[0].shape == (2, 128)
