"""Several continuations of one prompt where caches are large, tensors lie together, weights are kept and calls are refused (ops.beams, serve.PagedCache, serve.BeamSearch)."""
import json
import math
import os
import random
import subprocess
import sys

import pytest
import torch

from rustral_b200 import ops
from rustral_b200.models.config import preset
from rustral_b200.serve import BeamSearch, CacheLayer, CacheQuantization, ModelRunner, PagedCache
from test_beam_search import scores_are_their_tokens, sharp
from test_beams import attend64, bound, choose, forked, same_choice
from test_serving_e4m3 import Ranks

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
I32 = torch.int32


@pytest.fixture
def watched(request):
    """On a GPU: fails the test where a wait of a kernel ran out."""
    if request.node.callspec.params["device"] != "cpu":
        request.getfixturevalue("cuda_status")


# ---- selection -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 900), (torch.bfloat16, 1000), (torch.float32, 20000), (torch.bfloat16, 20001)])
def test_beam_select_of_more_equal_candidates_than_a_list_holds(device, dtype, vocab, watched):
    """Equal rows with 100 equal best tokens each: of 1600 equal candidates the first rows' first tokens, an ended beam's and dead beams' places between them."""
    x = torch.linspace(-2.0, 1.0, vocab)[torch.randperm(vocab, generator=torch.Generator().manual_seed(vocab))]
    x[torch.randperm(vocab, generator=torch.Generator().manual_seed(1))[:100]] = 3.0
    x = x.to(dtype).expand(16, vocab).contiguous()
    scores, ended = torch.full((1, 16), -2.5), torch.zeros(1, 16, dtype=torch.bool)
    for count in (128, 101, 7):
        same_choice(ops.beam_select(x.to(device), scores.to(device), count), choose(x, scores, count))
    scores[0, 1], scores[0, 3], ended[0, 2], ended[0, 5] = -math.inf, math.nan, True, True
    for count in (128, 120):
        same_choice(ops.beam_select(x.to(device), scores.to(device), count, ended.to(device), 11), choose(x, scores, count, ended, 11))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_beam_select_of_many_rows_waits_for_its_copies(dtype, cuda_status):
    """Rows that come by bulk copies, twice over them where there are infinities."""
    x = torch.empty(600, 50008, device="cuda").normal_(0.0, 2.5, generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    x[7, 123] = math.inf
    x[300:304] = math.nan
    scores = -torch.rand(150, 4, device="cuda")
    got, want = ops.beam_select(x, scores, 8), ops.beam_select(x.cpu(), scores.cpu(), 8)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])


@pytest.mark.parametrize("device", DEVICES)
def test_beam_select_of_groups_without_a_live_beam(device, watched):
    x = torch.randn(9, 50, generator=torch.Generator().manual_seed(3))
    scores, ended = torch.full((3, 3), -math.inf), torch.zeros(3, 3, dtype=torch.bool)
    scores[1], scores[2, 1] = torch.tensor([math.nan, -math.inf, -math.inf]), -4.0
    ended[2, 1] = ended[0, 0] = True
    for count in (1, 5, 120):
        same_choice(ops.beam_select(x.to(device), scores.to(device), count, ended.to(device), 49), choose(x, scores, count, ended, 49))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,vocab,skip", [(torch.bfloat16, 9_000_001, 1), (torch.float32, 1 << 26, 0), (torch.float16, 5_000_000, 0)])
def test_beam_select_of_long_rows(dtype, vocab, skip, cuda_status):
    """One row in thousands of pieces.  Its sum of exponentials is checked by the definition on the host; see there for what a score may be off."""
    x = torch.empty(1, vocab + 8, device="cuda").normal_(0.0, 2.5, generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)[:, skip:vocab + skip]
    scores = torch.tensor([[-3.0]])
    got = ops.beam_select(x, scores.cuda(), 128)
    row = x[0].cpu().double()
    row -= torch.logsumexp(row, 0) + 3.0
    best = torch.topk(row, 1000)
    order = sorted(zip((-best.values).tolist(), best.indices.tolist()))
    last = order[127][0]                                           # all that are as good as the last one, in the order of their tokens
    order = sorted([p for p in order if p[0] < last] + [(last, i) for i in (row == -last).nonzero()[:, 0].tolist()])[:128]
    assert got[2].tolist() == [[i for _, i in order]] and got[1].tolist() == [[0] * 128]
    want = -torch.tensor([p for p, _ in order], dtype=torch.float64)
    assert ((got[0][0].cpu().double() - want).abs() <= 2.0 ** -17 + want.abs() * 2.0 ** -24).all()


@pytest.mark.gpu
def test_a_step_of_beams_captured_and_replayed(cuda_status):
    """Selection and what the selected inherit in one graph, on a stream of its own, twice with other logits, beside the same on another stream."""
    beams, vocab = 6, 3001
    g = torch.Generator().manual_seed(9)
    draws = [torch.randn(2 * beams, vocab, generator=g).bfloat16() for _ in range(3)]
    held = torch.randn(2 * beams, 40, generator=g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    done = []
    for stream in streams:
        with torch.cuda.stream(stream):
            x, s, h, c = draws[0].cuda(), torch.zeros(2, beams, device="cuda"), held.cuda(), torch.arange(30.0, device="cuda").view(10, 3)
            best = ops.beam_select(x, s, beams)                    # kernels are set up before the capture
            ops.reorder_rows_([h.clone()], best[1].view(-1), group=beams)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                best = ops.beam_select(x, s, beams)
                ops.reorder_rows_([h], best[1].view(-1), group=beams)
                ops.copy_blocks_([c], [1, 2], [5, 7])
            done.append((graph, x, h, c, best))
    torch.cuda.synchronize()
    for d in draws[1:]:
        for stream, (graph, x, h, c, _) in zip(streams, done):
            with torch.cuda.stream(stream):
                x.copy_(d.cuda())
                c[1] += 1
                graph.replay()
        torch.cuda.synchronize()
        want = ops.beam_select(d, torch.zeros(2, beams), beams)
        held = held[want[1].view(-1)]
        for _, _, h, c, best in done:
            assert torch.equal(best[1].cpu(), want[1]) and torch.equal(best[2].cpu(), want[2]) and torch.equal(h.cpu(), held)
            assert torch.equal(c[5], c[1]) and torch.equal(c[7], c[2])


# ---- attention over a shared prefix ------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dim,more", [(64, 1 << 20), (128, 1 << 21)])
def test_attention_shared_in_a_larger_cache_at_the_same_address(dim, more, cuda_status):
    """A cache of 2^19 tokens, then one at its address with `more` tokens behind them: keys and values behind the smaller one's end are read.  Weights and rounding: see `bound`."""
    n, bs, lens = 20, 16, [21 + i for i in range(20)]
    blocks = [(1 << 19) // bs, ((1 << 19) + more) // bs]
    k, v = (torch.zeros(blocks[1], bs, 1, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(dim)
    q = torch.randn(n, dim, generator=g).bfloat16()
    groups, shared = ops.PrefixGroups([n], "cuda"), torch.tensor([bs], dtype=I32, device="cuda")
    for count in blocks:
        pages = count - 1 - torch.randperm(1 + 2 * n, generator=g)       # the last ones
        t = torch.cat([pages[:1].expand(n, 1), pages[1:].view(n, 2)], 1).to(I32)
        held = [torch.randn(1 + 2 * n, bs, 1, dim, generator=g).bfloat16() for _ in range(2)]
        for x, h in zip((k, v), held):
            x[pages.cuda()] = h.cuda()
        got = ops.paged_attention_shared(q.cuda(), k[:count], v[:count], groups, shared, t.cuda(), torch.tensor(lens, dtype=I32, device="cuda"))
        place = torch.empty(count, dtype=torch.int64)
        place[pages] = torch.arange(len(pages))
        want, most = attend64(q, *held, place[t.long()], lens, 1.0 / math.sqrt(dim))
        assert ((got.cpu().double() - want).abs() <= bound(want, most, torch.bfloat16)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [4, 40])
def test_attention_shared_of_one_row_for_all_and_into_rows_apart(device, n):
    """A query that is one row for every sequence; results into rows of a wider tensor, columns of a transposed one, and none whose rows share memory."""
    sizes, shared, lens, dim = [n], [33], [34 + i % 9 for i in range(n)], 64
    k, v, t = forked(sizes, shared, lens, 16, 2, dim, torch.bfloat16, n, hole=0.0)
    q = torch.randn(1, 4 * dim, generator=torch.Generator().manual_seed(n)).bfloat16()
    want, most = attend64(q.expand(n, -1), k, v, t, lens, 1.0 / math.sqrt(dim))
    tensors = (k.to(device), v.to(device), ops.PrefixGroups(sizes, device), *(torch.tensor(x, dtype=I32, device=device) for x in (shared, t.tolist(), lens)))
    limit = bound(want, most, torch.bfloat16)
    whole = torch.zeros(n, 4 * dim + 8, dtype=torch.bfloat16, device=device)
    columns = torch.zeros(4 * dim, n, dtype=torch.bfloat16, device=device)
    apart = torch.zeros(n, 8 * dim, dtype=torch.bfloat16, device=device)
    for out in (None, whole[:, 8:], whole[:, 5:-3], columns.t(), apart[:, ::2]):
        got = ops.paged_attention_shared(q.to(device).expand(n, -1), *tensors, out=out)
        assert ((got.cpu().double() - want).abs() <= limit).all() and (out is None or got is out)
    assert not apart[:, 1::2].any()
    flat = torch.zeros(n * 4 * dim, dtype=torch.bfloat16, device=device)
    for out in (flat[:4 * dim].expand(n, -1), flat.as_strided((n, 4 * dim), (8, 1)), flat[:n].view(n, 1).expand(n, 4 * dim)):
        with pytest.raises(ValueError):
            ops.paged_attention_shared(q.to(device).expand(n, -1), *tensors, out=out)
    assert not flat.any()


MORE = [
    # group sizes, shared tokens, own tokens of every sequence, block size, KV heads, heads of each, head size, type, scale (None: as a rule)
    ([30], [203], [1 + i for i in range(30)], 8, 2, 4, 64, torch.bfloat16, None),
    ([7, 25], [64, 517], [3 * i for i in range(32)], 8, 1, 4, 128, torch.float16, None),
    ([20], [500], [1 + 17 * i for i in range(20)], 384, 1, 4, 128, torch.bfloat16, None),
    ([20, 3], [385, 900], [100] * 23, 384, 2, 2, 64, torch.float16, None),
    ([20], [300], [1 + i for i in range(20)], 16, 2, 4, 64, torch.bfloat16, 0.0),
    ([20], [300], [1 + i for i in range(20)], 16, 2, 4, 128, torch.bfloat16, -0.1),
    ([3], [300], [1, 40, 200], 16, 2, 4, 64, torch.float16, 0.0),
    ([3], [300], [1, 40, 200], 16, 2, 4, 128, torch.bfloat16, -0.1),
    ([704], [200], [2] * 704, 16, 1, 1, 64, torch.bfloat16, None),
    ([705], [200], [2] * 705, 16, 1, 1, 64, torch.bfloat16, None),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(MORE)))
def test_attention_shared_of_other_pages_and_scales(device, case, watched):
    sizes, shared, mine, bs, kv, per, dim, dtype, scale = MORE[case]
    owner = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [shared[g] + n for g, n in zip(owner, mine)]
    k, v, t = forked(sizes, shared, lens, bs, kv, dim, dtype, 50 + case)
    q = (torch.randn(len(lens), kv * per * dim, generator=torch.Generator().manual_seed(case)) * 2).to(dtype)
    want, most = attend64(q, k, v, t, lens, 1.0 / math.sqrt(dim) if scale is None else scale)
    got = ops.paged_attention_shared(*(x.to(device) for x in (q, k, v)), ops.PrefixGroups(sizes, device),
                                     *(x.to(device) for x in (torch.tensor(shared, dtype=I32), t, torch.tensor(lens, dtype=I32))), scale=scale)
    assert ((got.cpu().double() - want).abs() <= bound(want, most, dtype)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,bs,dim", [(4, 16, 64), (24, 16, 64), (24, 8, 128), (24, 128, 64), (24, 256, 128)])
def test_attention_shared_of_tables_that_name_no_block(device, n, bs, dim, watched):
    """Entries below zero and behind the last block count as block 0, of shared tokens and of a sequence's own."""
    shared, lens = 3 * bs, [3 * bs + 1 + (7 * i) % (2 * bs) for i in range(n)]
    k, v, t = forked([n], [shared], lens, bs, 1, dim, torch.bfloat16, n + bs, width=5, hole=0.5)
    blocks, bad = k.shape[0], torch.tensor([-1, -1 << 31, k.shape[0], (1 << 31) - 1], dtype=I32)
    t[0, 1], t[1, 3], t[2, 3:5], t[3, 3] = bad[0], bad[1], bad[2:4], bad[3]
    clean = torch.where((t >= 0) & (t < blocks), t, 0)
    clean[:, :3] = clean[0, :3]                                    # the first one's table is the group's
    q = torch.randn(n, 4 * dim, generator=torch.Generator().manual_seed(n)).bfloat16()
    want, most = attend64(q, k, v, clean, lens, 1.0 / math.sqrt(dim))
    got = ops.paged_attention_shared(*(x.to(device) for x in (q, k, v)), ops.PrefixGroups([n], device),
                                     *(x.to(device) for x in (torch.tensor([shared], dtype=I32), t, torch.tensor(lens, dtype=I32))))
    assert ((got.cpu().double() - want).abs() <= bound(want, most, torch.bfloat16)).all()


@pytest.mark.gpu
def test_checking_build_reports_tables_that_name_no_block():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, RUSTRAL_BOUNDS="1", PYTHONPATH=root + os.pathsep + os.environ.get("PYTHONPATH", ""))
    res = subprocess.run([sys.executable, os.path.join(root, "tests", "bounds_continuations_worker.py")], env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-2000:]
    out = json.loads(res.stdout.strip().splitlines()[-1])
    for name in ("few", "many"):
        assert out.pop(name + "_ok") == [[0, 0, True]]
        for kind in ("shared", "own"):
            assert out.pop(f"{name}_{kind}") == [[8, 104, True]] * 4
    assert not out


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 20])
def test_attention_shared_past_four_gigabytes(n, cuda_status):
    """Pages behind 2^31 numbers of a cache, shared ones and a sequence's own."""
    bs, kv, per, dim, blocks = 16, 8, 4, 128, 140000
    lens = [40 + i for i in range(n)]
    small = forked([n], [32], lens, bs, kv, dim, torch.bfloat16, n, hole=0.0)
    k, v = (torch.zeros(blocks, bs, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pages = blocks - 1 - torch.arange(small[0].shape[0])
    k[pages.cuda()], v[pages.cuda()] = small[0].cuda(), small[1].cuda()
    t = pages[small[2].clamp(max=len(pages) - 1).long()].to(I32)
    q = torch.randn(n, kv * per * dim, generator=torch.Generator().manual_seed(n)).bfloat16()
    want, most = attend64(q, small[0], small[1], small[2], lens, 1.0 / math.sqrt(dim))
    got = ops.paged_attention_shared(q.cuda(), k, v, ops.PrefixGroups([n], "cuda"), torch.tensor([32], dtype=I32, device="cuda"), t.cuda(),
                                     torch.tensor(lens, dtype=I32, device="cuda"))
    assert ((got.cpu().double() - want).abs() <= bound(want, most, torch.bfloat16)).all()


@pytest.mark.gpu
def test_attention_shared_while_the_cache_of_tensor_maps_turns_over(cuda_status):
    """More queries at addresses of their own than there is room for maps: each has the result of a copy of it at one address, bit for bit."""
    n, dim, calls = 20, 64, 2 * 65536 + 2000
    k, v, t = (x.cuda() for x in forked([n], [33], [40] * n, 16, 1, dim, torch.bfloat16, 5, hole=0.0))
    plan, shared, lens = ops.PrefixGroups([n], "cuda"), torch.tensor([33], dtype=I32, device="cuda"), torch.full((n,), 40, dtype=I32, device="cuda")
    base = torch.randn(n * dim + 8 * calls, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    out, again, copy = (torch.empty(n, dim, dtype=torch.bfloat16, device="cuda") for _ in range(3))
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(calls):
        q = base[8 * i:8 * i + n * dim].view(n, dim)
        ops.paged_attention_shared(q, k, v, plan, shared, t, lens, out=out)
        if i % 300 == 0 or i % 65536 < 20 or i % 65536 > 65480:
            ops.paged_attention_shared(copy.copy_(q), k, v, plan, shared, t, lens, out=again)
            differ += (out != again).sum()
    assert int(differ) == 0


# ---- shared blocks -----------------------------------------------------------------------------------------------------------------------------
def weighed(blocks, device="cpu", bs=16):
    return PagedCache(blocks, bs, 2, 2, 64, device=device, quantization=CacheQuantization.FP8, attention_weights=True)


@pytest.mark.parametrize("device", DEVICES)
def test_evict_leaves_what_loses_no_tokens(device):
    """Only sequences that lose tokens get blocks of their own, and those only for the tokens that are kept; without room for all of them nothing changes."""
    c = weighed(5, device)
    c.allocate(1, 48)
    for p in c.pages:
        p.weight.copy_(torch.arange(p.weight.numel()).view(p.weight.shape))
        p.k.view(torch.uint8).random_(0, 127), p.v.view(torch.uint8).random_(0, 127)
    assert c.fork([1, 1], [2, 3], [48, 32])
    tables = [c.block_table(s) for s in (1, 2, 3)]
    state = [[t.clone() for t in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.weight)] for p in c.pages]

    def unchanged():
        assert [c.block_table(s) for s in (1, 2, 3)] == tables and c.free_blocks == 2 and c.shared_blocks == 3 and not c.thinned
        assert all(torch.equal(a, b) for p, was in zip(c.pages, state) for a, b in zip((p.k.view(torch.uint8), p.v.view(torch.uint8), p.weight), was))
    assert c.evict([1, 2, 3], [48, 48, 32], 48) == [48, 48, 32]
    unchanged()
    for bad in (dict(keep=0), dict(keep=16, recent=9, keep_first=8), dict(keep=16, recent=-1)):
        with pytest.raises(ValueError):
            c.evict([1], [48], **bad)
        unchanged()
    with pytest.raises(RuntimeError):
        c.evict([1, 3], [48, 32], 31)                              # the first would get two blocks, the other ones two
    unchanged()
    assert c.evict([1, 3], [48, 32], 32, recent=32) == [32, 32]    # the second stays; the last 32 tokens of the first
    assert c.block_table(3) == tables[2] and c.block_table(2) == tables[1] and not set(c.block_table(1)) & set(tables[1]) and c.thinned == {1}
    for p, (k, v, w) in zip(c.pages, state):
        for new, old in zip(c.block_table(1), tables[0][1:]):
            assert torch.equal(p.weight[new], w[old])
        for b in tables[1]:
            assert torch.equal(p.weight[b], w[b]) and torch.equal(p.k.view(torch.uint8)[b], k[b]) and torch.equal(p.v.view(torch.uint8)[b], v[b])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seed", range(3))
def test_blocks_of_their_own_for_several_sequences_or_none(device, seed):
    rng = random.Random(seed)
    c = PagedCache(20, 4, num_layers=1, num_kv_heads=1, head_dim=8, dtype=torch.float32, device=device)
    c.allocate(0, 40)
    c.k.copy_(torch.arange(20.0).view(1, 20, 1, 1, 1).expand_as(c.k))
    first = [float(c.k[0, b, 0, 0, 0]) for b in c.block_table(0)]
    assert c.fork([0] * 4, [1, 2, 3, 4], [rng.randrange(4, 40, 4) for _ in range(4)])
    refused = 0
    for _ in range(40):
        some = rng.sample(range(5), rng.randint(1, 4))
        spans = []
        for s in some:
            room = 4 * len(c.block_table(s))
            lo = rng.randrange(room)
            spans.append((lo, rng.randint(0, min(room - lo, 9))))
        before, free, shared = [c.block_table(s) for s in range(5)], c.free_blocks, c.shared_blocks
        try:
            c.own_all(some, [lo for lo, _ in spans], [n for _, n in spans])
        except RuntimeError:
            refused += 1
            assert [c.block_table(s) for s in range(5)] == before and (c.free_blocks, c.shared_blocks) == (free, shared)
            s = rng.randint(1, 4)                                  # room for the next ones
            c.free(s)
            assert c.fork([0], [s], [rng.randrange(4, 40, 4)])
            continue
        tables = [c.block_table(s) for s in range(5)]
        for s, (lo, n) in zip(some, spans):
            for i in range(lo // 4, (lo + n - 1) // 4 + 1 if n else 0):
                assert sum(tables[s][i] in t for t in tables) == 1
        assert all([float(c.k[0, b, 0, 0, 0]) for b in t] == first[:len(t)] for t in tables)
        assert c.num_blocks - c.free_blocks == len(set().union(*map(set, tables)))
    assert refused
    with pytest.raises(IndexError):
        c.own_all([0, 1, 77], [0, 0, 0], [1, 1, 1])
    c.own_all([77], [0], [0])


class Elsewhere:
    """A tensor as one on the second of two devices looks to the host."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 1

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("layers", [None, [CacheLayer(1, 8, 8)], [CacheLayer(state=(("z", (7,), None),))]])
def test_a_cache_on_another_device_is_refused_before_tables_change(layers, monkeypatch):
    c = PagedCache(6, 4, num_kv_heads=1, head_dim=8, dtype=torch.float32, layers=layers)
    c.allocate(1, 8), c.allocate(2, 6)
    assert c.fork([2], [3], [4])
    c.free(1)
    if layers is None:
        c.k, c.v = Elsewhere(c.k), Elsewhere(c.v)
    else:
        c.k, c.v = ([Elsewhere(t) for t in ts] for ts in (c.k, c.v)) if layers[0].kv_heads else (c.k, c.v)
        c.state = [{n: Elsewhere(t) for n, t in d.items()} for d in c.state]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    tables, free = [c.block_table(s) for s in (2, 3)], c.free_blocks
    for call in (lambda: c.fork([2], [4], [6]), lambda: c.own(3, 0, 4), lambda: c.own_all([2, 3], [0, 0], [6, 4]), c.compact):
        with pytest.raises(ValueError, match="device"):
            call()
        assert [c.block_table(s) for s in (2, 3)] == tables and c.block_table(4) == [] and (c.free_blocks, c.shared_blocks) == (free, 1)


# ---- attention weights of forked sequences -----------------------------------------------------------------------------------------------------
def weighing_runner(device, blocks=64):
    kw = dict(n_head=8, n_kv_head=2, d_model=512) if device == "cuda" else {}
    return ModelRunner(preset("llama-test", **kw), device=device, num_blocks=blocks, block_size=16, seed=2, kv_quantization=CacheQuantization.FP8, kv_weights=True)


def sums(r, seq, n):
    """The weights of a sequence's first n tokens, [layers, KV heads, n]."""
    table = r.cache.block_table(seq)
    return torch.stack([torch.cat(list(p.weight[table].transpose(0, 1).flatten(1)[:, :n]), 0) for p in r.cache.pages]).cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mixed", [False, True])
def test_forked_sequences_sum_weights_of_their_own(device, mixed):
    """Parent and children decoded together sum what sequences that never shared a block sum: the same operations on the same numbers, bit for bit."""
    prompt, more, last = list(range(3, 40)), list(range(60, 66)), [7, 300, 11, 500]
    got = []
    for forked in (False, True):
        r = weighing_runner(device)
        r.cache.allocate(1, 38)
        r.prefill(1, prompt)
        r.decode([1], [9], [38])
        if forked:
            assert r.cache.fork([1] * 3, [2, 3, 4], [38] * 3) and r.cache.shared_blocks == 2
        else:
            for s in (2, 3, 4):
                r.cache.allocate(s, 38)
                r.prefill(s, prompt)
                r.decode([s], [9], [38])
        for s in (1, 2, 3):
            r.cache.allocate(s, 48)
        for step in range(2):
            n = [39 + step] * 3
            if mixed:
                r.cache.allocate(9, 8)
                r.step_mixed([(9, more, 0, True)], [1, 2, 3], last[:3], n)
            else:
                r.decode([1, 2, 3], last[:3], n)
        got.append([sums(r, s, 40 if s < 4 else 38) for s in (1, 2, 3, 4)])
        assert r.cache.shared_blocks == 0 and r.cache.evict([1, 4], [40, 38], 20, recent=4) == [20, 20]
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_beam_search_where_weights_are_kept():
    r = weighing_runner("cpu", blocks=3 * 4)
    plain = ModelRunner(preset("llama-test"), device="cpu", num_blocks=64, block_size=16, seed=2, kv_quantization=CacheQuantization.FP8)
    prompt = list(range(20, 53))
    with pytest.raises(ValueError, match="blocks"):
        BeamSearch(r, 4).generate([prompt], 20)
    found = BeamSearch(r, 3).generate([prompt], 20)[0]            # every block that there is
    assert [h.tokens for h in found] == [h.tokens for h in BeamSearch(plain, 3).generate([prompt], 20)[0]] and r.cache.free_blocks == 12


# ---- moves -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
def test_blocks_are_numbers_not_bytes(device):
    t = torch.arange(8.0, device=device).view(4, 2)
    for bad in (bytes, bytearray):
        for src, dst in ((bad(4), [1]), ([0], bad(b"\1\0\0\0")), (bad(4), bad(b"\1\0\0\0"))):
            with pytest.raises(ValueError):
                ops.copy_blocks_([t], src, dst)
    assert t.flatten().tolist() == list(range(8))
    ops.copy_blocks_([t], torch.tensor([0]), (1,))
    assert t[1].tolist() == [0, 1]


def bytes_of(t, base):
    """The addresses of a tensor's bytes, relative to `base`'s first."""
    at = torch.arange(t.element_size())
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s * t.element_size()).flatten()
    return (at + t.data_ptr() - base.data_ptr()).tolist()


def cut(base, rng, rows):
    """A view of `rows` rows (dimension 1) somewhere in a flat tensor, its rows pieces at equal distances."""
    pitch = rng.choice((24, 24, 40, 48, 60))
    piece, segs = rng.randint(1, 6), rng.randint(1, 3)
    apart = rng.randint(piece, 12)
    outer = rng.randint(1, 2)
    first = rng.randrange(200)
    return base.as_strided((outer, rows, segs, piece), (rows * pitch + rng.choice((0, 7)), pitch, apart, 1), first)


@pytest.mark.parametrize("seed", range(8))
def test_moves_refuse_tensors_that_share_memory_and_no_others(seed):
    """Views of one tensor at random places, against the set of their bytes."""
    rng, base = random.Random(seed), torch.arange(2000, dtype=torch.int32)
    rows, met, index = 4, [0, 0], torch.tensor([1, 0, 3, 3])
    for _ in range(250):
        ts = [cut(base, rng, rows) for _ in range(rng.choice((2, 2, 3)))]
        every = [b for t in ts for b in bytes_of(t, base)]
        together = len(set(every)) < len(every)                   # two tensors, or two rows of one
        met[together] += 1
        was, want = base.clone(), base.clone()
        if together:
            with pytest.raises(ValueError):
                ops.reorder_rows_(ts, index, dim=1)
            with pytest.raises(ValueError):
                ops.copy_blocks_(ts, [1], [0], dim=1)
        else:
            for t in ts:
                v = want.as_strided(t.shape, t.stride(), t.storage_offset())
                v.copy_(v[:, index].clone())
            ops.reorder_rows_(ts, index, dim=1)
        assert torch.equal(base, want)
        base.copy_(was)
    assert min(met) > 20


@pytest.mark.parametrize("device", DEVICES)
def test_moves_of_parts_of_one_tensor(device):
    """Overlapping parts are refused, keys and values of all layers in one tensor of blocks are not; an index in memory of theirs is."""
    x = torch.arange(48.0, device=device).view(6, 8)
    was, i = x.clone(), torch.tensor([1, 0, 3, 2], device=device)
    for a, b in ((x[:4], x[2:]), (x[:4, :5], x[1:5, 4:]), (x[:4], x[1:5, 3:4]), (x[:4, ::4], x[:4, 4:])):
        with pytest.raises(ValueError):
            ops.reorder_rows_([a, b], i)
        with pytest.raises(ValueError):
            ops.copy_blocks_([a, b], [0], [3])
    longs = torch.arange(20, device=device).view(4, 5)
    with pytest.raises(ValueError):
        ops.reorder_rows_([longs[:2]], longs.view(-1)[7:9])
    with pytest.raises(ValueError):
        ops.reorder_rows_([longs], longs[1, :4])
    assert torch.equal(x, was) and longs.flatten().tolist() == list(range(20))
    inside = torch.tensor([[7, 7, 1, 0], [8, 8, 9, 9]], device=device)               # the index between its rows' columns
    ops.reorder_rows_([inside[:, :2]], inside[0, 2:])
    assert inside.tolist() == [[8, 8, 1, 0], [7, 7, 9, 9]]
    ops.reorder_rows_([x[:4, :4], x[:4, 4:]], i)
    assert torch.equal(x, was[[1, 0, 3, 2, 4, 5]])
    packed = torch.randn(5, 8, 2, 3, device=device)                # [blocks, layers, keys and values, ...]
    want = packed.clone()
    want[4] = want[1]
    ops.copy_blocks_([packed[:, l, j] for l in range(8) for j in range(2)], [1], [4])
    assert torch.equal(packed, want)


@pytest.mark.parametrize("device", DEVICES)
def test_moves_refuse_leaves_that_require_a_gradient(device):
    w, i = torch.nn.Parameter(torch.arange(12.0, device=device).view(4, 3)), torch.tensor([3, 2, 1, 0], device=device)
    other = torch.zeros(4, 2, device=device)
    for t in (w, w[:, 1:], w.view(4, 3, 1)):
        with pytest.raises(ValueError):
            ops.reorder_rows_([other, t], i)
        with pytest.raises(ValueError):
            ops.copy_blocks_([other, t], [0], [1])
    assert w.flatten().tolist() == list(range(12))
    with torch.no_grad():
        ops.reorder_rows_([w], i)
        ops.copy_blocks_([w[:, 1:]], [0], [1])
    assert w.tolist() == [[9, 10, 11], [6, 10, 11], [3, 4, 5], [0, 1, 2]]
    cache = torch.zeros(4, 3, device=device)                       # a dense cache that was filled where gradients are recorded
    cache[:2] = w[:2] * 2
    ops.reorder_rows_([cache], i)
    assert cache.tolist() == [[0, 0, 0], [0, 0, 0], [12, 20, 22], [18, 20, 22]]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 20])
def test_reorder_rows_past_four_gigabytes(rows):
    """Distances of rows and of copies that do not fit 32 bits."""
    size = (1 << 32) // rows + 4096
    t = torch.zeros(2, rows, size // 16 * 16, dtype=torch.uint8, device="cuda")
    t[:, :, -5000::7] = torch.arange(1, 2 * rows + 1, dtype=torch.uint8, device="cuda").view(2, rows, 1)
    index = torch.arange(rows, device="cuda").flip(0)
    ops.reorder_rows_([t], index, dim=1)
    want = torch.arange(1, 2 * rows + 1, dtype=torch.uint8, device="cuda").view(2, rows, 1).flip(1)
    assert bool((t[:, :, -5000::7] == want).all()) and not t[:, :, -4999::7].any() and not t[:, :, :4096].any()


# ---- scratch -----------------------------------------------------------------------------------------------------------------------------------
def test_scratch_is_sized_for_the_device_of_the_call(monkeypatch):
    """Two devices with different numbers of SMs, in turn: how work is cut, and so the scratch, goes by them."""
    from rustral_b200 import _native as N
    from rustral_b200.ops import beams, paged_e4m3
    now = []

    class Kernels:
        def rb_beam_select_scratch_bytes(self, groups, beams, vocab, count, kind):
            return 1000 * now[-1] + groups

        def rb_shared_prefix_scratch_bytes(self, batch, groups, heads, kv_heads, dim, bs, most):
            return 2000 * now[-1] + batch

        def rb_e4m3_decode_scratch_floats(self, batch, heads, kv_heads, dim, width, bs, accumulate):
            return 3000 * now[-1] + batch
    monkeypatch.setattr(N, "kernels", Kernels)
    sizes = {0: 148, 1: 160}
    for dev in (0, 1, 0, 1):
        now.append(sizes[dev])
        assert beams._select_bytes(dev, 7, 4, 1009, 8, 0) == 1000 * sizes[dev] + 7
        assert beams._shared_bytes(dev, 9, 2, 4, 2, 64, 16, 5) == 2000 * sizes[dev] + 9
        assert paged_e4m3._scratch_floats(dev, 11, 4, 2, 64, 33, 16, True) == 3000 * sizes[dev] + 11
    for cached in (beams._select_bytes, beams._shared_bytes, paged_e4m3._scratch_floats):
        cached.cache_clear()                                       # nothing of this stays


# ---- the search ------------------------------------------------------------------------------------------------------------------------------------
def test_length_penalties_that_are_no_powers_are_refused_first(monkeypatch):
    """Before a prompt is computed; a server answers that the request is bad."""
    from rustral_b200.serve import ServingEngine
    from rustral_b200.serve.http_server import BadRequest, engine_generate_fn
    r = ModelRunner(preset("gpt2-test"), device="cpu", num_blocks=32, block_size=4, seed=2)
    want = {}
    for alpha in (-30.0, -1, 0, 1, 60.0):
        found = BeamSearch(r, 3, length_penalty=alpha).generate([[5, 6, 7]], 6)[0]
        assert all(h.ranked == h.score / 6.0 ** alpha for h in found)
        want[alpha] = [h.tokens for h in found]
    assert len({str(w) for w in want.values()}) == 1               # all are six tokens long
    monkeypatch.setattr(ModelRunner, "step_mixed", lambda *a, **k: 1 / 0)
    for alpha in (math.nan, math.inf, -math.inf, 1e6, -1e6, 10 ** 6):
        with pytest.raises(ValueError):
            BeamSearch(r, 2, length_penalty=alpha).generate([[5, 6]], 5)
    fn = engine_generate_fn(ServingEngine(r))
    bad = [{"length_penalty": x} for x in (math.nan, 1e6, -1e6, "long", None, [1.0], 10 ** 400)] + [{"beams": x} for x in (None, [2], "two", math.inf, math.nan)]
    for body in bad:
        with pytest.raises(BadRequest):
            fn({"prompt": [1, 2], "max_tokens": 5, "beams": 2, **body})
    assert r.cache.free_blocks == 32


def test_two_ranks_search_alike():
    """Two tensor-parallel ranks find the same continuations, and their scores are what the whole model gives these tokens."""
    from concurrent.futures import ThreadPoolExecutor
    from rustral_b200.serve.weights import InferenceWeights
    cfg = preset("llama-test", seq_len=512, n_layer=2, d_model=256, n_head=4, ffn_dim=256, n_kv_head=2)
    whole = sharp(ModelRunner(cfg, device="cpu", num_blocks=64, seed=3), 4)
    ranks = Ranks(2)
    shards = [ModelRunner(cfg, params=InferenceWeights.shard_of(whole.params, cfg, i, 2), device="cpu", num_blocks=64, tp=ranks.of(i)) for i in range(2)]
    prompts = [[5, 300, 17, 44, 9], list(range(100, 140))]
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(lambda r: BeamSearch(r, 3, eos_id=7).generate(prompts, 6), shards))
    assert got[0] == got[1] and all(r.cache.free_blocks == 64 for r in shards)
    for p, found in zip(prompts, got[0]):
        assert len(found) == 3
        scores_are_their_tokens(whole, p, found, 1e-3)
