"""Serving over a cache in e4m3: what the runner stores, reads and attends over, against the oracle of the pages; graphs, the engine, eviction."""
import pytest
import torch

from paged_e4m3_oracle import Cache
from rustral_b200 import ops
from rustral_b200.core.errors import InvalidArgument
from rustral_b200.models.config import preset
from rustral_b200.ops import paged_e4m3 as e4m3_ops
from rustral_b200.serve import CacheQuantization, ModelRunner, PagedCache, ServingEngine
from rustral_b200.serve.model_runner import load_runner

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
FP8 = CacheQuantization.FP8


def runner_of(name, device, **kw):
    # heads of 64, as the kernels have them
    cfg = preset(name, seq_len=512, n_layer=2, d_model=256, n_head=4, ffn_dim=256, **({"n_kv_head": 2} if name == "llama-test" else {}))
    return ModelRunner(cfg, device=device, num_blocks=64, seed=3, kv_quantization=FP8, **kw)


def tokens(cfg, n, seed):
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Watch:
    """Follows every call of the cache's operators with an oracle of each layer's pages."""

    def __init__(self, monkeypatch, runner):
        self.oracles = {id(p): Cache(p) for p in runner.cache.pages}
        self.calls = {"append": 0, "read": 0, "attend": 0}
        append, read, attend = e4m3_ops.kv_append_e4m3, e4m3_ops.kv_read_e4m3, e4m3_ops.paged_attention_decode_e4m3

        def watched_append(pages, k, v, tables, lens, starts=None):
            append(pages, k, v, tables, lens, starts)
            o = self.oracles[id(pages)]
            o.append(k.cpu(), v.cpu(), tables.cpu(), lens.tolist(), list(range(k.shape[0] + 1)) if starts is None else starts.tolist())
            o.same(pages)
            self.calls["append"] += 1

        def watched_read(pages, tables, lens, starts, rows, dtype=torch.bfloat16, out=None):
            got = read(pages, tables, lens, starts, rows, dtype, out)
            o, n = self.oracles[id(pages)], lens.tolist()
            assert starts.tolist() == [sum(n[:i]) for i in range(len(n) + 1)] and rows == sum(n)
            for x, name in zip(got, "kv"):
                ref = torch.cat([o.tokens(name, tables.cpu(), b, m).reshape(m, -1) for b, m in enumerate(n)])
                assert torch.equal(x.cpu().double(), ref)
            self.calls["read"] += 1
            return got

        def watched_attend(q, pages, tables, lens, scale=None, out=None, accumulate=False):
            o = self.oracles[id(pages)]
            got = attend(q, pages, tables, lens, scale, out, accumulate)
            ref, err, _, _ = o.attend(q.cpu(), tables.cpu(), lens.tolist(), scale)
            assert bool(((got.cpu().double() - ref).abs() <= err + ref.abs() * torch.finfo(q.dtype).eps / 2 + 1e-30).all())
            if accumulate:
                o.w = pages.weight.cpu().double()
            self.calls["attend"] += 1
            return got

        for name, f in (("kv_append_e4m3", watched_append), ("kv_read_e4m3", watched_read), ("paged_attention_decode_e4m3", watched_attend)):
            monkeypatch.setattr(e4m3_ops, name, f)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["gpt2-test", "llama-test"])
def test_steps_follow_the_pages(device, name, monkeypatch):
    r = runner_of(name, device)
    r.use_graphs = False
    watch, cfg = Watch(monkeypatch, r), r.cfg
    a, b, c = tokens(cfg, 60, 1), tokens(cfg, 21, 2), tokens(cfg, 37, 3)
    for s, n in ((1, 70), (2, 30), (3, 40)):
        assert r.cache.allocate(s, n)
    r.step_mixed([(1, a[:25], 0, False), (2, b, 0, True)], [], [], [])
    assert watch.calls == {"append": 2, "read": 0, "attend": 0}
    # a later portion beside a whole prompt and a decoded sequence
    out, dec = r.step_mixed([(1, a[25:], 25, True), (3, c[:30], 0, False)], [2], [5], [22])
    assert watch.calls == {"append": 4, "read": 2, "attend": 2} and out[0].shape == dec[0].shape
    r.step_mixed([(3, c[30:], 30, True)], [1, 2], [7, 8], [61, 23])
    r.decode([1, 2, 3], [1, 2, 3], [62, 24, 38])
    assert watch.calls == {"append": 8, "read": 4, "attend": 6}


@pytest.mark.parametrize("device", DEVICES)
def test_portions_read_in_groups(device, monkeypatch):
    """More gathered keys than the limit: the same logits from several reads."""
    from rustral_b200.serve import model_runner
    logits = []
    for most in (model_runner.MOST_GATHERED, 1):
        monkeypatch.setattr(model_runner, "MOST_GATHERED", most)
        r = runner_of("llama-test", device)
        parts = []
        for s, n in ((1, 40), (2, 33), (3, 17)):
            assert r.cache.allocate(s, 60)
            r.step_mixed([(s, tokens(r.cfg, n, s), 0, False)], [], [], [])
            parts.append((s, tokens(r.cfg, 11, s + 9), n, True))
        assert r.cache.allocate(4, 20)
        out, _ = r.step_mixed(parts + [(4, tokens(r.cfg, 9, 8), 0, True)], [], [], [])
        logits.append(torch.stack(out))
    assert torch.equal(*logits)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gpt2-test", "llama-test"])
def test_graphs_give_what_eager_steps_give(name, cuda_status):
    got = []
    for graphs in (True, False):
        r = runner_of(name, "cuda", kv_weights=True)
        r.use_graphs = graphs
        for s in (1, 2):
            assert r.cache.allocate(s, 100)
            r.prefill(s, tokens(r.cfg, 20 + s, s))
        lens, logits = [21, 22], []
        for step in range(4):
            lens = [n + 1 for n in lens]
            logits.append(r.decode([1, 2], [step, step + 1], lens).clone())
        lens = r.cache.evict([1, 2], lens, 16, 4, 1)
        assert lens == [16, 16] and r.cache.allocate(1, 20) and r.cache.allocate(2, 20)
        for step in range(4):
            lens = [n + 1 for n in lens]
            logits.append(r.decode([1, 2], [step, step + 1], lens, [25 + step, 26 + step]).clone())
        got.append((torch.stack(logits), torch.stack([p.weight for p in r.cache.pages])))
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gpt2-test", "llama-test"])
def test_gpu_logits_match_cpu(name, cuda_status):
    """As the runner with a bf16 cache is held to the CPU's (tests/test_gpu_serving.py), with the same cache of codes on either side: its keys differ by the
    bf16 rounding of the projections, which moves a number by a step of its code, 2^-3 of it, where it lies beside a border."""
    gpu, cpu = runner_of(name, "cuda"), runner_of(name, "cpu")
    cpu.params.master.copy_(gpu.params.lowp.float().cpu())
    cpu.params.sync_lowp()
    prompt = tokens(gpu.cfg, 37, 0)
    for r in (gpu, cpu):
        assert r.cache.allocate(1, 50)
    lg, lc = gpu.prefill(1, prompt), cpu.prefill(1, prompt)
    assert (lg.float().cpu() - lc).abs().max() < 0.05 * lc.abs().max() + 0.02
    tok = int(lc[:gpu.cfg.vocab_size].argmax())
    for step in range(3):
        dg, dc = gpu.decode([1], [tok], [38 + step]), cpu.decode([1], [tok], [38 + step])
        assert (dg.float().cpu() - dc).abs().max() < 0.05 * dc.abs().max() + 0.02
        tok = int(dc[0, :gpu.cfg.vocab_size].argmax())


@pytest.mark.parametrize("device", DEVICES)
def test_engine_completes_and_frees(device):
    r = runner_of("llama-test", device, kv_weights=True)
    eng = ServingEngine(r, max_batch_size=4, prefill_chunk=16)
    ids = [eng.submit(tokens(r.cfg, n, n), 6) for n in (3, 30, 64, 17, 5)]
    done = eng.run_to_completion()
    assert sorted(x.id for x in done) == ids and all(len(x.generated) == 6 for x in done)
    assert r.cache.free_blocks == 64


@pytest.mark.parametrize("device", DEVICES)
def test_eviction_in_a_runner(device):
    r = runner_of("llama-test", device, kv_weights=True)
    r.use_graphs = False
    assert r.cache.allocate(1, 120) and r.cache.allocate(2, 40)
    r.prefill(1, tokens(r.cfg, 100, 1))
    r.prefill(2, tokens(r.cfg, 20, 2))
    lens = [100, 20]
    for step in range(3):
        lens = [n + 1 for n in lens]
        logits = r.decode([1, 2], [3, 4], lens)
    grown = torch.stack([p.weight.sum() for p in r.cache.pages]).cpu()
    # every step adds one for each of two sequences and four heads
    torch.testing.assert_close(grown, torch.full((2,), 3.0 * 2 * 4), rtol=1e-5, atol=0)
    # a budget that all sequences keep changes nothing but the blocks behind their tokens
    assert r.cache.evict([1, 2], lens, 200) == lens and len(r.cache.block_table(1)) == 7 and len(r.cache.block_table(2)) == 2
    before = r.cache.free_blocks
    assert r.cache.evict([1, 2], lens, 32, 8, 2) == [32, 23]
    assert r.cache.free_blocks == before + 5 and len(r.cache.block_table(1)) == 2
    assert r.cache.allocate(1, 33)
    logits = r.decode([1, 2], [5, 6], [33, 24], [103, 23])
    assert bool(torch.isfinite(logits).all())


def test_positions_apart_from_lengths_are_those_without():
    """Positions that are the lengths less one: the same logits as without them, from a cache in e4m3 (both architectures)."""
    for name in ("gpt2-test", "llama-test"):
        out = []
        for given in (False, True):
            r = runner_of(name, "cpu")
            assert r.cache.allocate(1, 40)
            r.prefill(1, tokens(r.cfg, 20, 1))
            out.append(r.decode([1], [4], [21], [20] if given else None))
        assert torch.equal(*out)


def test_trim():
    c = PagedCache(8, 16, allocate_storage=False)
    assert c.allocate(1, 70) and c.block_table(1) == [0, 1, 2, 3, 4] and c.free_blocks == 3
    assert c.trim(1, 33) == 2 and c.block_table(1) == [0, 1, 2] and c.free_blocks == 5
    assert c.trim(1, 100) == 0 and c.trim(1, 0) == 3 and c.free_blocks == 8
    assert c.allocate(1, 17) and len(c.block_table(1)) == 2
    with pytest.raises(InvalidArgument):
        c.trim(9, 1)


def test_refusals():
    with pytest.raises(InvalidArgument):
        PagedCache(4, 16, quantization=CacheQuantization.INT8)
    with pytest.raises(InvalidArgument):
        PagedCache(4, 16, attention_weights=True)
    with pytest.raises(ValueError):
        ModelRunner(preset("dolurax-test"), device="cpu", kv_quantization=FP8)
    c = PagedCache(4, 16, head_dim=64, quantization=FP8)
    with pytest.raises(InvalidArgument):
        c.evict([1], [1], 1)                                          # no weights
    c = PagedCache(4, 16, head_dim=64, quantization=FP8, attention_weights=True)
    assert c.allocate(1, 20) and c.evict([], [], 4) == []
    for ids, lens in (([1], [33]), ([1], [-1]), ([1, 1], [4, 4]), ([1], []), ([2], [4])):
        with pytest.raises(InvalidArgument):
            c.evict(ids, lens, 4)
    assert c.memory_bytes() == 4 * (2 * 16 * 64 + 2 + 16 * 4)
    assert ops.PagesE4M3.zeros(4, 16, 1, 64).memory_bytes() == 4 * (2 * 16 * 64 + 2)
    r = ModelRunner(preset("llama-test"), device="cpu", num_blocks=8)
    with pytest.raises(ValueError):
        r.decode([1], [1], [1], [0])                                  # positions without a cache in e4m3


def test_a_loaded_runner_keeps_weights():
    r = load_runner("llama-test", device="cpu", num_blocks=4, kv_quantization=FP8, kv_weights=True)
    assert r.kv_weights and all(p.weight is not None for p in r.cache.pages)
    with pytest.raises(InvalidArgument):
        load_runner("llama-test", device="cpu", num_blocks=4, kv_weights=True)


def thinned(name, device, graphs=False):
    """A runner with 41 tokens of sequence 1 brought down to 16."""
    r = runner_of(name, device, kv_weights=True)
    r.use_graphs = graphs
    assert r.cache.allocate(1, 60)
    r.prefill(1, tokens(r.cfg, 40, 1))
    r.decode([1], [3], [41])
    assert r.cache.evict([1], [41], 16, 4, 1) == [16] and r.cache.thinned == {1}
    assert r.cache.allocate(1, 60) and r.cache.allocate(2, 40)
    return r


def keys_of(r, toks, positions):
    """Keys of layer 0 in 64 bits from the weights, and how far 16-bit activations may take them: the embedding and the norm's output are rounded (2^-8 each, the
    first also through the norm's statistics), and so are the product and the rotation."""
    P, cfg = r.params, r.cfg
    w = lambda n: P.w(n).double().cpu()  # noqa: E731
    pos, H, G, D = torch.tensor(positions), cfg.n_head, cfg.n_kv_head, cfg.head_dim
    x = w("tok_embed.embed")[torch.tensor(toks)]
    if cfg.arch == "gpt2":
        x = x + w("pos_embed.embed")[pos]
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + cfg.norm_eps) * w("layers.0.ln1.weight")
    x = x + (w("layers.0.ln1.bias") if cfg.arch == "gpt2" else 0.0)
    W = w("layers.0.attn.wqkv.weight")[H * D:(H + G) * D]
    k = x @ W.t() + (w("layers.0.attn.wqkv.bias")[H * D:(H + G) * D] if cfg.arch == "gpt2" else 0.0)
    off = 3 * 2.0 ** -8 * (x.abs() @ W.abs().t()) + 2.0 ** -8 * k.abs()
    if cfg.arch == "llama":
        a, b = k.view(-1, G, 2, D // 2).unbind(2)
        angle = pos.double()[:, None, None] * cfg.rope_theta ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
        k = torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], 2).view(-1, G * D)
        off = off.view(-1, G, 2, D // 2).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(-1, G * D)
        # the rotation's own rounding, and of a 32-bit angle 2^-24 of it and of its cosine's argument
        off = off + k.abs() * 2.0 ** -8 + pos.double()[:, None] * 2.0 ** -22 * k.abs().amax()
    return k, off


def holds_keys(r, seq, place, toks, positions):
    """The pages' keys of tokens at places `place` on are those of tokens `toks` at `positions`, and not those at their places."""
    pages, n = r.cache.pages[0], place + len(toks)
    t = torch.tensor([r.cache.block_table(seq)], dtype=torch.int32, device=r.device)
    lens, starts = (torch.tensor(x, dtype=torch.int32, device=r.device) for x in ([n], [0, n]))
    got = ops.kv_read_e4m3(pages, t, lens, starts, n, dtype=torch.float32)[0][place:].double().cpu()
    e = pages.k_exp[t[0].long()][torch.arange(place, n) // 16].double().cpu().repeat_interleave(r.cfg.head_dim, 1)
    rounded = lambda k: k.abs() * 2.0 ** -3 + torch.exp2(e - 9)  # noqa: E731  half a step of a code, twice where its page's exponent grew
    want, off = keys_of(r, toks, positions)
    assert bool(((got - want).abs() <= off + rounded(want)).all())
    for i, p in enumerate(positions):
        if p != place + i:
            other, off2 = keys_of(r, toks[i:i + 1], [place + i])
            assert bool(((got[i] - other[0]).abs() > off2[0] + rounded(other)[i]).any())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["gpt2-test", "llama-test"])
def test_positions_decide_the_keys(name, graphs, device):
    """Steps of all kinds after an eviction: the stored keys are those of the positions that were given, formed apart from the runner."""
    r = thinned(name, device, graphs)
    for i, (tok, pos) in enumerate(((7, 41), (9, 42), (11, 90))):     # with graphs: captured, then replayed
        r.decode([1], [tok], [17 + i], [pos])
        holds_keys(r, 1, 16 + i, [tok], [pos])
    r.step([], [1], [5], [20], {1: 91})
    holds_keys(r, 1, 19, [5], [91])
    more = tokens(r.cfg, 23, 9)
    logits, decoded = r.step([(2, more, 0, True)], [1], [6], [21], {1: 92})
    assert bool(torch.isfinite(logits[0]).all()) and bool(torch.isfinite(decoded).all())
    holds_keys(r, 1, 20, [6], [92])
    holds_keys(r, 2, 0, more, list(range(23)))
    r.step_mixed([(1, more[:5], 21, True)], [2], [8], [24], {1: 93})
    holds_keys(r, 1, 21, more[:5], [93, 94, 95, 96, 97])
    holds_keys(r, 2, 23, [8], [23])
    r.step_mixed([], [1, 2], [4, 4], [27, 25], {1: 98})
    holds_keys(r, 1, 26, [4], [98])
    holds_keys(r, 2, 24, [4], [24])


@pytest.mark.parametrize("device", DEVICES)
def test_a_mixed_step_gives_what_decoding_gives(device):
    """A decoded row beside a portion of another sequence, after an eviction: the logits of a decoding step at the same position."""
    out = []
    for mixed in (False, True):
        r = thinned("llama-test", device)
        if mixed:
            out.append(r.step([(2, tokens(r.cfg, 9, 2), 0, True)], [1], [6], [17], {1: 41})[1][0])
        else:
            out.append(r.decode([1], [6], [17], [41])[0])
    off = (out[0] - out[1]).abs().max()                               # products of other numbers of rows may add up in another order
    assert float(off) <= float(out[0].abs().max()) * (2.0 ** -5 if device == "cuda" else 1e-5)


def test_sequences_that_tokens_have_left_ask_for_positions():
    r = thinned("llama-test", "cpu")
    more = tokens(r.cfg, 5, 2)
    for call in (lambda: r.decode([1], [4], [17]), lambda: r.step([], [1], [4], [17]), lambda: r.step([], [1], [4], [17], {2: 0}),
                 lambda: r.step([(2, more, 0, True)], [1], [4], [17]), lambda: r.step_mixed([(1, more, 16, True)], [], [], []),
                 lambda: r.decode([1], [4], [17], []), lambda: r.decode([1], [4], [17], [-1])):
        before = r.cache.pages[0].k.view(torch.uint8).clone()
        with pytest.raises(ValueError):
            call()
        assert torch.equal(before, r.cache.pages[0].k.view(torch.uint8))
    assert r.cache.evict([1], [16], 12) == [12] and r.cache.allocate(2, 40)
    r.prefill(2, more)
    r.decode([2], [4], [6])
    assert r.cache.evict([2], [6], 3) == [3]
    with pytest.raises(ValueError):
        r.step([(2, more, 0, True)], [1], [4], [13])                  # 2 would begin anew, but nothing is done without a position of 1
    assert r.cache.thinned == {1, 2}
    r.cache.free(2)
    r.cache.free(1)
    assert not r.cache.thinned and r.cache.allocate(1, 60)
    r.prefill(1, tokens(r.cfg, 40, 1))
    r.decode([1], [4], [41])
    assert r.cache.evict([1], [41], 50) == [41] and not r.cache.thinned                  # nothing left
    assert r.cache.evict([1], [41], 20) == [20] and r.cache.trim(1, 0) == 2 and not r.cache.thinned
    assert r.cache.allocate(1, 60)
    r.prefill(1, more)
    r.decode([1], [4], [6])
    assert r.cache.evict([1], [6], 3) == [3] and r.cache.allocate(1, 60)
    r.prefill(1, more)                                                # a portion that begins at 0
    r.decode([1], [4], [6])
    g = thinned("gpt2-test", "cpu")
    with pytest.raises(ValueError):
        g.decode([1], [4], [17], [g.cfg.seq_len])                     # no such learned position
    plain = ModelRunner(preset("llama-test"), device="cpu", num_blocks=8)
    assert plain.cache.allocate(1, 4)
    for call in (lambda: plain.step([], [1], [1], [1], {1: 3}), lambda: plain.step_mixed([], [1], [1], [1], {1: 3})):
        with pytest.raises(ValueError):
            call()


def test_evict_refuses_before_it_drops():
    """A sequence that is not there, or a budget that is none: nothing has been dropped or given back."""
    c = PagedCache(8, 16, num_layers=2, head_dim=64, quantization=FP8, attention_weights=True)
    assert c.allocate(1, 60)
    for p in c.pages:
        p.weight.uniform_()
    before = [p.weight.clone() for p in c.pages]
    for ids, lens, keep, recent in (([1, 9], [60, 0], 16, 0), ([1], [60], 0, 0), ([1], [60], 4, 5)):
        with pytest.raises((InvalidArgument, ValueError)):
            c.evict(ids, lens, keep, recent)
        assert all(torch.equal(p.weight, w) for p, w in zip(c.pages, before)) and len(c.block_table(1)) == 4 and not c.thinned
    assert c.allocate(2, 0) and c.evict([1, 2], [60, 0], 16) == [16, 0]             # a sequence without tokens is one
    assert not any(torch.equal(p.weight, w) for p, w in zip(c.pages, before))


@pytest.mark.parametrize("device", DEVICES)
def test_evict_all_sequences_right_after_their_prompts(device):
    """Weights of zero in every layer: the earliest tokens stay beside the last."""
    lens, keep, recent, G = [20 + 7 * b % 90 for b in range(40)], 18, 6, 8
    c = PagedCache(sum((n + 15) // 16 for n in lens), 16, 2, G, 64, device=device, quantization=FP8, attention_weights=True)
    g, want = torch.Generator().manual_seed(1), []
    ids = list(range(len(lens)))
    assert all(c.allocate(s, n) for s, n in zip(ids, lens))
    table = torch.empty((len(lens), max((n + 15) // 16 for n in lens)), dtype=torch.int32)
    c.fill_tables(ids, table)
    starts = torch.tensor([0, *lens], dtype=torch.int32).cumsum(0, dtype=torch.int32)
    for p in c.pages:
        k = torch.randn(sum(lens), G * 64, generator=g).bfloat16().to(device)
        ops.kv_append_e4m3(p, k, -k, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device), starts.to(device))
        want.append(Cache(p))
    assert c.evict(ids, lens, keep, recent) == [keep] * len(lens) and c.thinned == set(ids)
    for p, o in zip(c.pages, want):
        o.evict(table, lens, keep, recent, 0)
        o.same(p)
    assert all(len(c.block_table(s)) == 2 for s in ids)


class Ranks:
    """Ranks of one process, a thread each, with the calls that a step makes of parallel.tp_inference.TPInferenceComm."""

    def __init__(self, world):
        import threading
        self.world, self.meet, self.staged = world, threading.Barrier(world, timeout=60), [None] * world

    def of(self, rank):
        ranks = self

        class Comm:
            world = ranks.world
            transport = "threads"

            def __init__(self):
                self.rank = rank

            def staging(self, rows, cols):
                ranks.staged[rank] = torch.empty(rows, cols)
                return ranks.staged[rank]

            def _all(self):
                ranks.meet.wait()
                got = [t.clone() for t in ranks.staged]
                ranks.meet.wait()
                return got

            def all_reduce(self, rows, cols, residual=None):
                total = sum(self._all())
                return total if residual is None else total + residual

            def all_gather_cols(self, rows, cols):
                return torch.cat(self._all(), 1)

            def end_step(self):
                pass
        return Comm()


def test_ranks_cache_their_heads_in_e4m3():
    """Two tensor-parallel ranks: a page's exponents are a head's own, so that every rank holds the codes that the whole model has for its heads, also after an
    eviction, and all have its logits."""
    from concurrent.futures import ThreadPoolExecutor
    from rustral_b200.serve.weights import InferenceWeights
    cfg = preset("llama-test", seq_len=512, n_layer=2, d_model=256, n_head=4, ffn_dim=256, n_kv_head=2)
    whole = ModelRunner(cfg, device="cpu", num_blocks=32, seed=3, kv_quantization=FP8, kv_weights=True)
    ranks = Ranks(2)
    shards = [ModelRunner(cfg, params=InferenceWeights.shard_of(whole.params, cfg, i, 2), device="cpu", num_blocks=32, tp=ranks.of(i),
                          kv_quantization=FP8, kv_weights=True) for i in range(2)]
    a, b = tokens(cfg, 50, 1), tokens(cfg, 20, 2)

    @torch.no_grad()
    def steps(r):
        assert r.cache.allocate(1, 80) and r.cache.allocate(2, 40)
        out = [r.step([(1, a[:30], 0, False), (2, b, 0, True)], [], [], [])[0][1][None]]
        logits, decoded = r.step([(1, a[30:], 30, True)], [2], [5], [21])
        out += [logits[0][None], decoded]
        out.append(r.decode([1, 2], [6, 7], [51, 22]))
        before = [p.k.float() * torch.exp2(p.k_exp.float())[..., None, None] for p in r.cache.pages]
        lens = r.cache.evict([1, 2], [51, 22], 30, 8, 2)
        out.append(r.decode([1, 2], [8, 9], [lens[0] + 1, lens[1] + 1], [51, 22]))
        return torch.cat(out), before

    want, keys = steps(whole)
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(steps, shards))
    assert torch.equal(got[0][0], got[1][0])
    for i, (logits, k) in enumerate(got):
        assert k[0].shape[1] == 1
        # sums of two ranks add up in another order: a number beside a border of its code may take the other code, a step of 2^-3 of it
        for x, y in zip(keys, k):
            assert bool(((x[:, i] - y[:, 0]).abs() <= x[:, i].abs() * 2.0 ** -3 + 1e-4).all())
            assert float((x[:, i] != y[:, 0]).float().mean()) < 0.01
        torch.testing.assert_close(logits[:, :cfg.vocab_size], want[:, :cfg.vocab_size], rtol=0, atol=0.05 * float(want.abs().max()) + 0.02)
