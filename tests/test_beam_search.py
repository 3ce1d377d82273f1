"""Sequences that share blocks (PagedCache.fork, own, compact), beam search over them, and dense caches in the order of selected beams."""
import random

import pytest
import torch

from rustral_b200 import ops
from rustral_b200.core.errors import InvalidArgument
from rustral_b200.models.config import preset
from rustral_b200.ops import beams as beam_ops
from rustral_b200.serve import (BatchedCache, BeamSearch, CacheConfig, CacheQuantization, KVCache, ModelRunner, PagedCache, ServingEngine, SlidingWindowCache)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ---- shared blocks -----------------------------------------------------------------------------------------------------------------------------
def write(cache, seq, first, n, value):
    """Tokens first .. first + n - 1 hold `value` in every layer, as a step would store them."""
    cache.own(seq, first, n)
    for i in range(first, first + n):
        b, o = divmod(cache.slot(seq, i), cache.block_size)
        cache.k[:, b, o], cache.v[:, b, o] = value, -value


def held(cache, seq, n):
    return [float(cache.k[l, cache.slot(seq, i) // cache.block_size, cache.slot(seq, i) % cache.block_size, 0, 0]) for i in range(n) for l in (0,)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("seed", range(4))
def test_forked_sequences_never_see_each_others_tokens(device, seed):
    """Random forks, writes anywhere, trims, frees and compactions against lists of numbers."""
    rng = random.Random(seed)
    cache = PagedCache(24, 4, num_layers=2, num_kv_heads=1, head_dim=8, dtype=torch.float32, device=device)
    want, ids, value = {}, iter(range(10 ** 6)), 1.0
    for _ in range(250):
        act = rng.choice(("new", "fork", "fork", "append", "append", "write", "trim", "free", "compact"))
        s = rng.choice(sorted(want)) if want else None
        if act == "new" or s is None:
            s, n = next(ids), rng.randint(0, 9)
            if cache.allocate(s, n):
                write(cache, s, 0, n, value)
                want[s] = [value] * n
        elif act == "fork":
            children, sizes = [next(ids) for _ in range(rng.randint(1, 3))], []
            sizes = [rng.randint(0, len(want[s])) for _ in children]
            free = cache.free_blocks
            if cache.fork([s] * len(children), children, sizes):
                for c, n in zip(children, sizes):
                    want[c] = want[s][:n]
                assert cache.free_blocks == free - sum(n % 4 != 0 for n in sizes)
            else:
                assert cache.free_blocks == free and all(cache.block_table(c) == [] for c in children)
        elif act == "append":
            n = len(want[s]) + rng.randint(1, 5)
            if cache.allocate(s, n) and cache.free_blocks >= 2:
                write(cache, s, len(want[s]), n - len(want[s]), value)
                want[s] += [value] * (n - len(want[s]))
        elif act == "write" and want[s]:
            a = rng.randrange(len(want[s]))
            n = rng.randint(1, len(want[s]) - a)
            if cache.free_blocks >= n // 4 + 2:
                write(cache, s, a, n, value)
                want[s][a:a + n] = [value] * n
        elif act == "trim":
            n = rng.randint(0, len(want[s]))
            cache.trim(s, n)
            want[s] = want[s][:n]
        elif act == "free":
            cache.free(s)
            del want[s]
        elif act == "compact":
            used = cache.num_blocks - cache.free_blocks
            cache.compact()
            assert all(b < used for q in want for b in cache.block_table(q)) and cache.num_blocks - cache.free_blocks == used
        value += 1.0
        tables = [set(cache.block_table(q)) for q in want]
        every = set().union(*tables) if tables else set()
        assert len(every) == cache.num_blocks - cache.free_blocks
        assert cache.shared_blocks == sum(sum(b in t for t in tables) > 1 for b in every)
        for q in want:
            assert held(cache, q, len(want[q])) == want[q]
    for q in list(want):
        cache.free(q)
    assert cache.free_blocks == cache.num_blocks and cache.shared_blocks == 0


def test_fork_refuses():
    c = PagedCache(4, 4, head_dim=8, dtype=torch.float32)
    c.allocate(1, 6)
    for parents, children, n in (([2], [3], [1]), ([1], [1], [4]), ([1], [3], [9]), ([1], [3], [-1]), ([1, 1], [3, 3], [1, 1]), ([1], [3, 4], [1]), ([1, 3], [3, 4], [1, 1])):
        with pytest.raises(InvalidArgument):
            c.fork(parents, children, n)
    assert c.fork([1, 1, 1], [3, 4, 5], [6, 6, 6]) is False and c.free_blocks == 2 and c.shared_blocks == 0
    assert c.fork([1, 1], [3, 4], [6, 5]) and c.free_blocks == 0
    with pytest.raises(RuntimeError):
        c.own(3, 0, 1)                                            # the shared block has no free one to be copied to
    with pytest.raises(IndexError):
        c.own(3, 8, 1)
    c.free(1), c.free(3)
    assert c.shared_blocks == 0 and c.own(4, 0, 5) is None
    assert c.fork([4], [9], [0]) and c.block_table(9) == []
    assert c.compact() >= 0


@pytest.mark.parametrize("device", DEVICES)
def test_fork_copies_codes_exponents_weights_and_states(device):
    c = PagedCache(8, 16, 2, 3, 64, device=device, quantization=CacheQuantization.FP8, attention_weights=True)
    c.allocate(1, 20)
    for p in c.pages:
        for t in (p.k, p.v):
            t.view(torch.uint8).random_(0, 127)
        p.k_exp.random_(-9, 9), p.v_exp.random_(-9, 9), p.weight.uniform_()
    c.thinned.add(1)
    assert c.fork([1, 1], [2, 3], [20, 32]) and {2, 3} <= c.thinned
    a, b, d = c.block_table(1), c.block_table(2), c.block_table(3)
    assert a[0] == b[0] and a[1] != b[1] and d == a
    for p in c.pages:
        for t in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.k_exp, p.v_exp, p.weight):
            assert torch.equal(t[a[1]], t[b[1]])
    new = c.evict([3], [32], 16)                                  # moves tokens inside its pages: they become its own
    assert new == [16] and c.block_table(1) == a and not set(c.block_table(3)) & set(a)
    from rustral_b200.serve import CacheLayer
    c = PagedCache(8, 4, dtype=torch.float32, device=device, num_slots=3,
                   layers=[CacheLayer(2, 8, 4, (("s", (3, 5), torch.float32),)), CacheLayer(1, 8, 4, joint=True), CacheLayer(2, 8, 4, kv_of=0), CacheLayer(state=(("z", (7,), None),))])
    c.allocate(1, 6)
    for d in c.state:
        for t in d.values():
            t.normal_()
    for t in (c.k[0], c.v[0], c.k[1]):
        t.normal_()
    assert c.fork([1, 1], [2, 3], [6, 4]) and not c.fork([1], [4], [4])                     # no slot
    for d in c.state:
        for t in d.values():
            assert torch.equal(t[c.state_slot(1)], t[c.state_slot(2)]) and torch.equal(t[c.state_slot(1)], t[c.state_slot(3)])
    a, b = c.block_table(1), c.block_table(2)
    for t in (c.k[0], c.v[0], c.k[1]):
        assert torch.equal(t[a[1]], t[b[1]])


def test_a_step_that_begins_a_forked_sequence_anew_leaves_the_others():
    cfg = preset("gpt2-test")
    r = ModelRunner(cfg, device="cpu", num_blocks=32, block_size=4, seed=1)
    prompt = list(range(5, 15))
    r.cache.allocate(1, 11)
    r.prefill(1, prompt)
    want = r.decode([1], [3], [11])
    r.cache.trim(1, 10)
    assert r.cache.fork([1], [2], [10])
    r.step_mixed([(2, list(range(40, 48)), 0, True)], [], [], [])                       # writes blocks that sequence 1 has too
    r.cache.allocate(1, 11)
    assert torch.allclose(r.decode([1], [3], [11]), want, atol=1e-5)


# ---- the search ------------------------------------------------------------------------------------------------------------------------------------
def log_probs(r, tokens):
    """Logarithmic probabilities of the next token behind these, through a sequence of its own."""
    r.cache.allocate(7, len(tokens))
    logits = r.prefill(7, tokens)[:r.cfg.vocab_size].double().cpu()
    r.cache.free(7)
    return torch.log_softmax(logits, -1)


def plain_search(r, prompt, beams, max_tokens, eos, alpha):
    """Beam search with a whole pass for every beam and step."""
    live, done = [([], 0.0)], []
    finish = lambda t, s: done.append((s / len(t) ** alpha, t, s))  # noqa: E731
    for step in range(max_tokens):
        cand = []
        for t, s in live:
            lp = log_probs(r, prompt + t)
            cand += [(s + float(x), t + [int(i)]) for x, i in zip(*lp.topk(2 * beams))]
        cand.sort(key=lambda c: -c[0])
        live = []
        for j, (s, t) in enumerate(cand[:2 * beams]):
            if t[-1] == eos:
                if j < beams:
                    finish(t, s)
            elif len(live) < beams:
                live.append((t, s))
        done.sort(key=lambda h: -h[0])
        if len(done) >= beams and max(s for _, s in live) / (step + 1) ** alpha <= done[beams - 1][0]:
            live = []
            break
    for t, s in live:
        finish(t, s)
    done.sort(key=lambda h: -h[0])
    return done[:beams]


def sharp(r, seed):
    """Wider embeddings, so that continuations differ by more than rounding."""
    w = r.params.w("tok_embed.embed") if r.cfg.tie_embeddings else r.params.w("head.weight")
    with torch.no_grad():
        w.mul_(torch.exp2(torch.rand(w.shape[0], 1, generator=torch.Generator().manual_seed(seed)) * 3 + 2).to(w))
    return r


@pytest.mark.parametrize("name", ["gpt2-test", "llama-test"])
@pytest.mark.parametrize("beams,max_tokens,alpha", [(1, 6, 1.0), (3, 8, 1.0), (5, 7, 0.0), (4, 1, 1.0)])
def test_beam_search_is_the_plain_search(name, beams, max_tokens, alpha):
    r = sharp(ModelRunner(preset(name), device="cpu", num_blocks=96, block_size=4, seed=3), 4)
    g = torch.Generator().manual_seed(beams)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 12)]
    # a token that searches do meet ends them
    eos = plain_search(r, prompts[0], beams, 3, None, alpha)[-1][1][-1] if max_tokens > 1 else None
    free = r.cache.free_blocks
    got = BeamSearch(r, beams, eos, alpha).generate(prompts, max_tokens)
    assert r.cache.free_blocks == free and r.cache.shared_blocks == 0
    for p, found in zip(prompts, got):
        want = plain_search(r, p, beams, max_tokens, eos, alpha)
        assert [h.tokens for h in found] == [t for _, t, _ in want]
        assert all(abs(h.score - s) < 1e-3 and h.ended == (t[-1] == eos) for h, (_, t, s) in zip(found, want))


def scores_are_their_tokens(r, prompt, found, tol):
    for h in found:
        total = 0.0
        for i, t in enumerate(h.tokens):
            total += float(log_probs(r, prompt + h.tokens[:i])[t])
        assert abs(total - h.score) <= tol * len(h.tokens), (total, h.score)
    assert [h.ranked for h in found] == sorted((h.ranked for h in found), reverse=True)
    assert len({tuple(h.tokens) for h in found}) == len(found)


def test_beam_search_with_recurrent_states_and_with_e4m3_pages():
    r = ModelRunner(preset("vafodra-test"), device="cpu", num_blocks=64, num_slots=8)
    prompt = [3, 14, 15, 92, 65]
    found = BeamSearch(r, 3).generate([prompt, prompt[:2]], 5)
    scores_are_their_tokens(r, prompt, found[0], 1e-3)
    assert r.cache.free_slots == 8 and r.cache.free_blocks == 64
    with pytest.raises(ValueError, match="slots"):
        BeamSearch(r, 9).generate([prompt], 5)
    r = ModelRunner(preset("llama-test"), device="cpu", num_blocks=64, block_size=4, kv_quantization=CacheQuantization.FP8)
    found = BeamSearch(r, 3).generate([prompt], 9)[0]
    assert len(found) == 3 and all(len(h.tokens) == 9 for h in found) and r.cache.free_blocks == 64


def test_beam_search_refuses_and_gives_everything_back(monkeypatch):
    r = ModelRunner(preset("gpt2-test"), device="cpu", num_blocks=12, block_size=4)
    for bad in (lambda: BeamSearch(r, 0), lambda: BeamSearch(r, 65), lambda: BeamSearch(r).generate([[1], []], 3), lambda: BeamSearch(r).generate([[1]], 0),
                lambda: BeamSearch(r).generate([[1] * 120], 20), lambda: BeamSearch(r, 4).generate([[1] * 9], 8)):
        with pytest.raises(ValueError):
            bad()
    assert BeamSearch(r).generate([], 3) == []
    calls = []

    def failing(*a, **k):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("step failed")
        return ModelRunner.decode(r, *a, **k)
    monkeypatch.setattr(r, "decode", failing)
    with pytest.raises(RuntimeError, match="step failed"):
        BeamSearch(r, 2).generate([[1, 2, 3]], 6)
    assert r.cache.free_blocks == 12 and r.cache.num_sequences() == 0


def test_engine_and_server_search_beside_running_requests():
    from rustral_b200.serve.http_server import BadRequest, EngineLoop, engine_generate_fn
    r = sharp(ModelRunner(preset("gpt2-test"), device="cpu", num_blocks=64, block_size=4, seed=2), 1)
    eng = ServingEngine(r, max_batch_size=4)
    alone = eng.generate([4, 5, 6, 7], 8)
    found = eng.beam_search([9, 8, 7], 6, beams=3)
    rid = eng.submit([4, 5, 6, 7], 8)
    eng.step(), eng.step()
    assert [h.tokens for h in eng.beam_search([9, 8, 7], 6, beams=3)] == [h.tokens for h in found]
    eng.run_to_completion()
    assert eng.scheduler.get(rid).generated == alone
    loop = EngineLoop(eng)
    fn = engine_generate_fn(eng, loop)
    out = fn({"prompt": [9, 8, 7], "max_tokens": 6, "beams": 3})
    assert out["tokens"] == found[0].tokens and [b["tokens"] for b in out["beams"]] == [h.tokens for h in found]
    assert fn({"prompt": [4, 5, 6, 7], "max_tokens": 8}) == {"tokens": alone}
    for bad in ({"beams": 0}, {"beams": 1000}, {"max_tokens": 0, "beams": 2}, {"max_tokens": 4000, "beams": 2}):
        with pytest.raises(BadRequest):
            fn({"prompt": [1, 2], **bad})
    loop.shutdown()
    assert engine_generate_fn(eng)({"prompt": [9, 8, 7], "max_tokens": 6, "beams": 3}) == out


def test_decode_with_groups_asks_for_their_lengths():
    r = ModelRunner(preset("gpt2-test"), device="cpu", num_blocks=16)
    r.cache.allocate(1, 4)
    r.prefill(1, [1, 2, 3])
    for groups, shared in ((ops.PrefixGroups([2]), [1]), (ops.PrefixGroups([1]), None), (ops.PrefixGroups([1]), [1, 2])):
        with pytest.raises(ValueError):
            r.decode([1], [4], [4], groups=groups, shared_lens=shared)


@pytest.mark.gpu
@pytest.mark.parametrize("name,kw", [("gpt2-test", {}), ("llama-test", dict(n_head=8, n_kv_head=2, d_model=512))])
def test_beam_search_on_a_gpu(name, kw, monkeypatch):
    """Graphed decoding that reads the prompt once for all beams: every continuation's score is the sum of its tokens' logarithmic probabilities as whole passes give them, with and without
    the shared reading.  bf16 activations: logits of a few units are off by 2^-8 of themselves here and there, so a token's by less than 0.05."""
    cfg = preset(name, **kw)
    r = sharp(ModelRunner(cfg, device="cuda", num_blocks=128, block_size=16, seed=3), 4)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (70, 33)]
    used = []
    real = beam_ops.paged_attention_shared
    monkeypatch.setattr(beam_ops, "paged_attention_shared", lambda *a, **k: used.append(1) or real(*a, **k))
    for pays in (0, 1 << 60):
        monkeypatch.setattr(beam_ops, "SHARED_PAYS", pays)
        for beams in (4, 12):
            found = BeamSearch(r, beams, eos_id=5).generate(prompts, 12)
            for p, f in zip(prompts, found):
                assert len(f) == beams
                scores_are_their_tokens(r, p, f[:3], 0.05)
        assert bool(used) == (pays == 0)
        used.clear()
    assert r.cache.free_blocks == 128


# ---- dense caches, encoder and decoder -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("quant", [CacheQuantization.FP32, CacheQuantization.BF16, CacheQuantization.INT8, CacheQuantization.FP8])
def test_dense_caches_take_the_order_of_beams(device, quant):
    cfg = CacheConfig(num_heads=3, head_dim=8, max_seq_len=12, batch_size=6, quantization=quant)
    index = torch.tensor([2, 0, 0, 5, 5, 1])
    g = torch.Generator().manual_seed(0)
    for cache in (KVCache(cfg, device), SlidingWindowCache(cfg, 5, device)):
        for n in (4, 3):
            cache.append(torch.randn(6, 3, n, 8, generator=g).to(device), torch.randn(6, 3, n, 8, generator=g).to(device))
        want = [t[index.to(device)].clone() for t in cache.get()]
        cache.reorder(index.to(device))
        assert all(torch.equal(a, b) for a, b in zip(cache.get(), want))
    both = BatchedCache(2, cfg, device)
    for l in range(2):
        both.append(l, torch.randn(6, 3, 4, 8, generator=g).to(device), torch.randn(6, 3, 4, 8, generator=g).to(device))
    want = [[t[index.to(device)].clone() for t in both.get(l)] for l in range(2)]
    both.reorder(index.to(device))
    assert all(torch.equal(a, b) for l in range(2) for a, b in zip(both.get(l), want[l]))


@pytest.mark.parametrize("device", DEVICES)
def test_encoder_decoder_generates_with_beams(device):
    from rustral_b200.core import ForwardCtx
    from rustral_b200.core.backend import B200Backend, CpuBackend
    from rustral_b200.nn.transformer import TransformerEncoderConfig, TransformerEncoderDecoder
    backend = CpuBackend() if device == "cpu" else B200Backend()
    cfg = TransformerEncoderConfig(64, 4, 2, 128) if device == "cpu" else TransformerEncoderConfig(128, 2, 2, 256)
    m = TransformerEncoderDecoder.new(backend, cfg, 20, 30)
    ctx = ForwardCtx.inference(backend)
    src = torch.tensor([[1, 2, 3, 4, 5]])
    memory = m.encoder.forward(src, ctx)

    def score(tokens):
        x = torch.log_softmax(m.decoder.forward(torch.tensor([tokens[:-1]]), ctx, memory)[0].double().cpu(), -1)
        return float(sum(x[i, t] for i, t in enumerate(tokens[1:]))) / (len(tokens) - 1)
    greedy = m.generate(src, ctx, bos=1, eos=2, max_len=5)
    out = m.generate(src, ctx, bos=1, eos=2, max_len=5, beams=8)
    assert out[0] == 1 and 2 <= len(out) <= 6 and (len(out) == 6 or out[-1] == 2)
    if device == "cpu":
        # eight beams of thirty tokens hold the greedy path unless eight better ones push it out; the best found is no worse than it
        assert score(out) >= score(greedy) - 1e-5
        # two tokens: as many beams as the vocabulary has see every continuation
        best = max(([1, a] if a == 2 else [1, a, b] for a in range(30) for b in range(30)), key=score)
        assert abs(score(m.generate(src, ctx, bos=1, eos=2, max_len=2, beams=30)) - score(best)) < 1e-5
