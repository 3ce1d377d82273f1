"""Beam search over a serving runner: the beams of a prompt are sequences of the paged cache that share the prompt's pages.

A step is one decode pass over the beams of all prompts, which reads what a prompt's beams share once (`ModelRunner.decode` with groups), one selection over beams and vocabulary on the device
(`ops.beam_select`), and, for beams with several children, a fork of the parent's sequence (`PagedCache.fork`): full pages are shared, the page that is still filling is copied for all
layers of all new beams by one launch.  What a beam without children has is freed.

The reference decodes greedily, one sequence at a time (crates/nn/src/transformer.rs:837-862).
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

from .. import ops
from .model_runner import ModelRunner

MOST_PENALTY = 600.0                                              # length ** length_penalty is a power of e between -600 and 600: a 64-bit number, like a sum over it


@dataclass
class Hypothesis:
    """A continuation: its tokens (the end-of-sequence token among them), the sum of their logarithmic probabilities and that sum by the length penalty."""
    tokens: list
    score: float
    ranked: float
    ended: bool


@dataclass
class _Group:
    """The search over one prompt: its beams (sequence, tokens so far, score) and its finished continuations, best first."""
    prompt: list
    beams: list = field(default_factory=list)
    done: list = field(default_factory=list)
    over: bool = False


class BeamSearch:
    """`beams` continuations of every prompt are kept; a continuation that ends with `eos_id` among a step's best `beams` is finished.  Finished ones are ranked by
    score / length ** length_penalty; a prompt's search is over when `beams` of them rank above what its best beam has now, or at `max_tokens`.

    The runner's cache holds the beams while `generate` runs, beside the sequences of others (sequence ids from `first_seq` on are this search's).  With a
    tensor-parallel runner all ranks search alike."""

    def __init__(self, runner: ModelRunner, beams: int = 4, eos_id: int | None = None, length_penalty: float = 1.0, first_seq: int = 1 << 40):
        if not 1 <= beams <= ops.beams.MOST_COUNT // 2:
            raise ValueError(f"BeamSearch: 1 to {ops.beams.MOST_COUNT // 2} beams")
        if not math.isfinite(length_penalty):
            raise ValueError(f"BeamSearch: a length penalty of {length_penalty}")
        self.runner, self.beams, self.eos_id, self.length_penalty = runner, beams, eos_id, float(length_penalty)
        self.vocab = runner.cfg.vocab_size
        self._next = first_seq

    def _new_ids(self, n: int) -> list:
        ids = list(range(self._next, self._next + n))
        self._next += n
        return ids

    def blocks_needed(self, prompt_lens: list, max_tokens: int) -> int:
        """Blocks of the cache that a search over these prompts can take at most: a prompt's full blocks once and the others for every beam (where attention weights are summed: all)."""
        c = self.runner.cache
        if self.runner.kv_weights:
            return sum(self.beams * c.blocks_needed(n + max_tokens) for n in prompt_lens)
        return sum(n // c.block_size + self.beams * (c.blocks_needed(n + max_tokens) - n // c.block_size) for n in prompt_lens)

    @torch.no_grad()
    def generate(self, prompts: list, max_tokens: int) -> list:
        """For every prompt (a list of token ids) its best `beams` continuations of up to `max_tokens` tokens, best first (fewer where no more are possible)."""
        cache, cfg = self.runner.cache, self.runner.cfg
        if max_tokens < 1 or not all(len(p) for p in prompts):
            raise ValueError("BeamSearch: prompts of a token at least and max_tokens of at least 1")
        if abs(self.length_penalty) * math.log(max_tokens) > MOST_PENALTY:
            raise ValueError(f"BeamSearch: a length penalty of {self.length_penalty} for up to {max_tokens} tokens")
        for p in prompts:
            if len(p) + max_tokens > cfg.seq_len:
                raise ValueError(f"prompt + max_tokens exceeds the model's context of {cfg.seq_len}")
        if not prompts:
            return []
        need = self.blocks_needed([len(p) for p in prompts], max_tokens)
        if need > cache.free_blocks:
            raise ValueError(f"the search can take {need} KV blocks of {cache.block_size} tokens, {cache.free_blocks} are free")
        if cache.num_slots and len(prompts) * self.beams > cache.free_slots:
            raise ValueError(f"the search takes {len(prompts) * self.beams} state slots, {cache.free_slots} are free")
        groups = [_Group(list(p)) for p in prompts]
        self._held: set = set()
        try:
            self._first_step(groups)
            plan = ops.PrefixGroups([self.beams] * len(groups), self.runner.device)
            shared = [len(g.prompt) for g in groups]
            for made in range(1, max_tokens):
                if all(g.over for g in groups):
                    break
                self._step(groups, plan, shared, made)
            for g in groups:
                if not g.over:
                    for _, tokens, score in g.beams:
                        if score > float("-inf"):
                            self._finish(g, tokens, score, False)
        finally:
            for s in self._held:
                cache.free(s)
        return [g.done[:self.beams] for g in groups]

    def _finish(self, g: _Group, tokens: list, score: float, ended: bool) -> None:
        g.done.append(Hypothesis(tokens, score, score / len(tokens) ** self.length_penalty, ended))
        g.done.sort(key=lambda h: -h.ranked)

    def _first_step(self, groups: list) -> None:
        """Prompts into the cache, and their best first tokens."""
        cache, ids = self.runner.cache, self._new_ids(len(groups))
        for s, g in zip(ids, groups):
            if not cache.allocate(s, len(g.prompt)):
                raise RuntimeError("BeamSearch: out of KV blocks")
            self._held.add(s)
        logits, _ = self.runner.step_mixed([(s, g.prompt, 0, True) for s, g in zip(ids, groups)], [], [], [])
        for s, g in zip(ids, groups):
            g.beams = [(s, [], 0.0)]
        self._select(groups, torch.stack(logits), 1)

    def _step(self, groups: list, plan, shared: list, made: int) -> None:
        """One token more for every beam.  The beams of a search that is over stay as they are, so that the batch keeps its shape: their last token is computed again."""
        cache = self.runner.cache
        ids, last, lens = [], [], []
        for g in groups:
            for s, tokens, _ in g.beams:
                n = len(g.prompt) + len(tokens)
                if not cache.allocate(s, n):
                    raise RuntimeError("BeamSearch: out of KV blocks")
                ids.append(s)
                last.append(tokens[-1])
                lens.append(n)
        self._select(groups, self.runner.decode(ids, last, lens, groups=plan, shared_lens=shared), made + 1)

    def _select(self, groups: list, logits: torch.Tensor, length: int) -> None:
        """The next beams of every group from the logits of the present ones."""
        cache, K, per = self.runner.cache, self.beams, len(groups[0].beams)
        scores = torch.tensor([[b[2] for b in g.beams] for g in groups], dtype=torch.float32).to(logits.device)
        count = min(2 * K, per * self.vocab)
        best, rows, tokens = ops.beam_select(logits[:, :self.vocab], scores, count)
        best, (rows, tokens) = best.tolist(), torch.stack([rows, tokens]).tolist()
        forks, keeping, dropped = [], [], []
        for i, g in enumerate(groups):
            if g.over:
                continue
            chosen = []                                           # (parent, token, score) of the next beams
            for j in range(count):
                if best[i][j] == float("-inf") or len(chosen) == K:
                    break
                parent, token = rows[i][j] - i * per, tokens[i][j]
                if self.eos_id is not None and token == self.eos_id:
                    if j < K:
                        self._finish(g, g.beams[parent][1] + [token], best[i][j], True)
                else:
                    chosen.append((parent, token, best[i][j]))
            self._settle(g, chosen, length)
            chosen += [(chosen[0][0] if chosen else 0, 0, float("-inf"))] * (K - len(chosen))          # beams that are not there
            kept = {p for p, _, _ in chosen}
            dropped += [s for p, (s, _, _) in enumerate(g.beams) if p not in kept]
            heirs, beams = set(), []
            for parent, token, score in chosen:
                s, before, _ = g.beams[parent]
                if parent in heirs:                               # the first child takes the parent's place
                    forks.append((s, len(g.prompt) + len(before), len(beams), g))
                    s = None
                heirs.add(parent)
                beams.append((s, before + [token], score))
            g.beams = beams
        for s in dropped:                                         # their blocks are free for the copies
            cache.free(s)
            self._held.discard(s)
        if forks:
            new = self._new_ids(len(forks))
            if not cache.fork([f[0] for f in forks], new, [f[1] for f in forks]):
                raise RuntimeError("BeamSearch: out of KV blocks")
            self._held.update(new)
            for s, (_, _, at, g) in zip(new, forks):
                g.beams[at] = (s, *g.beams[at][1:])

    def _settle(self, g: _Group, chosen: list, length: int) -> None:
        """Whether the search over a prompt is over: no beam is left, or `beams` finished continuations rank above the best beam."""
        if not chosen:
            g.over = True
        elif len(g.done) >= self.beams:
            g.over = max(c[2] for c in chosen) / length ** self.length_penalty <= g.done[self.beams - 1].ranked
