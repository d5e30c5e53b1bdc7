"""Several continuations of one prompt, ranked by their log probability.

``best_of`` prefills the prompt once, forks its cache pages (``KVPagePool.fork``:
whole pages are shared, the partly filled one is copied), decodes all
continuations as one batch whose attention reads the shared pages once
(``shared_prefix_attention``; ``window_attention`` in windowed layers), and keeps
each token's log probability, entropy and best alternatives (``token_logprobs``).
Pages that every layer's window has passed are given back as it goes, a finished
continuation's pages at once, and the pool is compacted at the end of the batch's
life or when it has become sparse.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from .decode import Layout
from .kv_pages import KVPagePool
from .scoring import token_logprobs


@dataclass
class Continuation:
    tokens: list[int] = field(default_factory=list)
    logprobs: list[float] = field(default_factory=list)       # of the tokens
    entropies: list[float] = field(default_factory=list)      # of their distributions, nats
    top: list[list[tuple[int, float]]] = field(default_factory=list)   # (token, logprob), best first
    finished: bool = False                                     # ended with the stop token

    @property
    def mean_logprob(self) -> float:
        return float(np.mean(self.logprobs)) if self.logprobs else 0.0


def _sample(model, logits, temperature: float, generator):
    """One token per row: the first maximum, or the exponential race over
    softmax(logits / T).  Drawn tokens are rank 0's on every rank."""
    if temperature <= 0.0:
        return logits.argmax(dim=-1)
    probs = torch.softmax(logits / temperature, dim=-1)
    race = torch.empty_like(probs).exponential_(1.0, generator=generator).clamp_min(1e-10)
    return model.of_rank0((probs / race).argmax(dim=-1))


def best_of(model, prompt: list[int], n: int, max_new_tokens: int, *, block_size: int = 16,
            temperature: float = 1.0, top: int = 0, stop_token: int | None = None,
            seed: int = 0) -> list[Continuation]:
    """``n`` continuations of ``prompt`` of at most ``max_new_tokens`` tokens, the
    highest mean log probability first.  ``top`` alternatives are kept per token.
    The log probabilities are those of the model (temperature 1)."""
    if n < 1 or max_new_tokens < 1 or not prompt:
        raise ValueError("best_of needs a prompt, at least one continuation and one new token")
    per = -(-(len(prompt) + max_new_tokens) // block_size)
    whole = len(prompt) // block_size
    num_blocks = per + n * (per - whole) + 1
    k_caches, v_caches = model.allocate_caches(num_blocks, block_size)
    pool = KVPagePool(k_caches, v_caches, block_size)
    gen = torch.Generator(device=model.device)
    gen.manual_seed(seed)

    parent = pool.new(len(prompt))
    layout = Layout(list(prompt), list(range(len(prompt))),
                    [pool.slot(parent, i) for i in range(len(prompt))], [len(prompt)],
                    [len(prompt)], [pool.pages(parent)], True, shared_prefix_len=0)
    hidden = model.forward(layout, k_caches, v_caches, block_size)
    logits = model.logits_on_device(hidden, layout.query_lens).expand(n, -1)

    seqs = pool.fork(parent, n)
    pool.free(parent)
    shared = whole * block_size
    window = max(model.windows) if all(model.windows) else 0
    out = [Continuation() for _ in range(n)]
    live = list(range(n))            # continuation of each row of the batch
    for step in range(max_new_tokens):
        tokens = _sample(model, logits, temperature, gen)
        scores = token_logprobs(logits, tokens, top=top)
        ids = tokens.tolist()
        lp, ent = scores.logprobs.tolist(), scores.entropy.tolist()
        best = list(zip(scores.top_tokens.tolist(), scores.top_logprobs.tolist()))
        for row, i in enumerate(live):
            c = out[i]
            c.tokens.append(ids[row])
            c.logprobs.append(lp[row])
            c.entropies.append(ent[row])
            c.top.append(list(zip(*best[row])))
            c.finished = ids[row] == stop_token
        done = [i for i in live if out[i].finished]
        if done:
            pool.free([seqs[i] for i in done])
            live = [i for i in live if not out[i].finished]
            if live and pool.free_pages > pool.num_pages // 2:
                pool.compact()
        if not live or step + 1 == max_new_tokens:
            break
        ids, pos, slots = [], [], []
        for i in live:
            if window:       # the next token's window starts here
                pool.trim(seqs[i], window, model.sinks)
            pool.append(seqs[i])
            p = pool.length(seqs[i]) - 1
            ids.append(out[i].tokens[-1])
            pos.append(p)
            slots.append(pool.slot(seqs[i], p))
        rows = [pool.pages(seqs[i]) for i in live]
        layout = Layout(ids, pos, slots, [p + 1 for p in pos], [1] * len(live), rows, False,
                        shared_prefix_len=shared)
        hidden = model.forward(layout, k_caches, v_caches, block_size)
        logits = model.logits_on_device(hidden, layout.query_lens)
    if live:
        pool.free([seqs[i] for i in live])
    return sorted(out, key=lambda c: -c.mean_logprob)
