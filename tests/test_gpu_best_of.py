"""``best_of``: one prompt's continuations over forked cache pages, through the
shared-prefix and windowed attention kernels and the token log probabilities.

* f32: at temperature 0 every continuation is the plain greedy generation, and the
  log probabilities are those of the plain model's logits along it.
* f16: the same model with the attention computed in f64 from its definition (only
  the rounding of the softmax weights to f16 and of the output differ, a few parts in
  1e3 of an attention output) gives log probabilities within the f16 block
  tolerance of this suite, 2e-2 -- whole context, windows in some layers, windows
  in all of them (whose passed pages are given back).
* Sampling, stop tokens and the order of the result."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import pytest
import torch

import ie_tpq.model
from ie_tpq.best_of import best_of
from ie_tpq.decode import Layout, greedy_generate
from ie_tpq.model import QuantizedTransformer
from oracle import model_oracle as mo
from tests.attention_oracle import attention

pytestmark = pytest.mark.gpu


@dataclass
class Config(mo.Config):
    windows: tuple[int, ...] | None = None
    sinks: int = 0


def source(windows=None, sinks=0, layers=2, head_dim=64):
    cfg = Config(vocab_size=300, hidden_size=256, num_layers=layers, num_heads=4, num_kv_heads=2,
                 head_dim=head_dim, intermediate_size=256, windows=windows, sinks=sinks)
    model = mo.Model(cfg, seed=7)
    model.config = cfg
    return model


PROMPT = [int(t) for t in np.random.default_rng(3).integers(0, 300, 43)]


def logits_along(model, tokens):
    """The plain model's logits after every token (one prefill on contiguous pages)."""
    n = len(tokens)
    blocks = -(-n // 16)
    k, v = model.allocate_caches(blocks, 16)
    layout = Layout(list(tokens), list(range(n)), list(range(n)), [n], [n], [list(range(blocks))],
                    True)
    hidden = model.forward(layout, k, v, 16)
    return torch.log_softmax(model.logits_on_device(hidden, [1] * n).double(), -1).cpu().numpy()


def test_greedy_f32_is_the_plain_generation():
    model = QuantizedTransformer(source(), scheme="int8", dtype=torch.float32)
    want = greedy_generate(model, [PROMPT], 12)[0]
    got = best_of(model, PROMPT, 3, 12, temperature=0.0, top=4)
    logp = logits_along(model, PROMPT + want)[len(PROMPT) - 1:-1]
    for c in got:
        assert c.tokens == want and not c.finished
        np.testing.assert_allclose(c.logprobs, logp[np.arange(12), want], atol=1e-4)
        ent = -(np.exp(logp) * logp).sum(-1)
        np.testing.assert_allclose(c.entropies, ent, atol=1e-4)
        for row, best in zip(logp, c.top):
            assert best[0][0] == int(row.argmax()) and len(best) == 4
            np.testing.assert_allclose([lp for _, lp in best], np.sort(row)[::-1][:4], atol=1e-4)


def plain(q, k, v, tables, ctx, block, *, window=0, sinks=0, prefix=0, cu_seqlens_q=None,
          scale=None, **_):
    query = None if cu_seqlens_q is None else cu_seqlens_q.diff().tolist()
    out, _, _ = attention(q, k, v, tables, ctx.tolist(), block, query=query, window=window,
                          sinks=sinks, prefix=prefix, scale=scale)
    return torch.from_numpy(out).to(q)


@pytest.mark.parametrize("windows,sinks", [(None, 0), ((0, 24), 2), ((20, 33), 5)])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_f16_matches_attention_in_64_bits(monkeypatch, windows, sinks, temperature):
    model = QuantizedTransformer(source(windows, sinks), scheme="int8", dtype=torch.float16)
    got = best_of(model, PROMPT, 3, 10, temperature=temperature, top=2, seed=1)
    calls = {"window": 0, "prefix": 0}

    def window_plain(*a, **kw):
        calls["window"] += 1
        return plain(*a, **kw)

    def prefix_plain(q, k, v, tables, ctx, prefix, block, **kw):
        calls["prefix"] += 1
        assert prefix == 32
        return plain(q, k, v, tables, ctx, block, prefix=prefix, **kw)

    monkeypatch.setattr(ie_tpq.model, "window_attention", window_plain)
    monkeypatch.setattr(ie_tpq.model, "shared_prefix_attention", prefix_plain)
    want = best_of(model, PROMPT, 3, 10, temperature=temperature, top=2, seed=1)
    full = sum(w == 0 for w in windows) if windows else 2
    assert calls["prefix"] == 9 * full and calls["window"] == 10 * (2 - full) + full
    # a token drawn on the edge may differ; up to it the distributions agree
    for a in got:
        b = max(want, key=lambda c: sum(x == y for x, y in zip(a.tokens, c.tokens)))
        same = next((i for i, (x, y) in enumerate(zip(a.tokens, b.tokens)) if x != y), 10)
        assert same > 0
        np.testing.assert_allclose(a.logprobs[:same], b.logprobs[:same], atol=2e-2)
        np.testing.assert_allclose(a.entropies[:same], b.entropies[:same], atol=2e-2)


def test_windowed_layers_forget_what_the_window_has_passed():
    """With every layer windowed, tokens that no layer can reach any more do not
    change the continuation: what a layer sees reaches back one window a layer."""
    model = QuantizedTransformer(source((6, 5), 0), scheme="int8", dtype=torch.float32)
    other = [(t + 1) % 300 for t in PROMPT[:20]] + PROMPT[20:]
    a = best_of(model, PROMPT, 2, 8, temperature=0.0)
    b = best_of(model, other, 2, 8, temperature=0.0)
    assert [c.tokens for c in a] == [c.tokens for c in b]
    np.testing.assert_allclose(a[0].logprobs, b[0].logprobs, atol=1e-4)


def test_sampling_is_seeded_and_ranked():
    model = QuantizedTransformer(source(), scheme="int8", dtype=torch.float16)
    a = best_of(model, PROMPT, 6, 10, temperature=1.5, seed=5)
    b = best_of(model, PROMPT, 6, 10, temperature=1.5, seed=5)
    assert [c.tokens for c in a] == [c.tokens for c in b]
    assert len({tuple(c.tokens) for c in a}) > 1
    means = [c.mean_logprob for c in a]
    assert means == sorted(means, reverse=True)


def test_stop_token_ends_a_continuation_and_frees_its_pages():
    model = QuantizedTransformer(source(), scheme="int8", dtype=torch.float32)
    free = best_of(model, PROMPT, 8, 40, temperature=2.0, seed=2)
    stop = free[0].tokens[5]
    got = best_of(model, PROMPT, 8, 40, temperature=2.0, seed=2, stop_token=stop)
    assert any(c.finished for c in got)
    for c in got:
        assert c.finished == (c.tokens[-1] == stop) and stop not in c.tokens[:-1]
        assert len(c.tokens) == len(c.logprobs) == len(c.entropies) == len(c.top)
        assert c.finished or len(c.tokens) == 40
        logp = logits_along(model, PROMPT + c.tokens)[len(PROMPT) - 1:-1]
        np.testing.assert_allclose(c.logprobs, logp[np.arange(len(c.tokens)), c.tokens], atol=1e-4)


@pytest.mark.parametrize("prompt", [PROMPT[:1], PROMPT[:16], PROMPT[:32], PROMPT[:33]])
def test_prompts_around_the_page_size(prompt):
    model = QuantizedTransformer(source(), scheme="int8", dtype=torch.float32)
    want = greedy_generate(model, [prompt], 5)[0]
    for c in best_of(model, prompt, 2, 5, temperature=0.0):
        assert c.tokens == want


def test_refusals():
    model = QuantizedTransformer(source(layers=1), scheme="int8", dtype=torch.float32)
    for args in (([], 1, 1), (PROMPT, 0, 1), (PROMPT, 1, 0)):
        with pytest.raises(ValueError):
            best_of(model, *args)
    with pytest.raises(ValueError):
        best_of(model, PROMPT, 1, 1, top=301)
    with pytest.raises(ValueError):
        QuantizedTransformer(source((4,), 0), scheme="int8", dtype=torch.float32)
    windowed = QuantizedTransformer(source((4, 4), 0), scheme="int8", dtype=torch.float32)
    k, v = windowed.allocate_caches(1, 16)
    with pytest.raises(ValueError):       # a plan made without the window would ignore it
        windowed.run(torch.zeros(1, dtype=torch.long, device="cuda"),
                     torch.zeros(1, dtype=torch.long, device="cuda"), None, {"flash": False},
                     None, k, v, 16)


@pytest.mark.parametrize("windows", [(6, 5), (0, 7)])
def test_a_windowed_model_runs_a_captured_decode_step(windows):
    """``run`` with a plan of device tensors that a caller made, captured in a graph:
    the steps of ``forward``, whole and windowed layers alike."""
    model = QuantizedTransformer(source(windows, 2), scheme="int8", dtype=torch.float16)
    block, n = 256, len(PROMPT)
    long = dict(device="cuda", dtype=torch.long)
    i32 = dict(device="cuda", dtype=torch.int32)

    def prefilled():
        k, v = model.allocate_caches(2, block)
        layout = Layout(PROMPT + PROMPT, list(range(n)) * 2,
                        [*range(n), *range(block, block + n)], [n, n], [n, n], [[0], [1]], True)
        model.forward(layout, k, v, block)
        return k, v

    def layout_at(p):
        return Layout([1, 2], [p, p], [p, block + p], [p + 1, p + 1], [1, 1], [[0], [1]], False)

    k, v = prefilled()
    want = [model.forward(layout_at(p), k, v, block).clone() for p in range(n, n + 4)]
    k, v = prefilled()
    tokens, positions = torch.tensor([1, 2], **long), torch.tensor([n, n], **long)
    slots, lens = torch.tensor([n, block + n], **long), torch.tensor([n + 1, n + 1], **i32)
    tables = torch.tensor([[0], [1]], **long)
    plan = {"flash": True, "scale": 64 ** -0.5, "slots": slots, "context_lens": lens, "cu_q": None,
            "cu_k": None, "paged_tables": None, "tables32": tables.to(torch.int32)}
    step = lambda: model.run(tokens, positions, tables, plan, layout_at(n), k, v, block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        graph.replay()
        torch.testing.assert_close(out, want[i], rtol=2e-2, atol=2e-2)
        for t in (positions, slots, lens):
            t += 1
    with pytest.raises(ValueError):
        model.run(tokens, positions, tables, {**plan, "context_lens": None}, layout_at(n), k, v,
                  block)
