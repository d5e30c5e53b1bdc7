"""``token_logprobs`` against f64: types, vocabulary sizes around the vector and
iteration edges, row strides and alignments, ties, masks, NaN and infinities,
and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ie_tpq.scoring import token_logprobs

pytestmark = pytest.mark.gpu


def check(logits, tokens, top):
    x = logits.double().cpu().numpy()
    rows, vocab = x.shape
    got = token_logprobs(logits, tokens, top=top)
    t = tokens.cpu().numpy()
    for r in range(rows):
        m = x[r].max()
        p = np.exp(x[r] - m)
        s = p.sum()
        logp = x[r] - m - np.log(s)
        ent = np.log(s) - np.where(p > 0, p * np.where(p > 0, x[r] - m, 0), 0).sum() / s
        # f32: a difference of logits rounded once, weights 2^(x log2 e - c) with an
        # argument rounded once (|x - m| up to a few hundred matter: e^-x x < 1) and an
        # exponential of 2^-22, and sums of positive terms, in several hundred steps
        # of a thread at most
        tol = 2.0 ** -23 * (np.abs(x[r][np.isfinite(x[r])]).max() + 300) + 1e-6
        if 0 <= t[r] < vocab:
            want = logp[t[r]]
            if np.isinf(want):
                assert got.logprobs[r].item() == want
            else:
                assert abs(got.logprobs[r].item() - want) <= tol
        else:
            assert got.logprobs[r].item() == -np.inf
        assert abs(got.entropy[r].item() - ent) <= tol * (1 + ent)
        order = np.lexsort((np.arange(vocab), -x[r]))[:top]
        assert got.top_tokens[r].tolist() == order.tolist()
        best = got.top_logprobs[r].double().cpu().numpy()
        finite = np.isfinite(logp[order])
        assert np.all(np.abs(best[finite] - logp[order][finite]) <= tol)
        assert np.all(best[~finite] == -np.inf)
    return got


def make(rows, vocab, dtype, seed=0, std=2.5):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=gen, device="cuda") * std).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=gen, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (3, 1), (5, 7), (2, 64), (4, 8191),
                                        (3, 8192), (3, 8193), (2, 50257), (1, 16385),
                                        (300, 1000), (600, 33), (2, 262147)])
def test_sizes(dtype, rows, vocab):
    x, t = make(rows, vocab, dtype, seed=vocab)
    check(x, t, min(20, vocab))
    check(x, t, 0)


@pytest.mark.parametrize("top", [1, 2, 31, 32, 33, 63, 64])
def test_top(top):
    x, t = make(3, 20000, torch.bfloat16, seed=top)     # bf16: many equal logits
    check(x, t, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows", [2, 700])
def test_ties(dtype, rows):
    x = torch.full((rows, 9000), 1.25, dtype=dtype, device="cuda")
    t = torch.arange(rows, device="cuda")
    check(x, t, 64)
    x[:, 8999] = 2.0
    x[:, 17:19] = 2.0
    check(x, t, 5)
    x.zero_()
    x[:, ::3] = -0.0
    check(x, t, 9)


@pytest.mark.parametrize("order", ["up", "down", "blocks"])
@pytest.mark.parametrize("rows", [1, 600])
def test_orders(order, rows):
    """Sorted logits crowd the largest into neighbouring vectors."""
    v = torch.linspace(-20, 20, 60000, device="cuda")
    if order == "down":
        v = v.flip(0)
    if order == "blocks":
        v = v.view(-1, 3000).flip(0).reshape(-1)
    x = v.repeat(rows, 1)
    got = check(x[:2], torch.arange(min(rows, 2), device="cuda"), 64)
    every = token_logprobs(x, torch.zeros(rows, dtype=torch.long, device="cuda"), top=64)
    assert torch.equal(every.top_tokens[-1], got.top_tokens[0])


def test_crowded_candidates():
    """Thousands of elements above every other thread's best: the list is found rank
    by rank."""
    x = torch.zeros((2, 100000), device="cuda")
    lane = torch.arange(100000, device="cuda") // 4 % 512
    x[:, lane < 260] = torch.rand((2, int((lane < 260).sum())), device="cuda",
                                  generator=torch.Generator(device="cuda").manual_seed(1)) + 1
    check(x, torch.tensor([0, 99999], device="cuda"), 64)
    x[:, lane >= 252] = 0      # 63 groups of four lanes hold all that is not zero
    check(x, torch.tensor([0, 99999], device="cuda"), 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("allowed", [1, 3, 500])
def test_vocabulary_mask(dtype, allowed):
    x, t = make(4, 70001, dtype, seed=allowed)
    keep = torch.randperm(70001, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(2))[:allowed]
    masked = torch.full_like(x, -float("inf"))
    masked[:, keep] = x[:, keep]
    t[0] = keep[0]
    check(masked, t, 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lowest_values_and_large_logits(dtype):
    x, t = make(3, 5000, dtype, seed=3)
    x[:, ::2] = torch.finfo(dtype).min if dtype != torch.float32 else -1e30
    check(x, t, 8)
    x, t = make(3, 5000, torch.float32, seed=4)
    check(x + 5000.0, t, 8)


def check_masked(logits, tokens, top):
    """As ``check``, with a tolerance that knows nothing of masked logits: with
    d = x - max, only terms of |d| < 200 reach the sums (e^-200 is below every f32 sum's
    last bit); their arguments are rounded once (2^-24 |d| log2 e), their exponential is
    good to 2^-22 and they are summed in several hundred steps; a result beyond that
    range is a difference of logits, rounded twice."""
    x = logits.double().cpu().numpy()
    got = token_logprobs(logits, tokens, top=top)
    t = tokens.cpu().numpy()
    for r in range(x.shape[0]):
        d = x[r] - x[r].max()
        p = np.exp(d)
        s = p.sum()
        logp = d - np.log(s)
        near = d > -200
        ent = np.log(s) - (p[near] * d[near]).sum() / s
        tol = 2.0 ** -23 * (-d[near].min() + 300) + 1e-6
        bound = tol + 2.0 ** -22 * np.abs(logp)

        def held(value, at):
            if logp[at] <= -(2.0 ** 128 - 2.0 ** 103):      # rounds to -inf in f32
                return value == -np.inf
            return abs(value - logp[at]) <= bound[at]

        assert held(got.logprobs[r].item(), t[r])
        assert abs(got.entropy[r].item() - ent) <= tol * (1 + ent)
        order = np.lexsort((np.arange(x.shape[1]), -x[r]))[:top]
        assert got.top_tokens[r].tolist() == order.tolist()
        best = got.top_logprobs[r].double().cpu().numpy()
        assert all(held(b, at) for b, at in zip(best, order))


MASKS = [-1e9, -5e9, -1e10, -1e30, "lowest"]


def mask_of(value, dtype):
    low = torch.finfo(dtype).min
    return low if value == "lowest" else max(value, low)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", MASKS)
@pytest.mark.parametrize("rows,vocab", [(2, 128256), (3, 5000), (600, 3000)])
def test_finite_masks_over_whole_runs(dtype, value, rows, vocab):
    """A mask that leaves a few neighbouring tokens: most threads see masked logits alone."""
    x, t = make(rows, vocab, dtype, seed=vocab)
    masked = torch.full_like(x, mask_of(value, dtype))
    for r, n in zip(range(rows), (1, 700, 40) * rows):
        at = (r * 997) % (vocab - n)
        masked[r, at:at + n] = x[r, at:at + n]
        t[r] = at if r % 2 else t[r]
    check_masked(masked[:3], t[:3], 20)
    whole = token_logprobs(masked, t, top=20)
    for a, b in zip(whole, token_logprobs(masked[-3:], t[-3:], top=20)):
        torch.testing.assert_close(a[-3:], b, rtol=1e-6, atol=1e-4)
        assert not torch.isnan(a.float()).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", MASKS)
@pytest.mark.parametrize("rows,vocab", [(2, 128256), (3, 33), (600, 3000)])
def test_rows_that_a_finite_mask_covers_whole(dtype, value, rows, vocab):
    x = torch.full((rows, vocab), mask_of(value, dtype), dtype=dtype, device="cuda")
    t = torch.arange(rows, device="cuda") % vocab
    check_masked(x[:3], t[:3], 5)
    got = token_logprobs(x, t, top=5)
    torch.testing.assert_close(got.entropy, torch.full_like(got.entropy, np.log(vocab)),
                               rtol=0, atol=4e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("size", [2.0 ** 20 - 64, 2.0 ** 20, 2.0 ** 20 + 64, 3e9, 1e30, 3e38])
def test_maxima_of_any_size(dtype, scale, size):
    """Logits around a large value of either sign, spread over the type's last bits,
    beside masked ones."""
    step = max(abs(torch.finfo(dtype).eps * size), 0.25)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = scale * size + torch.randint(-8, 9, (3, 20000), generator=gen, device="cuda") * step
    x = x.to(dtype)
    t = torch.randint(0, 20000, (3,), generator=gen, device="cuda")
    check_masked(x, t, 8)
    x[:, 3000:19000] = torch.finfo(dtype).min
    check_masked(x, t, 8)
    x[:, :5] = 0.0
    check_masked(x, t, 8)


def test_not_finite():
    x, t = make(5, 3001, torch.float32, seed=5)
    clean = token_logprobs(x, t, top=4)
    x[1, 7] = float("nan")
    x[2] = -float("inf")
    x[3, 9] = float("inf")
    got = token_logprobs(x, t, top=4)
    for r in (1, 2, 3):
        assert torch.isnan(got.logprobs[r]) and torch.isnan(got.entropy[r])
    assert got.top_tokens[2].tolist() == [0, 1, 2, 3] and got.top_tokens[3, 0] == 9
    y = x[1].clone()
    y[7] = -float("inf")
    assert got.top_tokens[1].tolist() == torch.topk(y, 4).indices.tolist()
    for r in (0, 4):
        for a, b in zip(clean, got):
            assert torch.equal(a[r], b[r])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("part", [0, 5, 7])
def test_one_part_holds_the_allowed_tokens(dtype, part):
    """A split row whose other parts are all masked, and one whose parts all hold less
    than the wanted number."""
    x, t = make(2, 128000, dtype, seed=part)
    x[0, :part * 16000] = float("-inf")
    x[0, (part + 1) * 16000:] = float("-inf")
    x[1] = float("-inf")
    x[1, part::16000] = torch.arange(8, device="cuda").to(dtype)
    check(x, t, 20)
    check(x, t, 64)


def test_tokens_outside_the_vocabulary():
    x, _ = make(4, 100, torch.float32)
    check(x, torch.tensor([-1, 100, 2 ** 40, 99], device="cuda"), 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5])
def test_strides_and_alignments(dtype, shift):
    big, t = make(6, 1207, dtype, seed=shift)
    check(big[:, shift:shift + 1100], t % 1100, 6)
    check(big[::2, shift:shift + 1100], t[:3] % 1100, 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [2097152, 2097151, 2097150, 2097149])
def test_largest_vocabulary(dtype, vocab):
    x, t = make(2, vocab + 3, dtype, seed=8)
    for row in (x[:1, :vocab], x[1:, 3:]):      # aligned, and from an odd element on
        check(row, t[:1] % vocab, 64)
        check(row, t[:1] % vocab, 0)


def test_one_row_for_many_tokens():
    x, t = make(1, 3000, torch.float32, seed=9)
    check(x.expand(5, -1), torch.arange(5, device="cuda") * 500, 3)


def test_streams_and_empty():
    x, t = make(4, 30000, torch.float32, seed=6)
    a = token_logprobs(x, t, top=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b = token_logprobs(x, t, top=3, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    none = token_logprobs(x[:0], t[:0], top=3)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 3)


def test_refusals():
    x, t = make(4, 100, torch.float32)
    for args, kw in [((x[0], t), {}), ((x.double(), t), {}), ((x.T, t), {}), ((x, t[:3]), {}),
                     ((x, t.int()), {}), ((x, t), dict(top=65)), ((x, t), dict(top=-1)),
                     ((x[:, :5], t), dict(top=6)), ((x.cpu(), t), {}), ((x, t.cpu()), {}),
                     ((torch.zeros((1, 2097153), device="cuda"), t[:1]), {})]:
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)
