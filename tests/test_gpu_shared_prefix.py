"""``shared_prefix_attention`` against the f64 definition: decode and several
queries a sequence, prefixes around page and tile edges, sequences shorter than
the prefix, NaN where nothing may be read, and refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ie_tpq.kv_attention import shared_prefix_attention, window_attention
from tests.attention_oracle import Batch, assert_close

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(b, **kw):
    got = shared_prefix_attention(b.q, b.k, b.v, b.tables, b.ctx, b.prefix, b.block,
                                  **{**b.lens(), **kw})
    want, weight, largest = b.oracle(prefix=b.prefix)
    assert_close(got, want, weight, largest, b.q.shape[2])
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (64, 8, 128), (14, 2, 64), (4, 4, 128),
                                         (4, 2, 8), (5, 1, 80)])
def test_decode(dtype, heads, kv, hd):
    check(Batch([200, 161, 250, 330], heads, kv, hd, dtype, 16, prefix=160, seed=hd))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 127, 128, 129, 300, 1000, 2048])
def test_prefix_lengths(prefix):
    """Prefixes that end inside a page: the shared part is read through the first
    row, the rest of that page through each sequence's own."""
    check(Batch([prefix + n for n in (1, 9, 140)], 8, 2, 128, BF16, 16, prefix=prefix,
                seed=prefix))


@pytest.mark.parametrize("seqs", [1, 2, 31, 33, 70])
def test_batch_sizes(seqs):
    check(Batch([140 + i for i in range(seqs)], 8, 2, 64, F16, 16, prefix=130, seed=seqs))


# rows (sequences times kv heads) times prefix beyond what the decode kernel takes on alone
@pytest.mark.parametrize("seqs,heads,kv,hd,dtype,prefix", [
    (24, 32, 8, 128, BF16, 901), (24, 64, 8, 128, F16, 1100), (90, 14, 2, 64, F16, 1000),
    (90, 8, 2, 64, BF16, 928), (3, 8, 8, 128, BF16, 8191), (9, 34, 2, 64, F16, 5000)])
@pytest.mark.parametrize("own", [1, 40, 700])
def test_prefix_beyond_one_launch(seqs, heads, kv, hd, dtype, prefix, own):
    lens = [prefix + 1 + (i * 37) % own for i in range(seqs)]
    lens[1], lens[2] = prefix - 3, 0        # one shorter than the prefix, one empty
    b = Batch(lens, heads, kv, hd, dtype, 16, prefix=prefix, seed=own)
    got = check(b)
    assert torch.count_nonzero(got[2]) == 0
    assert torch.equal(check(b), got)


def test_prefix_beyond_one_launch_in_a_graph_and_beside_a_nan():
    b = Batch([1000 + i for i in range(24)], 32, 8, 128, BF16, 16, prefix=1000, seed=12)
    b.ctx[0] = 500
    call = lambda: shared_prefix_attention(b.q, b.k, b.v, b.tables, b.ctx, 1000, 16, **b.lens())
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    assert torch.equal(out, want)
    b.v[int(b.tables[0, 50]) * 16] = float("nan")      # position 800
    graph.replay()
    assert torch.equal(out[0], want[0])                 # its context ends before
    assert torch.isnan(out[1:]).all()


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
def test_several_queries(hd, dtype):
    query = [1, 7, 40, 0, 3]
    check(Batch([100 + n for n in query], 8, 2, hd, dtype, 16, query=query, prefix=96, seed=hd))


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
@pytest.mark.parametrize("lead,tail", [(0, 2), (0, 200), (5, 0), (140, 3)])
def test_tokens_of_no_sequence_are_zeros(hd, dtype, lead, tail):
    query = [7, 40, 3]
    b = Batch([1300, 1240, 1203], 8, 2, hd, dtype, 16, query=query, prefix=1200, seed=hd)
    want, weight, largest = b.oracle(prefix=1200)
    q = torch.randn((lead + 50 + tail, 8, hd), device="cuda").to(dtype)
    q[lead:lead + 50] = b.q
    out = torch.full_like(q, float("nan"))
    shared_prefix_attention(q, b.k, b.v, b.tables, b.ctx, 1200, 16, out=out,
                            cu_seqlens_q=b.cu + lead, max_query_len=40, max_context_len=1300)
    assert_close(out[lead:lead + 50], want, weight, largest, hd)
    assert torch.count_nonzero(out[:lead]) == 0 and torch.count_nonzero(out[lead + 50:]) == 0


def test_sequences_shorter_than_the_prefix():
    b = Batch([100, 20, 1, 0, 64], 8, 2, 64, BF16, 16, prefix=64, seed=3)
    got = check(b)
    assert torch.count_nonzero(got[3]) == 0
    check(Batch([100, 20, 60], 8, 2, 128, BF16, 16, query=[10, 20, 30], prefix=64, seed=4))


def test_the_first_row_names_the_prefix():
    b = Batch([90, 95, 70], 8, 2, 128, BF16, 16, prefix=64, seed=5)
    want = check(b)
    b.tables[1:, :4] = -1        # not read
    assert torch.equal(check(b), want)


def test_equal_to_attention_over_whole_tables():
    b = Batch([700, 650, 640], 8, 2, 128, BF16, 16, prefix=640, seed=6)
    check(b)
    got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, **b.lens())
    want, weight, largest = b.oracle(prefix=640)
    assert_close(got, want, weight, largest, 128)


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
def test_values_that_a_sequence_does_not_see(hd, dtype):
    """A value that is NaN poisons the sequences whose context reaches it alone."""
    b = Batch([60, 30, 64], 8, 2, hd, dtype, 16, prefix=48, seed=7)
    want, weight, largest = b.oracle(prefix=48)
    slot = int(b.tables[0, 2]) * 16 + 8                    # position 40
    b.v[slot] = float("nan")
    got = shared_prefix_attention(b.q, b.k, b.v, b.tables, b.ctx, 48, 16, **b.lens())
    assert_close(got[1:2], want[1:2], weight[1:2], largest, hd)
    assert torch.isnan(got[0]).all() and torch.isnan(got[2]).all()


@pytest.mark.parametrize("lens", [dict(max_query_len=0, max_context_len=0),
                                  dict(max_query_len=1, max_context_len=1),
                                  dict(max_query_len=999, max_context_len=99999)])
@pytest.mark.parametrize("query", [None, [3, 40]])
def test_lengths_unknown_or_wrong_give_the_same(lens, query):
    check(Batch([500, 800], 8, 2, 128, F16, 16, query=query, prefix=400, seed=8), **lens)


def test_large_scores_and_same_bits():
    b = Batch([1500, 1600, 1501], 32, 8, 128, F16, 16, prefix=1400, seed=9, std=20.0)
    assert torch.equal(check(b), check(b))


def test_graph_capture():
    b = Batch([300, 290], 8, 2, 128, BF16, 16, prefix=256, seed=10)
    call = lambda: shared_prefix_attention(b.q, b.k, b.v, b.tables, b.ctx, 256, 16, **b.lens())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    b.q.copy_(b.q.flip(0))
    graph.replay()
    want, weight, largest = b.oracle(prefix=256)
    assert_close(out, want, weight, largest, 128)


def test_refusals():
    b = Batch([50, 60], 4, 2, 64, BF16, 16, prefix=32, seed=11)
    args = (b.q, b.k, b.v, b.tables, b.ctx)
    for prefix in (-1, 65, 2 ** 40):
        with pytest.raises(ValueError):
            shared_prefix_attention(*args, prefix, 16)
    with pytest.raises(ValueError):
        shared_prefix_attention(*args, 32, 0)
    with pytest.raises(ValueError):
        shared_prefix_attention(b.q[:1], *args[1:], 32, 16)
    assert np.isfinite(b.q.float().cpu().numpy()).all()


@pytest.mark.parametrize("block", [1, 5, 20, 48, 256])
@pytest.mark.parametrize("heads,kv,hd,dtype", [(16, 8, 128, BF16), (8, 4, 64, F16)])
@pytest.mark.parametrize("query", [None, [3, 1, 40, 0, 17]])
def test_pages_of_any_size(block, heads, kv, hd, dtype, query):
    """A prefix long enough for the row tiles, in pages that are gathered or taken in boxes."""
    if query is None:
        b = Batch([1301 + 3 * i for i in range(40)], heads, kv, hd, dtype, block, prefix=1300,
                  seed=block)
        b.context[1], b.ctx[1] = 700, 700
    else:
        b = Batch([1300 + n for n in (9, 1, 40, 0, 90)], heads, kv, hd, dtype, block, query=query,
                  prefix=1300, seed=block)
    assert torch.equal(check(b), check(b))
