"""``window_attention`` against the f64 definition (tests/attention_oracle.py):
decode and ragged prefill, every type, head layouts and sizes, windows and
sinks around their edges, pages that end inside a tile, rows that see nothing,
NaN where nothing may be read, strides, streams and refusals."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from ie_tpq import _lib
from ie_tpq.kv_attention import window_attention
from tests.attention_oracle import Batch, as_f64, assert_close, attention

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(b, window=0, sinks=0, **kw):
    got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, b.block, window=window, sinks=sinks,
                           **b.lens(), **kw)
    want, weight, largest = b.oracle(window=window, sinks=sinks)
    assert_close(got, want, weight, largest, b.q.shape[2])
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (14, 2, 64), (8, 8, 128), (4, 2, 8),
                                         (20, 1, 64), (5, 1, 80), (3, 3, 256)])
def test_decode(dtype, heads, kv, hd):
    b = Batch([300, 1, 0, 77, 128, 129], heads, kv, hd, dtype, 16, seed=hd)
    check(b)
    check(b, window=50, sinks=3)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (14, 2, 64), (2, 2, 128), (4, 2, 8),
                                         (20, 1, 64), (5, 1, 80)])
def test_prefill(dtype, heads, kv, hd):
    b = Batch([70, 1, 0, 133, 40], heads, kv, hd, dtype, 16, query=[70, 1, 0, 5, 33], seed=hd)
    check(b)
    check(b, window=31, sinks=2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 200), (16, 0), (100, 4), (128, 128),
                                          (129, 17), (200, 1), (201, 5), (100000, 7),
                                          (1 << 40, 1 << 40)])
@pytest.mark.parametrize("query", [None, [1, 200, 30]])
def test_window_edges(window, sinks, query):
    b = Batch([64, 200, 199], 8, 2, 128, BF16, 16, query=query, seed=window % 97)
    check(b, window=window, sinks=sinks)


@pytest.mark.parametrize("block", [1, 5, 16, 48, 128, 256])
@pytest.mark.parametrize("query", [None, [100, 3, 260]])
def test_pages(block, query):
    b = Batch([100, 1000, 300], 4, 2, 64, F16, block, query=query, seed=block)
    check(b)
    check(b, window=90, sinks=4)


@pytest.mark.parametrize("context", [1, 127, 128, 129, 511, 2049])
def test_decode_splits(context):
    """One sequence: its keys are split over the SMs and joined."""
    b = Batch([context], 8, 2, 128, BF16, 16, seed=context)
    check(b)
    check(b, window=max(1, context // 2), sinks=4)


def test_chunked_prefill_equals_whole_prefill_rows():
    """The last queries of a prompt attend alike as a chunk and within the whole."""
    whole = Batch([300], 8, 2, 128, BF16, 16, query=[300], seed=5)
    got = check(whole, window=100, sinks=4)
    part = window_attention(whole.q[260:], whole.k, whole.v, whole.tables, whole.ctx, 16,
                            window=100, sinks=4, max_query_len=40, max_context_len=300,
                            cu_seqlens_q=torch.tensor([0, 40], dtype=torch.int32, device="cuda"))
    want, weight, largest = whole.oracle(window=100, sinks=4)
    assert_close(part, want[260:], weight[260:], largest, 128)
    assert got.shape == whole.q.shape


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("query", [None, [2, 4]])
def test_lengths_unknown_or_wrong_give_the_same(dtype, hd, query):
    b = Batch([500, 300], 8, 2, hd, dtype, 16, query=query, seed=2)
    want, weight, largest = b.oracle()
    for lens in (dict(), dict(max_query_len=1, max_context_len=1),
                 dict(max_query_len=10000, max_context_len=100000)):
        got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, cu_seqlens_q=b.cu, **lens)
        assert_close(got, want, weight, largest, hd)


@pytest.mark.parametrize("query", [None, [7, 9]])
def test_query_longer_than_its_context_sees_nothing_before_it(query):
    b = Batch([40, 3], 8, 2, 64, BF16, 16, query=query, seed=3)
    got = check(b)
    if query:
        assert torch.count_nonzero(got[7:13]) == 0 and torch.count_nonzero(got[13:]) > 0


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
@pytest.mark.parametrize("query", [None, [60]])
def test_entries_outside_the_cache_hide_their_keys(hd, dtype, query):
    b = Batch([200], 8, 2, hd, dtype, 16, query=query, seed=4)
    b.tables[0, 3] = -1
    b.tables[0, 5] = b.k.shape[0] // 16
    b.tables[0, 9] = 2 ** 31 - 1
    check(b)
    b.tables[0, :] = -1
    assert torch.count_nonzero(check(b)) == 0


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_behind_the_mask_do_not_matter(hd, dtype, bad):
    """A broken key or value poisons only the queries that see it."""
    b = Batch([180], 8, 2, hd, dtype, 16, query=[180], seed=6)
    want, weight, largest = b.oracle(window=40, sinks=2)
    at = 100
    slot = int(b.tables[0, at // 16]) * 16 + at % 16
    b.v[slot] = bad
    b.k[slot, 0] = float("nan")
    got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, window=40, sinks=2, **b.lens())
    blind = np.r_[0:at, at + 40:180]
    assert_close(got[blind], want[blind], weight[blind], largest, hd)
    assert not torch.isfinite(got[at:at + 40]).any()


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16)])
@pytest.mark.parametrize("window", [0, 1900])
def test_values_behind_the_mask_of_split_rows_do_not_matter(hd, dtype, window):
    """Rows in parts: what is computed again replaces the part's first result."""
    b = Batch([2000], 4, 1, hd, dtype, 16, query=[300], seed=30)
    out = torch.empty_like(b.q)
    assert _lib.lib().ie_attention_workspace_size(ctypes.byref(c_args(b, out, window=window))) > 0
    want, weight, largest = b.oracle(window=window, sinks=2)
    for at in (1750, 1999):
        b.v[int(b.tables[0, at // 16]) * 16 + at % 16] = float("nan")
    for _ in range(20):
        got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, window=window, sinks=2,
                               **b.lens())
        assert_close(got[:50], want[:50], weight[:50], largest, hd)
        assert torch.isnan(got[50:]).all()


@pytest.mark.parametrize("context,at,bad", [
    (400000, 100, float("nan")), (400000, 100, float("inf")), (400000, -300, float("nan")),
    (400000, -300, float("inf")), (1500000, -300, float("nan"))])
def test_a_broken_value_in_a_long_context(context, at, bad):
    """1024 queries over a long context (pages in turn), all in one CTA: a value that is
    not finite reaches the queries that see it, and the others are right, however long it
    takes to tell them apart (in the longest case more than the limit of a wait)."""
    block, hd, n = 256, 64, 1024
    gen = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda").to(BF16)
    k, v, q = rnd(9 * block, 1, hd), rnd(9 * block, 1, hd), rnd(n, 1, hd)
    at %= context
    table = torch.arange(-(-context // block), device="cuda", dtype=torch.int32) % 8
    table[at // block] = 8                   # a page of its own
    slot = table.long()[torch.arange(context, device="cuda") // block] * block \
        + torch.arange(context, device="cuda") % block
    rows = torch.arange(3, n, 50, device="cuda")
    score = q[rows, 0].double() @ k[slot, 0].double().T * hd ** -0.5
    score.masked_fill_(torch.arange(context, device="cuda")[None]
                       > (context - n + rows)[:, None], -float("inf"))
    p = torch.softmax(score, -1)
    want, weight = (p @ x[slot, 0].double() for x in (v, v.abs()))
    blind = (context - n + rows < at).cpu().numpy()
    v[8 * block + at % block] = bad
    ctx = torch.tensor([context], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 77.0)
    window_attention(q, k, v, table[None], ctx, block, cu_seqlens_q=cu, max_query_len=256,
                     max_context_len=128, out=out)
    status = ctypes.c_uint32()
    _lib.check(_lib.lib().ie_kernel_status(ctypes.byref(status), 1))
    assert status.value == 0
    assert blind.any() == (at != 100)
    if blind.any():
        # |q|_1 |k|_inf bounds a score's rounding as in the oracle
        largest = float((q[rows, 0].double().abs() @ k[slot, 0].double().abs().T).max()) / hd ** 0.5
        assert_close(out[rows, 0][blind], want.cpu().numpy()[blind], weight.cpu().numpy()[blind],
                     largest, hd)
    sees = out[context - n + torch.arange(n) >= at] if at != 100 else out
    assert not torch.isfinite(sees).any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_scores(dtype):
    """Scores of several hundred: the maximum is subtracted before the exponential,
    and a maximum that grows late rescales what was summed before."""
    for query in (None, [150, 170]):
        b = Batch([150, 400], 8, 2, 128, dtype, 16, query=query, seed=8, std=20.0)
        check(b)
    b = Batch([700], 4, 1, 64, dtype, 16, query=[700], seed=9)
    ramp = torch.linspace(0, 6, 700, device="cuda")
    order = (b.tables[0].long()[torch.arange(700, device="cuda") // 16] * 16
             + torch.arange(700, device="cuda") % 16)
    b.k[order] = (b.k[order].float() + ramp[:, None, None] * b.q[-1, 0].float()).to(dtype)
    check(b)


@pytest.mark.parametrize("dtype,hd", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("query", [None, [3]])
def test_a_long_flat_tail(dtype, hd, query):
    """A key of weight 1 before some 65000 of 2.48 * 2^-24, 1 % of the sum: an f16 weight
    that small is off by a fifth (two bounds of the sum), unless it is taken relative to a
    smaller maximum.  The lengths given make the rows one part; of one query's eight warps
    each has its large key and its tail.  (With more keys the f32 sums' own roundings, of a
    sixteen keys' 2^-19 beside 1, come near the bound.)"""
    context, peaks = (520000, torch.arange(0, 128, 16)) if query is None else (70000, [0])
    b = Batch([context], 2, 1, hd, dtype, 256, query=query, seed=18, spare=0)
    b.q.zero_()
    b.q[:, :, 0] = hd ** 0.5                    # a score is the key's first element
    first = int(b.tables[0, 0]) * 256
    b.k.zero_()
    b.k[:, :, 0] = -15.7266
    b.v = (b.v.nan_to_num(0.0).float() * 0.1 + 1).to(dtype)
    for at in peaks:
        b.k[first + int(at)] = 0.0
        b.v[first + int(at)] = -1.0
    got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 256, cu_seqlens_q=b.cu,
                           max_query_len=3, max_context_len=64)
    want, weight, largest = b.oracle()
    assert_close(got, want, weight, largest, hd)


def test_strides():
    """q as a slice of the fused projection, caches as halves of one tensor, a table
    that is a slice, and an output with wider rows."""
    b = Batch([90, 33], 8, 2, 64, BF16, 16, query=[20, 33], seed=10)
    want, weight, largest = b.oracle(window=30, sinks=1)
    wide = torch.zeros((53, 12, 64), dtype=BF16, device="cuda")
    wide[:, 2:10] = b.q
    both = torch.stack([b.k, b.v], dim=1)
    tables = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    tables[:, 3:3 + b.tables.shape[1]] = b.tables
    out = torch.zeros((53, 10, 64), dtype=BF16, device="cuda")[:, 1:9]
    got = window_attention(wide[:, 2:10], both[:, 0], both[:, 1],
                           tables[:, 3:3 + b.tables.shape[1]], b.ctx, 16, window=30, sinks=1,
                           out=out, **b.lens())
    assert got is out
    assert_close(got, want, weight, largest, 64)


@pytest.mark.parametrize("query", [None, [20, 33]])
def test_rows_that_are_not_aligned(query):
    b = Batch([90, 33], 4, 2, 64, F16, 16, query=query, seed=11)
    want, weight, largest = b.oracle()
    flat = torch.zeros(b.q.numel() + 1, dtype=F16, device="cuda")
    q = flat[1:].view(b.q.shape)
    q.copy_(b.q)
    got = window_attention(q, b.k, b.v, b.tables, b.ctx, 16, **b.lens())
    assert_close(got, want, weight, largest, 64)


def test_scale():
    b = Batch([90, 33], 4, 2, 64, BF16, 16, seed=12)
    got = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, scale=0.3)
    want, weight, largest = b.oracle(scale=0.3)
    assert_close(got, want, weight, largest, 64)


def test_cache_beyond_32_bit_offsets():
    """A page behind the first 2^31 elements (and 2^32 bytes) of the cache."""
    block, kv, hd = 256, 8, 128
    slots = (2 ** 31 // (kv * hd) // block + 4) * block
    k = torch.zeros((slots, kv, hd), dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    pages = slots // block
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device="cuda")
    for page in (pages - 1, 0, pages - 3):
        for c in (k, v):
            c[page * block:(page + 1) * block].normal_(generator=gen)
    for n in (1, 50):
        q = torch.randn((n, 32, hd), generator=gen, device="cuda").to(BF16)
        ctx = torch.tensor([700], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        got = window_attention(q, k, v, table, ctx, block, window=500, sinks=4, cu_seqlens_q=cu,
                               max_query_len=n)
        near = torch.cat([k[(pages - 1) * block:], k[:block], k[(pages - 3) * block:][:block]])
        nearv = torch.cat([v[(pages - 1) * block:], v[:block], v[(pages - 3) * block:][:block]])
        want, weight, largest = attention(q, near, nearv, torch.tensor([[0, 1, 2]]), [700], block,
                                          query=[n], window=500, sinks=4)
        assert_close(got, want, weight, largest, hd)


@pytest.mark.parametrize("several", [False, True])
def test_windows_and_sinks_beyond_2_to_the_30(several):
    """A context of 2^30 + 2^17 keys (three pages in turn) in which one key outweighs all
    others: it is seen or not by one position more or less of the window or the sinks."""
    block, hd = 1 << 16, 64
    context = (1 << 30) + (1 << 17)
    gen = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn((3 * block, 1, hd), generator=gen, device="cuda").to(BF16)
    v = torch.randn((3 * block, 1, hd), generator=gen, device="cuda").to(BF16)
    q = torch.randn((1, 1, hd), generator=gen, device="cuda").to(BF16)
    big = q[0, 0].double() * (60 * hd ** 0.5 / q.double().square().sum())
    k[block + 3, 0] = big.to(BF16)               # a score of 60 against N(0, 1)
    k[2 * block + 5, 0] = big.to(BF16)
    ctx = torch.tensor([context], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda") if several else None
    table = torch.zeros((1, context // block), dtype=torch.int32, device="cuda")

    def sees(slot, **kw):
        got = window_attention(q, k, v, table, ctx, block, cu_seqlens_q=cu, max_query_len=1,
                               max_context_len=context, **kw)
        # 2^31 keys of e^6 at most against e^59: below bf16's last bit
        return bool((got[0, 0] - v[slot, 0]).abs().max() <= 2.0 ** -7 * v[slot].abs().max())

    table[0, 0] = 1                              # the key at position 3
    assert sees(block + 3) and sees(block + 3, window=context)
    assert sees(block + 3, window=context - 3) and not sees(block + 3, window=context - 4)
    table[0, 0], table[0, 1 << 14] = 0, 2        # the key at position 2^30 + 5
    at = (1 << 30) + 5
    assert sees(2 * block + 5, window=10, sinks=at + 1)
    assert not sees(2 * block + 5, window=10, sinks=at)
    assert sees(2 * block + 5, window=10, sinks=1 << 40)


@pytest.mark.parametrize("n", [3, 200])
def test_one_item_may_take_longer_than_a_wait(n):
    """Two heads' queries over 2^28 keys (one page over and over) as one part, because the
    lengths given are far too small: seconds of key tiles for one CTA, in which the roles
    that have nothing to do must not give up.  A key at the end outweighs the others."""
    block, hd, context = 1 << 16, 64, 1 << 28
    k = torch.zeros((2 * block, 2, hd), dtype=BF16, device="cuda")
    v = torch.ones_like(k)
    q = torch.zeros((n, 2, hd), dtype=BF16, device="cuda")
    q[:, :, 0] = hd ** 0.5
    k[2 * block - n, :, 0], v[2 * block - n] = 40.0, -2.0     # seen by every query
    table = torch.zeros((1, context // block), dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    out = torch.full_like(q, float("nan"))
    window_attention(q, k, v, table, torch.tensor([context], dtype=torch.int32, device="cuda"),
                     block, max_query_len=1, max_context_len=128, out=out,
                     cu_seqlens_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    status = ctypes.c_uint32()
    _lib.check(_lib.lib().ie_kernel_status(ctypes.byref(status), 1))
    assert status.value == 0
    assert torch.all(out == -2.0)       # the others weigh 2^28 e^-40 together


def test_same_bits_twice_and_on_another_stream():
    b = Batch([700, 3000], 8, 2, 128, BF16, 16, seed=13)
    a = check(b, window=1000, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c = window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, window=1000, sinks=4, stream=side,
                         **b.lens())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, c)


@pytest.mark.parametrize("query", [None, [20, 90]])
def test_graph_capture_follows_the_lengths(query):
    b = Batch([300, 90], 8, 2, 128, BF16, 16, query=query, seed=14)
    lens = b.lens()
    call = lambda: window_attention(b.q, b.k, b.v, b.tables, b.ctx, 16, window=64, sinks=4, **lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    b.context = [211, 90]
    b.ctx.copy_(torch.tensor(b.context, dtype=torch.int32))
    graph.replay()
    want, weight, largest = b.oracle(window=64, sinks=4)
    assert_close(out, want, weight, largest, 128)


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (64, F16), (64, F32)])
@pytest.mark.parametrize("context,query", [([500, 300], [40, 9]), ([2000, 64], [5, 3]),
                                           ([70, 0], [70, 0])])
@pytest.mark.parametrize("lead,tail", [(0, 1), (0, 300), (3, 0), (150, 5)])
@pytest.mark.parametrize("lens", [True, False])
def test_tokens_of_no_sequence_are_zeros(hd, dtype, context, query, lead, tail, lens):
    """A batch of a fixed number of tokens of which the lengths cover a part, whole or in
    parts."""
    b = Batch(context, 4, 2, hd, dtype, 16, query=query, seed=33)
    want, weight, largest = b.oracle(window=400, sinks=2)
    n = sum(query)
    q = torch.randn((lead + n + tail, 4, hd), device="cuda").to(dtype)
    q[lead:lead + n] = b.q
    out = torch.full_like(q, float("nan"))
    window_attention(q, b.k, b.v, b.tables, b.ctx, 16, window=400, sinks=2, out=out,
                     cu_seqlens_q=b.cu + lead, max_query_len=max(query) if lens else 0,
                     max_context_len=max(context) if lens else 0)
    assert_close(out[lead:lead + n], want, weight, largest, hd)
    assert torch.count_nonzero(out[:lead]) == 0 and torch.count_nonzero(out[lead + n:]) == 0


def test_empty_batches():
    b = Batch([5], 4, 2, 64, BF16, 16, seed=15)
    none = torch.empty((0,), dtype=torch.int32, device="cuda")
    out = window_attention(b.q[:0], b.k, b.v, b.tables[:0], none, 16)
    assert out.shape == (0, 4, 64)
    got = window_attention(b.q, b.k, b.v, b.tables[:, :0], b.ctx, 16)
    assert torch.count_nonzero(got) == 0
    got = window_attention(b.q, b.k[:0], b.v[:0], b.tables, b.ctx, 16)
    assert torch.count_nonzero(got) == 0


def test_refusals():
    b = Batch([50, 20], 4, 2, 64, BF16, 16, seed=16)
    ok = (b.q, b.k, b.v, b.tables, b.ctx, 16)
    window_attention(*ok)
    bad = [
        (b.q[0], *ok[1:]), (b.q.half(), *ok[1:]), (b.q[:, :3], *ok[1:]), (b.q[..., :32], *ok[1:]),
        (b.q, b.k[:, :1], *ok[2:]), (b.q, b.k, b.v.half(), *ok[3:]),
        (*ok[:3], b.tables.long(), *ok[4:]), (*ok[:3], b.tables[0], *ok[4:]),
        (*ok[:4], b.ctx.long(), 16), (*ok[:4], b.ctx[:1], 16), (*ok[:5], 0),
        (b.q[:1], *ok[1:]), (b.q.cpu(), *ok[1:]), (*ok[:4], b.ctx.cpu(), 16),
        (*ok[:5], 2 ** 30),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            window_attention(*args)
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=float("nan")), dict(max_query_len=-1),
               dict(cu_seqlens_q=b.ctx), dict(out=b.q[:1]), dict(window=1.5)):
        with pytest.raises(ValueError):
            window_attention(*ok, **kw)
    big = torch.zeros((1, 2, 512), dtype=BF16, device="cuda")
    with pytest.raises(ValueError):
        window_attention(big, big.expand(16, 2, 512).contiguous(),
                         big.expand(16, 2, 512).contiguous(), b.tables[:1], b.ctx[:1], 16)


def c_args(b, out, window=0, sinks=0, prefix=0):
    a = _lib.AttentionArgs()
    a.q, a.q_token_stride, a.q_head_stride = b.q.data_ptr(), b.q.stride(0), b.q.stride(1)
    a.k_cache, a.v_cache, a.cache_slots = b.k.data_ptr(), b.v.data_ptr(), b.k.shape[0]
    a.slot_stride, a.head_stride = b.k.stride(0), b.k.stride(1)
    a.block_tables, a.table_stride, a.table_width = (b.tables.data_ptr(), b.tables.stride(0),
                                                     b.tables.shape[1])
    a.context_lens = b.ctx.data_ptr()
    a.cu_seqlens_q = None if b.cu is None else b.cu.data_ptr()
    a.out, a.out_token_stride = out.data_ptr(), out.stride(0)
    a.tokens, a.seqs = b.q.shape[0], len(b.context)
    lens = b.lens()
    a.max_query_len, a.max_context_len = lens["max_query_len"], lens["max_context_len"]
    a.window, a.sinks, a.prefix_len = window, sinks, prefix
    a.dtype = {BF16: _lib.IE_DT_BF16, F16: _lib.IE_DT_F16, F32: _lib.IE_DT_F32}[b.q.dtype]
    a.heads, a.kv_heads, a.head_dim = b.q.shape[1], b.k.shape[1], b.q.shape[2]
    a.block_size, a.scale = b.block, b.q.shape[2] ** -0.5
    return a


@pytest.mark.parametrize("case", ["split", "twin", "decode", "prefix", "f32"])
def test_a_workspace_needs_16_bytes_of_alignment(case):
    """The parts of split rows in a workspace that starts 16 bytes past a 32-byte boundary."""
    entry, prefix = "ie_window_attention", 0
    if case == "split":
        b = Batch([2000], 4, 1, 128, BF16, 16, query=[300], seed=20)
    elif case == "twin":
        b = Batch([1500, 700], 4, 2, 64, F16, 16, query=[5, 9], seed=21)
    elif case == "decode":
        b = Batch([20001], 2, 1, 128, BF16, 16, seed=22)
    elif case == "prefix":
        entry, prefix = "ie_shared_prefix_attention", 901
        b = Batch([901 + i for i in range(24)], 32, 8, 128, BF16, 16, prefix=901, seed=23)
    else:
        b = Batch([3000, 500], 4, 2, 64, F32, 16, seed=24)
    out = torch.full_like(b.q, float("nan"))
    a = c_args(b, out, prefix=prefix)
    need = _lib.lib().ie_attention_workspace_size(ctypes.byref(a))
    assert need > 0
    room = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    assert room.data_ptr() % 32 == 0
    for offset in (0, 16):
        out.fill_(float("nan"))
        _lib.check(getattr(_lib.lib(), entry)(ctypes.byref(a), room.data_ptr() + offset, need,
                                              _lib.stream_ptr()))
        want, weight, largest = b.oracle(prefix=prefix)
        assert_close(out, want, weight, largest, b.q.shape[2])


@pytest.mark.parametrize("hd", [1, 33, 127, 255])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_odd_head_sizes_split_into_parts(hd, dtype):
    for query in (None, [3]):
        b = Batch([200], 1, 1, hd, dtype, 16, query=query, seed=hd)
        out = torch.empty_like(b.q)
        assert _lib.lib().ie_attention_workspace_size(ctypes.byref(c_args(b, out))) > 0
        check(b)
        check(b, window=150, sinks=3)


def workspace(b, **kw):
    return _lib.lib().ie_attention_workspace_size(ctypes.byref(c_args(b, torch.empty_like(b.q),
                                                                      **kw)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("context,heads,kv,hd", [
    ([20001], 4, 1, 128), ([20000, 0], 2, 2, 64), ([9973, 20003], 3, 1, 128),
    ([30000, 5], 20, 1, 64)])
def test_decode_rows_in_parts_and_their_join(dtype, context, heads, kv, hd):
    """Rows long enough to go through the workspace, beside short and empty ones."""
    b = Batch(context, heads, kv, hd, dtype, 16, seed=hd)
    assert workspace(b) > 0 and workspace(b, window=15000, sinks=4) > 0
    check(b)
    check(b, window=15000, sinks=4)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("seqs", [38, 56, 74])
def test_decode_of_a_batch_that_a_window_makes_even(dtype, hd, seqs):
    """297 to 592 rows of one part: CTAs of two warps."""
    b = Batch([64 + 5 * i for i in range(seqs)], 16, 8, hd, dtype, 16, seed=seqs)
    b.context[3] = 0
    b.ctx[3] = 0
    assert workspace(b, window=48, sinks=2) == 0
    check(b, window=48, sinks=2)
    check(b, window=17)


@pytest.mark.parametrize("seqs,kv", [(1, 4), (2, 8), (3, 8), (5, 8), (9, 8), (20, 8), (40, 8)])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_in_clusters_of_every_size(seqs, kv, hd):
    check(Batch([1500 - 3 * i for i in range(seqs)], kv, kv, hd, BF16, 16, seed=seqs))


@pytest.mark.parametrize("heads,kv", [(130, 1), (260, 2)])
@pytest.mark.parametrize("query", [None, [9, 3]])
def test_more_than_128_query_heads_a_kv_head(heads, kv, query):
    b = Batch([200, 77], heads, kv, 64, BF16, 16, query=query, seed=heads)
    check(b)
    check(b, window=60, sinks=3)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("block", [1, 3, 5, 20, 24, 40, 96])
def test_pages_of_any_size_under_row_tiles(dtype, hd, block):
    """Pages that no TMA box fits are gathered; others take boxes of 8, 16 or 32 rows."""
    b = Batch([100, 1000, 300], 4, 2, hd, dtype, block, query=[100, 3, 260], seed=block)
    check(b)
    check(b, window=90, sinks=4)
