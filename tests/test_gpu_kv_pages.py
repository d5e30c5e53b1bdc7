"""``KVPagePool``: page copies on the device against plain indexing, and the books:
sharing, copies of partly filled pages, trimming, compaction, refusals that
change nothing."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from ie_tpq.kv_pages import KVPagePool, OutOfPages

pytestmark = pytest.mark.gpu


def caches(layers, pages, block, kv=2, hd=64, dtype=torch.bfloat16, seed=0, lead=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    out = []
    for _ in range(2 * layers):
        flat = torch.randn(lead + pages * block * kv * hd, generator=gen, device="cuda").to(dtype)
        out.append(flat[lead:].view(pages * block, kv, hd))
    return out[:layers], out[layers:]


@pytest.mark.parametrize("layers,pages,block,kv,hd,dtype,lead", [
    (1, 4, 1, 1, 1, torch.bfloat16, 0), (2, 9, 16, 2, 64, torch.bfloat16, 0),
    (3, 5000, 1, 2, 8, torch.float16, 0), (2, 64, 7, 3, 5, torch.float16, 0),
    (2, 33, 16, 8, 128, torch.float32, 0), (2, 12, 16, 2, 64, torch.bfloat16, 3),
    (150, 6, 2, 1, 8, torch.bfloat16, 0), (1, 5, 256, 8, 128, torch.float16, 0)])
def test_copies(layers, pages, block, kv, hd, dtype, lead):
    k, v = caches(layers, pages, block, kv, hd, dtype, seed=pages, lead=lead)
    pool = KVPagePool(k, v, block)
    order = np.random.default_rng(pages).permutation(pages)
    n = pages // 2
    for src, dst in ((order[:n], order[n:2 * n]), (order[:1].repeat(n), order[1:1 + n]),
                     ([], []), ([int(order[0])], [int(order[-1])])):
        want = []
        for c in k + v:
            w = c.clone().view(pages, -1)
            w[torch.as_tensor(np.asarray(dst, dtype=np.int64), device="cuda")] = \
                w[torch.as_tensor(np.asarray(src, dtype=np.int64), device="cuda")]
            want.append(w)
        pool.copy_pages(src, dst)
        for c, w in zip(k + v, want):
            assert torch.equal(c.view(pages, -1), w)


def test_long_lists_take_several_launches():
    k, v = caches(1, 20000, 1, 1, 8)
    pool = KVPagePool(k, v, 1)
    before = k[0].clone()
    pool.copy_pages(np.arange(9000), np.arange(11000, 20000))
    assert torch.equal(k[0][11000:], before[:9000]) and torch.equal(k[0][:11000], before[:11000])


def test_copies_on_a_stream_and_in_a_graph():
    k, v = caches(2, 10, 16)
    pool = KVPagePool(k, v, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pool.copy_pages([0], [5], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(k[1][:16], k[1][80:96])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.copy_pages([1, 2], [6, 7])
    k[0][16:32] = 3.0
    graph.replay()
    assert torch.equal(k[0][96:112], k[0][16:32])


def test_fork_shares_whole_pages_and_copies_the_last():
    k, v = caches(3, 12, 4)
    pool = KVPagePool(k, v, 4)
    a = pool.new(10)                                   # 2 whole pages, one of 2 tokens
    assert pool.pages(a) == [0, 1, 2] and pool.free_pages == 9
    b, c = pool.fork(a, 2)
    assert pool.pages(b) == [0, 1, 3] and pool.pages(c) == [0, 1, 4]
    for x in k + v:
        assert torch.equal(x[8:12], x[12:16]) and torch.equal(x[8:12], x[16:20])
    pool.append(b, 3)                                  # 13 tokens: one more page
    assert pool.pages(b) == [0, 1, 3, 5] and pool.length(b) == 13
    assert pool.slot(b, 12) == 20 and pool.slot(c, 9) == 17
    assert pool.tables([a, b]).tolist() == [[0, 1, 2, -1], [0, 1, 3, 5]]
    pool.free(a)                                       # its own page comes back, the shared stay
    assert pool.free_pages == 7
    assert pool.pages(pool.new(4)) == [2]
    pool.free([b, c])
    assert pool.free_pages == 11
    whole = pool.new(8)
    d = pool.fork(whole)[0]                            # nothing to copy
    assert pool.pages(d) == pool.pages(whole)
    e = pool.fork(pool.new(0), 2)
    assert [pool.pages(x) for x in e] == [[], []] and pool.tables(e).shape == (2, 1)


def test_trim_gives_back_what_the_window_hides():
    k, v = caches(1, 20, 4)
    pool = KVPagePool(k, v, 4)
    a = pool.new(40)
    # the next query is at position 40 and sees 31 .. 40 and the sinks 0 .. 4
    assert pool.trim(a, window=10, sinks=5) == 5
    assert pool.pages(a) == [0, 1, -1, -1, -1, -1, -1, 7, 8, 9] and pool.free_pages == 15
    assert pool.trim(a, window=10, sinks=5) == 0
    with pytest.raises(ValueError):
        pool.slot(a, 12)
    b = pool.fork(a)[0]
    pool.free(a)
    assert pool.free_pages == 15
    pool.append(b, 4)
    assert pool.trim(b, window=10, sinks=5) == 1
    pool.free(b)
    assert pool.free_pages == 20


def test_compact_moves_live_pages_down():
    k, v = caches(2, 40, 4, seed=3)
    pool = KVPagePool(k, v, 4)
    seqs = [pool.new(4 * n + 1) for n in (1, 3, 2, 5, 4)]
    forks = pool.fork(seqs[3], 2)
    content = {}
    for s in (seqs[1], seqs[3], *forks):
        content[s] = [[x[pool.slot(s, i)].clone() for i in range(pool.length(s))] for x in k + v]
    pool.free([seqs[0], seqs[2], seqs[4]])
    live = 40 - pool.free_pages
    assert pool.compact() > 0
    assert 40 - pool.free_pages == live
    used = set()
    for s, want in content.items():
        used |= set(pool.pages(s))
        for x, rows in zip(k + v, want):
            for i, row in enumerate(rows):
                assert torch.equal(x[pool.slot(s, i)], row)
    assert used == set(range(live)) and pool.compact() == 0
    assert pool.pages(pool.new(4)) == [live]


def test_random_books():
    """Pages are held exactly as often as they are counted, through many calls."""
    k, v = caches(1, 60, 4, seed=4)
    pool = KVPagePool(k, v, 4)
    rng, seqs = np.random.default_rng(0), []
    for _ in range(400):
        what = rng.integers(0, 6)
        try:
            if what == 0 or not seqs:
                seqs.append(pool.new(int(rng.integers(0, 20))))
            elif what == 1:
                seqs += pool.fork(seqs[rng.integers(len(seqs))], int(rng.integers(0, 4)))
            elif what == 2:
                pool.append(seqs[rng.integers(len(seqs))], int(rng.integers(0, 6)))
            elif what == 3:
                pool.free(seqs.pop(rng.integers(len(seqs))))
            elif what == 4:
                pool.trim(seqs[rng.integers(len(seqs))], int(rng.integers(1, 12)), 2)
            else:
                pool.compact()
        except OutOfPages:
            pool.free(seqs.pop(0))
        held = [p for s in seqs for p in pool.pages(s) if p >= 0]
        assert pool.free_pages == 60 - len(set(held))
        # a page that may still be written has one owner
        for s in seqs:
            if pool.length(s) % 4:
                assert held.count(pool.pages(s)[-1]) == 1


def test_refusals_change_nothing():
    k, v = caches(2, 8, 4)
    pool = KVPagePool(k, v, 4)
    before = [c.clone() for c in k + v]
    for src, dst in (([0], [8]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]),
                     ([0, 1], [2]), ([[0]], [[1]])):
        with pytest.raises(ValueError):
            pool.copy_pages(src, dst)
    for c, w in zip(k + v, before):
        assert torch.equal(c, w)
    a = pool.new(18)
    with pytest.raises(OutOfPages):
        pool.fork(a, 4)
    with pytest.raises(OutOfPages):
        pool.new(13)
    with pytest.raises(OutOfPages):
        pool.append(a, 15)
    assert pool.free_pages == 3 and pool.length(a) == 18
    for call in (lambda: pool.fork(99), lambda: pool.fork(a, -1), lambda: pool.free([a, a]),
                 lambda: pool.free(99), lambda: pool.trim(a, 0), lambda: pool.new(-1),
                 lambda: pool.append(a, -1), lambda: pool.slot(a, 18),
                 lambda: KVPagePool(k, v[:1], 4), lambda: KVPagePool(k, v, 5),
                 lambda: KVPagePool([], [], 4), lambda: KVPagePool([k[0].cpu()], [v[0].cpu()], 4),
                 lambda: KVPagePool([k[0], k[1].float()], v, 4)):
        with pytest.raises(ValueError):
            call()
    assert pool.free_pages == 3
