"""Paged attention from its definition in f64, one query at a time, and the bound
that the kernels' outputs are held to."""
from __future__ import annotations

import numpy as np
import torch


def as_f64(t):
    return t.detach().double().cpu().numpy()


def attention(q, k_cache, v_cache, tables, context, block, *, query=None, window=0, sinks=0,
              prefix=0, scale=None):
    """(out, weight) as f64 [tokens, heads, head_dim]: the attention output and
    sum_j p_j |v_j|, the scale of its rounding errors; also the largest
    sum_d |q_d k_d| * scale of a visible score.  ``query``: query lengths."""
    q, k, v = as_f64(q), as_f64(k_cache), as_f64(v_cache)
    tables = tables.cpu().numpy()
    tokens, heads, hd = q.shape
    kv = k.shape[1]
    group = heads // kv
    scale = hd ** -0.5 if scale is None else scale
    pages = k.shape[0] // block
    out, weight, largest = np.zeros_like(q), np.zeros_like(q), 0.0
    t = 0
    for s, ctx in enumerate(context):
        n = 1 if query is None else query[s]
        for i in range(n):
            pos = ctx - n + i
            keys = np.arange(0, max(pos + 1, 0))
            if window:
                keys = keys[(keys > pos - window) | (keys < sinks)]
            row = np.where(keys < prefix, 0, s)
            keys, row = keys[keys // block < tables.shape[1]], row[keys // block < tables.shape[1]]
            page = tables[row, keys // block]
            ok = (page >= 0) & (page < pages)
            slot = (page * block + keys % block)[ok].astype(np.int64)
            if slot.size:
                for h in range(heads):
                    prod = k[slot, h // group] * q[t, h] * scale
                    sc = prod.sum(-1)
                    largest = max(largest, np.abs(prod).sum(-1).max())
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    out[t, h] = p @ v[slot, h // group]
                    weight[t, h] = p @ np.abs(v[slot, h // group])
            t += 1
    assert t == tokens
    return out, weight, largest


def assert_close(got, want, weight, largest, hd):
    """Elementwise bound.  With u the unit roundoff of the output type: the output
    is rounded once (u |o|); every softmax weight is rounded once to that type
    before it meets V (u sum p |v|); and the f32 scores of hd products, the
    exponential (2^-21) and the running sums move the weights by at most
    e = 2 (hd + 4) 2^-24 (1 + largest) + 2^-19 relative.  f32 has no rounding of
    the weights."""
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}[got.dtype]
    e = 2 * (hd + 4) * 2.0 ** -24 * (1 + largest) + 2.0 ** -19
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 1e-30      # subnormal outputs
    bound = u * np.abs(want) + (u + e) * weight + tiny
    err = np.abs(as_f64(got) - want)
    assert np.all(np.isfinite(as_f64(got)))
    worst = np.max(err / bound) if err.size else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the bound"


class Batch:
    """A random paged batch on the device; cache rows that no sequence holds are NaN."""

    def __init__(self, context, heads, kv, hd, dtype, block, *, query=None, seed=0, spare=3,
                 prefix=0, width=None, std=1.5):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.context, self.query, self.block, self.prefix = list(context), query, block, prefix
        width = width or max(1, -(-max(context) // block))
        need = [-(-c // block) for c in context]
        shared = prefix // block
        rows = np.full((len(context), width), -1, dtype=np.int64)
        used = 0
        for s, n in enumerate(need):
            for b in range(n):
                if b < shared and s > 0 and rows[0, b] >= 0:
                    rows[s, b] = rows[0, b]
                else:
                    rows[s, b] = used
                    used += 1
        pages = used + spare
        perm = np.random.default_rng(seed).permutation(pages)
        live = rows >= 0
        rows[live] = perm[rows[live]]
        self.tables = torch.from_numpy(rows.astype(np.int32)).cuda()
        rnd = lambda *sh, std=1.0: torch.randn(sh, generator=gen, device="cuda") * std
        self.k = rnd(pages * block, kv, hd).to(dtype)
        self.v = rnd(pages * block, kv, hd).to(dtype)
        written = np.zeros(pages * block, dtype=bool)
        for s, c in enumerate(context):
            j = np.arange(c)
            written[rows[s, j // block] * block + j % block] = True
        bad = torch.from_numpy(~written).cuda()
        self.k[bad] = float("nan")
        self.v[bad] = float("nan")
        tokens = len(context) if query is None else sum(query)
        self.q = rnd(tokens, heads, hd, std=std).to(dtype)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.ctx = torch.tensor(self.context, **i32)
        self.cu = None if query is None else torch.tensor(np.cumsum([0, *query]), **i32)

    def lens(self):
        return dict(cu_seqlens_q=self.cu, max_context_len=max(self.context),
                    max_query_len=1 if self.query is None else max(self.query))

    def oracle(self, **kw):
        return attention(self.q, self.k, self.v, self.tables, self.context, self.block,
                         query=self.query, **kw)
